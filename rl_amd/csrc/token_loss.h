// Launch interface of the token-level language-model losses
// (token_loss.hip): plain structs, no C++ exceptions across the boundary.
// Every launcher returns the hipError_t of its launches as an int.
#pragma once

// Element types of operands that a kernel reads by a runtime code.
enum RlDtype : int {
  RL_F32 = 0,
  RL_BF16 = 1,
  RL_F16 = 2,
  RL_U8 = 3,   // bool / uint8
  RL_I32 = 4,
  RL_I64 = 5,
  RL_I8 = 6,
  RL_I16 = 7,
  RL_F64 = 8,
};

struct TokenLogProbArgs {
  const void* logits;   // [rows / width][width][vocab], last dim dense
  long stride_batch, stride_row;  // in elements
  long rows, width;
  int vocab;
  int dtype;            // RL_F32 / RL_BF16 / RL_F16
  const void* tokens;   // [rows], int64 or int32
  int tokens_i32;
  long ignore_index;
  float inv_temperature;
  float* log_probs;     // [rows], forward
  float* stats;         // [rows][2]: the max and the sum of exp2; may be null in forward
  float* parts;         // [rows][token_log_probs_parts()][2] where that is above 1, forward
  const float* upstream;  // [rows], backward
  void* grad;           // [rows][vocab] dense, backward
};

// One operand of the policy loss seen as [rows][cols] with strides.
struct PolicyOperand {
  const void* ptr;  // null: absent
  long stride_row, stride_col;
  int dtype;
};

struct PolicyLossArgs {
  PolicyOperand log_probs, old_log_probs, advantage, mask, ref;
  long rows, cols;
  unsigned cols_magic;     // the launcher's: reciprocal of cols
  int cols_shift;
  int variant;             // 0: clipped surrogate, 1: clipped weight
  double log_low, log_high;    // borders of the log ratio
  double log_off;              // upper border of the clip_fraction count
  double low, high;            // the clipped ratio's values: 1 - low, 1 + high
  double kl_coeff, entropy_coeff;
  int mean;                // 1: divide by the mask's sum, 0: plain sums
  double* partials;        // [blocks][8]
  int blocks;
  float* out;              // 7 scalars
  float* scale;            // for the backward pass: 1 / denominator; log2 of the ess'
                           // sum(r) / sum(r^2); whether sum(r^2) is above its floor
  // backward
  const float* g_total;    // upstream scalars; null: zero
  const float* g_objective;
  const float* g_kl;
  const float* g_entropy;
  const float* g_ess;
  void* grad;              // [rows][cols] dense, log_probs' type
};

extern "C" {
int token_log_probs_parts(const TokenLogProbArgs* a);
int launch_token_log_probs_fwd(const TokenLogProbArgs* a, void* stream);
int launch_token_log_probs_bwd(const TokenLogProbArgs* a, void* stream);
int policy_loss_blocks(long n);
int launch_policy_loss_fwd(const PolicyLossArgs* a, void* stream);
int launch_policy_loss_bwd(const PolicyLossArgs* a, void* stream);
}
