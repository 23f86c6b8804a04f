// Token-level language-model losses for CDNA4 (gfx950).
//
// token_log_probs.  For a row of logits z, a token t and a temperature T
//
//   lp      = z_t / T - log sum_j exp(z_j / T)
//   dlp/dz  = (onehot(t) - softmax(z / T)) / T
//
// With c = log2(e) / T, m = max_j z_j and s = sum_j exp2(c (z_j - m)) this is
// lp = (z_t - m) / T - ln s and softmax_j = exp2(c (z_j - m)) / s.  The forward
// pass reads the row once, each thread carrying a running (m, s) that is
// rescaled when m grows, and leaves (m, s) for the backward pass, which reads
// the row a second time and writes the gradient once.  z - m is taken before
// the product with c: c m overflows for rows masked with the type's lowest
// value.  Bound by HBM: one read forward, one read and one write backward.
//
// token_policy_loss.  See the section below.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>

#include "token_loss.h"

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) {
  return __builtin_amdgcn_exp2f(x);  // v_exp_f32, 1 ulp
}

template <typename T>
struct Vec16 {  // 16 bytes of T
  static constexpr int N = 16 / sizeof(T);
};

// 16 bytes from or to an address that is aligned to T only: the target allows
// unaligned wide global accesses and the compiler emits one dwordx4.
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&x)[Vec16<T>::N]);

template <>
__device__ __forceinline__ void load16<float>(const float* p, float (&x)[4]) {
  __builtin_memcpy(x, p, 16);
}

__device__ __forceinline__ float bf16_lo(unsigned u) {
  return __uint_as_float(u << 16);
}
__device__ __forceinline__ float bf16_hi(unsigned u) {
  return __uint_as_float(u & 0xffff0000u);
}

template <>
__device__ __forceinline__ void load16<__bf16>(const __bf16* p, float (&x)[8]) {
  unsigned u[4];
  __builtin_memcpy(u, p, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(u[i]);
    x[2 * i + 1] = bf16_hi(u[i]);
  }
}

template <>
__device__ __forceinline__ void load16<_Float16>(const _Float16* p, float (&x)[8]) {
  _Float16 h[8];
  __builtin_memcpy(h, p, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&x)[Vec16<T>::N]) {
  T h[Vec16<T>::N];
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) h[i] = (T)x[i];
  __builtin_memcpy(__builtin_assume_aligned(p, 16), h, 16);
}

struct MaxSum {
  float m, s;
};

// Joins two running (max, sum of exp2(c (z - max))) pairs.  A side that saw
// nothing above -inf has s = 0 and does not contribute.
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float sa = a.s == 0.f ? 0.f : a.s * exp2_hw((a.m - m) * c);
  const float sb = b.s == 0.f ? 0.f : b.s * exp2_hw((b.m - m) * c);
  return {m, sa + sb};
}

template <int U, int N>
__device__ __forceinline__ void absorb(MaxSum& r, const float (&x)[U][N], float c) {
  float top = x[0][0];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, x[u][i]);
  if (top > r.m) {
    r.s *= r.m == -INFINITY ? 0.f : exp2_hw((r.m - top) * c);
    r.m = top;
  }
  // while everything seen is -inf any finite offset keeps exp2 at zero
  const float off = r.m == -INFINITY ? 0.f : r.m;
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2_hw((x[u][i] - off) * c);
  r.s += s;
}

__device__ __forceinline__ long token_at(const TokenLogProbArgs& a, long n) {
  return a.tokens_i32 ? (long)((const int*)a.tokens)[n] : ((const long*)a.tokens)[n];
}

// TPR threads share a row; BLOCK / TPR rows share a workgroup.
template <typename T, int TPR, int BLOCK, int U>
__global__ __launch_bounds__(BLOCK) void token_log_probs_fwd_k(const TokenLogProbArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int ROWS = BLOCK / TPR;
  __shared__ MaxSum part[BLOCK / 64];
  const int t = threadIdx.x % TPR;
  const float c = a.inv_temperature * kLog2e;
  for (long first = (long)blockIdx.x * ROWS; first < a.rows; first += (long)gridDim.x * ROWS) {
    const long n = first + threadIdx.x / TPR;
    const bool live = n < a.rows;
    const long tok = live ? token_at(a, n) : a.ignore_index;
    if (TPR > 64 ? tok == a.ignore_index : false) {  // the whole workgroup's row
      if (t == 0) {
        a.log_probs[n] = 0.f;
        if (a.stats) {
          a.stats[2 * n] = 0.f;
          a.stats[2 * n + 1] = 1.f;
        }
      }
      continue;
    }
    MaxSum r = {-INFINITY, 0.f};
    const T* row = nullptr;
    if (tok != a.ignore_index) {
      row = (const T*)a.logits + (n / a.width) * a.stride_batch + (n % a.width) * a.stride_row;
      const int mis = (int)(((size_t)row & 15) / sizeof(T));
      const int head = min(mis ? N - mis : 0, a.vocab);
      const int vecs = (a.vocab - head) / N;
      const int tail = a.vocab - head - vecs * N;
      const T* body = row + head;
      float edge[1][1];
      if (t < head) {
        edge[0][0] = (float)row[t];
        absorb<1, 1>(r, edge, c);
      }
      if (TPR - 1 - t < tail) {
        edge[0][0] = (float)row[a.vocab - (TPR - t)];
        absorb<1, 1>(r, edge, c);
      }
      int v = t;
      for (; v + (U - 1) * TPR < vecs; v += U * TPR) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load16<T>(body + (long)(v + u * TPR) * N, x[u]);
        absorb<U, N>(r, x, c);
      }
      for (; v < vecs; v += TPR) {
        float x[1][N];
        load16<T>(body + (long)v * N, x[0]);
        absorb<1, N>(r, x, c);
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      MaxSum o = {__shfl_xor(r.m, off, 64), __shfl_xor(r.s, off, 64)};
      r = join(r, o, c);
    }
    if (TPR > 64) {
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r;
      __syncthreads();
      if (threadIdx.x == 0)
        for (int w = 1; w < TPR / 64; ++w) r = join(r, part[w], c);
      __syncthreads();  // part is written again for the next row
    }
    if (t == 0 && live) {
      float lp = 0.f, s = 1.f;
      if (tok != a.ignore_index) {
        // a row of -inf alone has no distribution: NaN, as 0 / 0
        s = r.s == 0.f ? NAN : r.s;
        lp = tok >= 0 && tok < a.vocab
                 ? fmaf((float)row[tok] - r.m, a.inv_temperature, -__builtin_amdgcn_logf(s) * kLn2)
                 : NAN;
      }
      a.log_probs[n] = lp;
      if (a.stats) {
        a.stats[2 * n] = r.m;
        a.stats[2 * n + 1] = s;
      }
    }
  }
}

template <typename T, int TPR, int BLOCK, int U>
__global__ __launch_bounds__(BLOCK) void token_log_probs_bwd_k(const TokenLogProbArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int ROWS = BLOCK / TPR;
  const int t = threadIdx.x % TPR;
  const float c = a.inv_temperature * kLog2e;
  for (long first = (long)blockIdx.x * ROWS; first < a.rows; first += (long)gridDim.x * ROWS) {
    // last rows first: what the forward pass read last is still in the cache
    const long n = a.rows - 1 - (first + threadIdx.x / TPR);
    if (n < 0) continue;
    const long tok = token_at(a, n);
    const float g = tok == a.ignore_index ? 0.f : a.upstream[n] * a.inv_temperature;
    T* out = (T*)a.grad + n * a.vocab;
    const T* row = (const T*)a.logits + (n / a.width) * a.stride_batch + (n % a.width) * a.stride_row;
    // aligned to the row that is written; reads may be unaligned
    const int mis = (int)(((size_t)out & 15) / sizeof(T));
    const int head = min(mis ? N - mis : 0, a.vocab);
    const int vecs = (a.vocab - head) / N;
    const int tail = a.vocab - head - vecs * N;
    T* obody = out + head;
    if (g == 0.f) {  // a masked token: exact zeros, and its logits are not read
      const float zero[N] = {};
      if (t < head) out[t] = (T)0.f;
      if (TPR - 1 - t < tail) out[a.vocab - (TPR - t)] = (T)0.f;
      for (int v = t; v < vecs; v += TPR) store16<T>(obody + (long)v * N, zero);
      continue;
    }
    const bool known = tok >= 0 && tok < a.vocab;
    const float m = a.stats[2 * n];
    const float scale = known ? -g / a.stats[2 * n + 1] : NAN;
    const T* body = row + head;
    auto one = [&](int j) {
      const float d = scale * exp2_hw(((float)row[j] - m) * c);
      out[j] = (T)(j == tok ? d + g : d);
    };
    if (t < head) one(t);
    if (TPR - 1 - t < tail) one(a.vocab - (TPR - t));
    const long hot = tok - head;  // the token's place in the body
    auto finish = [&](int v, float (&x)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = scale * exp2_hw((x[i] - m) * c);
      const long at = hot - (long)v * N;
      if (at >= 0 && at < N) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i == at) x[i] += g;
      }
      store16<T>(obody + (long)v * N, x);
    };
    int v = t;
    for (; v + (U - 1) * TPR < vecs; v += U * TPR) {
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) load16<T>(body + (long)(v + u * TPR) * N, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) finish(v + u * TPR, x[u]);
    }
    for (; v < vecs; v += TPR) {
      float x[N];
      load16<T>(body + (long)v * N, x);
      finish(v, x);
    }
  }
}

constexpr long kMaxBlocks = 1 << 20;

template <typename T, int TPR, int BLOCK, int U>
int log_probs_launch(const TokenLogProbArgs& a, bool bwd, hipStream_t st) {
  const long rows = BLOCK / TPR;
  const long need = (a.rows + rows - 1) / rows;
  const dim3 grid((unsigned)(need < kMaxBlocks ? need : kMaxBlocks));
  if (bwd)
    hipLaunchKernelGGL((token_log_probs_bwd_k<T, TPR, BLOCK, U>), grid, dim3(BLOCK), 0, st, a);
  else
    hipLaunchKernelGGL((token_log_probs_fwd_k<T, TPR, BLOCK, U>), grid, dim3(BLOCK), 0, st, a);
  return (int)hipGetLastError();
}

template <typename T>
int log_probs_dispatch(const TokenLogProbArgs& a, bool bwd, hipStream_t st) {
  const long bytes = (long)a.vocab * (long)sizeof(T);
  if (bytes <= 4096) return log_probs_launch<T, 64, 256, 4>(a, bwd, st);
  if (a.rows >= 1024) return log_probs_launch<T, 256, 256, 4>(a, bwd, st);
  return log_probs_launch<T, 1024, 1024, 4>(a, bwd, st);
}

int log_probs_any(const TokenLogProbArgs* a, bool bwd, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  switch (a->dtype) {
    case RL_F32:
      return log_probs_dispatch<float>(*a, bwd, st);
    case RL_BF16:
      return log_probs_dispatch<__bf16>(*a, bwd, st);
    case RL_F16:
      return log_probs_dispatch<_Float16>(*a, bwd, st);
  }
  return (int)hipErrorInvalidValue;
}

// ---------------------------------------------------------------------------
// token_policy_loss: with x = lp - old, r = exp(x), weights w of the mask and
// D = max(1, sum w) (or 1 for sums)
//
//   clip:   gain = min(r A, clip(r, 1 - low, 1 + high) A)
//           dgain/dlp = r A, or 0 where the ratio is clipped against A
//   cispo:  gain = clip(r) x A, dgain/dlp = clip(r) A  (clip(r) is a constant)
//   kl:     e^y - 1 - y with y = ref - lp;  d/dlp = 1 - e^y
//   entropy term: + lp (the sampled estimate of -H); d/dlp = 1
//   objective = -sum w gain / D, and the rest likewise
//
// Whether a ratio is clipped is decided in double on x against the borders'
// logarithms: x is then exact for fp32 inputs, and an element next to a border
// falls on the same side as in the definition.  e^y - 1 - y cancels near 0: a
// series there.  Sums are in double (the loop is bound by its loads).
//
// One workgroup does everything up to 16K tokens; above, partial sums of many
// and a second launch that joins them in a fixed order: no atomics, the result
// does not depend on the order of execution.  Launch bound below ~1M tokens.
// ---------------------------------------------------------------------------

__device__ __forceinline__ double operand(const PolicyOperand& o, long r, long c) {
  const long i = r * o.stride_row + c * o.stride_col;
  switch (o.dtype) {
    case RL_F32:
      return ((const float*)o.ptr)[i];
    case RL_BF16:
      return (float)((const __bf16*)o.ptr)[i];
    case RL_F16:
      return (float)((const _Float16*)o.ptr)[i];
    case RL_U8:
      return ((const unsigned char*)o.ptr)[i];
    case RL_I32:
      return ((const int*)o.ptr)[i];
    case RL_I64:
      return (double)((const long*)o.ptr)[i];
    case RL_I8:
      return ((const signed char*)o.ptr)[i];
    case RL_I16:
      return ((const short*)o.ptr)[i];
    default:
      return ((const double*)o.ptr)[i];
  }
}

// e^y - 1 - y
__device__ __forceinline__ float kl3(float y) {
  if (fabsf(y) > 0.5f) return expf(y) - 1.f - y;
  // y^2 (1/2! + y/3! + y^2/4! + ...), remainder below 2^-25 of the sum at 1/2
  float p = 1.f / 3628800.f;
  p = fmaf(p, y, 1.f / 362880.f);
  p = fmaf(p, y, 1.f / 40320.f);
  p = fmaf(p, y, 1.f / 5040.f);
  p = fmaf(p, y, 1.f / 720.f);
  p = fmaf(p, y, 1.f / 120.f);
  p = fmaf(p, y, 1.f / 24.f);
  p = fmaf(p, y, 1.f / 6.f);
  p = fmaf(p, y, 0.5f);
  return y * y * p;
}

struct PolicyToken {
  bool above, below;
  float x, ratio;
};

__device__ __forceinline__ PolicyToken policy_token(const PolicyLossArgs& a, double x) {
  PolicyToken t;
  t.above = x > a.log_high;
  t.below = x < a.log_low;
  t.x = (float)x;
  t.ratio = expf(t.x);
  return t;
}

__device__ __forceinline__ bool clipped_against(const PolicyToken& t, float adv) {
  return (t.above && adv > 0.f) || (t.below && adv < 0.f);
}

enum { S_GAIN, S_KL, S_LP, S_W, S_R, S_RR, S_OFF, S_COUNT };

__device__ __forceinline__ void policy_finish(const PolicyLossArgs& a, const double (&s)[S_COUNT]) {
  const double n = (double)a.rows * (double)a.cols;
  const double inv = a.mean ? 1.0 / (s[S_W] > 1.0 || isnan(s[S_W]) ? s[S_W] : 1.0) : 1.0;
  const double objective = -s[S_GAIN] * inv;
  const double kl = s[S_KL] * inv;
  const double entropy = a.entropy_coeff * (s[S_LP] * inv);
  a.out[0] = (float)(objective + a.kl_coeff * kl + entropy);
  a.out[1] = (float)objective;
  a.out[2] = (float)(a.kl_coeff * kl);
  a.out[3] = (float)entropy;
  a.out[4] = (float)kl;
  a.out[5] = (float)(s[S_OFF] / n);
  a.out[6] = (float)(s[S_R] * s[S_R] / fmax(s[S_RR], 1e-9) / n);
  *a.scale = (float)inv;
}

template <int BLOCK>
__device__ __forceinline__ bool block_sums(double (&s)[S_COUNT]) {
  __shared__ double part[BLOCK / 64][S_COUNT];
#pragma unroll
  for (int k = 0; k < S_COUNT; ++k)
    for (int off = 32; off > 0; off >>= 1) s[k] += __shfl_xor(s[k], off, 64);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) part[threadIdx.x >> 6][k] = s[k];
  __syncthreads();
  if (threadIdx.x != 0) return false;
  for (int w = 1; w < BLOCK / 64; ++w)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) s[k] += part[w][k];
  return true;
}

template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void policy_loss_fwd_k(const PolicyLossArgs a) {
  double s[S_COUNT] = {};
  const long n = a.rows * a.cols;
  for (long i = (long)blockIdx.x * BLOCK + threadIdx.x; i < n; i += (long)gridDim.x * BLOCK) {
    const long r = i / a.cols, c = i - r * a.cols;
    const double lp = operand(a.log_probs, r, c);
    const double x = lp - operand(a.old_log_probs, r, c);
    const PolicyToken t = policy_token(a, x);
    s[S_R] += t.ratio;
    s[S_RR] += (double)t.ratio * t.ratio;
    s[S_OFF] += (x > a.log_off || t.below) ? 1.0 : 0.0;
    const double w = a.mask.ptr ? operand(a.mask, r, c) : 1.0;
    if (w == 0.0) continue;  // a masked token may hold anything, NaN too
    const float adv = (float)operand(a.advantage, r, c);
    const float bound = t.above ? a.high : t.below ? a.low : t.ratio;
    float gain;
    if (a.variant == 0)
      gain = (clipped_against(t, adv) ? bound : t.ratio) * adv;
    else
      gain = bound * t.x * adv;
    s[S_GAIN] += w * gain;
    s[S_W] += w;
    s[S_LP] += w * lp;
    if (a.ref.ptr) s[S_KL] += w * kl3((float)(operand(a.ref, r, c) - lp));
  }
  if (!block_sums<BLOCK>(s)) return;
  if (gridDim.x == 1) {
    policy_finish(a, s);
    return;
  }
#pragma unroll
  for (int k = 0; k < S_COUNT; ++k) a.partials[(long)blockIdx.x * 8 + k] = s[k];
}

__global__ __launch_bounds__(256) void policy_loss_join_k(const PolicyLossArgs a) {
  double s[S_COUNT] = {};
  for (int b = threadIdx.x; b < a.blocks; b += 256)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) s[k] += a.partials[(long)b * 8 + k];
  if (block_sums<256>(s)) policy_finish(a, s);
}

template <typename T>
__global__ __launch_bounds__(256) void policy_loss_bwd_k(const PolicyLossArgs a) {
  const float inv = *a.scale;
  const float total = a.g_total ? *a.g_total : 0.f;
  const float go = (total + (a.g_objective ? *a.g_objective : 0.f)) * inv;
  const float gk = (total + (a.g_kl ? *a.g_kl : 0.f)) * a.kl_coeff * inv;
  const float ge = (total + (a.g_entropy ? *a.g_entropy : 0.f)) * a.entropy_coeff * inv;
  const long n = a.rows * a.cols;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / a.cols, c = i - r * a.cols;
    const float w = a.mask.ptr ? (float)operand(a.mask, r, c) : 1.f;
    float d = 0.f;
    if (w != 0.f) {
      const double lp = operand(a.log_probs, r, c);
      const PolicyToken t = policy_token(a, lp - operand(a.old_log_probs, r, c));
      const float adv = (float)operand(a.advantage, r, c);
      float dgain;
      if (a.variant == 0)
        dgain = clipped_against(t, adv) ? 0.f : t.ratio * adv;
      else
        dgain = (t.above ? a.high : t.below ? a.low : t.ratio) * adv;
      d = ge - go * dgain;
      if (a.ref.ptr && a.kl_coeff != 0.f) d -= gk * expm1f((float)(operand(a.ref, r, c) - lp));
      d *= w;
    }
    ((T*)a.grad)[i] = (T)d;
  }
}

}  // namespace

extern "C" int launch_token_log_probs_fwd(const TokenLogProbArgs* a, void* stream) {
  return log_probs_any(a, false, stream);
}

extern "C" int launch_token_log_probs_bwd(const TokenLogProbArgs* a, void* stream) {
  return log_probs_any(a, true, stream);
}

extern "C" int policy_loss_blocks(long n) {
  if (n <= 16384) return 1;
  const long b = (n + 2047) / 2048;
  return (int)(b < 1024 ? b : 1024);
}

extern "C" int launch_policy_loss_fwd(const PolicyLossArgs* a, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (a->blocks == 1) {
    if (a->rows * a->cols <= 256)
      hipLaunchKernelGGL((policy_loss_fwd_k<256>), dim3(1), dim3(256), 0, st, *a);
    else
      hipLaunchKernelGGL((policy_loss_fwd_k<1024>), dim3(1), dim3(1024), 0, st, *a);
  } else {
    hipLaunchKernelGGL((policy_loss_fwd_k<256>), dim3(a->blocks), dim3(256), 0, st, *a);
    hipLaunchKernelGGL(policy_loss_join_k, dim3(1), dim3(256), 0, st, *a);
  }
  return (int)hipGetLastError();
}

extern "C" int launch_policy_loss_bwd(const PolicyLossArgs* a, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  const long n = a->rows * a->cols;
  const long need = (n + 255) / 256;
  const dim3 grid((unsigned)(need < 4096 ? need : 4096));
  switch (a->log_probs.dtype) {
    case RL_F32:
      hipLaunchKernelGGL((policy_loss_bwd_k<float>), grid, dim3(256), 0, st, *a);
      break;
    case RL_BF16:
      hipLaunchKernelGGL((policy_loss_bwd_k<__bf16>), grid, dim3(256), 0, st, *a);
      break;
    case RL_F16:
      hipLaunchKernelGGL((policy_loss_bwd_k<_Float16>), grid, dim3(256), 0, st, *a);
      break;
    default:
      return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}
