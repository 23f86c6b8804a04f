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
// value.  Bound by HBM: one read forward, one read and one write backward
// (8192 x 50257 bf16: 140 us at 5.9 TB/s, 299 us at 5.5 TB/s).
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

template <bool STREAM, typename T>
__device__ __forceinline__ void store16(T* p, const float (&x)[Vec16<T>::N]) {
  typedef unsigned U4 __attribute__((ext_vector_type(4)));
  T h[Vec16<T>::N];
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) h[i] = (T)x[i];
  U4 u;
  __builtin_memcpy(&u, h, 16);
  if (STREAM)
    __builtin_nontemporal_store(u, (U4*)p);
  else
    *(U4*)p = u;
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

// The row's log-prob and statistics from its joined (max, sum).
template <typename T>
__device__ __forceinline__ void write_row(const TokenLogProbArgs& a, long n, long tok, const T* row,
                                          MaxSum r) {
  float lp = 0.f, s = 1.f;
  if (tok != a.ignore_index) {
    // a row of -inf alone has no distribution: NaN, as 0 / 0
    s = r.s == 0.f ? NAN : r.s;
    lp = tok >= 0 && tok < a.vocab
             ? fmaf((float)row[tok] - r.m, a.inv_temperature, -__builtin_amdgcn_logf(s) * kLn2)
             : NAN;
  } else {
    r.m = 0.f;
  }
  a.log_probs[n] = lp;
  if (a.stats) {
    a.stats[2 * n] = r.m;
    a.stats[2 * n + 1] = s;
  }
}

template <typename T>
__device__ __forceinline__ const T* row_at(const TokenLogProbArgs& a, long n) {
  return (const T*)a.logits + (n / a.width) * a.stride_batch + (n % a.width) * a.stride_row;
}

// TPR threads share a row; BLOCK / TPR rows share a workgroup, or with
// gridDim.y > 1 that many workgroups share one row and leave their parts.
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
    if (TPR > 64 && tok == a.ignore_index) {  // the whole workgroup's row
      if (t == 0 && gridDim.y == 1) write_row<T>(a, n, tok, nullptr, {0.f, 1.f});
      continue;
    }
    MaxSum r = {-INFINITY, 0.f};
    const T* row = nullptr;
    if (tok != a.ignore_index) {
      row = row_at<T>(a, n);
      const int mis = (int)(((size_t)row & 15) / sizeof(T));
      const int head = min(mis ? N - mis : 0, a.vocab);
      const int vecs = (a.vocab - head) / N;
      const int tail = a.vocab - head - vecs * N;
      const T* body = row + head;
      float edge[1][1];
      if (t < head && blockIdx.y == 0) {
        edge[0][0] = (float)row[t];
        absorb<1, 1>(r, edge, c);
      }
      if (TPR - 1 - t < tail && blockIdx.y == gridDim.y - 1) {
        edge[0][0] = (float)row[a.vocab - (TPR - t)];
        absorb<1, 1>(r, edge, c);
      }
      const int end = (int)((long)vecs * (blockIdx.y + 1) / gridDim.y);
      int v = (int)((long)vecs * blockIdx.y / gridDim.y) + t;
      for (; v + (U - 1) * TPR < end; v += U * TPR) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load16<T>(body + (long)(v + u * TPR) * N, x[u]);
        absorb<U, N>(r, x, c);
      }
      if (v < end) {  // what is left, all loads at once: the last vector again for none
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load16<T>(body + (long)min(v + u * TPR, end - 1) * N, x[u]);
#pragma unroll
        for (int u = 1; u < U; ++u)
          if (v + u * TPR >= end)
#pragma unroll
            for (int i = 0; i < N; ++i) x[u][i] = -INFINITY;
        absorb<U, N>(r, x, c);
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
      if (gridDim.y == 1) {
        write_row<T>(a, n, tok, row, r);
      } else {
        a.parts[2 * (n * gridDim.y + blockIdx.y)] = r.m;
        a.parts[2 * (n * gridDim.y + blockIdx.y) + 1] = r.s;
      }
    }
  }
}

// A wave joins the parts of a row, in order.
template <typename T>
__global__ __launch_bounds__(64) void token_log_probs_join_k(const TokenLogProbArgs a, int parts) {
  const long n = blockIdx.x;
  const long tok = token_at(a, n);
  const float c = a.inv_temperature * kLog2e;
  MaxSum r = {-INFINITY, 0.f};
  if (tok != a.ignore_index && (int)threadIdx.x < parts)
    r = {a.parts[2 * (n * parts + threadIdx.x)], a.parts[2 * (n * parts + threadIdx.x) + 1]};
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    MaxSum o = {__shfl_xor(r.m, off, 64), __shfl_xor(r.s, off, 64)};
    r = join(r, o, c);
  }
  if (threadIdx.x == 0) write_row<T>(a, n, tok, row_at<T>(a, n), r);
}

template <typename T, int TPR, int BLOCK, int U, bool STREAM>
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
    const T* row = row_at<T>(a, n);
    // aligned to the row that is written; reads may be unaligned
    const int mis = (int)(((size_t)out & 15) / sizeof(T));
    const int head = min(mis ? N - mis : 0, a.vocab);
    const int vecs = (a.vocab - head) / N;
    const int tail = a.vocab - head - vecs * N;
    T* obody = out + head;
    // gridDim.y workgroups take a share of the row each
    const bool has_head = t < head && blockIdx.y == 0;
    const bool has_tail = TPR - 1 - t < tail && blockIdx.y == gridDim.y - 1;
    const int end = (int)((long)vecs * (blockIdx.y + 1) / gridDim.y);
    int v = (int)((long)vecs * blockIdx.y / gridDim.y) + t;
    if (g == 0.f) {  // a masked token: exact zeros, and its logits are not read
      const float zero[N] = {};
      if (has_head) out[t] = (T)0.f;
      if (has_tail) out[a.vocab - (TPR - t)] = (T)0.f;
      for (; v < end; v += TPR) store16<STREAM, T>(obody + (long)v * N, zero);
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
    if (has_head) one(t);
    if (has_tail) one(a.vocab - (TPR - t));
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
      store16<STREAM, T>(obody + (long)v * N, x);
    };
    for (; v + (U - 1) * TPR < end; v += U * TPR) {
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) load16<T>(body + (long)(v + u * TPR) * N, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) finish(v + u * TPR, x[u]);
    }
    if (v < end) {  // what is left, all loads at once
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) load16<T>(body + (long)min(v + u * TPR, end - 1) * N, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + u * TPR < end) finish(v + u * TPR, x[u]);
    }
  }
}

constexpr long kMaxBlocks = 1 << 20;

// A gradient that the last-level cache (256 MB) cannot hold next to its logits is
// written past it: what it would push out is what the passes around it read, and
// its own reader finds it in memory either way.  (A variant of the kernel, not a
// branch: the compiler joins the two stores into an ordinary one.)
constexpr long kStreamBytes = 128L << 20;

template <typename T, int TPR, int BLOCK, int U>
int log_probs_fwd(const TokenLogProbArgs& a, int parts, hipStream_t st) {
  const long rows = BLOCK / TPR;
  const long need = (a.rows + rows - 1) / rows;
  const dim3 grid((unsigned)(need < kMaxBlocks ? need : kMaxBlocks), parts);
  hipLaunchKernelGGL((token_log_probs_fwd_k<T, TPR, BLOCK, U>), grid, dim3(BLOCK), 0, st, a);
  if (parts > 1)
    hipLaunchKernelGGL((token_log_probs_join_k<T>), dim3((unsigned)a.rows), dim3(64), 0, st, a, parts);
  return (int)hipGetLastError();
}

template <typename T, int TPR, int BLOCK, int U>
int log_probs_bwd(const TokenLogProbArgs& a, int parts, hipStream_t st) {
  const long rows = BLOCK / TPR;
  const long need = (a.rows + rows - 1) / rows;
  const dim3 grid((unsigned)(need < kMaxBlocks ? need : kMaxBlocks), parts);
  if (a.rows * a.vocab * (long)sizeof(T) > kStreamBytes)
    hipLaunchKernelGGL((token_log_probs_bwd_k<T, TPR, BLOCK, U, true>), grid, dim3(BLOCK), 0, st, a);
  else
    hipLaunchKernelGGL((token_log_probs_bwd_k<T, TPR, BLOCK, U, false>), grid, dim3(BLOCK), 0, st, a);
  return (int)hipGetLastError();
}

// Workgroups to a long row where rows are few: as many as give every CU one, with
// 16 KB each at least (bf16, 1 / 8 / 64 rows of 100 KB, backward: 7.8 / 8.1 / 8.8 us
// with one, 6.3 / 6.3 / 7.2 shared; twice as many workgroups 6.3 / 6.3 / 9.1).
int shares_of_row(long bytes, long rows) {
  const long share = bytes / 16384, fill = 256 / rows;
  const long n = share < fill ? share : fill;
  return n < 1 ? 1 : n < 64 ? (int)n : 64;
}

// Threads to a row, by the row's bytes (MI355X, bf16, 8192 rows, forward /
// backward, us):
//             64 threads   256      512      1024
//    2.4 KB    14 / 13   18 / 19  35 / 41   55 / 63
//     10 KB    24 / 30   25 / 29  48 / 48   74 / 74
//     32 KB    47 / 98   46 / 89  57 / 98   91 / 117
//     64 KB    97 / 193  99 / 188 90 / 173 111 / 170
//    100 KB   146 / 311 146 / 301 137 / 287 158 / 270
// and for 256 rows of 10 KB, too few for a wave each, 7.4 / 7.4 with 64 threads
// and 6.2 / 6.3 with 256.
template <typename T>
int log_probs_dispatch(const TokenLogProbArgs& a, bool bwd, hipStream_t st) {
  const long bytes = (long)a.vocab * (long)sizeof(T);
  if (bytes <= 4096 || (bytes <= 8192 && a.rows >= 1024))
    return bwd ? log_probs_bwd<T, 64, 256, 8>(a, 1, st) : log_probs_fwd<T, 64, 256, 8>(a, 1, st);
  if (bytes <= 40960)
    return bwd ? log_probs_bwd<T, 256, 256, 4>(a, 1, st) : log_probs_fwd<T, 256, 256, 4>(a, 1, st);
  if (!bwd) return log_probs_fwd<T, 512, 512, 4>(a, a.parts ? token_log_probs_parts(&a) : 1, st);
  return log_probs_bwd<T, 1024, 1024, 4>(a, shares_of_row(bytes, a.rows), st);
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
//   ess = S^2 / (Q n) over all n places, S = sum r, Q = sum r^2;
//           dess/dlp = 2 / n (t - t^2) with t = r S / Q
//
// Whether a ratio is clipped is decided in double on x against the borders'
// logarithms, so that an element next to a border is treated as in the definition.
// e^y - 1 - y cancels near 0: a series there.  The objective's terms and all sums
// are in double, the exponential too: gains of either sign cancel, by 1e5 where
// advantages are few, and what float32 leaves in each would show (it costs 0.8 us
// of 18.8 at 4M tokens).  A gradient stands by itself and is computed in float32.
//
// One workgroup does everything up to 16K tokens (two launches cost more than
// its few passes); above, partial sums of many and a second launch that joins
// them in a fixed order: no atomics, the result does not depend on the order of
// execution.  Dense operands take 4 tokens to an access; any other strides or
// types go one by one through the runtime codes.  The row of a token (for an
// advantage per row) comes from a multiplication by the column count's
// reciprocal; 64-bit divisions took longer than the loads.  4M tokens with all
// terms: 19 + 4 us forward (54 MB; 2.9 TB/s in the first kernel), 17 us backward
// (71 MB, 4.3 TB/s); 8192 tokens 10 us forward, 4 backward.
// ---------------------------------------------------------------------------

__device__ __forceinline__ float operand(const PolicyOperand& o, long r, long c) {
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
      return (float)((const int*)o.ptr)[i];
    case RL_I64:
      return (float)((const long*)o.ptr)[i];
    case RL_I8:
      return ((const signed char*)o.ptr)[i];
    case RL_I16:
      return ((const short*)o.ptr)[i];
    default:
      return (float)((const double*)o.ptr)[i];
  }
}

// e^y - 1 - y
__device__ __forceinline__ float kl3(float y) {
  if (fabsf(y) > 0.5f) return exp2_hw(y * kLog2e) - 1.f - y;
  // y^2 (1/2! + y/3! + y^2/4! + ...), remainder below 2^-25 of the sum at 1/2
  float p = 1.f / 362880.f;
  p = fmaf(p, y, 1.f / 40320.f);
  p = fmaf(p, y, 1.f / 5040.f);
  p = fmaf(p, y, 1.f / 720.f);
  p = fmaf(p, y, 1.f / 120.f);
  p = fmaf(p, y, 1.f / 24.f);
  p = fmaf(p, y, 1.f / 6.f);
  p = fmaf(p, y, 0.5f);
  return y * y * p;
}

// e^y - 1, which stays -1 for y down to -inf.
__device__ __forceinline__ float kl3_slope(float y) {
  return fabsf(y) > 0.5f ? exp2_hw(y * kLog2e) - 1.f : kl3(y) + y;
}

struct PolicyToken {
  bool above, below;
  double x;
};

__device__ __forceinline__ PolicyToken policy_token(const PolicyLossArgs& a, float lp, float old) {
  PolicyToken t;
  t.x = (double)lp - (double)old;
  t.above = t.x > a.log_high;
  t.below = t.x < a.log_low;
  return t;
}

__device__ __forceinline__ bool clipped_against(const PolicyToken& t, float adv) {
  return (t.above && adv > 0.f) || (t.below && adv < 0.f);
}

enum { S_GAIN, S_KL, S_LP, S_W, S_R, S_RR, S_OFF, S_COUNT };

// One token's terms.
__device__ __forceinline__ void policy_terms(const PolicyLossArgs& a, float lp, float old, float adv,
                                             float w, float ref, bool has_ref, double (&s)[S_COUNT]) {
  const PolicyToken t = policy_token(a, lp, old);
  const double ratio = exp(t.x);
  s[S_R] += ratio;
  s[S_RR] += ratio * ratio;
  s[S_OFF] += t.x > a.log_off || t.below ? 1.0 : 0.0;
  if (w == 0.f) return;  // a masked token may hold anything, NaN too
  const double bound = t.above ? a.high : t.below ? a.low : ratio;
  const double gain = a.variant == 0 ? (clipped_against(t, adv) ? bound : ratio) * adv
                                     : bound * t.x * adv;
  s[S_GAIN] += w * gain;
  s[S_W] += w;
  s[S_LP] += (double)w * lp;
  if (has_ref) s[S_KL] += (double)w * kl3(ref - lp);
}

// The upstream gradients with their coefficients and 1 / D, or 2 / n.
struct PolicyUpstream {
  float go, gk, ge;
  float ess, ess_log2, ess_live;
};

__device__ __forceinline__ float policy_grad(const PolicyLossArgs& a, float lp, float old, float adv,
                                             float w, float ref, bool has_ref,
                                             const PolicyUpstream& u) {
  float e = 0.f;
  if (u.ess != 0.f) {  // of masked tokens too
    const float t = exp2_hw(fmaf((float)((double)lp - (double)old), kLog2e, u.ess_log2));
    e = u.ess * (t - u.ess_live * t * t);
  }
  if (w == 0.f) return e;
  const PolicyToken t = policy_token(a, lp, old);
  const float ratio = exp2_hw((float)t.x * kLog2e);
  const float dgain = a.variant == 0 ? (clipped_against(t, adv) ? 0.f : ratio * adv)
                                     : (t.above ? (float)a.high : t.below ? (float)a.low : ratio) * adv;
  float d = u.ge - u.go * dgain;
  if (has_ref) d -= u.gk * kl3_slope(ref - lp);
  return fmaf(d, w, e);
}

__device__ __forceinline__ void policy_finish(const PolicyLossArgs& a, const double (&s)[S_COUNT]) {
  const double n = (double)a.rows * (double)a.cols;
  const double inv = a.mean ? 1.0 / (s[S_W] > 1.0 || isnan(s[S_W]) ? s[S_W] : 1.0) : 1.0;
  const double objective = -s[S_GAIN] * inv;
  const double kl = s[S_KL] * inv;
  // a term without weight is left out: an infinite one times 0 would be NaN
  const double loss_kl = a.kl_coeff == 0.0 ? 0.0 : a.kl_coeff * kl;
  const double entropy = a.entropy_coeff == 0.0 ? 0.0 : a.entropy_coeff * (s[S_LP] * inv);
  a.out[0] = (float)(objective + loss_kl + entropy);
  a.out[1] = (float)objective;
  a.out[2] = (float)loss_kl;
  a.out[3] = (float)entropy;
  a.out[4] = (float)kl;
  a.out[5] = (float)(s[S_OFF] / n);
  a.out[6] = (float)(s[S_R] * s[S_R] / fmax(s[S_RR], 1e-9) / n);
  a.scale[0] = (float)inv;
  a.scale[1] = (float)log2(s[S_R] / fmax(s[S_RR], 1e-9));
  a.scale[2] = s[S_RR] >= 1e-9 ? 1.f : 0.f;
}

template <int BLOCK>
__device__ __forceinline__ bool block_sums(double (&s)[S_COUNT]) {
  __shared__ double part[BLOCK / 64][S_COUNT];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) s[k] += __shfl_xor(s[k], off, 64);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) part[threadIdx.x >> 6][k] = s[k];
  __syncthreads();
  if (threadIdx.x != 0) return false;
#pragma unroll
  for (int w = 1; w < BLOCK / 64; ++w)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) s[k] += part[w][k];
  return true;
}

// n / cols for n < 2^31.
__device__ __forceinline__ unsigned row_of(const PolicyLossArgs& a, unsigned n) {
  return (__umulhi(a.cols_magic, n) + n) >> a.cols_shift;
}

// Four tokens of dense operands.
struct Four {
  float lp[4], old[4], ref[4], adv[4], w[4];
};

template <typename T>
__device__ __forceinline__ void load4(const void* p, unsigned i, float (&x)[4]) {
  struct alignas(4 * sizeof(T)) Q {
    T x[4];
  };
  const Q q = *(const Q*)((const T*)p + i);
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = (float)q.x[k];
}

template <typename T>
__device__ __forceinline__ void load_four(const PolicyLossArgs& a, unsigned i, unsigned n, Four& f) {
  if (i + 4 <= n) {
    load4<T>(a.log_probs.ptr, i, f.lp);
    load4<T>(a.old_log_probs.ptr, i, f.old);
    if (a.ref.ptr) load4<T>(a.ref.ptr, i, f.ref);
    if (a.mask.ptr) load4<unsigned char>(a.mask.ptr, i, f.w);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned j = i + k < n ? i + k : n - 1;
      f.lp[k] = (float)((const T*)a.log_probs.ptr)[j];
      f.old[k] = (float)((const T*)a.old_log_probs.ptr)[j];
      if (a.ref.ptr) f.ref[k] = (float)((const T*)a.ref.ptr)[j];
      if (a.mask.ptr) f.w[k] = ((const unsigned char*)a.mask.ptr)[j];
    }
  }
  if (!a.mask.ptr) f.w[0] = f.w[1] = f.w[2] = f.w[3] = 1.f;
  if (a.advantage.stride_col) {  // one for each token
    const float* adv = (const float*)a.advantage.ptr;
    if (i + 4 <= n) {
      load4<float>(adv, i, f.adv);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) f.adv[k] = adv[i + k < n ? i + k : n - 1];
    }
    return;
  }
  // one for each row: a single value unless the four cross into the next
  unsigned r = row_of(a, i), c = i - r * (unsigned)a.cols;
  const float* adv = (const float*)a.advantage.ptr;
  f.adv[0] = adv[(long)r * a.advantage.stride_row];
  if (c + 4 <= (unsigned)a.cols) {
    f.adv[1] = f.adv[2] = f.adv[3] = f.adv[0];
  } else {
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      if (++c == (unsigned)a.cols) c = 0, ++r;
      f.adv[k] = adv[(long)(r < (unsigned)a.rows ? r : 0) * a.advantage.stride_row];
    }
  }
}

template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void policy_loss_dense_fwd_k(const PolicyLossArgs a) {
  double s[S_COUNT] = {};
  const unsigned n = (unsigned)(a.rows * a.cols);
  const bool has_ref = a.ref.ptr != nullptr;
  for (unsigned i = 4 * (blockIdx.x * BLOCK + threadIdx.x); i < n; i += 4 * gridDim.x * BLOCK) {
    Four f;
    load_four<T>(a, i, n, f);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n)
        policy_terms(a, f.lp[k], f.old[k], f.adv[k], f.w[k], has_ref ? f.ref[k] : 0.f, has_ref, s);
  }
  if (!block_sums<BLOCK>(s)) return;
  if (gridDim.x == 1) {
    policy_finish(a, s);
    return;
  }
#pragma unroll
  for (int k = 0; k < S_COUNT; ++k) a.partials[(long)blockIdx.x * 8 + k] = s[k];
}

template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void policy_loss_fwd_k(const PolicyLossArgs a) {
  double s[S_COUNT] = {};
  const long n = a.rows * a.cols;
  const bool has_ref = a.ref.ptr != nullptr;
  for (long i = (long)blockIdx.x * BLOCK + threadIdx.x; i < n; i += (long)gridDim.x * BLOCK) {
    const long r = n < (1L << 31) ? row_of(a, (unsigned)i) : i / a.cols, c = i - r * a.cols;
    policy_terms(a, operand(a.log_probs, r, c), operand(a.old_log_probs, r, c),
                 operand(a.advantage, r, c), a.mask.ptr ? operand(a.mask, r, c) : 1.f,
                 has_ref ? operand(a.ref, r, c) : 0.f, has_ref, s);
  }
  if (!block_sums<BLOCK>(s)) return;
  if (gridDim.x == 1) {
    policy_finish(a, s);
    return;
  }
#pragma unroll
  for (int k = 0; k < S_COUNT; ++k) a.partials[(long)blockIdx.x * 8 + k] = s[k];
}

__global__ __launch_bounds__(512) void policy_loss_join_k(const PolicyLossArgs a) {
  double s[S_COUNT] = {};
  for (int b = threadIdx.x; b < a.blocks; b += 512)
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) s[k] += a.partials[(long)b * 8 + k];
  if (block_sums<512>(s)) policy_finish(a, s);
}

__device__ __forceinline__ PolicyUpstream policy_upstream(const PolicyLossArgs& a) {
  const float inv = *a.scale;
  const float total = a.g_total ? *a.g_total : 0.f;
  return {(total + (a.g_objective ? *a.g_objective : 0.f)) * inv,
          (float)((total + (a.g_kl ? *a.g_kl : 0.f)) * a.kl_coeff * inv),
          (float)((total + (a.g_entropy ? *a.g_entropy : 0.f)) * a.entropy_coeff * inv),
          (a.g_ess ? *a.g_ess : 0.f) * (float)(2.0 / ((double)a.rows * (double)a.cols)), a.scale[1],
          a.scale[2]};
}

template <typename T>
__global__ __launch_bounds__(256) void policy_loss_dense_bwd_k(const PolicyLossArgs a) {
  const PolicyUpstream u = policy_upstream(a);
  const unsigned n = (unsigned)(a.rows * a.cols);
  const bool has_ref = a.ref.ptr != nullptr && a.kl_coeff != 0.f;
  struct alignas(4 * sizeof(T)) Q {
    T x[4];
  };
  for (unsigned i = 4 * (blockIdx.x * 256 + threadIdx.x); i < n; i += 4 * gridDim.x * 256) {
    Four f;
    load_four<T>(a, i, n, f);
    Q q;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      q.x[k] = (T)policy_grad(a, f.lp[k], f.old[k], f.adv[k], f.w[k], has_ref ? f.ref[k] : 0.f, has_ref,
                              u);
    if (i + 4 <= n) {
      *(Q*)((T*)a.grad + i) = q;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) ((T*)a.grad)[i + k] = q.x[k];
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void policy_loss_bwd_k(const PolicyLossArgs a) {
  const PolicyUpstream u = policy_upstream(a);
  const long n = a.rows * a.cols;
  const bool has_ref = a.ref.ptr != nullptr && a.kl_coeff != 0.f;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = n < (1L << 31) ? row_of(a, (unsigned)i) : i / a.cols, c = i - r * a.cols;
    ((T*)a.grad)[i] = (T)policy_grad(a, operand(a.log_probs, r, c), operand(a.old_log_probs, r, c),
                                     operand(a.advantage, r, c), a.mask.ptr ? operand(a.mask, r, c) : 1.f,
                                     has_ref ? operand(a.ref, r, c) : 0.f, has_ref, u);
  }
}

// Whether the dense kernels may take the operands: 4 tokens to an access.
bool policy_dense(const PolicyLossArgs& a) {
  const long n = a.rows * a.cols;
  auto dense = [&](const PolicyOperand& o, int dtype, long align) {
    return o.dtype == dtype && (o.stride_col == 1 || a.cols == 1) &&
           (o.stride_row == a.cols || a.rows == 1) && (size_t)o.ptr % align == 0;
  };
  const int t = a.log_probs.dtype;
  const long align = t == RL_F32 ? 16 : 8;
  return n < (1L << 31) - (1L << 22) && dense(a.log_probs, t, align) && dense(a.old_log_probs, t, align) &&
         (!a.ref.ptr || dense(a.ref, t, align)) && (!a.mask.ptr || dense(a.mask, RL_U8, 4)) &&
         (dense(a.advantage, RL_F32, 16) ||
          (a.advantage.dtype == RL_F32 && a.advantage.stride_col == 0));
}

// The reciprocal for row_of: with s = ceil(log2 d), magic = 2^32 (2^s - d) / d + 1.
void policy_divisor(PolicyLossArgs* a) {
  const unsigned long d = (unsigned long)a->cols;
  if (d >= (1ul << 31)) return;  // no 32-bit index is used then
  int s = 0;
  while ((1ul << s) < d) ++s;
  a->cols_shift = s;
  a->cols_magic = (unsigned)(((1ul << 32) * ((1ul << s) - d)) / d + 1);
}

template <typename T>
int policy_bwd(const PolicyLossArgs& a, hipStream_t st) {
  const long n = a.rows * a.cols;
  const bool dense = policy_dense(a);
  const long need = dense ? (n + 1023) / 1024 : (n + 255) / 256;
  const dim3 grid((unsigned)(need < 4096 ? need : 4096));
  if (dense)
    hipLaunchKernelGGL((policy_loss_dense_bwd_k<T>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((policy_loss_bwd_k<T>), grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

template <int BLOCK>
void policy_fwd_block(const PolicyLossArgs& a, bool dense, hipStream_t st) {
  const dim3 grid(a.blocks), block(BLOCK);
  if (!dense)
    hipLaunchKernelGGL((policy_loss_fwd_k<BLOCK>), grid, block, 0, st, a);
  else if (a.log_probs.dtype == RL_F32)
    hipLaunchKernelGGL((policy_loss_dense_fwd_k<float, BLOCK>), grid, block, 0, st, a);
  else if (a.log_probs.dtype == RL_BF16)
    hipLaunchKernelGGL((policy_loss_dense_fwd_k<__bf16, BLOCK>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((policy_loss_dense_fwd_k<_Float16, BLOCK>), grid, block, 0, st, a);
}

}  // namespace

// Workgroups that share a row forward.  A second launch joins them, so only rows
// long enough to pay for it are split (bf16, 8 / 64 rows, one workgroup each ->
// shared and joined, us): 100 KB 8.8 / 9.0 -> 9.3 / 9.9, 160 KB 10.4 / 10.7 ->
// 9.3 / 10.6, 256 KB 12.4 / 12.7 -> 9.3 / 11.0, 320 KB 14.1 / 14.5 -> 9.2 / 11.4; the
// second launch also takes the host 2 us.
extern "C" int token_log_probs_parts(const TokenLogProbArgs* a) {
  const long bytes = (long)a->vocab * (a->dtype == RL_F32 ? 4 : 2);
  if (bytes <= (192L << 10) || a->rows > 64 || a->rows < 1) return 1;
  return shares_of_row(bytes, a->rows);
}

extern "C" int launch_token_log_probs_fwd(const TokenLogProbArgs* a, void* stream) {
  return log_probs_any(a, false, stream);
}

extern "C" int launch_token_log_probs_bwd(const TokenLogProbArgs* a, void* stream) {
  return log_probs_any(a, true, stream);
}

extern "C" int policy_loss_blocks(long n) {
  if (n <= 16384) return 1;
  const long b = (n + 2047) / 2048;
  return (int)(b < 512 ? b : 512);
}

extern "C" int launch_policy_loss_fwd(const PolicyLossArgs* args, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  PolicyLossArgs a = *args;
  policy_divisor(&a);
  const bool dense = policy_dense(a);
  if (a.blocks > 1) {
    policy_fwd_block<512>(a, dense, st);
    hipLaunchKernelGGL(policy_loss_join_k, dim3(1), dim3(512), 0, st, a);
  } else if (a.rows * a.cols <= 1024) {
    policy_fwd_block<256>(a, dense, st);
  } else {
    policy_fwd_block<1024>(a, dense, st);
  }
  return (int)hipGetLastError();
}

extern "C" int launch_policy_loss_bwd(const PolicyLossArgs* args, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  PolicyLossArgs a = *args;
  policy_divisor(&a);
  switch (a.log_probs.dtype) {
    case RL_F32:
      return policy_bwd<float>(a, st);
    case RL_BF16:
      return policy_bwd<__bf16>(a, st);
    case RL_F16:
      return policy_bwd<_Float16>(a, st);
  }
  return (int)hipErrorInvalidValue;
}
