// Paged key-value cache kernels for CDNA4 (gfx950): the append with its
// position rotation, and attention of one new token per sequence.
//
// The cache is [pages][kv_heads][page_size][dim]: one head's page is one dense
// run of page_size * dim elements, so the attention streams whole pages, and a
// page id (32 bits) times the page's stride is the only 64-bit offset.
//
// paged_append.  Dims (i, i + R/2) (or (2i, 2i + 1) when interleaved) of a key
// or query at position p turn by the angle whose cosine and sine stand in row p
// of the tables:  a' = a cos - b sin,  b' = b cos + a sin, in fp32, rounded once
// to the cache's type.  A thread owns a pair of chunks of `vec` elements (the
// two halves of a rotation, or two plain ones) at the same place of every head
// it visits, and keeps its cosines and sines for all of them.  Bound by HBM (it
// reads and writes everything once), by the launch for single tokens.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>

#include "paged_kv.h"
#include "token_loss.h"

namespace {

__device__ __forceinline__ long whole(const void* p, int i64, long i) {
  return i64 ? ((const long*)p)[i] : (long)((const int*)p)[i];
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T x[VEC];
};

// One lane's place within a head: two chunks, rotated against each other
// (interleaved: each within itself) or copied.
struct Place {
  int first, second;  // element offsets; second < 0: none
  bool turn;
  int angle0, angle1;  // first column of the tables for each chunk
};

template <int VEC>
__device__ __forceinline__ Place place_of(int item, int dim, int rotary, int interleaved) {
  Place p;
  const int turning = rotary / 2 / VEC;
  p.turn = item < turning;
  if (p.turn && !interleaved) {
    p.first = item * VEC;
    p.second = p.first + rotary / 2;
    p.angle0 = p.angle1 = item * VEC;
  } else if (p.turn) {
    p.first = 2 * item * VEC;
    p.second = p.first + VEC;
    p.angle0 = item * VEC;
    p.angle1 = item * VEC + VEC / 2;
  } else {
    p.first = rotary + 2 * (item - turning) * VEC;
    p.second = p.first + VEC < dim ? p.first + VEC : -1;
    p.angle0 = p.angle1 = 0;
  }
  return p;
}

template <int VEC>
__device__ __forceinline__ int places(int dim, int rotary) {
  return rotary / 2 / VEC + ((dim - rotary) / VEC + 1) / 2;
}

// LANES lanes share a head; 256 / LANES heads are worked on at once, of one
// token, or of several when a token has fewer heads than that.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void paged_append_k(const PagedAppendArgs a, int lanes_shift,
                                                      int tokens_shift) {
  using C = Chunk<T, VEC>;
  const int lanes = 1 << lanes_shift;
  const int item = threadIdx.x & (lanes - 1);
  const int slots = 256 >> lanes_shift;             // heads at once
  const int per_token = slots >> tokens_shift;      // heads of one token at once
  const int slot = threadIdx.x >> lanes_shift;
  const int rows = a.q ? a.heads : 0;
  const int all = rows + 2 * a.kv_heads;
  const int page_size = 1 << a.cache.page_shift;
  const long tokens = a.batch * a.width;
  const long token = ((long)blockIdx.x << tokens_shift) + slot / per_token;
  if (token >= tokens) return;
  const long b = token / a.width;
  const int t = (int)(token - b * a.width);
  const long length = a.lengths ? whole(a.lengths, a.lengths_i64, b) : a.width;
  const bool live = t < length;
  if (!live && !rows) return;
  const long pos = whole(a.start, a.start_i64, b) + t;
  // where the token's keys and values go; page < 0: nowhere
  long page = -1;
  if (live && pos >= 0 && (pos >> a.cache.page_shift) < a.cache.table_cols) {
    page = a.cache.table[b * a.cache.table_stride + (pos >> a.cache.page_shift)];
    if (page >= a.cache.pages) page = -1;
  }
  const int in_page = (int)(pos & (page_size - 1));

  const int turned = places<VEC>(a.dim, a.rotary);
  const int plain = places<VEC>(a.dim, 0);
  const Place rot = place_of<VEC>(item, a.dim, a.rotary, a.interleaved);
  const Place copy = place_of<VEC>(item, a.dim, 0, 0);
  float cs0[VEC], sn0[VEC], cs1[VEC], sn1[VEC];
  if (a.rotary && rot.turn && item < turned && live) {
    const bool inside = pos >= 0 && pos < a.positions;
    const long row = inside ? pos * (a.rotary / 2) : 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      // interleaved: element i of a chunk belongs to pair i / 2
      const int j0 = a.interleaved ? rot.angle0 + i / 2 : rot.angle0 + i;
      cs0[i] = inside ? a.cos[row + j0] : NAN;
      sn0[i] = inside ? a.sin[row + j0] : NAN;
      if (a.interleaved) {
        const int j1 = rot.angle1 + i / 2;
        cs1[i] = inside ? a.cos[row + j1] : NAN;
        sn1[i] = inside ? a.sin[row + j1] : NAN;
      }
    }
  }
  for (int h = slot % per_token; h < all; h += per_token) {
    const bool is_q = h < rows, is_v = h >= rows + a.kv_heads;
    const Place p = is_v ? copy : rot;
    if (item >= (is_v ? plain : turned)) continue;
    const T* src;
    T* dst;
    if (is_q) {
      src = (const T*)a.q + b * a.q_batch + t * a.q_token + h * a.q_head;
      dst = (T*)a.q_out + (token * a.heads + h) * a.dim;
    } else {
      if (page < 0) continue;
      if (is_v) {
        const int g = h - rows - a.kv_heads;
        src = (const T*)a.v + b * a.v_batch + t * a.v_token + g * a.v_head;
        dst = (T*)a.cache.v + page * a.cache.v_page + g * a.cache.v_head +
              in_page * a.cache.v_slot;
      } else {
        const int g = h - rows;
        src = (const T*)a.k + b * a.k_batch + t * a.k_token + g * a.k_head;
        dst = (T*)a.cache.k + page * a.cache.k_page + g * a.cache.k_head +
              in_page * a.cache.k_slot;
      }
    }
    C x{}, y{};
    if (live) {
      x = *(const C*)(src + p.first);
      if (p.second >= 0) y = *(const C*)(src + p.second);
    }
    if (live && !is_v && p.turn) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i + 1 < VEC; i += 2) {
          const float p0 = (float)x.x[i], p1 = (float)x.x[i + 1];
          x.x[i] = (T)(p0 * cs0[i] - p1 * sn0[i]);
          x.x[i + 1] = (T)(p1 * cs0[i] + p0 * sn0[i]);
          const float r0 = (float)y.x[i], r1 = (float)y.x[i + 1];
          y.x[i] = (T)(r0 * cs1[i] - r1 * sn1[i]);
          y.x[i + 1] = (T)(r1 * cs1[i] + r0 * sn1[i]);
        }
        if (VEC == 1) {  // a pair is the two chunks
          const float p0 = (float)x.x[0], p1 = (float)y.x[0];
          x.x[0] = (T)(p0 * cs0[0] - p1 * sn0[0]);
          y.x[0] = (T)(p1 * cs0[0] + p0 * sn0[0]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float p0 = (float)x.x[i], p1 = (float)y.x[i];
          x.x[i] = (T)(p0 * cs0[i] - p1 * sn0[i]);
          y.x[i] = (T)(p1 * cs0[i] + p0 * sn0[i]);
        }
      }
    }
    *(C*)(dst + p.first) = x;
    if (p.second >= 0) *(C*)(dst + p.second) = y;
  }
}

template <typename T, int VEC>
int append_launch(const PagedAppendArgs& a, hipStream_t st) {
  const int rot = a.rotary / 2 / VEC + ((a.dim - a.rotary) / VEC + 1) / 2;
  const int plain = (a.dim / VEC + 1) / 2;
  const int most = rot > plain ? rot : plain;
  int lanes_shift = 0;
  while ((1 << lanes_shift) < most) ++lanes_shift;  // dim <= 512: at most 256
  const int all = (a.q ? a.heads : 0) + 2 * a.kv_heads;
  int tokens_shift = 0;  // whole tokens that fit the workgroup's head slots
  while ((256 >> lanes_shift >> (tokens_shift + 1)) >= all) ++tokens_shift;
  const long tokens = a.batch * a.width;
  const long blocks = (tokens + (1L << tokens_shift) - 1) >> tokens_shift;
  hipLaunchKernelGGL((paged_append_k<T, VEC>), dim3((unsigned)blocks), dim3(256), 0, st, a,
                     lanes_shift, tokens_shift);
  return (int)hipGetLastError();
}

template <typename T, int WIDE>
int append_vec(const PagedAppendArgs& a, hipStream_t st) {
  if (a.vec >= WIDE) return append_launch<T, WIDE>(a, st);
  return append_launch<T, 1>(a, st);
}

// ---------------------------------------------------------------------------
// paged_attend, the simple form: one workgroup per (sequence, head), its four
// waves over every fourth key, 64 lanes over the dims, the running maximum and
// sum of the softmax in fp32, and one join at the end.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void paged_attend_simple_k(const PagedAttendArgs a) {
  constexpr int MAXD = 8;  // dim <= 512
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long b = blockIdx.x / a.heads;
  const int h = (int)(blockIdx.x % a.heads);
  const int kv = h / (a.heads / a.kv_heads);
  long len = whole(a.lengths, a.lengths_i64, b);
  const long room = (long)a.cache.table_cols << a.cache.page_shift;
  len = len < room ? len : room;
  const T* q = (const T*)a.q + b * a.q_batch + h * a.q_head;
  float qv[MAXD], acc[MAXD] = {};
#pragma unroll
  for (int i = 0; i < MAXD; ++i) qv[i] = lane + 64 * i < a.dim ? (float)q[lane + 64 * i] : 0.f;
  float m = -INFINITY, l = 0.f;
  for (long key = wave; key < len; key += 4) {
    const long page = a.cache.table[b * a.cache.table_stride + (key >> a.cache.page_shift)];
    if (page < 0 || page >= a.cache.pages) continue;
    const long slot = key & ((1 << a.cache.page_shift) - 1);
    const T* k = (const T*)a.cache.k + page * a.cache.k_page + kv * a.cache.k_head + slot * a.cache.k_slot;
    const T* v = (const T*)a.cache.v + page * a.cache.v_page + kv * a.cache.v_head + slot * a.cache.v_slot;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < MAXD; ++i)
      if (lane + 64 * i < a.dim) s += qv[i] * (float)k[lane + 64 * i];
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    s *= a.scale;
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
    const float p = s == -INFINITY ? 0.f : exp2f(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < MAXD; ++i)
      if (lane + 64 * i < a.dim) acc[i] = acc[i] * keep + p * (float)v[lane + 64 * i];
  }
  __shared__ float sm[4], sl[4], sacc[4][512];
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < MAXD; ++i)
    if (lane + 64 * i < a.dim) sacc[wave][lane + 64 * i] = acc[i];
  __syncthreads();
  float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], total = 0.f;
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - top);
    total += f[w] * sl[w];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* out = (T*)a.out + (b * a.heads + h) * a.dim;
  for (int d = threadIdx.x; d < a.dim; d += 256) {
    float o = 0.f;
    for (int w = 0; w < 4; ++w) o += f[w] * sacc[w][d];
    out[d] = (T)(o * inv);
  }
}

template <typename T>
int attend_simple(const PagedAttendArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((paged_attend_simple_k<T>), dim3((unsigned)(a.batch * a.heads)), dim3(256), 0,
                     st, a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int launch_paged_append(const PagedAppendArgs* a, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  switch (a->dtype) {
    case RL_F32:
      return append_vec<float, 4>(*a, st);
    case RL_BF16:
      return append_vec<__bf16, 8>(*a, st);
    case RL_F16:
      return append_vec<_Float16, 8>(*a, st);
  }
  return (int)hipErrorInvalidValue;
}

extern "C" int launch_paged_attend(const PagedAttendArgs* a, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  switch (a->dtype) {
    case RL_F32:
      return attend_simple<float>(*a, st);
    case RL_BF16:
      return attend_simple<__bf16>(*a, st);
    case RL_F16:
      return attend_simple<_Float16>(*a, st);
  }
  return (int)hipErrorInvalidValue;
}
