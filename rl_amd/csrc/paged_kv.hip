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
// (interleaved: each within itself) or copied.  Either way the two belong to the
// angles [item * VEC, (item + 1) * VEC).
struct Place {
  int first, second;  // element offsets; second < 0: none
  bool turn;
};

template <int VEC>
__device__ __forceinline__ Place place_of(int item, int dim, int rotary, int interleaved) {
  const int turning = rotary / 2 / VEC;
  Place p;
  p.turn = item < turning;
  if (p.turn) {
    p.first = interleaved ? 2 * item * VEC : item * VEC;
    p.second = interleaved ? p.first + VEC : p.first + rotary / 2;
  } else {
    p.first = rotary + 2 * (item - turning) * VEC;
    p.second = p.first + VEC < dim ? p.first + VEC : -1;
  }
  return p;
}

template <int VEC>
__host__ __device__ constexpr int places(int dim, int rotary) {
  return rotary / 2 / VEC + ((dim - rotary) / VEC + 1) / 2;
}

// 1 << lanes_shift lanes share a head; the workgroup's slots take `per_token`
// heads of a token at a time, and `tokens_here` tokens where those are all.  One
// head on the way per thread and many threads: two or three heads at a time cost
// registers and ran at 4.2 and 4.1 TB/s where this runs at 5.0 (32768 tokens of
// 32 + 16 heads of 128, bf16).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void paged_append_k(const PagedAppendArgs a, int lanes_shift,
                                                      int per_token, int tokens_here) {
  using C = Chunk<T, VEC>;
  const int item = threadIdx.x & ((1 << lanes_shift) - 1);
  const int slot = threadIdx.x >> lanes_shift;
  const int rows = a.q ? a.heads : 0;
  const int all = rows + 2 * a.kv_heads;
  const int page_size = 1 << a.cache.page_shift;
  const long tokens = a.batch * a.width;
  const int sub = tokens_here > 1 ? slot / per_token : 0;
  const long token = (long)blockIdx.x * tokens_here + sub;
  if (token >= tokens || sub >= tokens_here) return;
  const long b = (unsigned)token / (unsigned)a.width;  // at most 2^24 tokens
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
  float cs[VEC], sn[VEC];
  if (a.rotary && rot.turn && live) {
    if (pos >= 0 && pos < a.positions) {
      __builtin_memcpy(cs, a.cos + pos * (a.rotary / 2) + item * VEC, sizeof(cs));
      __builtin_memcpy(sn, a.sin + pos * (a.rotary / 2) + item * VEC, sizeof(sn));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) cs[i] = sn[i] = NAN;
    }
  }
  const T* qsrc = (const T*)a.q + b * a.q_batch + t * a.q_token;
  const T* ksrc = (const T*)a.k + b * a.k_batch + t * a.k_token;
  const T* vsrc = (const T*)a.v + b * a.v_batch + t * a.v_token;
  T* qdst = (T*)a.q_out + token * a.heads * a.dim;
  T* kdst = (T*)a.cache.k + page * a.cache.k_page + in_page * a.cache.k_slot;
  T* vdst = (T*)a.cache.v + page * a.cache.v_page + in_page * a.cache.v_slot;
  for (int h = slot - sub * per_token; h < all; h += per_token) {
    const bool is_q = h < rows, is_v = h >= rows + a.kv_heads;
    if (item >= (is_v ? plain : turned) || (!is_q && page < 0)) continue;
    const Place p = is_v ? copy : rot;
    const int g = is_q ? h : is_v ? h - rows - a.kv_heads : h - rows;
    const T* src = is_q ? qsrc + g * a.q_head : is_v ? vsrc + g * a.v_head : ksrc + g * a.k_head;
    T* dst = is_q ? qdst + g * a.dim : is_v ? vdst + g * a.cache.v_head : kdst + g * a.cache.k_head;
    C x{}, y{};
    if (live) {
      x = *(const C*)(src + p.first);
      if (p.second >= 0) y = *(const C*)(src + p.second);
      if (!is_v && p.turn) {
        if (a.interleaved && VEC > 1) {
#pragma unroll
          for (int i = 0; i + 1 < VEC; i += 2) {
            const float p0 = (float)x.x[i], p1 = (float)x.x[i + 1];
            x.x[i] = (T)(p0 * cs[i / 2] - p1 * sn[i / 2]);
            x.x[i + 1] = (T)(p1 * cs[i / 2] + p0 * sn[i / 2]);
            const float r0 = (float)y.x[i], r1 = (float)y.x[i + 1];
            y.x[i] = (T)(r0 * cs[VEC / 2 + i / 2] - r1 * sn[VEC / 2 + i / 2]);
            y.x[i + 1] = (T)(r1 * cs[VEC / 2 + i / 2] + r0 * sn[VEC / 2 + i / 2]);
          }
        } else {  // the two chunks against each other (VEC 1: an interleaved pair too)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float p0 = (float)x.x[i], p1 = (float)y.x[i];
            x.x[i] = (T)(p0 * cs[i] - p1 * sn[i]);
            y.x[i] = (T)(p1 * cs[i] + p0 * sn[i]);
          }
        }
      }
    }
    *(C*)(dst + p.first) = x;
    if (p.second >= 0) *(C*)(dst + p.second) = y;
  }
}

template <typename T, int VEC>
int append_launch(const PagedAppendArgs& a, hipStream_t st) {
  const int rot = places<VEC>(a.dim, a.rotary), plain = places<VEC>(a.dim, 0);
  const int most = rot > plain ? rot : plain;
  int lanes_shift = 0;
  while ((1 << lanes_shift) < most) ++lanes_shift;  // dim <= 256: at most 128 lanes
  const int all = (a.q ? a.heads : 0) + 2 * a.kv_heads;
  // the workgroup of 1 to 4 waves whose slots are idle least, the larger of equals
  int threads = 256, per_token = 256 >> lanes_shift, tokens_here = 1;
  long best = -1;
  for (int n = 64; n <= 256; n += 64) {
    const int slots = n >> lanes_shift;
    if (slots < 1) continue;
    const int here = slots >= all ? slots / all : 1;
    const int passes = (all + slots - 1) / slots;
    const long busy = 4096L * here * all / ((long)slots * passes);
    if (busy >= best) {
      best = busy;
      threads = n;
      tokens_here = here;
      per_token = here > 1 ? all : slots;
    }
  }
  const long tokens = a.batch * a.width;
  const long blocks = (tokens + tokens_here - 1) / tokens_here;
  hipLaunchKernelGGL((paged_append_k<T, VEC>), dim3((unsigned)blocks), dim3(threads), 0, st, a,
                     lanes_shift, per_token, tokens_here);
  return (int)hipGetLastError();
}

template <typename T, int WIDE>
int append_vec(const PagedAppendArgs& a, hipStream_t st) {
  if (a.vec >= WIDE) return append_launch<T, WIDE>(a, st);
  return append_launch<T, 1>(a, st);
}

// ---------------------------------------------------------------------------
// paged_attend: out = softmax(scale q k^T) v for one query token per sequence.
//
// The G = heads / kv_heads query heads that share a key head are the 16 columns
// of one matrix tile (padded; more than 16 take ceil(G / 16) blocks).  Both
// products are turned so that a lane keeps one query head throughout:
//
//   S^T [keys x heads] = K Q^T     A = K: lane l holds 16 bytes of key row l % 16,
//                                  straight from the cache, no shared memory
//   O^T [dims x heads] = V^T P^T   B = P: what the first product and the softmax
//                                  left in the lane's registers is its operand
//                                  (the order of the keys within a product is
//                                  free); A = V^T comes through shared memory
//                                  with a transposing read
//
// so the running maximum, the sum and the rescaling of the output are per lane,
// and a tile of keys costs two shuffles.  Weights enter the second product as
// two 16-bit parts (the rounded weight and what it left), so that they are not
// rounded to 8 bits for bfloat16; the matrix unit has the time, the kernel is
// bound by the cache's bytes.  float32 caches use the fp32 matrix instruction on
// tiles of 16 keys, with V's operand read directly.
//
// A wave owns whole tiles: while it computes one, the keys, values and page ids
// of the next are on their way in its registers.  No barrier in the loop.
//
// Work is split over the cache's length.  The tiles of all (sequence, key head)
// items form one line, and worker w of W takes the tiles [w n / W, (w + 1) n / W)
// of it, whatever items they belong to: ragged batches and single long sequences
// fill the card alike, without the host knowing a length.  A worker's first and
// last item may be shared with its neighbours; their parts (maximum, sum and
// unnormalised output) go to its two workspace slots and a second launch joins
// them in order.  Sequences of length 0 count one empty tile and get zeros.
// ---------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Matrix;

template <>
struct Matrix<__bf16> {
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Matrix<_Float16> {
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// A value that is the same in every lane of the wave, as the compiler's scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long uniform(long x) {
  const int lo = uniform((int)x), hi = uniform((int)(x >> 32));
  return ((long)hi << 32) | (unsigned)lo;
}

// An item that several workers shared; parts == 0: none begins here.
struct SharedItem {
  long b;
  int item, worker, parts, slot;  // the first part's worker and slot
};

struct AttendPlan {
  int workers;     // 0: one workgroup per item, nothing shared
  int blocks;      // head blocks of 16 per key head
  SharedItem* notes;  // [workers]
  float* part;     // [2 * workers][min(16, G)][dim] unnormalised outputs
  float* part_ms;  // [2 * workers][min(16, G)][2] maximum and sum
};

__device__ __forceinline__ int tiles_of(const PagedAttendArgs& a, long b, int tile) {
  long len = whole(a.lengths, a.lengths_i64, b);
  const long room = (long)a.cache.table_cols << a.cache.page_shift;
  len = len < room ? len : room;
  return len > 0 ? (int)((len + tile - 1) / tile) : 1;
}

// Where sequence `b` and its items lie on the line of all tiles.
struct Spot {
  long b;
  long first;  // place of its first tile
  int tiles;   // of one of its items
};

// The line as one wave sees it: up to 64 sequences in its lanes, more in passes.
struct Line {
  int mine;   // tiles of an item of sequence `lane` (batches up to 64)
  long upto;  // inclusive sum over sequences, times the items of a sequence
  long total;
};

__device__ __forceinline__ void line_pass(const PagedAttendArgs& a, long per, int tile, long b0,
                                          Line& x) {
  const int lane = threadIdx.x & 63;
  x.mine = b0 + lane < a.batch ? tiles_of(a, b0 + lane, tile) : 0;
  x.upto = (long)x.mine * per;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const long o = __shfl_up(x.upto, off, 64);
    if (lane >= off) x.upto += o;
  }
}

__device__ __forceinline__ Line line_of(const PagedAttendArgs& a, long per, int tile) {
  Line x;
  if (a.batch <= 64) {
    line_pass(a, per, tile, 0, x);
    x.total = uniform(__shfl(x.upto, 63, 64));
    return x;
  }
  long n = 0;
  for (long b = threadIdx.x & 63; b < a.batch; b += 64) n += tiles_of(a, b, tile);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  x.mine = 0;
  x.upto = 0;
  x.total = uniform(n) * per;
  return x;
}

// The sequence of tile `at`.
__device__ __forceinline__ Spot spot_of(const PagedAttendArgs& a, long per, int tile, Line x, long at) {
  const int lane = threadIdx.x & 63;
  long before = 0;
  for (long b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) line_pass(a, per, tile, b0, x);
    const bool here = b0 + lane < a.batch && before + x.upto > at;
    const unsigned long long hit = __ballot(here);
    if (hit) {
      const int l = __ffsll((long long)hit) - 1;
      const int tiles = uniform(__shfl(x.mine, l, 64));
      return {uniform(b0 + l), before + uniform(__shfl(x.upto, l, 64)) - (long)tiles * per, tiles};
    }
    before += uniform(__shfl(x.upto, 63, 64));
  }
  return {a.batch, before, 1};  // not reached: `at` < total
}

// x * y / z of whole numbers, 64-bit divisions only where 32 bits do not hold.
__device__ __forceinline__ long share(long x, long y, long z) {
  const long p = x * y;
  return (p | z) < (1L << 32) ? (long)((unsigned)p / (unsigned)z) : p / z;
}

// Workers that get work: at least one tile to each of a workgroup's waves.
__device__ __forceinline__ long busy_workers(long workers, long total, int waves) {
  const long most = (total + waves - 1) / waves;
  return workers < most ? workers : most;
}

// The dim that the next smaller DP takes: chunks below it are never past `dim`.
template <int DP>
constexpr int smaller_dim() {
  return DP <= 64 ? 0 : DP <= 96 ? 64 : DP <= 128 ? 96 : DP <= 192 ? 128 : 192;
}

// What one wave carries through its tiles of one item.
template <typename T, int DP>
struct Tiles;

// 16-bit caches: tiles of 32 keys.
template <typename T, int DP>
struct Tiles {
  using V8 = typename Matrix<T>::V8;
  static constexpr int KEYS = 32;
  static constexpr int J = DP / 32;
  // a row of V in shared memory, padded so that the transposing read of 16 rows
  // and the 16-byte writes of 16 rows both spread over all banks
  static constexpr int PITCH = DP + 16;
  static constexpr int LDS_BYTES = KEYS * PITCH * 2;
  // whether chunks of column block j can lie past `dim`
  static constexpr bool edge(int j) { return 32 * j + 32 > smaller_dim<DP>(); }
  V8 q[J], k[2][J], v[2][J];
  f32x4 acc[DP / 16];
  float m, l;

  __device__ __forceinline__ void start(const T* qrow, bool live, int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 8;
      q[j] = V8{};
      if (live && d < dim) q[j] = *(const V8*)(qrow + d);
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }

  template <bool EXACT>
  __device__ __forceinline__ void fetch(V8 (&x)[2][J], const T* base, const long (&row)[2], int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* p = base + row[h];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int d = (chunk + 4 * j) * 8;
        // columns past dim: the row's first ones again, cleared before use
        x[h][j] = *(const V8*)(p + (EXACT || !edge(j) || d < dim ? d : 0));
      }
    }
  }

  template <bool EXACT>
  __device__ __forceinline__ void scores(f32x4 (&s)[2], int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        V8 x = k[h][j];
        if (!EXACT && edge(j) && (chunk + 4 * j) * 8 >= dim) x = V8{};
        s[h] = Matrix<T>::mul(x, q[j], s[h]);
      }
    }
  }

  // `ok`: bit i of ok[h] says that key 16 h + i counts.
  __device__ __forceinline__ void weigh(f32x4 (&s)[2], float scale, const unsigned (&ok)[2], bool full,
                                        V8& hi, V8& lo) {
    const int group = (threadIdx.x & 63) >> 4;
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] *= scale;
        if (!full && !((ok[h] >> (4 * group + r)) & 1)) s[h][r] = -INFINITY;
        top = fmaxf(top, s[h][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m)) {
      const float next = fmaxf(m, top);
      const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) acc[i] *= keep;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(s[h][r] - off);
        l += p;
        hi[4 * h + r] = (T)p;
        lo[4 * h + r] = (T)(p - (float)hi[4 * h + r]);
      }
  }

  __device__ __forceinline__ void stage(T* lds, const unsigned (&ok)[2], bool full) {
    const int lane = threadIdx.x & 63, row = lane & 15, chunk = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool clear = !full && !((ok[h] >> row) & 1);
#pragma unroll
      for (int j = 0; j < J; ++j)
        *(V8*)(lds + (16 * h + row) * PITCH + (chunk + 4 * j) * 8) = clear ? V8{} : v[h][j];
    }
  }

  __device__ __forceinline__ void gather(const T* lds, V8 hi, V8 lo) {
    const int lane = threadIdx.x & 63, i = lane & 15, group = lane >> 4;
    const T* p = lds + (4 * group + i / 4) * PITCH + (i % 4) * 4;
    typedef __attribute__((address_space(3))) s16x4* Shared;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      union {
        s16x4 half[2];
        V8 all;
      } x;
      x.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(p + 16 * d));
      x.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(p + 16 * PITCH + 16 * d));
      acc[d] = Matrix<T>::mul(x.all, hi, acc[d]);
      acc[d] = Matrix<T>::mul(x.all, lo, acc[d]);
    }
  }
};

// Orders a wave's own shared-memory writes before its reads of other lanes'
// values, and the other way round.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename T, int DP, bool EXACT>
__device__ __forceinline__ void run_tiles(Tiles<T, DP>& w, const PagedAttendArgs& a, long b, int kv,
                                          int len, int t, int end, int step, T* lds) {
  constexpr int KEYS = Tiles<T, DP>::KEYS;
  const int row = threadIdx.x & 15;
  const int* table = a.cache.table + b * a.cache.table_stride;
  const T* kbase = (const T*)a.cache.k + kv * a.cache.k_head;
  const T* vbase = (const T*)a.cache.v + kv * a.cache.v_head;
  const int slot_mask = (1 << a.cache.page_shift) - 1;
  int page[2];
  unsigned ok[2], ok_next[2];
  long krow[2], vrow[2];
  auto pages = [&](int tile) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = tile * KEYS + 16 * h + row;
      page[h] = key < len ? table[key >> a.cache.page_shift] : -1;
    }
  };
  // rows to read of a tile; keys that do not count read the cache's first row
  auto resolve = [&](int tile, unsigned (&good)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = tile * KEYS + 16 * h + row;
      const bool fine = page[h] >= 0 && page[h] < a.cache.pages;
      const long slot = key & slot_mask;
      krow[h] = fine ? page[h] * a.cache.k_page + slot * a.cache.k_slot : 0;
      vrow[h] = fine ? page[h] * a.cache.v_page + slot * a.cache.v_slot : 0;
      good[h] = (unsigned)__ballot(fine) & 0xffffu;
    }
  };
  if (t >= end) return;
  pages(t);
  resolve(t, ok);
  if (t + step < end) pages(t + step);
  w.template fetch<EXACT>(w.k, kbase, krow, a.dim);
  w.template fetch<EXACT>(w.v, vbase, vrow, a.dim);
  for (; t < end; t += step) {
    const bool more = t + step < end;
    if (more) {
      resolve(t + step, ok_next);
      if (t + 2 * step < end) pages(t + 2 * step);  // ahead of the loads that follow
    }
    f32x4 s[2];
    typename Tiles<T, DP>::V8 hi, lo;
    w.template scores<EXACT>(s, a.dim);
    if (more) w.template fetch<EXACT>(w.k, kbase, krow, a.dim);
    const bool full = (ok[0] & ok[1]) == 0xffffu;
    w.weigh(s, a.scale, ok, full, hi, lo);
    w.stage(lds, ok, full);
    if (more) w.template fetch<EXACT>(w.v, vbase, vrow, a.dim);
    wave_sync();
    w.gather(lds, hi, lo);
    wave_sync();
    ok[0] = ok_next[0];
    ok[1] = ok_next[1];
  }
}

// float32 caches: tiles of 16 keys, the fp32 matrix instruction.
template <int DP>
struct Tiles<float, DP> {
  static constexpr int KEYS = 16;
  static constexpr int J = DP / 16;
  static constexpr int LDS_BYTES = 16 * (DP + 4) * 4;  // the join's only
  static constexpr bool edge(int j) { return 16 * j + 16 > smaller_dim<DP>(); }
  f32x4 q[J], k[J], v[J], acc[J];  // v[d][r]: dim 16 d + l % 16 of key 4 (l / 16) + r
  float m, l;

  __device__ __forceinline__ void start(const float* qrow, bool live, int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 4;
      q[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (live && d < dim) q[j] = *(const f32x4*)(qrow + d);
      acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    m = -INFINITY;
    l = 0.f;
  }
};

template <int DP, bool EXACT>
__device__ __forceinline__ void run_tiles_f32(Tiles<float, DP>& w, const PagedAttendArgs& a, long b,
                                              int kv, int len, int t, int end, int step) {
  constexpr int J = DP / 16;
  const int lane = threadIdx.x & 63, row = lane & 15, chunk = lane >> 4;
  const int* table = a.cache.table + b * a.cache.table_stride;
  const float* kbase = (const float*)a.cache.k + kv * a.cache.k_head;
  const float* vbase = (const float*)a.cache.v + kv * a.cache.v_head;
  const int slot_mask = (1 << a.cache.page_shift) - 1;
  int page = -1;
  unsigned ok = 0, ok_next = 0;
  long krow = 0, vrow = 0;
  auto pages = [&](int tile) {
    const int key = tile * 16 + row;
    page = key < len ? table[key >> a.cache.page_shift] : -1;
  };
  auto resolve = [&](int tile, unsigned& good) {
    const int key = tile * 16 + row;
    const bool fine = page >= 0 && page < a.cache.pages;
    const long slot = key & slot_mask;
    krow = fine ? page * a.cache.k_page + slot * a.cache.k_slot : 0;
    vrow = fine ? page * a.cache.v_page + slot * a.cache.v_slot : 0;
    good = (unsigned)__ballot(fine) & 0xffffu;
  };
  auto fetch_k = [&]() {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 4;
      w.k[j] = *(const f32x4*)(kbase + krow + (EXACT || !w.edge(j) || d < a.dim ? d : 0));
    }
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float* p = vbase + __shfl(vrow, 4 * chunk + r, 64);
#pragma unroll
      for (int d = 0; d < J; ++d) {
        const int col = 16 * d + row;
        w.v[d][r] = p[EXACT || !w.edge(d) || col < a.dim ? col : 0];
      }
    }
  };
  if (t >= end) return;
  pages(t);
  resolve(t, ok);
  if (t + step < end) pages(t + step);
  fetch_k();
  fetch_v();
  for (; t < end; t += step) {
    const bool more = t + step < end;
    if (more) {
      resolve(t + step, ok_next);
      if (t + 2 * step < end) pages(t + 2 * step);
    }
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      f32x4 x = w.k[j];
      if (!EXACT && w.edge(j) && (chunk + 4 * j) * 4 >= a.dim) x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], w.q[j][i], s, 0, 0, 0);
    }
    if (more) fetch_k();
    const bool full = ok == 0xffffu;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] *= a.scale;
      if (!full && !((ok >> (4 * chunk + r)) & 1)) s[r] = -INFINITY;
      top = fmaxf(top, s[r]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > w.m)) {
      const float next = fmaxf(w.m, top);
      const float keep = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - next);
      w.m = next;
      w.l *= keep;
#pragma unroll
      for (int i = 0; i < J; ++i) w.acc[i] *= keep;
    }
    const float off = w.m == -INFINITY ? 0.f : w.m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float p = __builtin_amdgcn_exp2f(s[r] - off);
      w.l += p;
      const bool gone = !full && !((ok >> (4 * chunk + r)) & 1);
#pragma unroll
      for (int d = 0; d < J; ++d)
        w.acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(gone ? 0.f : w.v[d][r], p, w.acc[d], 0, 0, 0);
    }
    if (more) fetch_v();
    ok = ok_next;
  }
}

// Waves to a SIMD that the registers are held to.
constexpr int resident_waves(int dim, int size) {
  return dim <= 96 ? 3 : dim <= 128 || (size == 2 && dim <= 192) ? 2 : 1;
}

template <typename T, int DP, bool EXACT, int NW>
__global__ __launch_bounds__(64 * NW, resident_waves(DP, sizeof(T))) void paged_attend_k(
    const PagedAttendArgs a, const AttendPlan plan) {
  using W = Tiles<T, DP>;
  constexpr int OUT = DP + 4;  // pitch of a head's output in shared memory
  static_assert(16 * OUT * 4 <= W::LDS_BYTES, "the join reuses the staging rows");
  __shared__ __attribute__((aligned(16))) char lds[NW][W::LDS_BYTES];
  __shared__ float sm[NW][16], sl[NW][16];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int group = a.heads / a.kv_heads;
  const int per = a.kv_heads * plan.blocks;  // items of a sequence
  const int rows = group < 16 ? group : 16;
  const long room = (long)a.cache.table_cols << a.cache.page_shift;

  long b;
  int item, tiles, at, left;  // `left`: tiles still to do, over items
  SharedItem note = {0, 0, 0, 0, 0};
  if (plan.workers == 0) {
    b = blockIdx.x / per;
    item = (int)(blockIdx.x % per);
    tiles = left = tiles_of(a, b, W::KEYS);
    at = 0;
  } else {
    const Line line = line_of(a, per, W::KEYS);
    const long busy = busy_workers(plan.workers, line.total, NW);
    if (blockIdx.x >= busy) {
      if (threadIdx.x == 0) plan.notes[blockIdx.x] = note;
      return;
    }
    const long lo = share(blockIdx.x, line.total, busy), hi = share(blockIdx.x + 1, line.total, busy);
    const Spot s = spot_of(a, per, W::KEYS, line, lo);
    b = s.b;
    tiles = s.tiles;
    item = (int)share(lo - s.first, 1, tiles);
    at = (int)(lo - s.first - (long)item * tiles);
    left = (int)(hi - lo);
    if (at > 0) {
      // the first border strictly inside an item answers for its join
      const long from = lo - at, before = share(blockIdx.x - 1, line.total, busy);
      if (before <= from) {
        // the worker of the item's last tile is the last whose range begins at or
        // before it: ceil(end * busy / total) - 1
        const long end = from + tiles, last = share(end, busy, line.total);
        const int w1 = (int)(last * line.total == end * busy ? last - 1 : last);
        note = {b, item, (int)blockIdx.x - 1, w1 - (int)blockIdx.x + 2,
                2 * ((int)blockIdx.x - 1) + (before == from ? 0 : 1)};
      }
    }
    if (threadIdx.x == 0) plan.notes[blockIdx.x] = note;
  }
  bool first = true;
  while (left > 0) {
    const int end = left < tiles - at ? at + left : tiles;
    long len = whole(a.lengths, a.lengths_i64, b);
    len = len < room ? len : room;
    const int kv = item / plan.blocks;
    const int head0 = kv * group + 16 * (item % plan.blocks);  // the first of this block
    const int heads = min(16, (kv + 1) * group - head0);
    W w;
    const bool live = (lane & 15) < heads;
    w.start((const T*)a.q + b * a.q_batch + (head0 + (live ? lane & 15 : 0)) * a.q_head, live, a.dim);
    if constexpr (sizeof(T) == 4)
      run_tiles_f32<DP, EXACT>(w, a, b, kv, (int)len, at + wave, end, NW);
    else
      run_tiles<T, DP, EXACT>(w, a, b, kv, (int)len, at + wave, end, NW, (T*)lds[wave]);
    w.l += __shfl_xor(w.l, 16, 64);
    w.l += __shfl_xor(w.l, 32, 64);
    wave_sync();
    float* mine = (float*)lds[wave] + (lane & 15) * OUT + 4 * (lane >> 4);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) *(f32x4*)(mine + 16 * d) = w.acc[d];
    if (lane < 16) {
      sm[wave][lane] = w.m;
      sl[wave][lane] = w.l;
    }
    __syncthreads();
    const bool shared = at > 0 || end < tiles;
    const long slot = 2 * (long)blockIdx.x + (first ? 0 : 1);
    for (int i = threadIdx.x; i < heads * a.dim; i += 64 * NW) {
      const int g = i / a.dim, d = i - g * a.dim;
      float top = sm[0][g];
#pragma unroll
      for (int o = 1; o < NW; ++o) top = fmaxf(top, sm[o][g]);
      float sum = 0.f, out = 0.f;
#pragma unroll
      for (int o = 0; o < NW; ++o) {
        const float f = sm[o][g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[o][g] - top);
        sum += f * sl[o][g];
        out += f * ((const float*)lds[o])[g * OUT + d];
      }
      if (shared) {
        plan.part[(slot * rows + g) * a.dim + d] = out;
        if (d == 0) {
          plan.part_ms[(slot * rows + g) * 2] = top;
          plan.part_ms[(slot * rows + g) * 2 + 1] = sum;
        }
      } else {
        ((T*)a.out)[(b * a.heads + head0 + g) * a.dim + d] = (T)(sum == 0.f ? 0.f : out / sum);
      }
    }
    first = false;
    left -= end - at;
    at = 0;
    if (left > 0) {
      __syncthreads();  // the rows above are staged into again
      if (++item == per) {
        item = 0;
        ++b;
        tiles = tiles_of(a, b, W::KEYS);
      }
    }
  }
}

// Joins the parts of an item that several workers shared, by the note that the
// first worker whose range begins inside the item left (blockIdx.x).  blockIdx.y
// takes 128 of the item's values (heads x dims), 4 to a lane; the 8 half-waves
// take every eighth part each, eight at a time, so that an item of 64 parts waits
// for its loads once.
template <typename T>
__global__ __launch_bounds__(256) void paged_attend_join_k(const PagedAttendArgs a, const AttendPlan plan) {
  __shared__ float sm[8][32], sl[8][32];
  __shared__ f32x4 so[8][32];
  const SharedItem note = plan.notes[blockIdx.x];
  if (note.parts == 0) return;
  const int group = a.heads / a.kv_heads;
  const int rows = group < 16 ? group : 16;
  const int kv = note.item / plan.blocks;
  const int head0 = kv * group + 16 * (note.item % plan.blocks);
  const int heads = min(16, (kv + 1) * group - head0);
  const int quads = a.dim / 4;
  const int half = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = blockIdx.y * 32 + lane;
  const int g = min(q / quads, heads - 1);  // lanes past the item repeat its last head
  const int quad = q % quads;
  float top = -INFINITY, sum = 0.f;
  f32x4 out = {0.f, 0.f, 0.f, 0.f};
  constexpr int N = 8;
  for (int i0 = half; i0 < note.parts; i0 += 8 * N) {
    float m[N], l[N];
    f32x4 x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = min(i0 + 8 * u, note.parts - 1);
      // all but the first part lie in their workers' first slots
      const long row = (i == 0 ? note.slot : 2 * (long)(note.worker + i)) * rows + g;
      m[u] = plan.part_ms[2 * row];
      l[u] = plan.part_ms[2 * row + 1];
      x[u] = *(const f32x4*)(plan.part + row * a.dim + 4 * quad);
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < N; ++u) next = fmaxf(next, m[u]);
    const float keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
    top = next;
    sum *= keep;
    out *= keep;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (i0 + 8 * u >= note.parts) continue;
      const float f = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
      sum += f * l[u];
      out += f * x[u];
    }
  }
  sm[half][lane] = top;
  sl[half][lane] = sum;
  so[half][lane] = out;
  __syncthreads();
  if (half != 0 || q >= heads * quads) return;
#pragma unroll
  for (int o = 1; o < 8; ++o) top = fmaxf(top, sm[o][lane]);
  sum = 0.f;
  out = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int o = 0; o < 8; ++o) {
    const float m = sm[o][lane];
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    sum += f * sl[o][lane];
    out += f * so[o][lane];
  }
  T* dst = (T*)a.out + (note.b * a.heads + head0 + g) * a.dim + 4 * quad;
#pragma unroll
  for (int r = 0; r < 4; ++r) dst[r] = (T)(sum == 0.f ? 0.f : out[r] / sum);
}

template <typename T, int DP, bool EXACT>
int attend_launch(const PagedAttendArgs& a, hipStream_t st) {
  const AttendPlan plan{a.workers, a.head_blocks, (SharedItem*)a.notes, a.part, a.part_ms};
  const int per = a.kv_heads * a.head_blocks;
  const long items = a.batch * per;
  const dim3 blocks((unsigned)(a.workers ? a.workers : items));
  if (a.waves == 1)
    hipLaunchKernelGGL((paged_attend_k<T, DP, EXACT, 1>), blocks, dim3(64), 0, st, a, plan);
  else
    hipLaunchKernelGGL((paged_attend_k<T, DP, EXACT, 4>), blocks, dim3(256), 0, st, a, plan);
  if (a.workers < 2) return (int)hipGetLastError();
  const int group = a.heads / a.kv_heads;
  const dim3 grid((unsigned)a.workers, (unsigned)(((group < 16 ? group : 16) * a.dim + 127) / 128));
  hipLaunchKernelGGL((paged_attend_join_k<T>), grid, dim3(256), 0, st, a, plan);
  return (int)hipGetLastError();
}

template <typename T, int DP>
int attend_dim(const PagedAttendArgs& a, hipStream_t st) {
  return a.dim == DP ? attend_launch<T, DP, true>(a, st) : attend_launch<T, DP, false>(a, st);
}

template <typename T>
int attend_any(const PagedAttendArgs& a, hipStream_t st) {
  if (a.dim <= 64) return attend_dim<T, 64>(a, st);
  if (a.dim <= 96) return attend_dim<T, 96>(a, st);
  if (a.dim <= 128) return attend_dim<T, 128>(a, st);
  if (a.dim <= 192) return attend_dim<T, 192>(a, st);
  return attend_dim<T, 256>(a, st);
}

}  // namespace

extern "C" long paged_attend_note_bytes(void) { return (long)sizeof(SharedItem); }

// How a call is split, by what the host knows: the table's columns bound every
// length.  Measured in us, 16-bit caches, the other choice in brackets:
//
// - Short tables take one workgroup per item and no join, of one wave where
//   there are items to fill the card: 2048 items of 16 tiles 99 [split: 108],
//   3072 of 16 74 [80]; 4096 of 4 tiles 57 [four waves: 74].  Longer ones are
//   split, for ragged batches: what a direct call wins at equal lengths (768
//   items of 32 tiles 39 [43]) it loses on the longest item of others.
// - A split call gives a CU one workgroup of 4 waves for dims above 96, where
//   their tiles on the way (128 dim bytes to a wave) cover the latency, and two
//   below: 1 x 131072 keys, 8 heads of 128: 101 [104 with two, 113 with three];
//   2 heads of 256, 65536 keys: 40 [54]; 48 x 4096, 12 heads of 64: 113 [120
//   with one].  More workers only add prologues and parts to join.
extern "C" void plan_paged_attend(PagedAttendArgs* a, int cus) {
  const int keys = a->dtype == RL_F32 ? 16 : 32;
  const long room = (long)a->cache.table_cols << a->cache.page_shift;
  const long most = (room + keys - 1) / keys;  // tiles of an item
  const int group = a->heads / a->kv_heads;
  a->head_blocks = (group + 15) / 16;
  const long items = a->batch * a->kv_heads * a->head_blocks;
  if (most <= 8 || (most <= 16 && items >= 1024)) {
    a->workers = 0;
    a->waves = items >= 1024 ? 1 : 4;
    return;
  }
  const long resident = (long)cus * (a->dim > 96 ? 1 : 2);
  const long worth = (items * most + 3) / 4;  // a tile to each wave
  a->workers = (int)(resident < worth ? resident : worth);
  a->waves = 4;
}

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
      return attend_any<float>(*a, st);
    case RL_BF16:
      return attend_any<__bf16>(*a, st);
    case RL_F16:
      return attend_any<_Float16>(*a, st);
  }
  return (int)hipErrorInvalidValue;
}
