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
// reads and writes everything once: 32768 tokens of 32 + 16 heads of 128 bf16, 805
// MB in 146 us, 5.5 TB/s; interleaved 153 us), by the launch for single tokens (256
// of 24 heads of 64: 3.8 us).

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
  if (a.vec >= 4) return append_launch<T, 4>(a, st);
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
// bound by the cache's bytes.  Halves end at 2^-24, where weights relative to the
// maximum would be cut off from 17 nats below it on and yet count in the sum, so
// float16 weights are all taken times 2^15, in sum, output and parts alike: each is
// right to 2^-22 of itself or 2^-40 of the largest weight, whichever is more
// (bfloat16, with float32's exponents: 2^-17 of itself).  float32 caches use the fp32
// matrix instruction on tiles of 16 keys, with V's operand read directly.
//
// A wave owns whole tiles: while it computes one, the keys and values of the next
// are on their way in its registers, and the page ids of the one after.  No barrier
// in the loop.
//
// Work is split over the cache's length.  The tiles of all (sequence, key head)
// items form one line, and worker w of W takes the tiles [w n / W, (w + 1) n / W)
// of it, whatever items they belong to: ragged batches and single long sequences
// fill the card alike, without the host knowing a length.  A worker is a wave where
// items are many, else a workgroup whose four waves take every fourth tile.  Its
// first and last item may be shared with its neighbours; those parts (maximum, sum
// and unnormalised output) go to its two workspace slots, and a second launch joins
// them in order.  Sequences of length 0 count one empty tile and get zeros.
//
// Measured (one MI355X, where a large copy runs at 4.9 TB/s): 1 x 131072 keys, 32 +
// 8 heads of 128 bf16, 98 us a call, 93 in the kernel (5.8 TB/s) and 5 in the join;
// 48 sequences of 1 to 8192 keys 152 us (5.3 TB/s); 256 of 65 to 96 keys, 12 heads of
// 64, 13.3 us (4.7 TB/s).  float32: 48 of 1 to 4096 keys, 32 + 8 heads of 128, 161 us
// (5.0 TB/s); 65536 keys 121 us (4.5 TB/s); 256 of 65 to 96, 12 heads of 64, 27 us (4.7
// TB/s).  Bound by HBM; small calls by three dependent loads (length,
// page id, key) and the launch.
// ---------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Matrix;

template <>
struct Matrix<__bf16> {
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static constexpr float WEIGHT = 1.f;
  static __device__ __forceinline__ f32x4 mul(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Matrix<_Float16> {
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static constexpr float WEIGHT = 32768.f;  // the largest power of two that is a half
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
  int workers;     // 0: one worker per item, nothing shared
  int blocks;      // head blocks of 16 per key head
  int group;       // query heads to a key head
  int per;         // items of a sequence: kv_heads * blocks
  SharedItem* notes;  // [workers]
  float* part;     // [2 * workers][min(16, G)][dim] unnormalised outputs
  float* part_ms;  // [2 * workers][min(16, G)][2] maximum and sum
};

__device__ __forceinline__ int length_of(const PagedAttendArgs& a, long b) {
  const long len = whole(a.lengths, a.lengths_i64, b);
  const long room = (long)a.cache.table_cols << a.cache.page_shift;
  return (int)(len < 0 ? 0 : len < room ? len : room);
}

__device__ __forceinline__ int tiles_in(int len, int tile) { return len > 0 ? (len + tile - 1) / tile : 1; }

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
  x.mine = b0 + lane < a.batch ? tiles_in(length_of(a, b0 + lane), tile) : 0;
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
  for (long b = threadIdx.x & 63; b < a.batch; b += 64) n += tiles_in(length_of(a, b), tile);
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

// Orders a wave's own shared-memory writes before its reads of other lanes'
// values, and the other way round.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The dim that the next smaller DP takes: chunks below it are never past `dim`.
template <int DP>
constexpr int smaller_dim() {
  return DP <= 64 ? 0 : DP <= 96 ? 64 : DP <= 128 ? 96 : DP <= 192 ? 128 : 192;
}

// One (sequence, key head, head block) as a wave sees it.
template <typename T>
struct Item {
  const int* table;
  const T *k, *v;  // the key head's part of the caches
  int len;
};

// What one wave carries through its tiles.  A tile goes through
//
//   pages     its page ids are asked for            (two tiles ahead)
//   resolve   they become row addresses, fetch_k    (one tile ahead)
//   scores    S = K Q^T; the key registers are free, fetch_k of the next tile
//   weigh     the softmax's step, and the values leave their registers;
//             fetch_v of the next tile
//   gather    O += P V
template <typename T, int DP, bool EXACT>  // EXACT: dim == DP
struct Tiles;

// 16-bit caches: tiles of 32 keys.
template <typename T, int DP, bool EXACT>
struct Tiles {
  using V8 = typename Matrix<T>::V8;
  static constexpr int KEYS = 32;
  static constexpr int J = DP / 32;
  // a row of V in shared memory, padded so that the transposing read of 16 rows
  // and the 16-byte writes of 16 rows both spread over all banks
  static constexpr int PITCH = DP + 16;
  static constexpr int LDS_BYTES = KEYS * PITCH * 2;
  // whether chunks of column block j can lie past `dim`
  static constexpr bool edge(int j) { return !EXACT && 32 * j + 32 > smaller_dim<DP>(); }
  struct Query {
    V8 x[J];
  };
  Query q;
  V8 k[2][J], v[2][J], hi, lo;
  f32x4 acc[DP / 16], s[2];
  float m, l;
  int page[2];
  unsigned ok[2], ok_next[2];  // bit i of [h]: key 16 h + i counts
  long krow[2], vrow[2];

  static __device__ __forceinline__ Query query(const T* row, bool live, int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
    Query q;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 8;
      q.x[j] = V8{};
      if (live && d < dim) q.x[j] = *(const V8*)(row + d);
    }
    return q;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }

  __device__ __forceinline__ void pages(const Item<T>& it, int shift, int tile) {
    const int row = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = tile * KEYS + 16 * h + row;
      page[h] = key < it.len ? it.table[key >> shift] : -1;
    }
  }

  // rows to read of a tile; keys that do not count read the cache's first row
  __device__ __forceinline__ void resolve(const PagedCache& c, int tile) {
    const int row = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = tile * KEYS + 16 * h + row;
      const bool fine = page[h] >= 0 && page[h] < c.pages;
      const long slot = key & ((1 << c.page_shift) - 1);
      krow[h] = fine ? page[h] * c.k_page + slot * c.k_slot : 0;
      vrow[h] = fine ? page[h] * c.v_page + slot * c.v_slot : 0;
      ok_next[h] = (unsigned)__ballot(fine) & 0xffffu;
    }
  }

  __device__ __forceinline__ void fetch(V8 (&x)[2][J], const T* base, const long (&row)[2], int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* p = base + row[h];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int d = (chunk + 4 * j) * 8;
        // columns past dim: the row's first ones again, cleared before use
        x[h][j] = *(const V8*)(p + (!edge(j) || d < dim ? d : 0));
      }
    }
  }
  __device__ __forceinline__ void fetch_k(const Item<T>& it, int dim) { fetch(k, it.k, krow, dim); }
  __device__ __forceinline__ void fetch_v(const Item<T>& it, int dim) { fetch(v, it.v, vrow, dim); }

  __device__ __forceinline__ void scores(int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        V8 x = k[h][j];
        if (edge(j) && (chunk + 4 * j) * 8 >= dim) x = V8{};
        s[h] = Matrix<T>::mul(x, q.x[j], s[h]);
      }
    }
  }

  __device__ __forceinline__ void weigh(float scale, T* lds) {
    const int lane = threadIdx.x & 63, row = lane & 15, group = lane >> 4;
    const bool full = (ok[0] & ok[1]) == 0xffffu;
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
        const float p = Matrix<T>::WEIGHT * __builtin_amdgcn_exp2f(s[h][r] - off);
        l += p;
        hi[4 * h + r] = (T)p;
        lo[4 * h + r] = (T)(p - (float)hi[4 * h + r]);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool gone = !full && !((ok[h] >> row) & 1);
#pragma unroll
      for (int j = 0; j < J; ++j)
        *(V8*)(lds + (16 * h + row) * PITCH + (group + 4 * j) * 8) = gone ? V8{} : v[h][j];
    }
  }

  __device__ __forceinline__ void gather(const T* lds) {
    const int lane = threadIdx.x & 63, i = lane & 15, group = lane >> 4;
    const T* p = lds + (4 * group + i / 4) * PITCH + (i % 4) * 4;
    typedef __attribute__((address_space(3))) s16x4* Shared;
    wave_sync();
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
    wave_sync();
  }

  __device__ __forceinline__ void turn_over() {
    ok[0] = ok_next[0];
    ok[1] = ok_next[1];
  }
};

// float32 caches: tiles of 16 keys, the fp32 matrix instruction, V's operand
// straight from the cache.
template <int DP, bool EXACT>
struct Tiles<float, DP, EXACT> {
  static constexpr int KEYS = 16;
  static constexpr int J = DP / 16;
  static constexpr int LDS_BYTES = 16 * (DP + 4) * 4;  // the join's only
  static constexpr bool edge(int j) { return !EXACT && 16 * j + 16 > smaller_dim<DP>(); }
  struct Query {
    f32x4 x[J];
  };
  Query q;
  f32x4 k[J], v[J], acc[J], s;  // v[d][r]: dim 16 d + l % 16 of key 4 (l / 16) + r
  float m, l;
  int page;
  unsigned ok, ok_next;
  long krow, vrow;

  static __device__ __forceinline__ Query query(const float* row, bool live, int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
    Query q;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 4;
      q.x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (live && d < dim) q.x[j] = *(const f32x4*)(row + d);
    }
    return q;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < J; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }

  __device__ __forceinline__ void pages(const Item<float>& it, int shift, int tile) {
    const int key = tile * KEYS + (threadIdx.x & 15);
    page = key < it.len ? it.table[key >> shift] : -1;
  }

  __device__ __forceinline__ void resolve(const PagedCache& c, int tile) {
    const int key = tile * KEYS + (threadIdx.x & 15);
    const bool fine = page >= 0 && page < c.pages;
    const long slot = key & ((1 << c.page_shift) - 1);
    krow = fine ? page * c.k_page + slot * c.k_slot : 0;
    vrow = fine ? page * c.v_page + slot * c.v_slot : 0;
    ok_next = (unsigned)__ballot(fine) & 0xffffu;
  }

  __device__ __forceinline__ void fetch_k(const Item<float>& it, int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int d = (chunk + 4 * j) * 4;
      k[j] = *(const f32x4*)(it.k + krow + (!edge(j) || d < dim ? d : 0));
    }
  }

  __device__ __forceinline__ void fetch_v(const Item<float>& it, int dim) {
    const int lane = threadIdx.x & 63, row = lane & 15, chunk = lane >> 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float* p = it.v + __shfl(vrow, 4 * chunk + r, 64);
#pragma unroll
      for (int d = 0; d < J; ++d) {
        const int col = 16 * d + row;
        v[d][r] = p[!edge(d) || col < dim ? col : 0];
      }
    }
  }

  __device__ __forceinline__ void scores(int dim) {
    const int chunk = (threadIdx.x & 63) >> 4;
    s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      f32x4 x = k[j];
      if (edge(j) && (chunk + 4 * j) * 4 >= dim) x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], q.x[j][i], s, 0, 0, 0);
    }
  }

  __device__ __forceinline__ void weigh(float scale, float*) {
    const int chunk = (threadIdx.x & 63) >> 4;
    const bool full = ok == 0xffffu;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] *= scale;
      if (!full && !((ok >> (4 * chunk + r)) & 1)) s[r] = -INFINITY;
      top = fmaxf(top, s[r]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m)) {
      const float next = fmaxf(m, top);
      const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= keep;
#pragma unroll
      for (int i = 0; i < J; ++i) acc[i] *= keep;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float p = __builtin_amdgcn_exp2f(s[r] - off);
      l += p;
      const bool gone = !full && !((ok >> (4 * chunk + r)) & 1);
#pragma unroll
      for (int d = 0; d < J; ++d)
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(gone ? 0.f : v[d][r], p, acc[d], 0, 0, 0);
    }
  }

  __device__ __forceinline__ void gather(const float*) {}
  __device__ __forceinline__ void turn_over() { ok = ok_next; }
};

// A place on the line of tiles.
struct Cursor {
  long b;
  int item, at, tiles;  // at < tiles of the item
  int len;              // of the sequence
};

template <typename T>
__device__ __forceinline__ Item<T> item_of(const PagedAttendArgs& a, const AttendPlan& plan,
                                           const Cursor& c) {
  const int kv = plan.blocks == 1 ? c.item : c.item / plan.blocks;
  return {a.cache.table + c.b * a.cache.table_stride, (const T*)a.cache.k + kv * a.cache.k_head,
          (const T*)a.cache.v + kv * a.cache.v_head, c.len};
}

// The first query head of an item and how many it has.
struct Heads {
  int first, count;
};

__device__ __forceinline__ Heads heads_of(const AttendPlan& plan, int item) {
  if (plan.blocks == 1) return {item * plan.group, plan.group};
  const int kv = item / plan.blocks, block = item - kv * plan.blocks;
  return {kv * plan.group + 16 * block, min(16, plan.group - 16 * block)};
}

template <typename W, typename T>
__device__ __forceinline__ typename W::Query query_of(const PagedAttendArgs& a, long b, Heads h) {
  const int mine = threadIdx.x & 15;
  const bool live = mine < h.count;
  return W::query((const T*)a.q + b * a.q_batch + (h.first + (live ? mine : 0)) * a.q_head, live, a.dim);
}

// The range of the line that worker `me` takes, and its note for the join.
struct Range {
  Cursor from;
  int count;
  SharedItem note;
};

__device__ __forceinline__ Range range_of(const PagedAttendArgs& a, const AttendPlan& plan, int keys,
                                          int waves) {
  Range x;
  x.note = {0, 0, 0, 0, 0};
  if (plan.workers == 0) {  // blockIdx: item, sequence
    const int len = length_of(a, blockIdx.y), tiles = tiles_in(len, keys);
    x.from = {(long)blockIdx.y, (int)blockIdx.x, 0, tiles, len};
    x.count = tiles;
    return x;
  }
  const long me = blockIdx.x;
  const int per = plan.per;
  const Line line = line_of(a, per, keys);
  const long busy = busy_workers(plan.workers, line.total, waves);
  x.count = 0;
  x.from = {0, 0, 0, 1, 0};
  if (me < busy) {
    const long lo = share(me, line.total, busy), hi = share(me + 1, line.total, busy);
    const Spot s = spot_of(a, per, keys, line, lo);
    const int item = (int)share(lo - s.first, 1, s.tiles);
    const int at = (int)(lo - s.first - (long)item * s.tiles);
    x.from = {s.b, item, at, s.tiles, length_of(a, s.b)};
    x.count = (int)(hi - lo);
    if (at > 0) {
      // the first border strictly inside an item answers for its join
      const long from = lo - at, before = share(me - 1, line.total, busy);
      if (before <= from) {
        // the worker of the item's last tile is the last whose range begins at or
        // before it: ceil(end * busy / total) - 1
        const long end = from + s.tiles, last = share(end, busy, line.total);
        const int w1 = (int)(last * line.total == end * busy ? last - 1 : last);
        x.note = {s.b, item, (int)me - 1, w1 - (int)me + 2, 2 * ((int)me - 1) + (before == from ? 0 : 1)};
      }
    }
  }
  if (threadIdx.x == 0) plan.notes[me] = x.note;
  return x;
}

// Waves to a SIMD that the registers are held to.
constexpr int resident_waves(int dim, int size) {
  return dim <= 96 ? 3 : dim <= 128 || (size == 2 && dim <= 192) ? 2 : 1;
}

// Many items: a wave is a worker by itself.  Its tiles run on over the borders of
// items, the next item's first keys on their way while the last one ends.
template <typename T, int DP, bool EXACT>
__global__ __launch_bounds__(64, resident_waves(DP, sizeof(T))) void paged_attend_wave_k(
    const PagedAttendArgs a, const AttendPlan plan) {
  using W = Tiles<T, DP, EXACT>;
  __shared__ __attribute__((aligned(16))) char lds[sizeof(T) == 2 ? W::LDS_BYTES : 16];
  const int lane = threadIdx.x;
  const int rows = plan.group < 16 ? plan.group : 16;
  const int shift = a.cache.page_shift;
  const Range range = range_of(a, plan, W::KEYS, 1);
  if (range.count == 0) return;

  auto after = [&](Cursor c) {
    if (++c.at == c.tiles) {
      c.at = 0;
      if (++c.item == plan.per) {
        c.item = 0;
        if (c.b + 1 < a.batch) {
          c.len = length_of(a, ++c.b);
          c.tiles = tiles_in(c.len, W::KEYS);
        }
      }
    }
    return c;
  };
  Cursor now = range.from, next = now, far;
  Item<T> it = item_of<T>(a, plan, now);
  Heads heads = heads_of(plan, now.item);
  W w;
  typename W::Query q;
  w.pages(it, shift, now.at);
  w.q = query_of<W, T>(a, now.b, heads);
  w.resolve(a.cache, now.at);
  w.turn_over();
  const Item<T> first = it;
  if (range.count > 1) {
    next = after(now);
    it = item_of<T>(a, plan, next);
    w.pages(it, shift, next.at);
  }
  w.fetch_k(first, a.dim);
  w.fetch_v(first, a.dim);
  far = range.count > 2 ? after(next) : next;
  w.clear();
  int begin = now.at;  // where this worker's part of the item begins
  long slot = 2 * (long)blockIdx.x;
  for (int i = 0; i < range.count; ++i) {
    const bool more = i + 1 < range.count;
    const bool last = !more || next.at == 0;  // of this item here
    const Item<T> ahead = it;                  // of `next`
    if (more) {
      w.resolve(a.cache, next.at);
      if (i + 2 < range.count) {
        it = item_of<T>(a, plan, far);
        w.pages(it, shift, far.at);  // ahead of the loads that follow
      }
      if (last) q = query_of<W, T>(a, next.b, heads_of(plan, next.item));
    }
    w.scores(a.dim);
    if (more) w.fetch_k(ahead, a.dim);
    w.weigh(a.scale, (T*)lds);
    if (more) w.fetch_v(ahead, a.dim);
    w.gather((const T*)lds);
    if (last) {
      float sum = w.l;
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      const int g = lane & 15, d0 = 4 * (lane >> 4);
      if (g < heads.count) {
        if (begin > 0 || now.at + 1 < now.tiles) {
          float* p = plan.part + (slot * rows + g) * a.dim + d0;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d)
            if (16 * d + d0 < a.dim) *(f32x4*)(p + 16 * d) = w.acc[d];
          if (lane < 16) {
            plan.part_ms[(slot * rows + g) * 2] = w.m;
            plan.part_ms[(slot * rows + g) * 2 + 1] = sum;
          }
        } else {
          T* p = (T*)a.out + (now.b * a.heads + heads.first + g) * a.dim + d0;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d)
            if (16 * d + d0 < a.dim) {
              Chunk<T, 4> o;
#pragma unroll
              for (int r = 0; r < 4; ++r) o.x[r] = (T)(sum == 0.f ? 0.f : w.acc[d][r] / sum);
              *(Chunk<T, 4>*)(p + 16 * d) = o;
            }
        }
      }
      if (more) {
        heads = heads_of(plan, next.item);
        w.q = q;
        w.clear();
        begin = 0;
        slot = 2 * (long)blockIdx.x + 1;
      }
    }
    w.turn_over();
    now = next;
    next = far;
    if (i + 3 < range.count) far = after(far);
  }
}

// Few items: the waves of a workgroup (four; one for short tables) share a worker's
// tiles and join what they have at the end of each item.
template <typename T, int DP, bool EXACT, int NW>
__global__ __launch_bounds__(64 * NW, resident_waves(DP, sizeof(T))) void paged_attend_group_k(
    const PagedAttendArgs a, const AttendPlan plan) {
  using W = Tiles<T, DP, EXACT>;
  constexpr int OUT = DP + 4;  // pitch of a head's output in shared memory
  static_assert(16 * OUT * 4 <= W::LDS_BYTES, "the join reuses the staging rows");
  __shared__ __attribute__((aligned(16))) char lds[NW][W::LDS_BYTES];
  __shared__ float sm[NW][16], sl[NW][16];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int rows = plan.group < 16 ? plan.group : 16;
  const int shift = a.cache.page_shift;
  const Range range = range_of(a, plan, W::KEYS, NW);
  Cursor now = range.from;
  int left = range.count;  // tiles still to do, over items
  bool first = true;
  while (left > 0) {
    const int end = left < now.tiles - now.at ? now.at + left : now.tiles;
    const Item<T> it = item_of<T>(a, plan, now);
    const Heads heads = heads_of(plan, now.item);
    W w;
    T* mine = (T*)lds[wave];
    int t = now.at + wave;
    w.clear();
    if (t < end) {
      w.pages(it, shift, t);
      w.q = query_of<W, T>(a, now.b, heads);
      w.resolve(a.cache, t);
      w.turn_over();
      if (t + NW < end) w.pages(it, shift, t + NW);
      w.fetch_k(it, a.dim);
      w.fetch_v(it, a.dim);
      for (; t < end; t += NW) {
        const bool more = t + NW < end;
        if (more) {
          w.resolve(a.cache, t + NW);
          if (t + 2 * NW < end) w.pages(it, shift, t + 2 * NW);  // ahead of the loads that follow
        }
        w.scores(a.dim);
        if (more) w.fetch_k(it, a.dim);
        w.weigh(a.scale, mine);
        if (more) w.fetch_v(it, a.dim);
        w.gather(mine);
        w.turn_over();
      }
    }
    w.l += __shfl_xor(w.l, 16, 64);
    w.l += __shfl_xor(w.l, 32, 64);
    float* put = (float*)lds[wave] + (lane & 15) * OUT + 4 * (lane >> 4);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) *(f32x4*)(put + 16 * d) = w.acc[d];
    if (lane < 16) {
      sm[wave][lane] = w.m;
      sl[wave][lane] = w.l;
    }
    __syncthreads();
    const bool shared = now.at > 0 || end < now.tiles;
    const long slot = 2 * (long)blockIdx.x + (first ? 0 : 1);
    for (int i = threadIdx.x; i < heads.count * a.dim; i += 64 * NW) {
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
        ((T*)a.out)[(now.b * a.heads + heads.first + g) * a.dim + d] = (T)(sum == 0.f ? 0.f : out / sum);
      }
    }
    first = false;
    left -= end - now.at;
    now.at = 0;
    if (left > 0) {
      __syncthreads();  // the rows above are staged into again
      if (++now.item == plan.per) {
        now.item = 0;
        now.len = length_of(a, ++now.b);
        now.tiles = tiles_in(now.len, W::KEYS);
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
  const int rows = plan.group < 16 ? plan.group : 16;
  const Heads heads = heads_of(plan, note.item);
  const int quads = a.dim / 4;
  const int half = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = blockIdx.y * 32 + lane;
  const int g = min(q / quads, heads.count - 1);  // lanes past the item repeat its last head
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
  if (half != 0 || q >= heads.count * quads) return;
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
  T* dst = (T*)a.out + (note.b * a.heads + heads.first + g) * a.dim + 4 * quad;
#pragma unroll
  for (int r = 0; r < 4; ++r) dst[r] = (T)(sum == 0.f ? 0.f : out[r] / sum);
}

// The same where single waves are the workers: items are many and their parts
// few, so a thread takes 4 values of an item and all its parts.
template <typename T>
__global__ __launch_bounds__(256) void paged_attend_join_few_k(const PagedAttendArgs a,
                                                               const AttendPlan plan) {
  const int rows = plan.group < 16 ? plan.group : 16;
  const unsigned quads = a.dim / 4, all = rows * quads;
  const unsigned id = blockIdx.x * 256 + threadIdx.x;
  if (id / all >= (unsigned)plan.workers) return;
  const SharedItem note = plan.notes[id / all];
  const int g = (int)(id % all / quads), quad = (int)(id % quads);
  const Heads heads = heads_of(plan, note.item);
  if (note.parts == 0 || g >= heads.count) return;
  float top = -INFINITY, sum = 0.f;
  f32x4 out = {0.f, 0.f, 0.f, 0.f};
  constexpr int N = 4;
  for (int i0 = 0; i0 < note.parts; i0 += N) {
    float m[N], l[N];
    f32x4 x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = min(i0 + u, note.parts - 1);
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
      if (i0 + u >= note.parts) continue;
      const float f = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
      sum += f * l[u];
      out += f * x[u];
    }
  }
  T* dst = (T*)a.out + (note.b * a.heads + heads.first + g) * a.dim + 4 * quad;
#pragma unroll
  for (int r = 0; r < 4; ++r) dst[r] = (T)(sum == 0.f ? 0.f : out[r] / sum);
}

template <typename T, int DP, bool EXACT>
void attend_kernel(const PagedAttendArgs& a, const AttendPlan& plan, hipStream_t st) {
  if (a.workers == 0) {
    const dim3 items(plan.per, (unsigned)a.batch);
    if (a.waves == 1)
      hipLaunchKernelGGL((paged_attend_group_k<T, DP, EXACT, 1>), items, dim3(64), 0, st, a, plan);
    else
      hipLaunchKernelGGL((paged_attend_group_k<T, DP, EXACT, 4>), items, dim3(256), 0, st, a, plan);
  } else if (a.waves == 1) {
    hipLaunchKernelGGL((paged_attend_wave_k<T, DP, EXACT>), dim3(a.workers), dim3(64), 0, st, a, plan);
  } else {
    hipLaunchKernelGGL((paged_attend_group_k<T, DP, EXACT, 4>), dim3(a.workers), dim3(256), 0, st, a,
                       plan);
  }
}

template <typename T>
int attend_any(const PagedAttendArgs& a, hipStream_t st) {
  const AttendPlan plan{a.workers, a.head_blocks, a.heads / a.kv_heads, a.kv_heads * a.head_blocks,
                        (SharedItem*)a.notes, a.part, a.part_ms};
  if (a.dim < 64)
    attend_kernel<T, 64, false>(a, plan, st);
  else if (a.dim == 64)
    attend_kernel<T, 64, true>(a, plan, st);
  else if (a.dim <= 96)
    attend_kernel<T, 96, false>(a, plan, st);
  else if (a.dim < 128)
    attend_kernel<T, 128, false>(a, plan, st);
  else if (a.dim == 128)
    attend_kernel<T, 128, true>(a, plan, st);
  else if (a.dim <= 192)
    attend_kernel<T, 192, false>(a, plan, st);
  else if (a.dim < 256)
    attend_kernel<T, 256, false>(a, plan, st);
  else
    attend_kernel<T, 256, true>(a, plan, st);
  if (a.workers < 2) return (int)hipGetLastError();
  const long quads = (long)(plan.group < 16 ? plan.group : 16) * (a.dim / 4);
  if (a.waves == 1)
    hipLaunchKernelGGL((paged_attend_join_few_k<T>), dim3((unsigned)((a.workers * quads + 255) / 256)),
                       dim3(256), 0, st, a, plan);
  else
    hipLaunchKernelGGL((paged_attend_join_k<T>), dim3((unsigned)a.workers, (unsigned)((quads + 31) / 32)),
                       dim3(256), 0, st, a, plan);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" long paged_attend_note_bytes(void) { return (long)sizeof(SharedItem); }

// How a call is split, by what the host knows: the table's columns bound every
// length.  Measured in us with the other choice in brackets (bf16, keys by page
// tables of 64):
//
// - Short tables take one worker per item and no join, whose launch costs 4: up to
//   2048 / dim tiles, below which a single CU streams an item (some 40 GB/s) in that
//   time.  8 items of dim 64, 500 / 800 / 1200 keys: 9.7 / 12.4 / 15.4 [split: 12.4 /
//   13.6 / 13.5]; of dim 128, 300 / 500 / 800: 10.6 / 13.3 / 18.2 [14.5 / 13.0 / 14.9];
//   200 items of dim 64, 800: 14 [19].  With single waves, up to 16 tiles: 2048 items
//   of 16 tiles, dim 128, 100 [106]; 4096 of 4 57 [65].
// - From 256 items on a worker is one wave, below a workgroup of four.  Ragged lengths of
//   1 to 8192, dim 128, 256 items 119 [130], 384 items 172 [184]; of 1 to 1024, 512 items
//   36 [60]; of 100 to 700, dim 64, 2048 items 54 [70].  Equal lengths are even: 384 items
//   of 4096, dim 128, 151 [154], 256 items 113 [112].  But 16 items of 1 to 30000 34 [83],
//   8 of 131072 105 [164].  In between single waves would do from some 128 items on: 128
//   and 192 items of 1 to 8192 81 and 108 [71 and 97].
// - Workers are as many as fill the card once, no more: each has a start of its
//   own, and shares items that must be joined.  Single waves two to a SIMD: 512
//   items of 1 to 1024, dim 128, 41 [49 with one, 44 with three].  Workgroups one
//   to a CU for dims from 96 on, whose tiles on the way (128 dim bytes to a wave)
//   cover the latency, and two below: 8 items of 131072, dim 128, 101 [104 with two,
//   113 with three]; 2 of 65536, dim 256, 40 [54]; 4 of 65536, dim 96, 26 [31]; 12 of
//   65536, dim 64, 45 [47 with one].
extern "C" void plan_paged_attend(PagedAttendArgs* a, int cus) {
  const int size = a->dtype == RL_F32 ? 4 : 2;
  const int keys = size == 4 ? 16 : 32;
  const long room = (long)a->cache.table_cols << a->cache.page_shift;
  // tiles of an item, one at least: no pages at all are an empty item's one tile
  const long most = room > 0 ? (room + keys - 1) / keys : 1;
  const int group = a->heads / a->kv_heads;
  a->head_blocks = (group + 15) / 16;
  const long items = a->batch * a->kv_heads * a->head_blocks;
  // (a grid's y takes 65535 sequences)
  const bool brief = most <= 8 || (items >= 1024 ? most <= 16 : most * a->dim <= 2048);
  if (brief && a->batch < 65536) {
    a->workers = 0;
    a->waves = items >= 1024 ? 1 : 4;
    return;
  }
  a->waves = items >= 256 ? 1 : 4;
  const int fit = resident_waves(a->dim, size);
  const long fill = (long)cus * (a->waves == 1 ? 4 * (fit < 2 ? fit : 2) : a->dim >= 96 ? 1 : 2);
  const long worth = (items * most + a->waves - 1) / a->waves;  // a tile to each wave
  a->workers = (int)(fill < worth ? fill : worth);
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
  // the parts are written and read 16 bytes at a time, the notes hold 8-byte numbers
  if (a->workers && ((size_t)a->part % 16 != 0 || (size_t)a->notes % 8 != 0))
    return (int)hipErrorInvalidValue;
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
