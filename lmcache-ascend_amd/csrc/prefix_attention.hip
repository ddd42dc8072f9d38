// Attention of a batch whose requests share a prefix, over paged K and V
// caches, on MI355X (gfx950).
//
//   o(t, h)   = sum_j softmax_j(scale q(t, h) . k(j)) v(j)
//   lse(t, h) = log sum_j exp(scale q(t, h) . k(j))
//
// over the keys j of token t's request up to the token's own position.  Keys
// before shared_len lie in the blocks of one list for the whole batch, the
// others in the request's row of the block table.
//
// One pass over the keys with the running maximum and sum of each row; the
// key range is cut into parts, whose sums (32 bits, with their maximum) a
// second launch joins:
//
//   * The prefix: rows of all requests together, a KV head's heads beside each
//     other, against one part of the shared keys.  With more than 64 rows a
//     KV head, tiles of 128 rows and blocks of 64 keys (attend_wide), bound by
//     the matrix cores and their operands from LDS; else 32 rows and a block
//     of 32 keys a wave (attend_narrow).
//   * Each request's own keys: a wave a part (attend_narrow), bound by the
//     bytes of K and V: 4 to 16 rows stand in tiles of 32, which costs less
//     than the loads do.
//
// S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 matrix instructions: a lane
// holds one row's weights for half of a block's keys, in the order in which
// the second product takes them, so that maximum, sum and weights stay in
// registers; K and V go from memory to LDS without registers between, and V
// is read from there transposed.
//
// The weights are rounded to the caches' type for the product with V: the
// matrix instructions take both operands in 16 bits (in 32 they have a
// sixteenth of the rate).  Scores, maximum, sum, lse and the sums of V stay in
// 32 bits.  A weight is then off by at most half a step of the type, in
// outputs of some thousand keys 0.0023 of their size against 64 bits, where
// 32-bit weights and the output's own rounding give 0.0017 (bf16).
//
// 256 requests, 32 heads over 8 KV heads of 128 bf16 dims, 16384 shared and 1
// to 1024 own keys: 154 to 158 us (71 GFLOP, 607 MB), of which 11 the join;
// calls of the prefix alone take 98 us (700 TFLOP/s), of the own keys alone
// 115 (4.7 TB/s).  64 requests over 4096 shared and the same own keys: 42 to
// 44 us.  4 requests over 1000 shared and 1 to 200 own keys: 12 us, the latency
// of two launches.
//
// Prompts: 512 new tokens of one request over 16384 shared keys take 192 us
// (730 TFLOP/s), 2048 take 764 (770).  Their own keys go at 32 rows a wave, to
// the request's end also where a tile's rows end before: 8192 new tokens
// without a prefix take 3.1 ms (180 TFLOP/s).
//
// Registers at 128 dims: 256 for wide tiles (2 of them spilled, 12 bytes of
// scratch, two waves a SIMD), 195 for narrow ones; at 64 dims 193 and 131; 192
// and 256 dims take accumulation registers too, a wave a SIMD.  48 to 60 scalar
// registers are kept in vector registers.
#include "rope_math.h"
#include "serving.h"

#include <cmath>
#include <limits>
#include <type_traits>

namespace lmc {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Keys of a part of a request's own ones where requests are many: 256 requests
// over 16384 shared and up to 1024 own keys take 151 us with 384, 156 with 256
// (more starts and ends) and 149 with 512, which takes 116 over 1024 shared keys
// against 112.  An equal share of all own keys for every wave, over the
// requests' borders, took as long (124 against 120 for the own keys alone) and
// cost small batches 2 of 12 us.
constexpr int kOwnChunk = 384;

struct AttnArgs {
  const void *q;
  int64_t q_token, q_head;  // elements
  void *o;
  int64_t o_token, o_head;
  float *lse;               // may be null
  int64_t lse_token, lse_head;
  const uint8_t *k, *v;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  uint32_t pages, block_size, block_mul, block_shift;
  const int32_t *shared;
  int shared_len;
  const int32_t *table;
  int64_t table_stride;
  uint32_t width, shared_width;
  const int32_t *seq_lens, *starts;
  int n_requests, n_tokens;
  int heads, kv_heads, group;
  int max_keys;             // that a request can have
  float scale2;             // scale * log2(e)
  // Partial results: [parts][tokens * heads] rows of D sums, and (m, l).
  float *part_o;
  float2 *part_ml;
  int prefix_parts, own_parts;
  int prefix_tiles;         // row tiles of one KV head's rows
  int prefix_chunk;         // keys of one prefix part
  int prefix_groups;        // groups of 8 workgroups, the first of the launch
  int own_tiles;            // row tiles of a request dealt to waves
  int own_want;             // parts of a request's own keys that fill the chip
  int own_items;
};

// Rows of zeros, read in the place of keys that nobody sees.
__device__ const uint4 zero_row[32] = {};

// MFMA operands of the two types: A rows are keys (or dims of V), B columns
// are query rows.
template <typename T> struct Mma;
template <> struct Mma<BF16> {
  using V8 = bf16x8;
  static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ __bf16 from(float x) { return static_cast<__bf16>(x); }
  static constexpr uint32_t kInf = 0x7f80;
};
template <> struct Mma<F16> {
  using V8 = f16x8;
  static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ _Float16 from(float x) { return static_cast<_Float16>(x); }
  static constexpr uint32_t kInf = 0x7c00;
};

// The value of the lane 32 away beside the own one: (lower half's, upper half's).
__device__ __forceinline__ float2 both_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 16 bytes a lane from global memory to LDS at `lds` (uniform) + 16 * lane:
// from base (uniform) + off, or from an address of the lane's.  No register
// is written; wait_loads<N>() waits until at most N loads are under way.
__device__ __forceinline__ uint64_t uniform(const void *p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// ONCE: a request's own keys, which its one tile of 32 rows reads once, so they
// need not stay in the caches: own keys alone, 256 requests of 1 to 1024, take
// 115 us so and 127 without, 64 requests with a prefix 43.5 and 50; the shared
// keys, which all row tiles read, take 4% longer.  A prompt's tiles read its own
// keys once each and would rather find them there: 2048 new tokens over 16384
// shared keys take 764 us so and 743 without, 8192 over none 3.1 ms and 2.3.
// The kernel is made for the former.  (m0 is reserved: nothing but these
// statements writes it in this file's kernels, each right before its load.)
template <bool ONCE> __device__ __forceinline__ void load_to_lds(const uint8_t *base, uint32_t off, uint32_t lds) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
                 "v"(off), "s"(uniform(base))
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off),
                 "s"(uniform(base))
                 : "memory");
}
__device__ __forceinline__ void load_to_lds(const uint8_t *at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(at) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// LDS reads have their data: what they read may be written again.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

typedef __attribute__((address_space(3))) s16x4 LdsS4;
typedef __attribute__((address_space(3))) s16x8 LdsS8;

// Tiles of K and V keep their rows as they are; 16-byte piece c of row r
// lies at piece c ^ swizzle(r), so that the 16 rows that one read of K
// touches, and the 4 rows x 64 bytes of a transposed read of V, fall on
// different banks.
template <int D> __device__ __forceinline__ constexpr uint32_t k_swizzle(uint32_t r) {
  return D % 128 == 0 ? r & 15 : D % 64 == 0 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D> __device__ __forceinline__ constexpr uint32_t v_swizzle(uint32_t r) {
  return D % 128 == 0 ? (r & 3) << 2 : D % 64 == 0 ? ((r >> 1) & 1) << 2 : 0;
}

// One wave's 32 query rows: column n = lane & 31 of S^T and O^T.
template <typename T, int D> struct Rows32 {
  typename Mma<T>::V8 q[D / 16];
  f32x16 o[D / 32];
  float m, l;   // m in powers of two; l of this lane's keys
  int limit;    // keys that the row sees; INT_MAX for a row that is none
  int row;      // token * heads + head, or -1
};

template <int D> struct Geometry {
  static constexpr int kPitch = 2 * D;           // bytes of a row
  static constexpr int kPieces = D / 8;          // 16-byte pieces of a row
};

// Whether a tile of V holds an infinity or a NaN.
template <typename T, int D, int KEYS>
__device__ __forceinline__ bool has_odd(uint32_t v) {
  bool bad = false;
  for (int i = threadIdx.x & 63; i < KEYS * D / 8; i += 64) {
    const s16x8 x = *reinterpret_cast<const LdsS8 *>(v + i * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) bad |= (static_cast<uint32_t>(x[e]) & Mma<T>::kInf) == Mma<T>::kInf;
  }
  return __any(bad);
}

// Takes the infinities and NaN out of a tile of V that holds keys which some
// rows see and others do not: a weight of zero would make NaN of them.  The
// rows that see such a key get its infinities and NaN added here.  SHARED:
// the four waves work on one tile, and all of them come here.
template <typename T, int D, int KEYS, bool SHARED>
__device__ __forceinline__ void take_odd_out(Rows32<T, D> &r, uint32_t v, int j0, uint64_t seen) {
  using M = Mma<T>;
  constexpr int kPitch = Geometry<D>::kPitch;
  const int lane = threadIdx.x & 63, hb = lane >> 5;
#pragma unroll 1
  for (int key = 0; key < KEYS; ++key) {
    const bool see = ((seen >> key) & 1) && j0 + key < r.limit;
    const uint32_t row = v + key * kPitch + 8 * hb, x = v_swizzle<D>(key) << 4;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const s16x4 y = *reinterpret_cast<const LdsS4 *>(row + ((64 * t + 16 * q) ^ x));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (see && (static_cast<uint32_t>(y[e]) & M::kInf) == M::kInf)
            r.o[t][4 * q + e] += to_f32<T>(static_cast<uint16_t>(y[e]));
        asm volatile("" ::: "memory");  // (few registers here)
      }
  }
  if constexpr (SHARED) __syncthreads();
#pragma unroll 1
  for (int i = lane; i < KEYS * D / 8; i += 64) {
    s16x8 x = *reinterpret_cast<const LdsS8 *>(v + i * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((static_cast<uint32_t>(x[e]) & M::kInf) == M::kInf) x[e] = 0;
    *reinterpret_cast<LdsS8 *>(v + i * 16) = x;
  }
  if constexpr (SHARED) __syncthreads();
  else wait_reads();
}

// The steps of a tile of NB * 32 keys, in LDS at k and v.

// S^T = K Q^T: lane (n, hb) gets the scores of row n with the keys 32 b + 8 i
// + 4 hb + j of s[b][4 i + j].
template <typename T, int D, int NB>
__device__ __forceinline__ void scores(const Rows32<T, D> &r, uint32_t k, f32x16 (&s)[NB]) {
  using M = Mma<T>;
  constexpr int kPitch = Geometry<D>::kPitch;
  const int lane = threadIdx.x & 63, n = lane & 31, hb = lane >> 5;
  const uint32_t krow = k + n * kPitch, kx = k_swizzle<D>(n);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) {
    const uint32_t at = krow + (((2 * kc + hb) ^ kx) << 4);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const s16x8 a = *reinterpret_cast<const LdsS8 *>(at + b * 32 * kPitch);
      s[b] = M::mul(__builtin_bit_cast(typename M::V8, a), r.q[kc], s[b]);
    }
  }
}

// Takes out the keys that the row does not see: those whose bit of `seen` is
// clear and those past its limit.
template <int NB> __device__ __forceinline__ void hide(f32x16 (&s)[NB], int limit, int j0, uint64_t seen) {
  const int hb = (threadIdx.x & 63) >> 5;
  // Bit 32 b + 8 i + j: key 4 hb further.
  uint64_t bits = seen >> (4 * hb);
  const int left = limit - j0 - 4 * hb;
  if (left < 64) bits &= left > 0 ? (uint64_t(1) << left) - 1 : 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t half = static_cast<uint32_t>(bits >> (32 * b));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(half & (1u << (8 * (i / 4) + i % 4)))) s[b][i] = -INFINITY;
  }
}

// The largest score of the row in the tile, in powers of two.
template <int NB> __device__ __forceinline__ float largest(const f32x16 (&s)[NB], float c) {
  float top = s[0][0];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
  const float2 tops = both_halves(top);
  return fmaxf(tops.x, tops.y) * c;
}

// The sums keep their reference point until a score passes it by 2^8: the
// weights stay below 256, where their relative rounding is the same.
template <typename T, int D> __device__ __forceinline__ void refer_to(Rows32<T, D> &r, float top) {
  if (__any(top > r.m + 8.f)) {
    const float m = fmaxf(r.m, top);
    const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
    r.l *= f;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[t][i] *= f;
    r.m = m;
  }
}

// Weights, rounded to the type once for the product with V, which takes 16
// bits (l sums them before the rounding, so lse has none of it).
template <typename T, int D>
__device__ __forceinline__ void weigh(Rows32<T, D> &r, const f32x16 &s, typename Mma<T>::V8 (&p)[2], float c) {
  const float base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float w = __builtin_amdgcn_exp2f(s[i] * c - base);
    r.l += w;
    p[i / 8][i % 8] = Mma<T>::from(w);
  }
}

// O^T += V^T P^T.  The sum over keys may take them in any order: the order in
// which a lane holds its 8 of 16 weights, keys 4 hb + {0..3, 8..11}.
template <typename T, int D>
__device__ __forceinline__ void add_values(Rows32<T, D> &r, uint32_t v, const typename Mma<T>::V8 (&p)[2]) {
  using M = Mma<T>;
  constexpr int kPitch = Geometry<D>::kPitch;
  const int lane = threadIdx.x & 63, hb = lane >> 5, a = lane & 15;
  const uint32_t vrow = 4 * hb + (a >> 2);
  const uint32_t vx = v_swizzle<D>(vrow);
  const uint32_t vcol = 2 * ((lane >> 4) & 1) + ((a & 3) >> 1);
  const uint32_t vbase = v + vrow * kPitch + (a & 1) * 8;
#pragma unroll
  for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      const uint32_t at = vbase + (((4 * t + vcol) ^ vx) << 4) + c2 * 16 * kPitch;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at + 8 * kPitch));
      const s16x8 x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      r.o[t] = M::mul(__builtin_bit_cast(typename M::V8, x), p[c2], r.o[t]);
    }
}

// Where a group of 16 keys lies: if it is whole, there and in one block of
// the caches, at k + i * k_token and v + i * v_token.
struct Place {
  const uint8_t *k, *v;
  bool whole;
};

// The keys [k0, k1) of one list of blocks for one KV head, in groups of 16:
// 32 keys every `stride` from `first` (a multiple of 16).  A lane looks up a
// group, so 64 of them at a time; each is then a few reads of a lane.
struct Keys {
  const AttnArgs &a;
  const int32_t *list;
  uint32_t n_list;
  int k0, k1, first, stride;
  int64_t k_off, v_off;  // of the head
  bool holes;            // blocks may lie outside the caches: ask for each key
  int base = 0;          // group of lane 0
  uint64_t groups = 0;   // which lanes' groups are whole
  uint64_t k = 0, v = 0;

  __device__ __forceinline__ uint32_t block_of(uint32_t j) const {
    return a.block_size == 1 ? j : __umulhi(j, a.block_mul) >> a.block_shift;
  }
  // The block of a lane's key, -1 without one.
  __device__ __forceinline__ int page(int j) const {
    if (j < k0 || j >= k1) return -1;
    const uint32_t b = block_of(j);
    const int p = b < n_list ? list[b] : -1;
    return static_cast<uint32_t>(p) < a.pages ? p : -1;
  }
  __device__ __forceinline__ int key(int g) const { return first + g / 2 * stride + g % 2 * 16; }
  // The entry of the list for this lane's group of the 64 from g, and what
  // follows from it (apart, so that other loads can be under way between).
  __device__ __forceinline__ int entry(int g) const {
    const uint32_t b = block_of(min(max(key(g + (threadIdx.x & 63)), k0), k1));
    return n_list ? list[min(b, n_list - 1)] : -1;
  }
  __device__ __forceinline__ void look_up(int g, int entry) {
    base = g;
    const int j = key(g + (threadIdx.x & 63));
    const bool in = j + 16 > k0 && j < k1;
    const int p = in && block_of(max(j, k0)) < n_list && static_cast<uint32_t>(entry) < a.pages ? entry : -1;
    const int at = j - static_cast<int>(block_of(j) * a.block_size);
    groups = __ballot(p >= 0 && j >= k0 && j + 16 <= k1 && a.block_size % 16 == 0);
    if (__any(in && p < 0)) holes = true;
    k = reinterpret_cast<uint64_t>(a.k + k_off) + p * a.k_page + at * a.k_token;
    v = reinterpret_cast<uint64_t>(a.v + v_off) + p * a.v_page + at * a.v_token;
  }
  static __device__ __forceinline__ const uint8_t *lane_of(uint64_t x, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), lane);
    return reinterpret_cast<const uint8_t *>((static_cast<uint64_t>(hi) << 32) | lo);
  }
  __device__ __forceinline__ Place place(int g) {
    if (g - base >= 64) look_up(g & ~63, entry(g & ~63));
    const int l = g - base;
    return {lane_of(k, l), lane_of(v, l), ((groups >> l) & 1) != 0};
  }
  // Whether all of the N keys from j0 are there; which of them are.
  template <int N> __device__ __forceinline__ bool all(int j0) const { return j0 >= k0 && j0 + N <= k1 && !holes; }
  template <int N> __device__ __forceinline__ uint64_t seen(int j0) const {
    uint64_t bits = N == 64 ? ~uint64_t(0) : (uint64_t(1) << N % 64) - 1;
    if (j0 < k0) bits &= k0 - j0 < 64 ? ~uint64_t(0) << (k0 - j0) : 0;
    if (j0 + 64 > k1) bits &= k1 > j0 ? ~uint64_t(0) >> (j0 + 64 - k1) : 0;
    if (holes) bits &= __ballot(page(j0 + (threadIdx.x & (N - 1))) >= 0);
    return bits;
  }
};

// Load i of the D / 32 loads of a group of 16 rows: this lane's row and
// piece of it, as an offset from the group's first row.
template <int D, bool V> __device__ __forceinline__ uint32_t row_offset(int i, int64_t token) {
  constexpr int kPieces = Geometry<D>::kPieces;
  const int x = i * 64 + (threadIdx.x & 63), row = x / kPieces;
  return static_cast<uint32_t>(row * token) + ((x % kPieces) ^ (V ? v_swizzle<D>(row) : k_swizzle<D>(row))) * 16;
}

// The D / 32 loads of the group of 16 rows from `key`, row by row: where it
// is not whole.  Rows of zeros stand for the keys that are not there.
template <int D, bool V> __device__ __forceinline__ void load_single_rows(const Keys &s, int key, uint32_t lds) {
  constexpr int kPieces = Geometry<D>::kPieces;
  const AttnArgs &a = s.a;
#pragma unroll 1
  for (int i = 0; i < D / 32; ++i) {
    const int x = i * 64 + (threadIdx.x & 63), row = x / kPieces, j = key + row;
    const uint32_t piece = ((x % kPieces) ^ (V ? v_swizzle<D>(row) : k_swizzle<D>(row))) * 16;
    const int p = s.page(j);
    const int at = j - static_cast<int>(s.block_of(j) * a.block_size);
    const uint8_t *from = reinterpret_cast<const uint8_t *>(zero_row);
    if (p >= 0) from = V ? a.v + s.v_off + p * a.v_page + at * a.v_token : a.k + s.k_off + p * a.k_page + at * a.k_token;
    load_to_lds(from + piece, lds + i * 1024);
  }
}

// A group's K or V to LDS, off[i] as row_offset gives it.
template <int D, bool V, bool ONCE>
__device__ __forceinline__ void load_group(const Keys &s, const Place &at, int key, const uint32_t (&off)[D / 32], uint32_t lds) {
  if (at.whole) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) load_to_lds<ONCE>(V ? at.v : at.k, off[i], lds + i * 1024);
  } else {
    load_single_rows<D, V>(s, key, lds);
  }
}

// The query rows are there: waited for here and not in the loops, where the
// wait would be for all loads under way.
template <typename T, int D> __device__ __forceinline__ void wait_rows(Rows32<T, D> &r) {
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) {
    s16x8 x = __builtin_bit_cast(s16x8, r.q[kc]);
    asm volatile("" : "+v"(x));
    r.q[kc] = __builtin_bit_cast(typename Mma<T>::V8, x);
  }
}

// Query rows to registers: row n of `m` (head-local row numbers).
template <typename T, int D> __device__ __forceinline__ void load_rows(const AttnArgs &a, Rows32<T, D> &r, int t, int head, int limit) {
  using S = typename T::S;
  const int hb = (threadIdx.x & 63) >> 5;
  const bool there = t >= 0;
  r.row = there ? t * a.heads + head : -1;
  r.limit = there && limit > 0 ? limit : INT32_MAX;
  const S *q = static_cast<const S *>(a.q) + (there ? t * a.q_token + head * a.q_head : 0);
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) {
    s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) x = *reinterpret_cast<const s16x8 *>(q + kc * 16 + hb * 8);
    r.q[kc] = __builtin_bit_cast(typename Mma<T>::V8, x);
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) r.o[i][e] = 0.f;
  r.m = -INFINITY;
  r.l = 0.f;
}

template <int D> struct Lds {
  static constexpr int kNarrow = 4 * 2 * 32 * D * 2;       // a block of 32 keys a wave
  static constexpr int kWide = 2 * 2 * 64 * D * 2;         // two blocks of 64 keys
  static constexpr int kSums = 4 * D * 33 * 4 + 4 * 32 * 8;  // O^T of four waves, and (m, l)
  static constexpr int kBytes = kNarrow > kSums ? (kNarrow > kWide ? kNarrow : kWide) : (kSums > kWide ? kSums : kWide);
};

// The four waves' sums to their part.  MERGE: the waves hold the same 32
// rows over different keys.  A row whose limit is 0 or less gets nothing.
template <typename T, int D, bool MERGE>
__device__ __forceinline__ void store_part(const AttnArgs &a, const Rows32<T, D> &r, bool dead, int part, uint8_t *lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hb = lane >> 5;
  float *sums = reinterpret_cast<float *>(lds);
  float2 *ml = reinterpret_cast<float2 *>(lds + 4 * D * 33 * 4);
  const float2 ls = both_halves(r.l);
  __syncthreads();
  float *own = sums + wave * D * 33;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) own[(32 * t + 8 * (i / 4) + 4 * hb + i % 4) * 33 + n] = r.o[t][i];
  if (hb == 0) ml[wave * 32 + n] = dead ? make_float2(-INFINITY, 0.f) : make_float2(r.m, ls.x + ls.y);
  __syncthreads();
  const int64_t rows = static_cast<int64_t>(a.n_tokens) * a.heads;
  constexpr int kQuads = D / 4;
  if constexpr (MERGE) {
    for (int x = threadIdx.x; x < 32 * kQuads; x += 256) {
      const int i = x / kQuads, d = x % kQuads * 4;
      const int row = __builtin_amdgcn_ds_bpermute(i * 4, r.row);
      if (row < 0) continue;
      float2 w[4];
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        w[g] = ml[g * 32 + i];
        top = fmaxf(top, w[g].x);
      }
      const float base = top == -INFINITY ? 0.f : top;
      float l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (w[g].y == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(w[g].x - base);
        l += f * w[g].y;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f * sums[(g * D + d + e) * 33 + i];
      }
      if (d == 0) a.part_ml[part * rows + row] = make_float2(top, l);
      if (l != 0.f) *reinterpret_cast<f32x4 *>(a.part_o + (part * rows + row) * D + d) = o;
    }
  } else {
    for (int x = lane; x < 32 * kQuads; x += 64) {
      const int i = x / kQuads, d = x % kQuads * 4;
      const int row = __builtin_amdgcn_ds_bpermute(i * 4, r.row);
      if (row < 0) continue;
      const float2 w = ml[wave * 32 + i];
      f32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = own[(d + e) * 33 + i];
      if (d == 0) a.part_ml[part * rows + row] = w;
      if (w.y != 0.f) *reinterpret_cast<f32x4 *>(a.part_o + (part * rows + row) * D + d) = o;
    }
  }
}

// One wave's sums to their part, straight from the registers.
template <typename T, int D>
__device__ __forceinline__ void store_rows(const AttnArgs &a, const Rows32<T, D> &r, bool dead, int part) {
  const int hb = (threadIdx.x & 63) >> 5;
  const float2 ls = both_halves(r.l);
  if (r.row < 0) return;
  const int64_t at = part * (static_cast<int64_t>(a.n_tokens) * a.heads) + r.row;
  const float l = dead ? 0.f : ls.x + ls.y;
  if (hb == 0) a.part_ml[at] = make_float2(dead ? -INFINITY : r.m, l);
  if (l == 0.f) return;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = r.o[t][4 * b + e];
      *reinterpret_cast<f32x4 *>(a.part_o + at * D + 32 * t + 8 * b + 4 * hb) = o;
    }
}

// One wave's 32 rows over the blocks of `keys`, in LDS of its own: few rows,
// bound by the bytes of K and V.  The next block's K is loaded once this
// one's has been read, while V is used, and its V after that, so some load is
// always under way.
template <typename T, int D, bool ONCE>
__device__ __forceinline__ void attend_narrow(const AttnArgs &a, Rows32<T, D> &r, Keys &keys, int entry, int least, uint32_t k) {
  constexpr int kPer = D / 32;  // loads of a group
  const uint32_t v = k + 32 * D * 2;
  int j0 = keys.first;
  if (j0 >= keys.k1) return;
  uint32_t k_off[kPer], v_off[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    k_off[i] = row_offset<D, false>(i, a.k_token);
    v_off[i] = row_offset<D, true>(i, a.v_token);
  }
  Place lo, hi;
  auto load_k = [&](int j) {
    load_group<D, false, ONCE>(keys, lo, j, k_off, k);
    load_group<D, false, ONCE>(keys, hi, j + 16, k_off, k + kPer * 1024);
  };
  auto load_v = [&](int j) {
    load_group<D, true, ONCE>(keys, lo, j, v_off, v);
    load_group<D, true, ONCE>(keys, hi, j + 16, v_off, v + kPer * 1024);
  };
  keys.look_up(0, entry);
  lo = keys.place(0);
  hi = keys.place(1);
  load_k(j0);
  load_v(j0);
  wait_rows<T, D>(r);
  for (int b = 0; j0 < keys.k1; j0 += keys.stride, ++b) {
    const int next = j0 + keys.stride;
    const bool more = next < keys.k1;
    const bool cut = least < min(j0 + 32, keys.k1);
    f32x16 s[1];
    typename Mma<T>::V8 p[2];
    wait_loads<2 * kPer>();
    scores<T, D, 1>(r, k, s);
    wait_reads();
    if (more) {
      lo = keys.place(2 * b + 2);
      hi = keys.place(2 * b + 3);
      load_k(next);
    }
    uint64_t seen = 0;
    if (cut || !keys.template all<32>(j0)) {
      seen = keys.template seen<32>(j0);
      hide<1>(s, r.limit, j0, seen);
    }
    refer_to<T, D>(r, largest<1>(s, a.scale2));
    weigh<T, D>(r, s[0], p, a.scale2);
    if (more) wait_loads<2 * kPer>();
    else wait_loads<0>();
    if (cut && has_odd<T, D, 32>(v)) take_odd_out<T, D, 32, false>(r, v, j0, seen);
    add_values<T, D>(r, v, p);
    wait_reads();
    if (more) load_v(next);
  }
}

// Four waves of 32 rows each over blocks of 64 keys that they share: many
// rows, bound by the matrix cores.  The scores of the next block are computed
// beside the weights of this one, and their maximum beside the product with
// V: a wave has a SIMD to itself, or shares it with one that waits for
// memory, and has to keep matrix and vector units busy.  K and V have two
// buffers each, K a block ahead.  Each wave loads a group of 16 keys.
template <typename T, int D>
__device__ __forceinline__ void attend_wide(const AttnArgs &a, Rows32<T, D> &r, Keys &keys, int entry, int least, uint32_t lds) {
  using M = Mma<T>;
  using V8 = typename M::V8;
  constexpr int kPer = D / 32, kSteps = D / 8, kPitch = Geometry<D>::kPitch;
  constexpr uint32_t kBlock = 64 * kPitch, kGroup = 16 * kPitch;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float c = a.scale2;
  const int k0 = keys.k0, k1 = keys.k1, n = (k1 - k0 + 63) / 64;
  uint32_t k_off[kPer], v_off[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    k_off[i] = row_offset<D, false>(i, a.k_token);
    v_off[i] = row_offset<D, true>(i, a.v_token);
  }
  const uint32_t own = lds + wave * kGroup;
  keys.look_up(0, entry);
  Place now = keys.place(wave), last;  // of the block whose K, and the one whose V is loaded
  load_group<D, false, false>(keys, now, k0 + 16 * wave, k_off, own);
  load_group<D, true, false>(keys, now, k0 + 16 * wave, v_off, own + 2 * kBlock);
  if (n > 1) {
    now = keys.place(4 + wave);
    load_group<D, false, false>(keys, now, k0 + 64 + 16 * wave, k_off, own + kBlock);
  }
  wait_rows<T, D>(r);
  wait_loads<0>();
  __syncthreads();
  f32x16 s[2];
  scores<T, D, 2>(r, lds, s);
  uint64_t seen = 0;
  bool cut = least < min(k0 + 64, k1);
  if (cut || !keys.template all<64>(k0)) {
    seen = keys.template seen<64>(k0);
    hide<2>(s, r.limit, k0, seen);
  }
  float top = largest<2>(s, c);
  const int lane = threadIdx.x & 63, row = lane & 31, hb = lane >> 5, al = lane & 15;
  const uint32_t vrow = 4 * hb + (al >> 2), vcol = 2 * ((lane >> 4) & 1) + ((al & 3) >> 1);
  // A lane's first row and 16-byte piece of K and V.
  uint32_t krow = row * kPitch, kpiece = hb ^ k_swizzle<D>(row);
  uint32_t vlane = vrow * kPitch + (al & 1) * 8, vpiece = vcol ^ v_swizzle<D>(vrow);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    // K of the next block and V of this one are there, and every wave has
    // read K of this one and V of the last one.
    wait_loads<0>();
    __syncthreads();
    const int j0 = k0 + 64 * j;
    const uint32_t odd = (j & 1) * kBlock;
    if (j + 1 < n) {
      last = now;
      if (j + 2 < n) {
        now = keys.place(4 * (j + 2) + wave);
        load_group<D, false, false>(keys, now, j0 + 128 + 16 * wave, k_off, own + odd);
      }
      load_group<D, true, false>(keys, last, j0 + 64 + 16 * wave, v_off, own + 2 * kBlock + (kBlock - odd));
    }
    const uint32_t k = lds + (kBlock - odd), v = lds + 2 * kBlock + odd;
    // (addresses are computed in each block and not kept in registers)
    asm volatile("" : "+v"(krow), "+v"(kpiece), "+v"(vlane), "+v"(vpiece));
    refer_to<T, D>(r, top);
    const float base = r.m == -INFINITY ? 0.f : r.m;
    auto read_k = [&](int x) {
      return *reinterpret_cast<const LdsS8 *>(k + krow + (((2 * (x / 2)) ^ kpiece) << 4) + x % 2 * 32 * kPitch);
    };
    auto read_v = [&](int c2, int t) {
      const uint32_t at = v + vlane + (((4 * t) ^ vpiece) << 4) + c2 * 16 * kPitch;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at + 8 * kPitch));
      return static_cast<s16x8>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    V8 p[4];
    auto weigh_one = [&](int i) {
      const float w = __builtin_amdgcn_exp2f(s[i / 16][i % 16] * c - base);
      r.l += w;
      p[i / 8][i % 8] = M::from(w);
    };
    s16x8 kf[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) kf[x] = read_k(x);
#pragma unroll
    for (int i = 0; i < 16; ++i) weigh_one(i);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 next[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) next[b][i] = 0.f;
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      next[x % 2] = M::mul(__builtin_bit_cast(V8, kf[x % 8]), r.q[x / 2], next[x % 2]);
      if (x + 8 < kSteps) kf[x % 8] = read_k(x + 8);
      // Between the products: the other half of the weights.
#pragma unroll
      for (int i = 16 + x * 16 / kSteps; i < 16 + (x + 1) * 16 / kSteps; ++i) weigh_one(i);
      __builtin_amdgcn_sched_barrier(0);
    }
    // (the weights are computed here, not where they are used)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      s16x8 y = __builtin_bit_cast(s16x8, p[x]);
      asm volatile("" : "+v"(y));
      p[x] = __builtin_bit_cast(V8, y);
    }
    if (cut && has_odd<T, D, 64>(v)) take_odd_out<T, D, 64, true>(r, v, j0, seen);
    s16x8 vf[2][kPer];
#pragma unroll
    for (int t = 0; t < kPer; ++t) vf[0][t] = read_v(0, t);
    s[0] = next[0];
    s[1] = next[1];
    cut = least < min(j0 + 128, k1);
    if (cut || !keys.template all<64>(j0 + 64)) {
      seen = keys.template seen<64>(j0 + 64);
      hide<2>(s, r.limit, j0 + 64, seen);
    }
    top = s[0][0];
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      const int t = x % kPer, c2 = x / kPer;
      r.o[t] = M::mul(__builtin_bit_cast(V8, vf[c2 % 2][t]), p[c2], r.o[t]);
      if (c2 < 3) vf[(c2 + 1) % 2][t] = read_v(c2 + 1, t);
      // Between the products: the next block's maximum.
#pragma unroll
      for (int i = x * 32 / kSteps; i < (x + 1) * 32 / kSteps; ++i) top = fmaxf(top, s[i / 16][i % 16]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const float2 tops = both_halves(top);
    top = fmaxf(tops.x, tops.y) * c;
  }
}

// Keys that token t sees of a request of `seq` keys whose tokens end at
// `stop`; there are none behind the table's row.
__device__ __forceinline__ int limit_of(const AttnArgs &a, int seq, int stop, int t) {
  const int64_t n = static_cast<int64_t>(seq) - stop + t + 1;
  return static_cast<int>(max(static_cast<int64_t>(0), min(n, static_cast<int64_t>(a.max_keys))));
}

// The request of a token: tried first as one token a request (a load of all
// that is needed then, before the answer is known), else by bisection.
struct Request {
  int r, start, stop, seq, end;

  __device__ __forceinline__ Request(const AttnArgs &a, int t) {
    r = min(max(t, 0), a.n_requests - 1);
    start = a.starts[r];
    stop = a.starts[r + 1];
    seq = a.seq_lens[r];
    end = a.starts[a.n_requests];
  }
  // False if token t is none of a request's.
  __device__ __forceinline__ bool find(const AttnArgs &a, int t) {
    if (start <= t && t < stop) return true;
    if (t >= end) return false;
    int lo = 0, hi = a.n_requests;  // the first of 0 .. R whose start lies behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] > t) hi = mid;
      else lo = mid + 1;
    }
    if (lo == 0) return false;
    r = lo - 1;
    stop = a.starts[lo];
    seq = a.seq_lens[r];
    return true;
  }
};

typedef const __attribute__((address_space(4))) int32_t *ScalarInts;

// The least limit of a wave's rows, or (ALL) of the four waves'.
template <bool ALL> __device__ __forceinline__ int least_limit(int limit, uint8_t *lds) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) limit = min(limit, __shfl_xor(limit, d));
  if constexpr (ALL) {
    int *w = reinterpret_cast<int *>(lds);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = limit;
    __syncthreads();
    limit = min(min(w[0], w[1]), min(w[2], w[3]));
    __syncthreads();
  }
  return __builtin_amdgcn_readfirstlane(limit);
}

// Keys of one part of a request with `own` keys of its own: parts enough to
// fill the chip, of one tile at least and 8 where requests are many (a part's
// start and end cost about two tiles' time), and no more than there are.
__device__ __forceinline__ int own_chunk(const AttnArgs &a, int own) {
  own = max(own, 1);
  const int most = (own + a.own_parts - 1) / a.own_parts, fill = min(kOwnChunk, (own + a.own_want - 1) / a.own_want);
  return (max(most, fill) + 31) / 32 * 32;
}

// The first workgroups take the prefix, the others the requests' own keys:
// the long ones start first, one on every other CU or so, and both kinds run
// beside each other (dealing them in turn instead put all prefix work on half
// of the CUs, since the dispatcher goes round the shader engines).  Of 8
// consecutive workgroups each runs on an XCD of its own; the row tiles of one
// (KV head, prefix part) go to one XCD, whose L2 then holds that part.
template <typename T, int D, bool WIDE> __global__ void __launch_bounds__(256, D > 128 ? 1 : 2) attend(AttnArgs a) {
  extern __shared__ uint8_t lds[];
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31;
  const int group = blockIdx.x / 8, xcd = blockIdx.x % 8;
  Rows32<T, D> r;
  if (group < a.prefix_groups) {
    const int pair = group / a.prefix_tiles * 8 + xcd, tile = group % a.prefix_tiles;
    if (pair >= a.kv_heads * a.prefix_parts) return;
    const int h = pair % a.kv_heads, part = pair / a.kv_heads;
    const int x = tile * (WIDE ? 128 : 32) + (WIDE ? wave * 32 : 0) + n;
    int t = x < a.n_tokens * a.group ? x / a.group : -1, limit = 0;
    const int k0 = part * a.prefix_chunk, k1 = min(a.shared_len, k0 + a.prefix_chunk);
    Keys keys{a, a.shared, a.shared_width, k0, k1, k0 + (WIDE ? 0 : 32 * wave), WIDE ? 32 : 128, h * a.k_head, h * a.v_head,
              a.block_size % 16 != 0};
    const int entry = keys.entry(0);
    Request q(a, t);
    if (t >= 0) {
      if (q.find(a, t)) limit = limit_of(a, q.seq, q.stop, t);
      else t = -1;
    }
    load_rows<T, D>(a, r, t, h * a.group + (t < 0 ? 0 : x % a.group), limit);
    const int least = least_limit<WIDE>(r.limit, lds);
    if constexpr (WIDE) attend_wide<T, D>(a, r, keys, entry, least, at);
    else attend_narrow<T, D, false>(a, r, keys, entry, least, at + wave * (2 * 32 * D * 2));
    store_part<T, D, !WIDE>(a, r, limit <= 0, part, lds);
    return;
  }
  // A request's own keys: a wave an item, on its own.  The KV heads of a
  // request are neighbours, so that a workgroup reads whole rows of tokens.
  const int item = ((blockIdx.x - a.prefix_groups * 8) * 4 + wave);
  if (item >= a.own_items) return;
  // (the parts that only long requests have come last: in turn they would
  // fall on some XCDs alone)
  const int h = item % a.kv_heads, y = item / a.kv_heads;
  const int first = y % a.own_tiles, z = y / a.own_tiles;
  const int q = z % a.n_requests, part = z / a.n_requests;
  const ScalarInts starts = (ScalarInts)(a.starts + q), seq_lens = (ScalarInts)(a.seq_lens + q);
  const int start = starts[0], stop = starts[1], seq = seq_lens[0];
  const int t0 = max(0, start), t1 = min(a.n_tokens, stop);
  const int n_rows = max(0, t1 - t0) * a.group;
  const int end = t1 > t0 ? limit_of(a, seq, stop, t1 - 1) : 0;
  // Parts from a multiple of 32 keys: only the first one begins inside a group.
  const int from = a.shared_len & ~31, chunk = own_chunk(a, end - from);
  const int k0 = from + min(part * chunk, max(0, end - from));
  for (int m = first * 32; m < n_rows; m += a.own_tiles * 32) {
    const int x = m + n;
    const int t = x < n_rows ? t0 + x / a.group : -1;
    const int limit = t >= 0 ? limit_of(a, seq, stop, t) : 0;
    const int head = h * a.group + (t < 0 ? 0 : x % a.group);
    Keys keys{a, a.table + q * a.table_stride, a.width, max(a.shared_len, k0), min(end, k0 + chunk), k0, 32, h * a.k_head,
              h * a.v_head, a.block_size % 16 != 0};
    if (keys.k0 >= keys.k1) {  // an empty part
      if (t >= 0 && lane < 32)
        a.part_ml[(a.prefix_parts + part) * (static_cast<int64_t>(a.n_tokens) * a.heads) + t * a.heads + head] =
            make_float2(-INFINITY, 0.f);
      continue;
    }
    const int entry = keys.entry(0);
    load_rows<T, D>(a, r, t, head, limit);
    attend_narrow<T, D, true>(a, r, keys, entry, least_limit<false>(r.limit, lds), at + wave * (2 * 32 * D * 2));
    store_rows<T, D>(a, r, limit <= 0, a.prefix_parts + part);
  }
}

// Joins the parts of a row: four waves take a quarter of them each, D / 4
// lanes a row.
template <typename T, int D> __global__ void __launch_bounds__(256) join_parts(AttnArgs a) {
  constexpr int kQuads = D / 4, kRows = 64 / kQuads;
  using S = typename T::S;
  __shared__ f32x4 sums[4][64];
  __shared__ float2 weights[4][kRows];
  const int64_t rows = static_cast<int64_t>(a.n_tokens) * a.heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane / kQuads, d = lane % kQuads * 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + i;
  const bool there = i < kRows && row < rows;
  const int t = there ? static_cast<int>(row / a.heads) : -1, h = static_cast<int>(row % a.heads);
  const int parts = a.prefix_parts + a.own_parts;
  auto weight = [&](int p) { return there && p < parts ? a.part_ml[p * rows + row] : make_float2(-INFINITY, 0.f); };
  float2 w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = weight(wave + 4 * k);
  const bool live = t >= a.starts[0] && t < a.starts[a.n_requests];
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    for (int p0 = wave; p0 < parts; p0 += 16) {
      f32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (w[k].y != 0.f) x[k] = *reinterpret_cast<const f32x4 *>(a.part_o + ((p0 + 4 * k) * rows + row) * D + d);
      float2 next[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) next[k] = weight(p0 + 16 + 4 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (w[k].y == 0.f) continue;
        const float top = fmaxf(m, w[k].x), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(w[k].x - base);
        l = l * f + w[k].y * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f + x[k][e] * g;
        m = top;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = next[k];
    }
    sums[wave][lane] = o;
    if (d == 0) weights[wave][i] = make_float2(m, l);
  }
  __syncthreads();
  if (wave != 0 || !live) return;
  float top = -INFINITY;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    w[g] = weights[g][i];
    top = fmaxf(top, w[g].x);
  }
  const float base = top == -INFINITY ? 0.f : top;
  l = 0.f;
  o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (w[g].y == 0.f) continue;
    const float f = __builtin_amdgcn_exp2f(w[g].x - base);
    const f32x4 x = sums[g][lane];
    l += f * w[g].y;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += f * x[e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  Pack<S, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y.v[e] = from_f32<T>(o[e] * inv);
  *reinterpret_cast<Pack<S, 4> *>(static_cast<S *>(a.o) + t * a.o_token + h * a.o_head + d) = y;
  if (a.lse && d == 0) a.lse[t * a.lse_token + h * a.lse_head] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.69314718056f;
}

template <typename T, int D> void launch(const AttnArgs &a, bool wide, uint32_t groups, hipStream_t s) {
  const void *fn = wide ? reinterpret_cast<const void *>(attend<T, D, true>) : reinterpret_cast<const void *>(attend<T, D, false>);
  if (Lds<D>::kBytes > 64 * 1024)
    hip_check(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, Lds<D>::kBytes), "attend shared memory");
  if (wide) hipLaunchKernelGGL((attend<T, D, true>), dim3(groups * 8), dim3(256), Lds<D>::kBytes, s, a);
  else hipLaunchKernelGGL((attend<T, D, false>), dim3(groups * 8), dim3(256), Lds<D>::kBytes, s, a);
  hip_check(hipGetLastError(), "attend launch");
  constexpr int kRows = 64 / (D / 4);
  const int64_t rows = static_cast<int64_t>(a.n_tokens) * a.heads;
  hipLaunchKernelGGL((join_parts<T, D>), dim3(static_cast<uint32_t>((rows + kRows - 1) / kRows)), dim3(256), 0, s, a);
  hip_check(hipGetLastError(), "join_parts launch");
}

template <typename T> void launch_dim(const AttnArgs &a, int64_t dim, bool wide, uint32_t groups, hipStream_t s) {
  switch (dim) {
  case 64: launch<T, 64>(a, wide, groups, s); break;
  case 96: launch<T, 96>(a, wide, groups, s); break;
  case 128: launch<T, 128>(a, wide, groups, s); break;
  case 192: launch<T, 192>(a, wide, groups, s); break;
  default: launch<T, 256>(a, wide, groups, s); break;
  }
}

// Key numbers and what is added to them stay far from 2^31.
constexpr int64_t kMaxKeys = int64_t(1) << 30;

// How a call's work is cut, from its sizes alone (the lengths are on the GPU).
struct Plan {
  bool wide;
  int prefix_tiles, prefix_parts, prefix_chunk;
  int own_tiles, own_parts, own_want;
};

Plan make_plan(int64_t T, int64_t R, int64_t kv_heads, int64_t group, int64_t shared_len, int64_t table_keys) {
  Plan p;
  const int64_t rows = T * group;  // of a KV head
  p.wide = rows > 64;
  const int64_t m = p.wide ? 128 : 32, tile = p.wide ? 64 : 128;
  p.prefix_tiles = static_cast<int>((rows + m - 1) / m);
  // Rows of a request, about.  (The lengths are on the GPU.  A request far above
  // the mean goes through its tiles in turn: 255 requests of one new token and
  // one of 2048, over 4096 shared keys, take 4.3 ms together and 0.12 + 0.39 in
  // two calls.)
  const int64_t per = (T + R - 1) / R * group;
  p.own_tiles = static_cast<int>(std::max<int64_t>(1, (per + 31) / 32));
  const int64_t own = std::max<int64_t>(0, table_keys - shared_len);
  const int64_t items = p.prefix_tiles * kv_heads, own_items = R * kv_heads * p.own_tiles;
  // Two workgroups fit a CU.  The prefix gets 3/2 of its share of those 512
  // places, at a key of its own in half of the time of a request's own key
  // (which comes from memory, while all row tiles read the prefix; requests
  // are taken to have half of their tables' keys, 512 at most), so that both
  // end together: 256 requests, 32 heads over 16384 keys, up to 1024 own: 151
  // to 155 us, with 7/4 of its share 160.  A part has four wide
  // blocks or one round of narrow ones at least: it costs a row of 32-bit
  // sums to write and read.  Under three parts are rounded up, since one
  // part's time is then the call's: 256 requests over 4096 and 8192 shared
  // keys take 118 and 126 us with 2 and 3, 134 and 135 with 1 and 2; above,
  // the nearest is better (12000 keys: 138 us with 3, 142 with 4).
  const double prefix_cost = static_cast<double>(items) * shared_len;
  const double own_cost = static_cast<double>(own_items) * std::min<int64_t>(own, 1024);
  const int64_t places = static_cast<int64_t>(std::min(512.0, 768 * prefix_cost / (prefix_cost + own_cost + 1)));
  const int64_t most = p.wide ? std::max<int64_t>(1, shared_len / (4 * tile)) : (shared_len + tile - 1) / tile;
  p.prefix_parts = shared_len == 0 ? 0 : static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, (places + (places < 3 * items ? items - 1 : items / 2)) / items)));
  p.prefix_chunk = 0;
  if (p.prefix_parts) {
    p.prefix_chunk = static_cast<int>(((shared_len + p.prefix_parts - 1) / p.prefix_parts + tile - 1) / tile * tile);
    p.prefix_parts = static_cast<int>((shared_len + p.prefix_chunk - 1) / p.prefix_chunk);
  }
  // Own keys: parts enough to fill the chip and of kOwnChunk keys at most, up
  // to 8, or to 64 where that makes 4096 waves; a request takes those that its
  // length calls for (own_chunk).
  p.own_want = static_cast<int>(std::max<int64_t>(1, (2048 + own_items - 1) / own_items));
  const int64_t own_most = std::min<int64_t>(std::max<int64_t>(8, std::min<int64_t>(64, 4096 / own_items)),
                                             std::max<int64_t>(p.own_want, (own + 31 + kOwnChunk - 1) / kOwnChunk));
  p.own_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(own_most, (own + 62) / 32)));
  return p;
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_shared_prefix_attention(const lmc_tensor *query, const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                                           const lmc_tensor *shared_blocks, int64_t shared_len,
                                           const lmc_tensor *block_table, const lmc_tensor *seq_lens,
                                           const lmc_tensor *query_start_loc, double scale, const lmc_tensor *output,
                                           const lmc_tensor *lse, const lmc_tensor *workspace, int64_t *workspace_bytes,
                                           int32_t kvcache_format, int32_t vllm_two_major, void *stream) {
  return guarded([&] {
    const lmc_tensor &q = deref(query, "query");
    const lmc_tensor &o = deref(output, "output");
    const lmc_tensor &sb = deref(shared_blocks, "shared_blocks");
    const lmc_tensor &bt = deref(block_table, "block_table");
    const lmc_tensor &sl = deref(seq_lens, "seq_lens");
    const lmc_tensor &qs = deref(query_start_loc, "query_start_loc");
    const PagedKv kv = paged_kv(vllm_kv_caches, n_caches, kvcache_format, vllm_two_major != 0, "shared_prefix_attention");
    const int dev = kv.device;
    if (kv.dtype != LMC_BF16 && kv.dtype != LMC_F16)
      fail(LMC_ERR_VALUE, "shared_prefix_attention takes bfloat16 or float16 caches only");
    check_on(q, "query", dev, kv.dtype);
    check_on(o, "output", dev, kv.dtype);
    check_vector(sb, "shared_blocks", dev, LMC_I32);
    check_on(bt, "block_table", dev, LMC_I32);
    check_vector(sl, "seq_lens", dev, LMC_I32);
    check_vector(qs, "query_start_loc", dev, LMC_I32);
    expect(kv.dim == 64 || kv.dim == 96 || kv.dim == 128 || kv.dim == 192 || kv.dim == 256,
                "shared_prefix_attention takes heads of 64, 96, 128, 192 or 256 dims");
    expect(q.ndim == 3 && o.ndim == 3, "query and output must be [tokens, heads, dim]");
    const int64_t T = q.sizes[0], R = sl.sizes[0], Hq = q.sizes[1];
    for (int i = 0; i < 3; ++i) {
      expect(q.sizes[i] == o.sizes[i], "query and output differ in shape");
      expect(q.strides[i] >= 0 && o.strides[i] >= 0, "negative strides unsupported");
    }
    expect(q.sizes[2] == kv.dim, "query heads are not of the caches' dim");
    expect(q.strides[2] == 1 && o.strides[2] == 1, "a head's dims must be adjacent");
    expect(Hq % kv.heads == 0, "query heads are not a multiple of the caches' heads");
    expect(qs.sizes[0] == R + 1, "query_start_loc must have one entry per request and one more");
    expect(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    expect(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    expect(shared_len >= 0 && shared_len <= kMaxKeys, "shared_len must be between 0 and 2^30");
    expect(bt.sizes[1] * kv.block_size <= kMaxKeys, "a block_table row spans more than 2^30 keys");
    expect((shared_len + kv.block_size - 1) / kv.block_size <= sb.sizes[0], "shared_blocks has too few blocks for shared_len");
    // (a scale of zero in 32 bits would make NaN of the keys that are not seen)
    const float scale2 = static_cast<float>(scale * 1.4426950408889634);
    expect(scale2 >= std::numeric_limits<float>::min() && std::isfinite(scale2), "scale must be positive and finite in 32 bits");
    AttnArgs a;
    std::memset(&a, 0, sizeof(a));
    if (lse) {
      const lmc_tensor &e = deref(lse, "lse");
      check_on(e, "lse", dev, LMC_F32);
      expect(e.ndim == 2 && e.sizes[0] == T && e.sizes[1] == Hq, "lse must be [tokens, heads]");
      expect(rows_apart({T, Hq}, {e.strides[0], e.strides[1]}), "lse has overlapping rows");
      a.lse = static_cast<float *>(e.data);
      a.lse_token = e.strides[0];
      a.lse_head = e.strides[1];
    }
    auto on_16 = [](int64_t x) { return x % 16 == 0; };
    // (the stride of a dim of one entry says nothing)
    auto steps_16 = [](int64_t n, int64_t stride) { return n <= 1 || stride % 16 == 0; };
    expect(on_16(reinterpret_cast<intptr_t>(kv.k)) && on_16(reinterpret_cast<intptr_t>(kv.v)) &&
                    steps_16(kv.pages, kv.k_page) && steps_16(kv.block_size, kv.k_token) && steps_16(kv.heads, kv.k_head) &&
                    steps_16(kv.pages, kv.v_page) && steps_16(kv.block_size, kv.v_token) && steps_16(kv.heads, kv.v_head),
                "the paged caches' rows must start on 16-byte boundaries");
    expect(on_16(reinterpret_cast<intptr_t>(q.data)) && steps_16(T, q.strides[0] * 2) && steps_16(Hq, q.strides[1] * 2) &&
                    on_16(reinterpret_cast<intptr_t>(o.data)) && steps_16(T, o.strides[0] * 2) && steps_16(Hq, o.strides[1] * 2),
                "rows of query and output must start on 16-byte boundaries");
    expect(rows_apart({T, Hq, kv.dim}, {o.strides[0], o.strides[1], 1}), "output has overlapping rows");
    // A lane's offset from the first of 16 rows has 32 bits.
    expect(kv.block_size == 1 || std::max(kv.k_token, kv.v_token) < (int64_t(1) << 27),
                "rows of the paged caches are 2^27 bytes or more apart");
    expect(T * Hq <= INT32_MAX / 128 && R <= INT32_MAX / 4096, "too many rows");
    const int64_t group = kv.heads ? Hq / kv.heads : 0;
    if (workspace_bytes) *workspace_bytes = 0;
    if (T == 0 || Hq == 0 || R == 0) return;
    const int64_t keys = bt.sizes[1] * kv.block_size;
    const Plan p = make_plan(T, R, kv.heads, group, shared_len, keys);
    const int64_t parts = p.prefix_parts + p.own_parts, rows = T * Hq;
    const int64_t bytes = parts * rows * (kv.dim * 4 + 8);
    // A launch has less than 2^32 threads along a dimension.
    const int64_t own_items = R * kv.heads * p.own_tiles * p.own_parts, own_groups = (own_items + 31) / 32;
    const int64_t prefix_groups = (kv.heads * p.prefix_parts + 7) / 8 * p.prefix_tiles;
    expect((own_groups + prefix_groups) * 8 <= UINT32_MAX / 256, "too many rows");
    if (workspace_bytes) {
      *workspace_bytes = bytes;
      return;
    }
    const lmc_tensor &ws = deref(workspace, "workspace");
    check_on(ws, "workspace", dev, LMC_U8);
    expect(ws.ndim == 1 && (ws.sizes[0] <= 1 || ws.strides[0] == 1) && ws.sizes[0] >= bytes &&
                    on_16(reinterpret_cast<intptr_t>(ws.data)),
                "workspace must be 1-D, contiguous, on a 16-byte boundary and of at least ", (bytes), " bytes");
    // The parts are joined in a launch of its own: output and lse may lie over query.
    expect(!lse || !may_share(o, *lse), "output and lse overlap");
    for (const lmc_tensor *out : {output, lse, workspace}) {
      if (!out) continue;
      expect(!extents_meet(*out, qs) && !extents_meet(*out, sl) && !extents_meet(*out, bt) && !extents_meet(*out, sb),
                  "output, lse or workspace overlap the tables or the lengths");
      for (int i = 0; i < n_caches; ++i)
        expect(!extents_meet(*out, vllm_kv_caches[i]), "output, lse or workspace overlap the paged caches");
    }
    expect(!extents_meet(ws, q) && !extents_meet(ws, o) && !(lse && extents_meet(ws, *lse)),
                "workspace overlaps query, output or lse");
    a.q = q.data;
    a.q_token = q.strides[0];
    a.q_head = q.strides[1];
    a.o = o.data;
    a.o_token = o.strides[0];
    a.o_head = o.strides[1];
    a.k = kv.k;
    a.v = kv.v;
    a.k_page = kv.k_page;
    a.k_token = kv.k_token;
    a.k_head = kv.k_head;
    a.v_page = kv.v_page;
    a.v_token = kv.v_token;
    a.v_head = kv.v_head;
    a.pages = static_cast<uint32_t>(kv.pages);
    // j / block_size = umulhi(j, mul) >> shift for j < 2^31 (block_size > 1).
    a.block_size = static_cast<uint32_t>(kv.block_size);
    if (kv.block_size > 1) {
      uint32_t log = 1;
      while ((int64_t(1) << log) < kv.block_size) ++log;
      a.block_mul = static_cast<uint32_t>((uint64_t(1) << (31 + log)) / kv.block_size + 1);
      a.block_shift = log - 1;
    }
    a.shared = static_cast<const int32_t *>(sb.data);
    a.shared_len = static_cast<int>(shared_len);
    a.shared_width = static_cast<uint32_t>(sb.sizes[0]);
    a.table = static_cast<const int32_t *>(bt.data);
    a.table_stride = bt.strides[0];
    a.width = static_cast<uint32_t>(bt.sizes[1]);
    a.seq_lens = static_cast<const int32_t *>(sl.data);
    a.starts = static_cast<const int32_t *>(qs.data);
    a.n_requests = static_cast<int>(R);
    a.n_tokens = static_cast<int>(T);
    a.heads = static_cast<int>(Hq);
    a.kv_heads = static_cast<int>(kv.heads);
    a.group = static_cast<int>(group);
    a.max_keys = static_cast<int>(std::max(shared_len, keys));
    a.scale2 = scale2;
    a.part_o = static_cast<float *>(ws.data);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + parts * rows * kv.dim);
    a.prefix_parts = p.prefix_parts;
    a.own_parts = p.own_parts;
    a.prefix_tiles = p.prefix_tiles;
    a.prefix_chunk = p.prefix_chunk;
    a.own_tiles = p.own_tiles;
    a.own_want = p.own_want;
    a.own_items = static_cast<int>(own_items);
    a.prefix_groups = static_cast<int>(prefix_groups);
    DeviceGuard guard(dev);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t groups = static_cast<uint32_t>(own_groups + prefix_groups);
    if (kv.dtype == LMC_BF16) launch_dim<BF16>(a, kv.dim, p.wide, groups, s);
    else launch_dim<F16>(a, kv.dim, p.wide, groups, s);
  });
}
