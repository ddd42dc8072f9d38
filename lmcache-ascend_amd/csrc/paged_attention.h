// Attention over paged K and V caches on the matrix cores of MI355X (gfx950):
// what the kernels of prefix_attention.hip and tree_attention.hip share.  The
// arguments of a call and their checks, tiles of keys from the caches to LDS,
// their infinities, masks and largest scores; and the steps of a tile that
// prefix_attention.hip takes (Rows32, has_odd, scores, refer_to, weigh,
// add_values: tree_attention.hip spreads a step over two products and has its
// own).
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
#pragma once

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

// What every kernel over the caches reads.
struct PagedArgs {
  const void *q;
  int64_t q_token, q_head;  // elements
  void *o;
  int64_t o_token, o_head;
  float *lse;               // may be null
  int64_t lse_token, lse_head;
  const uint8_t *k, *v;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  uint32_t pages, block_size, block_mul, block_shift;
  const int32_t *table;
  int64_t table_stride;
  uint32_t width;
  const int32_t *seq_lens, *starts;
  int n_requests, n_tokens;
  int heads, kv_heads, group;
  int max_keys;             // that a request can have
  float scale2;             // scale * log2(e)
};

// Read by scalar loads: addresses that are the same for a wave.
typedef const __attribute__((address_space(4))) int32_t *ScalarInts;

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
// That kernel, prefix_attention.hip's, is made for the former;
// tree_attention.hip's loads all keys so.  (m0 is reserved: nothing but these
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
template <typename T, int D> struct RowSums {
  typename Mma<T>::V8 q[D / 16];
  f32x16 o[D / 32];
  float m, l;   // m in powers of two; l of this lane's keys
  int row;      // token * heads + head, or -1
};

// Rows that see the keys before a limit.
template <typename T, int D> struct Rows32 : RowSums<T, D> {
  int limit;    // INT_MAX for a row that is none
  // Bit i: the row sees key j0 + i.
  __device__ __forceinline__ uint64_t visible(const PagedArgs &, int j0) const {
    const int left = limit - j0;
    return left >= 64 ? ~uint64_t(0) : left > 0 ? (uint64_t(1) << left) - 1 : 0;
  }
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

// Infinities and NaN in a tile of V that holds keys which some rows see and
// others do not: a weight of zero would make NaN of them.  The rows that see
// such a key (a bit of `seen`, of the lane's row) get its infinities and NaN
// added here; then they are taken out of the tile.
template <typename T, int D, int KEYS>
__device__ __forceinline__ void add_odd(RowSums<T, D> &r, uint32_t v, uint64_t seen) {
  using M = Mma<T>;
  constexpr int kPitch = Geometry<D>::kPitch;
  const int lane = threadIdx.x & 63, hb = lane >> 5;
#pragma unroll 1
  for (int key = 0; key < KEYS; ++key) {
    const bool see = (seen >> key) & 1;
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
}

// SHARED: all waves work on one tile, and all of them come here.
template <typename T, int D, int KEYS, bool SHARED> __device__ __forceinline__ void clear_odd(uint32_t v) {
  using M = Mma<T>;
  const int lane = threadIdx.x & 63;
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

template <typename T, int D, int KEYS, bool SHARED>
__device__ __forceinline__ void take_odd_out(RowSums<T, D> &r, uint32_t v, uint64_t seen) {
  add_odd<T, D, KEYS>(r, v, seen);
  clear_odd<T, D, KEYS, SHARED>(v);
}

// The steps of a tile of NB * 32 keys, in LDS at k and v.

// S^T = K Q^T: lane (n, hb) gets the scores of row n with the keys 32 b + 8 i
// + 4 hb + j of s[b][4 i + j].
template <typename T, int D, int NB>
__device__ __forceinline__ void scores(const RowSums<T, D> &r, uint32_t k, f32x16 (&s)[NB]) {
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
// clear.
template <int NB> __device__ __forceinline__ void hide(f32x16 (&s)[NB], uint64_t seen) {
  const int hb = (threadIdx.x & 63) >> 5;
  // Bit 32 b + 8 i + j: key 4 hb further.
  const uint64_t bits = seen >> (4 * hb);
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
template <typename T, int D> __device__ __forceinline__ void refer_to(RowSums<T, D> &r, float top) {
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
__device__ __forceinline__ void weigh(RowSums<T, D> &r, const f32x16 &s, typename Mma<T>::V8 (&p)[2], float c) {
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
__device__ __forceinline__ void add_values(RowSums<T, D> &r, uint32_t v, const typename Mma<T>::V8 (&p)[2]) {
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
  const PagedArgs &a;
  const int32_t *list;
  uint32_t n_list;
  int k0, k1, first, stride;
  int64_t k_off, v_off;  // of the head
  bool holes;            // blocks may lie outside the caches: ask for each key
  int base = 0;          // group of lane 0
  uint64_t groups = 0;   // which lanes' groups are whole
  uint64_t k = 0, v = 0;

  // Other keys of the same caches and head.
  __device__ __forceinline__ void turn_to(const int32_t *other, int from, int to, bool with_holes) {
    list = other;
    k0 = first = from;
    k1 = to;
    holes = with_holes;
  }

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
  __device__ __forceinline__ int entry(int g) const { return entry_of(list, key(g + (threadIdx.x & 63)), k0, k1); }
  // The entry of a list for a key of [from, to].
  __device__ __forceinline__ int entry_of(const int32_t *of, int j, int from, int to) const {
    const uint32_t b = block_of(min(max(j, from), to));
    return n_list ? of[min(b, n_list - 1)] : -1;
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
  const PagedArgs &a = s.a;
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
template <typename T, int D> __device__ __forceinline__ void wait_rows(RowSums<T, D> &r) {
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) {
    s16x8 x = __builtin_bit_cast(s16x8, r.q[kc]);
    asm volatile("" : "+v"(x));
    r.q[kc] = __builtin_bit_cast(typename Mma<T>::V8, x);
  }
}

// A lane's query row to registers: head `head` of token t, -1 without one.
template <typename T, int D> __device__ __forceinline__ void load_query(const PagedArgs &a, RowSums<T, D> &r, int t, int head) {
  using S = typename T::S;
  const int hb = (threadIdx.x & 63) >> 5;
  const bool there = t >= 0;
  const S *q = static_cast<const S *>(a.q) + (there ? t * a.q_token + head * a.q_head : 0);
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) {
    s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) x = *reinterpret_cast<const s16x8 *>(q + kc * 16 + hb * 8);
    r.q[kc] = __builtin_bit_cast(typename Mma<T>::V8, x);
  }
}

// Nothing summed up.
template <typename T, int D> __device__ __forceinline__ void clear_sums(RowSums<T, D> &r) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) r.o[i][e] = 0.f;
  r.m = -INFINITY;
  r.l = 0.f;
}

template <typename T, int D> __device__ __forceinline__ void load_rows(const PagedArgs &a, RowSums<T, D> &r, int t, int head) {
  r.row = t >= 0 ? t * a.heads + head : -1;
  load_query(a, r, t, head);
  clear_sums(r);
}

// Key numbers and what is added to them stay far from 2^31.
constexpr int64_t kMaxKeys = int64_t(1) << 30;

inline bool on_16(int64_t x) { return x % 16 == 0; }

// Sizes of a call whose arguments fit each other.
struct PagedSizes {
  PagedKv kv;
  int64_t tokens, requests, heads, group;
  int64_t keys;             // of a table row
};

// Checks what every attention over the caches is given, and fills the
// kernel's arguments (all but the workspace) from it.
inline PagedSizes paged_call(PagedArgs &a, const char *op, const lmc_tensor *query, const lmc_tensor *vllm_kv_caches,
                             int32_t n_caches, int32_t kvcache_format, bool two_major, const lmc_tensor *block_table,
                             const lmc_tensor *seq_lens, const lmc_tensor *query_start_loc, double scale,
                             const lmc_tensor *output, const lmc_tensor *lse) {
  const lmc_tensor &q = deref(query, "query");
  const lmc_tensor &o = deref(output, "output");
  const lmc_tensor &bt = deref(block_table, "block_table");
  const lmc_tensor &sl = deref(seq_lens, "seq_lens");
  const lmc_tensor &qs = deref(query_start_loc, "query_start_loc");
  const PagedKv kv = paged_kv(vllm_kv_caches, n_caches, kvcache_format, two_major, op);
  const int dev = kv.device;
  expect(kv.dtype == LMC_BF16 || kv.dtype == LMC_F16, op, " takes bfloat16 or float16 caches only");
  check_on(q, "query", dev, kv.dtype);
  check_on(o, "output", dev, kv.dtype);
  check_on(bt, "block_table", dev, LMC_I32);
  check_vector(sl, "seq_lens", dev, LMC_I32);
  check_vector(qs, "query_start_loc", dev, LMC_I32);
  expect(kv.dim == 64 || kv.dim == 96 || kv.dim == 128 || kv.dim == 192 || kv.dim == 256, op,
         " takes heads of 64, 96, 128, 192 or 256 dims");
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
  expect(bt.sizes[1] * kv.block_size <= kMaxKeys, "a block_table row spans more than 2^30 keys");
  // (a scale of zero in 32 bits would make NaN of the keys that are not seen)
  a.scale2 = static_cast<float>(scale * 1.4426950408889634);
  expect(a.scale2 >= std::numeric_limits<float>::min() && std::isfinite(a.scale2), "scale must be positive and finite in 32 bits");
  if (lse) {
    const lmc_tensor &e = deref(lse, "lse");
    check_on(e, "lse", dev, LMC_F32);
    expect(e.ndim == 2 && e.sizes[0] == T && e.sizes[1] == Hq, "lse must be [tokens, heads]");
    expect(rows_apart({T, Hq}, {e.strides[0], e.strides[1]}), "lse has overlapping rows");
    a.lse = static_cast<float *>(e.data);
    a.lse_token = e.strides[0];
    a.lse_head = e.strides[1];
  }
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
  const int64_t keys = bt.sizes[1] * kv.block_size;
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
  a.table = static_cast<const int32_t *>(bt.data);
  a.table_stride = bt.strides[0];
  a.width = static_cast<uint32_t>(bt.sizes[1]);
  a.seq_lens = static_cast<const int32_t *>(sl.data);
  a.starts = static_cast<const int32_t *>(qs.data);
  a.n_requests = static_cast<int>(R);
  a.n_tokens = static_cast<int>(T);
  a.heads = static_cast<int>(Hq);
  a.kv_heads = static_cast<int>(kv.heads);
  a.group = static_cast<int>(Hq / kv.heads);
  a.max_keys = static_cast<int>(keys);
  return {kv, T, R, Hq, Hq / kv.heads, keys};
}

// The caller's scratch: large enough, and apart from all that the call reads
// and writes; output and lse apart from the caches and from `inputs`, the call's
// tables and lengths.  Whether output or lse may lie over query is the call's to
// check: it depends on when the kernel writes them.
inline void check_outputs(const lmc_tensor *query, const lmc_tensor *output, const lmc_tensor *lse,
                          const lmc_tensor *workspace, int64_t bytes, int device, const lmc_tensor *vllm_kv_caches,
                          int32_t n_caches, std::initializer_list<const lmc_tensor *> inputs) {
  const lmc_tensor &ws = deref(workspace, "workspace");
  check_on(ws, "workspace", device, LMC_U8);
  expect(ws.ndim == 1 && (ws.sizes[0] <= 1 || ws.strides[0] == 1) && ws.sizes[0] >= bytes &&
             on_16(reinterpret_cast<intptr_t>(ws.data)),
         "workspace must be 1-D, contiguous, on a 16-byte boundary and of at least ", bytes, " bytes");
  expect(!lse || !may_share(*output, *lse), "output and lse overlap");
  for (const lmc_tensor *out : {output, lse, workspace}) {
    if (!out) continue;
    for (const lmc_tensor *in : inputs)
      expect(!extents_meet(*out, *in), "output, lse or workspace overlap the tables or the lengths");
    for (int i = 0; i < n_caches; ++i)
      expect(!extents_meet(*out, vllm_kv_caches[i]), "output, lse or workspace overlap the paged caches");
  }
  expect(!extents_meet(ws, *query) && !extents_meet(ws, *output) && !(lse && extents_meet(ws, *lse)),
         "workspace overlaps query, output or lse");
}

} // namespace

} // namespace lmc
