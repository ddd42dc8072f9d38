// Attention of drafted tokens over paged K and V caches on MI355X (gfx950).
//
//   o(t, h)   = sum_j softmax_j(scale q(t, h) . k(j)) v(j)
//   lse(t, h) = log sum_j exp(scale q(t, h) . k(j))
//
// over the keys j of token t's request that the token sees: all of the
// context, which is what lies before the request's drafted tokens, and those
// drafted tokens whose bit is set in the token's row of the mask.
//
// A tile is the rows of one request and KV head (drafted tokens times the
// heads of the group; 64, 128 or 256 of them) against blocks of 64 of the
// request's keys.  The lengths are on the GPU, so the cut is made there: a KV
// head's tiles, one request's behind the other's, are one line of key blocks,
// and each of its workgroups takes an equal piece of it, wherever requests
// begin and end.  A tile that lies in one piece is written at once; one that is
// cut leaves sums (32 bits, with their maximum) for every piece, which a second
// launch joins.  Each workgroup has two places for sums: one for a tile that an
// earlier workgroup began, one for a tile that a later one ends.
//
// Few rows are bound by the bytes of K and V, many by vector work beside the
// products (a wave's step of 32 keys at 128 dims: 16 products, about 96 vector
// instructions, of which 25 are addresses in LDS and 16 exponentials of four
// times the length) and by loads that are waited for once a block (below): 32
// requests of up to 8192 keys, 32 heads over 8 KV heads of 128 bf16 dims, take 95
// to 99 us with one token each (5.6 to 5.9 TB/s), 116 with 16, 147 to 152 with 32
// and 198 to 214 with 64 (663 to 725 TFLOP/s).  64 tokens over up to 16384 keys
// take 356 to 408 us: the clock falls to 1.6 GHz there.  2 requests of 8 tokens
// over 2000 keys: 15.0 us, the latency of two launches.  The join takes 10 us of
// 116 and 18 of 400.
//
// Registers at 128 dims: 255 for 64 rows, 256 for more (10 to 18 spilled outside of
// the loop over the keys), two waves a SIMD; at 96 dims 204 to 206; at 64 dims 176
// to 183, and 168 for 128 rows (three waves a SIMD, 6 or 7 spilled); at 192 and 256
// a wave a SIMD, with 128 to 204 accumulation registers.  111 to 155 scalar
// registers are kept in vector registers.
#include "paged_attention.h"

namespace lmc {

namespace {

struct TreeArgs : PagedArgs {
  const int64_t *mask;
  int64_t mask_token;
  int words;
  int pieces;               // of a KV head's line: workgroups [piece][KV head]
  // Sums of cut tiles: [piece][KV head][begun before, ended behind][rows].
  float *part_o;
  float2 *part_ml;
  // Of the place "ended behind": the pieces that follow (-1: nothing is there),
  // the tile's rows and the request's first token.
  struct Cut { int more, first_row, rows, start; } *cuts;
};

// How a call's work is cut, from its sizes alone (the lengths are on the GPU).
struct TreePlan {
  int64_t rows;                   // of a tile: 64, 128 or 256
  int64_t pieces, groups;         // of a KV head's line; workgroups
  int64_t cuts, join_groups;      // cut tiles at most; workgroups that share the rows of one
};

TreePlan make_plan(int64_t T, int64_t R, int64_t kv_heads, int64_t group, int64_t dim, int64_t keys) {
  TreePlan p;
  // Rows of a request and KV head, about.  A tile of up to 64 rows has a half of
  // each block's keys for each two waves, so that none idles; 128 rows of 128 dims
  // take 157 us with four row waves and halves, 220 as a tile of 256; 64 rows
  // take 128 us on 64 and 157 on 128.  At 64 dims 128 rows have workgroups of four
  // waves, three a CU (88 us; 100 with eight waves and halves).  192 dims do not
  // fit 256 rows' registers (two waves a SIMD), 256 dims not 128 rows' blocks in
  // LDS (five of 32 KB).  (The mean counts all rows, padding too: one wide tree
  // among many short ones reads its keys once for each 64 rows.)
  const int64_t per = (T + R - 1) / R * group;
  p.rows = per <= 64 || dim == 256 ? 64 : per <= 128 || dim == 192 ? 128 : 256;
  // Workgroups that the 256 CUs hold at once.
  const int64_t places = dim == 64 && p.rows == 128 ? 768 : dim <= 128 && p.rows == 64 ? 512 : 256;
  const int64_t tiles = T * group / p.rows + R;
  p.pieces = std::min(tiles * std::max<int64_t>(1, (keys + 63) / 64), std::max<int64_t>(1, places / kv_heads));
  p.groups = p.pieces * kv_heads;
  p.cuts = std::min(p.pieces - 1, tiles) * kv_heads;
  const int64_t step = 64 / (dim / 4);  // rows of a workgroup's turn
  p.join_groups = std::max<int64_t>(1, std::min((std::min(per, p.rows) + step - 1) / step, 8192 / std::max<int64_t>(1, p.cuts)));
  return p;
}

// Rows that see the context and the drafted tokens of their mask.
template <typename T, int D> struct TreeRows : RowSums<T, D> {
  int context;  // keys before the drafted tokens
  uint64_t word0;  // of the mask (loaded beside the query, not when it is needed)
  __device__ __forceinline__ void load_word(const TreeArgs &a, int t) {
    word0 = t >= 0 && a.words > 0 ? static_cast<uint64_t>(a.mask[t * a.mask_token]) : 0;
  }
  // Bit i: the row sees key j0 + i.
  __device__ __forceinline__ uint64_t visible(const PagedArgs &p, int j0) const {
    const TreeArgs &a = static_cast<const TreeArgs &>(p);
    const int d = j0 - context;
    if (d <= -64 || this->row < 0) return ~uint64_t(0);
    const int64_t *w = a.mask + static_cast<uint32_t>(this->row) / static_cast<uint32_t>(a.heads) * a.mask_token;
    auto word = [&](int i) { return i == 0 ? word0 : i < a.words ? static_cast<uint64_t>(w[i]) : 0; };
    if (d < 0) return (~uint64_t(0) >> (64 + d)) | (word(0) << -d);
    const int i = d >> 6, s = d & 63;
    return s ? (word(i) >> s) | (word(i + 1) << (64 - s)) : word(i);
  }
};

// What a tile's start and end take, in blocks of keys: units of the line that
// stand before the tile's first block, so that a piece with more tiles gets fewer
// blocks.  (Measured in a piece, a tile more takes 5 to 10 us, a block 2.6.)
// With 4: 32 requests of 16 tokens 125 us, trees of up to 77 45, of 64 over 16384
// keys 412; with 0: 128, 52, 430; with 8: 124, 46, 421.
constexpr int kStart = 4;

// One request's part of the line.
struct Span {
  int start, n_rows, context, end, blocks;  // rows of a KV head; keys; blocks of keys of a tile
  int64_t units;
};

template <int ROWS> __device__ __forceinline__ Span span_of(const TreeArgs &a, int start, int stop, int seq) {
  Span s;
  s.start = max(0, start);
  s.n_rows = max(0, min(a.n_tokens, stop) - s.start) * a.group;
  s.end = max(0, min(seq, a.max_keys));
  // (no mask reaches 2^29 tokens)
  s.context = static_cast<int>(max(static_cast<int64_t>(seq) - stop + start, -(int64_t(1) << 29)));
  // (rows without keys are written too)
  s.blocks = max(1, (s.end + 63) / 64);
  s.units = static_cast<int64_t>((s.n_rows + ROWS - 1) / ROWS) * (s.blocks + kStart);
  return s;
}
template <int ROWS> __device__ __forceinline__ Span span_of(const TreeArgs &a, int r) {
  return span_of<ROWS>(a, a.starts[r], a.starts[r + 1], a.seq_lens[r]);
}
// The same for a request that the wave has in common.
template <int ROWS> __device__ __forceinline__ Span span_of_all(const TreeArgs &a, int r) {
  const ScalarInts starts = (ScalarInts)(a.starts + r), seq_lens = (ScalarInts)(a.seq_lens + r);
  return span_of<ROWS>(a, starts[0], starts[1], seq_lens[0]);
}

// The request, and the unit of it, where a workgroup's piece begins.
struct Begin {
  int64_t each, left, unit;       // units of a piece, of this one; of the request before it
  int r;
  Span span;
};

// Blocks of a piece at least: a piece more for the join costs about as much as
// a block (2 requests of 8 tokens over 2000 keys: 17.5 us with 2, 18.3 with 1,
// 18.4 with 3, all before lengths were summed in registers).
constexpr int64_t kLeast = 2;

// All requests' units, summed: of up to 64 by each wave for itself, a request a
// lane (0.6 us less than through LDS), of more by the workgroup, a run of them a thread.
template <int ROWS, int THREADS> __device__ __forceinline__ Begin find_piece(const TreeArgs &a, int piece) {
  __shared__ int64_t sums[THREADS / 64];
  __shared__ Begin found;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // (the same in all lanes: to scalar registers)
  auto all32 = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto all64 = [&](int64_t x) {
    const uint32_t lo = all32(static_cast<int>(x)), hi = all32(static_cast<int>(x >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
  };
  // The sum of the lanes up to this one.
  auto sum_up = [&](int64_t x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t below = __shfl_up(x, d);
      if (lane >= d) x += below;
    }
    return x;
  };
  Begin b;
  b.left = b.unit = 0;
  b.r = 0;
  b.span = {0, 0, 0, 0, 1, 0};
  if (a.n_requests <= 64) {
    Span s = span_of<ROWS>(a, min(lane, a.n_requests - 1));
    if (lane >= a.n_requests) s.units = 0;
    const int64_t upto = sum_up(s.units), total = all64(__shfl(upto, 63));
    b.each = max((total + a.pieces - 1) / a.pieces, kLeast);
    const int64_t first = b.each * piece;
    const uint64_t here = __ballot(first >= upto - s.units && first < upto);
    if (here == 0) return b;
    const int from = __ffsll(static_cast<unsigned long long>(here)) - 1;
    b.left = min(b.each, total - first);
    b.unit = first - all64(__shfl(upto - s.units, from));
    b.r = from;
    b.span = {__builtin_amdgcn_readlane(s.start, from), __builtin_amdgcn_readlane(s.n_rows, from),
              __builtin_amdgcn_readlane(s.context, from), __builtin_amdgcn_readlane(s.end, from),
              __builtin_amdgcn_readlane(s.blocks, from), all64(__shfl(s.units, from))};
    return b;
  }
  const int per = (a.n_requests + THREADS - 1) / THREADS;
  const int r0 = min(a.n_requests, static_cast<int>(threadIdx.x) * per), r1 = min(a.n_requests, r0 + per);
  Span s;
  int64_t own = 0;
  for (int r = r0; r < r1; ++r) {
    s = span_of<ROWS>(a, r);
    own += s.units;
  }
  int64_t upto = sum_up(own);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) upto += sums[w];
    total += sums[w];
  }
  const int64_t each = max((total + a.pieces - 1) / a.pieces, kLeast), first = each * piece;
  if (first >= upto - own && first < upto) {
    int64_t at = upto - own;
    int r = r0;
    if (per > 1) {
      for (;; ++r) {
        s = span_of<ROWS>(a, r);
        if (r == r1 - 1 || first < at + s.units) break;
        at += s.units;
      }
    }
    found = {each, min(each, total - first), first - at, r, s};
  }
  __syncthreads();
  b.each = all64(each);
  if (all64(first) >= all64(total)) return b;
  const Begin f = found;
  b.left = all64(f.left);
  b.unit = all64(f.unit);
  b.r = all32(f.r);
  b.span = {all32(f.span.start), all32(f.span.n_rows), all32(f.span.context), all32(f.span.end), all32(f.span.blocks), all64(f.span.units)};
  return b;
}

// The sums of a wave's rows, divided, to the output.
template <typename T, int D> __device__ __forceinline__ void write_rows(const TreeArgs &a, RowSums<T, D> &r) {
  using M = Mma<T>;
  using O4 = decltype(M::from(0.f)) __attribute__((ext_vector_type(4)));
  const int hb = (threadIdx.x & 63) >> 5;
  const float2 ls = both_halves(r.l);
  if (r.row < 0) return;
  const float l = ls.x + ls.y, inv = l == 0.f ? 0.f : 1.f / l;
  const uint32_t t = static_cast<uint32_t>(r.row) / static_cast<uint32_t>(a.heads), h = r.row - t * a.heads;
  if (l == 0.f) {  // (a key of weight zero may have left its infinities)
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[x][i] = 0.f;
  }
  typename T::S *o = static_cast<typename T::S *>(a.o) + t * a.o_token + h * a.o_head;
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const O4 y = {M::from(r.o[x][4 * b] * inv), M::from(r.o[x][4 * b + 1] * inv), M::from(r.o[x][4 * b + 2] * inv),
                    M::from(r.o[x][4 * b + 3] * inv)};
      *reinterpret_cast<O4 *>(o + 32 * x + 8 * b + 4 * hb) = y;
    }
  if (a.lse && hb == 0)
    a.lse[t * a.lse_token + h * a.lse_head] = l == 0.f ? -INFINITY : (r.m + log2f(l)) * 0.69314718056f;
}

// The sums of a wave's rows to rows [at, at + 32) of the parts.
template <typename T, int D> __device__ __forceinline__ void write_part(const TreeArgs &a, const RowSums<T, D> &r, int64_t at) {
  const int n = threadIdx.x & 31, hb = (threadIdx.x & 63) >> 5;
  const float2 ls = both_halves(r.l);
  if (r.row < 0) return;
  if (hb == 0) a.part_ml[at + n] = make_float2(r.m, ls.x + ls.y);
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = r.o[x][4 * b + e];
      *reinterpret_cast<f32x4 *>(a.part_o + (at + n) * D + 32 * x + 8 * b + 4 * hb) = o;
    }
}

// Row waves x key waves: 32 rows a wave, all or half of each block of 64 keys,
// in steps of 32.  kNK and kNV: blocks of K and of V that LDS holds.
template <int D, int RW, int KW> struct Shape {
  static constexpr int kWaves = RW * KW, kRows = 32 * RW;
  static constexpr int kSteps = 2 / KW;  // of a block
  static constexpr int kNV = kWaves == 8 ? 4 : 2, kNK = kNV + kSteps - 1;
  static constexpr int kRing = (kNK + kNV) * 64 * D * 2;
  // Where waves of the same rows join: 32 dims of a row a lane pair, maximum and sum.
  static constexpr int kJoin = KW == 2 ? RW * (16 * 64 * 4 + 64 * 8) : 0;
  static constexpr int kBytes = kRing + kJoin;
  static_assert(KW == 1 || RW * 64 * 4 * D / 2 <= kRing, "all sums in the ring");
  static constexpr int kPerSimd = D > 128 ? 1 : D == 64 && RW == 4 ? 3 : 2;  // waves of a SIMD
};

// The other waves are here too, all that was read from LDS has arrived.
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Whether a block of V holds an infinity or a NaN: each wave looks at a part of
// it and says so at `odd`, which no wave writes again before all have read it.
template <typename T, int D, int WAVES> __device__ __forceinline__ bool any_odd(uint32_t v, uint32_t *odd) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u16x8 top = {0, 0, 0, 0, 0, 0, 0, 0};
  // (1024 bytes a turn of the wave, of 128 D)
  for (int i = wave; i < D / 8; i += WAVES) {
    const s16x8 x = *reinterpret_cast<const LdsS8 *>(v + i * 1024 + (threadIdx.x & 63) * 16);
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8, x) & static_cast<unsigned short>(0x7fff));
  }
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) bad |= top[e] >= Mma<T>::kInf;
  odd[wave] = __any(bad);
  meet();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all |= odd[w];
  return __builtin_amdgcn_readfirstlane(all) != 0;
}

// A workgroup's rows over keys, a block of 64 at a time, a wave's 32 keys a step.
// K runs a step ahead of V, and a step's softmax is spread over two products:
// beside the product with V of step i stand the maximum of step i + 1 and the
// first half of its weights, beside the scores of step i + 2 the other half.  So
// matrix and vector units have work at any time.  K and V have rings of blocks
// in LDS, loaded as soon as a place is free.  The waits for them are counted, but
// the compiler adds one for all loads to every block but the last: last() loads a
// register there, which has to be settled on the other path too.  So the blocks
// that are under way arrive together, and deep rings give less than they could;
// kNV and kStart were measured like that.
template <typename T, int D, int RW, int KW> struct Ring {
  using S = Shape<D, RW, KW>;
  static constexpr int kPer = D / 32, NK = S::kNK, NV = S::kNV;
  static constexpr uint32_t kBlock = 64 * Geometry<D>::kPitch, kGroup = 16 * Geometry<D>::kPitch;
  // Blocks that are under way; K of the block before is still read where a
  // block takes two steps.
  static constexpr int kAheadK = NV, kAheadV = NV - 1;
  // Of eight waves four load K and four V; of four each loads 16 keys of both.
  static constexpr bool kSplit = S::kWaves == 8;
  static_assert(S::kWaves == 4 || kSplit, "");

  Keys keys;
  uint32_t lds, own;              // the ring, this wave's first row of it
  int wave;                       // of four
  bool of_k, of_v;
  uint32_t k_off[kPer], v_off[kPer];
  uint32_t *odd;                  // two words for each wave

  __device__ __forceinline__ Ring(const PagedArgs &a, int h, uint32_t at, uint32_t *odd)
      : keys{a, nullptr, a.width, 0, 0, 0, 32, h * a.k_head, h * a.v_head, false}, lds(at), odd(odd) {
    const int any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wave = any & 3;
    of_k = !kSplit || any < 4;
    of_v = !kSplit || !of_k;
    own = lds + wave * kGroup;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      k_off[i] = row_offset<D, false>(i, a.k_token);
      v_off[i] = row_offset<D, true>(i, a.v_token);
      if constexpr (kSplit) k_off[i] = v_off[i] = of_k ? k_off[i] : v_off[i];
    }
  }
  __device__ __forceinline__ int blocks() const { return (keys.k1 - keys.k0 + 63) / 64; }
  // (Streaming loads: a request of one tile for each KV head reads its keys once.
  // Those of several tiles, more than 256 rows, are read so too.)
  __device__ __forceinline__ void load_k(int j, uint32_t slot) {
    load_group<D, false, true>(keys, keys.place(4 * j + wave), keys.k0 + 64 * j + 16 * wave, k_off, own + slot * kBlock);
  }
  __device__ __forceinline__ void load_v(int j, uint32_t slot) {
    load_group<D, true, true>(keys, keys.place(4 * j + wave), keys.k0 + 64 * j + 16 * wave, v_off, own + (NK + slot) * kBlock);
  }
  // The first blocks; every wave has read what was in the ring.
  __device__ __forceinline__ void begin(int entry) {
    const int n = blocks();
    keys.look_up(0, entry);
#pragma unroll
    for (int j = 0; j < kAheadK; ++j) {
      if (of_v && j > 0 && j - 1 < n) load_v(j - 1, j - 1);
      if (of_k && j < n) load_k(j, j);
    }
  }
  template <typename Last> __device__ __forceinline__ void run(const PagedArgs &a, TreeRows<T, D> &r, int least, const Last &last);
};

// The rows over all of the keys; last() is called in the last block, when the
// ring loads nothing more.
template <typename T, int D, int RW, int KW>
template <typename Last>
__device__ __forceinline__ void Ring<T, D, RW, KW>::run(const PagedArgs &a, TreeRows<T, D> &r, int least, const Last &last) {
  using M = Mma<T>;
  using V8 = typename M::V8;
  constexpr int kSteps = S::kSteps, kPitch = Geometry<D>::kPitch, kScores = D / 16, kAhead = 4;
  constexpr uint32_t kStep = 32 * kPitch;
  const int half = KW == 2 ? 32 * (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / RW) : 0;  // this wave's keys of a block
  const float c = a.scale2;
  const int k0 = keys.k0, k1 = keys.k1, n = blocks();
  wait_rows<T, D>(r);
  const int lane = threadIdx.x & 63, row = lane & 31, hb = lane >> 5, al = lane & 15;
  const uint32_t vrow = 4 * hb + (al >> 2), vcol = 2 * ((lane >> 4) & 1) + ((al & 3) >> 1);
  // A lane's first row and 16-byte piece of K and V.
  uint32_t krow = (half + row) * kPitch, kpiece = hb ^ k_swizzle<D>(row);
  uint32_t vlane = (half + vrow) * kPitch + (al & 1) * 8, vpiece = vcol ^ v_swizzle<D>(vrow);
  auto read_k = [&](uint32_t k, int x) { return *reinterpret_cast<const LdsS8 *>(k + krow + (((2 * x) ^ kpiece) << 4)); };
  auto read_v = [&](uint32_t v, int c2, int t) {
    const uint32_t at = v + vlane + (((4 * t) ^ vpiece) << 4) + c2 * 16 * kPitch;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsS4 *>(at + 8 * kPitch));
    return static_cast<s16x8>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  f32x16 s[1];
  V8 p[2];
  float base;
  auto weigh_one = [&](V8 &to, int i) {
    const float w = __builtin_amdgcn_exp2f(s[0][i] * c - base);
    r.l += w;
    to[i % 8] = M::from(w);
  };
  auto pin = [&](V8 &x) {  // (computed here, not where it is used)
    s16x8 y = __builtin_bit_cast(s16x8, x);
    asm volatile("" : "+v"(y));
    x = __builtin_bit_cast(V8, y);
  };
  // Takes out the keys from block j0 on (this wave's 32 from `from` on) that a
  // row does not see, or that the caches do not have.
  auto cut_at = [&](int j0) { return least < min(j0 + 64, k1); };
  auto hide_at = [&](int j0, int from) {
    if (cut_at(j0) || !keys.template all<64>(j0)) hide<1>(s, (keys.template seen<64>(j0) & r.visible(a, j0)) >> from);
  };
  constexpr int kFirst = (kSplit ? 1 : 2) * (kAheadK - 1) * kPer;  // loads behind those of K's first block
  static_assert(kFirst < 64, "");
  if (n >= kAheadK) wait_loads<kFirst>();
  else wait_loads<0>();
  meet();
#pragma unroll
  for (int i = 0; i < 16; ++i) s[0][i] = 0.f;
#pragma unroll
  for (int x = 0; x < kScores; ++x) s[0] = M::mul(__builtin_bit_cast(V8, read_k(lds, x)), r.q[x], s[0]);
  hide_at(k0, half);
  r.m = largest<1>(s, c);
  base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
  for (int i = 0; i < 8; ++i) weigh_one(p[0], i);
  s16x8 kf[kAhead];
  if constexpr (kSteps == 2) {
#pragma unroll
    for (int x = 0; x < kAhead; ++x) kf[x] = read_k(lds + kStep, x);
  }
  // Step i: the scores of the step behind it, whose K is at k; the product with
  // V at v; and the first reads of the K behind that, at k_next (where a
  // block takes two steps, it is there already).
  auto step = [&](uint32_t k, uint32_t k_next, uint32_t v, int j0_next, int from) {
    // (addresses are computed in each step and not kept in registers)
    asm volatile("" : "+v"(krow), "+v"(kpiece), "+v"(vlane), "+v"(vpiece));
    f32x16 next;
    s16x8 vf[2][kPer];
#pragma unroll
    for (int i = 0; i < 16; ++i) next[i] = 0.f;
    if constexpr (kSteps == 1) {
#pragma unroll
      for (int x = 0; x < kAhead; ++x) kf[x] = read_k(k, x);
    }
#pragma unroll
    for (int x = 0; x < kScores; ++x) {
      next = M::mul(__builtin_bit_cast(V8, kf[x % kAhead]), r.q[x], next);
      if (x + kAhead < kScores) kf[x % kAhead] = read_k(k, x + kAhead);
      else if (x + kAhead - kScores < kPer) vf[0][x + kAhead - kScores] = read_v(v, 0, x + kAhead - kScores);
#pragma unroll
      for (int i = x * 8 / kScores; i < (x + 1) * 8 / kScores; ++i) weigh_one(p[1], 8 + i);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = kAhead; t < kPer; ++t) vf[0][t] = read_v(v, 0, t);
    pin(p[1]);
    s[0] = next;
    hide_at(j0_next, from);
    float top = s[0][0], scale = 1.f;
    bool moved = false;
    V8 first;
    constexpr int kProducts = 2 * kPer, kTop = kProducts / 4, kRest = kProducts - kTop;
#pragma unroll
    for (int y = 0; y < kProducts; ++y) {
      const int t = y % kPer, c2 = y / kPer;
      r.o[t] = M::mul(__builtin_bit_cast(V8, vf[c2][t]), p[c2], r.o[t]);
      if (c2 == 0) vf[1][t] = read_v(v, 1, t);
      else if (kSteps == 2 && t < kAhead) kf[t] = read_k(k_next, t);
      if (y < kTop) {
#pragma unroll
        for (int i = y * 16 / kTop; i < (y + 1) * 16 / kTop; ++i) top = fmaxf(top, s[0][i]);
      }
      if (y == kTop - 1) {
        // The sums keep their reference point until a score passes it by 2^8:
        // the weights stay below 256, where their relative rounding is the
        // same.  What V's product adds meanwhile goes by the old point.
        const float2 tops = both_halves(top);
        top = fmaxf(tops.x, tops.y) * c;
        if (__any(top > r.m + 8.f)) {
          const float m = fmaxf(r.m, top);
          // (A row without a reference point has no sums yet, but may have
          // infinities from the other half of the block: zero times those
          // would be NaN.)
          scale = r.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
          r.l *= scale;
          r.m = m;
          base = m == -INFINITY ? 0.f : m;
          moved = true;
        }
      }
      if (y >= kTop) {
#pragma unroll
        for (int i = (y - kTop) * 8 / kRest; i < (y - kTop + 1) * 8 / kRest; ++i) weigh_one(first, i);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kSteps == 2) {
#pragma unroll
      for (int x = kPer; x < kAhead; ++x) kf[x] = read_k(k_next, x);
    }
    pin(first);
    p[0] = first;
    if (moved) {
#pragma unroll
      for (int t = 0; t < kPer; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) r.o[t][i] *= scale;
    }
  };
  uint32_t ks = 0, vs = 0;  // places of K of block j and of V of block j
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    // K of the next block and V of this one are there, and every wave has
    // read what the blocks loaded now take the place of.
    constexpr int kBehind = (kSplit ? 1 : 2) * (kAheadV - 1) * kPer;
    if (kBehind > 0 && j + kAheadK <= n) wait_loads<kBehind>();
    else wait_loads<0>();
    meet();
    const int j0 = k0 + 64 * j;
    if (j == n - 1) last();
    if (of_v && j + kAheadV < n) load_v(j + kAheadV, vs == 0 ? NV - 1 : vs - 1);
    if (of_k && j + kAheadK < n) load_k(j + kAheadK, kSteps == 1 ? ks : ks == 0 ? NK - 1 : ks - 1);
    const uint32_t k = lds + ks * kBlock;
    ks = ks + 1 == NK ? 0 : ks + 1;
    const uint32_t k_next = lds + ks * kBlock, v = lds + (NK + vs) * kBlock;
    vs = vs + 1 == NV ? 0 : vs + 1;
    if (cut_at(j0) && any_odd<T, D, S::kWaves>(v, odd + (j & 1) * S::kWaves)) {
      const uint64_t there = keys.template seen<64>(j0) & (KW == 2 ? uint64_t(0xffffffff) << half : ~uint64_t(0));
      take_odd_out<T, D, 64, true>(r, v, there & r.visible(a, j0));
    }
    if constexpr (kSteps == 1) {
      step(k_next, 0, v, j0 + 64, half);
    } else {
      step(k + kStep, k_next, v, j0, 32);
      step(k_next, k_next + kStep, v + kStep, j0 + 64, 0);
    }
  }
}

// The sums of two waves of the same rows, over different keys, to the first's:
// 32 dims at a time beside the ring, or all of them in it where nothing is loaded
// there any more (the last tile).
template <typename T, int D, int RW> __device__ __forceinline__ void join_halves(RowSums<T, D> &r, uint8_t *ring, uint8_t *beside, bool last) {
  // (192 and 256 dims have no registers for both ways: 1.3 times as long)
  const bool once = D <= 128 && last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 *at = reinterpret_cast<f32x4 *>(once ? ring : beside) + (wave % RW) * 256 + lane;
  float2 *ml = reinterpret_cast<float2 *>(beside + RW * 4096) + (wave % RW) * 64 + lane;
  const int step = once ? RW * 256 : 0;
  float f = 0.f, g = 0.f;
  auto give = [&](int t) {
    if (t == 0) *ml = make_float2(r.m, r.l);
#pragma unroll
    for (int b = 0; b < 4; ++b) at[t * step + b * 64] = f32x4{r.o[t][4 * b], r.o[t][4 * b + 1], r.o[t][4 * b + 2], r.o[t][4 * b + 3]};
  };
  auto take = [&](int t) {
    if (t == 0) {
      const float2 x = *ml;
      const float top = fmaxf(r.m, x.x), base = top == -INFINITY ? 0.f : top;
      f = __builtin_amdgcn_exp2f(r.m - base);
      g = __builtin_amdgcn_exp2f(x.x - base);
      r.m = top;
      r.l = r.l * f + x.y * g;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 x = at[t * step + b * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.o[t][4 * b + e] = r.o[t][4 * b + e] * f + x[e] * g;
    }
  };
  if (once) {
    if (wave >= RW)
#pragma unroll
      for (int t = 0; t < D / 32; ++t) give(t);
    meet();
    if (wave < RW)
#pragma unroll
      for (int t = 0; t < D / 32; ++t) take(t);
    return;
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    if (wave >= RW) give(t);
    meet();
    if (wave < RW) take(t);
    meet();
  }
}

template <typename T, int D, int RW, int KW>
__global__ void __launch_bounds__(64 * RW * KW, (Shape<D, RW, KW>::kPerSimd)) attend_tree(TreeArgs a) {
  using S = Shape<D, RW, KW>;
  extern __shared__ __align__(128) uint8_t lds[];
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % RW, n = threadIdx.x & 31;
  const int piece = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads, me = piece * a.kv_heads + h;
  const Begin begin = find_piece<S::kRows, 64 * S::kWaves>(a, piece);
  const int64_t each = begin.each;
  TreeArgs::Cut cut = {-1, 0, 0, 0};
  // The part of a tile that is worked on: `blocks` of its blocks from b0 on.
  Span s = begin.span;
  int q = begin.r, tile = 0, b0 = 0, blocks = 0;
  int64_t left = begin.left;
  if (left > 0) {
    tile = static_cast<int>(begin.unit / (s.blocks + kStart));
    b0 = static_cast<int>(begin.unit - static_cast<int64_t>(tile) * (s.blocks + kStart)) - kStart;
    if (b0 < 0) {
      left += b0;
      b0 = 0;
    }
    blocks = static_cast<int>(max(static_cast<int64_t>(0), min(left, static_cast<int64_t>(s.blocks - b0))));
    left -= blocks;
  }
  const bool odd_blocks = a.block_size % 16 != 0;
  __shared__ uint32_t odd[2 * S::kWaves];
  Ring<T, D, RW, KW> ring(a, h, at, odd);
  TreeRows<T, D> r;
  // The token of this lane's row of a tile, or -1, and its head.
  auto token = [&](const Span &x, int i) { return i < x.n_rows ? x.start + i / a.group : -1; };
  auto head = [&](const Span &x, int i) { return h * a.group + (i < x.n_rows ? i % a.group : 0); };
  auto turn_to = [&](const Span &x, int request, int from, int count) {
    ring.keys.turn_to(a.table + request * a.table_stride, from * 64, min(x.end, (from + count) * 64), odd_blocks);
  };
  if (blocks > 0) {
    const int i = tile * S::kRows + wave * 32 + n;
    turn_to(s, q, b0, blocks);
    const int entry = ring.keys.entry(0);
    load_rows<T, D>(a, r, token(s, i), head(s, i));
    r.load_word(a, token(s, i));
    ring.begin(entry);
  }
  while (blocks > 0) {
    r.context = s.context;
    // The tile behind this one, of this request or the next with rows.
    Span next = s;
    int next_q = q, next_tile = tile + 1, next_blocks = 0, entry = 0;
    left -= kStart;
    if (left > 0) {
      if (next_tile * S::kRows >= s.n_rows) {
        next_tile = 0;
        next.units = 0;
        while (next.units == 0 && next_q + 1 < a.n_requests) next = span_of_all<S::kRows>(a, ++next_q);
      }
      if (next.units > 0) next_blocks = static_cast<int>(min(left, static_cast<int64_t>(next.blocks)));
      left -= next_blocks;
    }
    const int32_t *list = a.table + next_q * a.table_stride;
    const int next_end = min(next.end, next_blocks * 64);
    if (ring.keys.k0 < ring.keys.k1)
      ring.run(a, r, s.context, [&] {
        if (next_blocks > 0) entry = ring.keys.entry_of(list, (threadIdx.x & 63) * 16, 0, next_end);
      });
    else if (next_blocks > 0) entry = ring.keys.entry_of(list, (threadIdx.x & 63) * 16, 0, next_end);
    // What follows is loaded while this one's sums are written (run() then waits
    // for all of it: the query, which it needs first, is loaded last).
    meet();
    const int i = next_tile * S::kRows + wave * 32 + n, next_t = token(next, i), next_h = head(next, i);
    if (next_blocks > 0) {
      turn_to(next, next_q, 0, next_blocks);
      ring.begin(entry);
      load_query<T, D>(a, r, next_t, next_h);
      r.load_word(a, next_t);
    }
    if constexpr (KW == 2) join_halves<T, D, RW>(r, lds, lds + S::kRing, next_blocks == 0);
    const bool ends = b0 + blocks < s.blocks && b0 == 0;
    if (KW == 1 || threadIdx.x < 64 * RW) {
      if (blocks == s.blocks) write_rows<T, D>(a, r);
      else write_part<T, D>(a, r, (static_cast<int64_t>(me) * 2 + ends) * S::kRows + wave * 32);
    }
    if (ends)
      cut = {static_cast<int>((s.blocks - blocks + each - 1) / each), tile * S::kRows, min(S::kRows, s.n_rows - tile * S::kRows), s.start};
    r.row = next_t >= 0 ? next_t * a.heads + next_h : -1;
    clear_sums(r);
    s = next;
    q = next_q;
    tile = next_tile;
    b0 = 0;
    blocks = next_blocks;
  }
  if (threadIdx.x == 0) a.cuts[me] = cut;
}

// Joins the pieces of the tiles that are cut: the k-th of a KV head to the
// workgroups (k, KV head, y), which find its first piece among the head's
// cuts.  D / 4 lanes a row.  Tiles of few pieces take a wave a row (or two or
// four), all pieces loaded together; those of many, four waves a row, with a
// quarter of the pieces each.
template <typename T, int D, int ROWS> __global__ void __launch_bounds__(256) join_tree(TreeArgs a) {
  constexpr int kQuads = D / 4, kStep = 64 / kQuads, kFew = 8;
  using M = Mma<T>;
  using O4 = decltype(M::from(0.f)) __attribute__((ext_vector_type(4)));
  __shared__ f32x4 sums[4][64];
  __shared__ float2 weights[4][kStep];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.kv_heads;
  int rank = blockIdx.x / a.kv_heads, piece = -1;
  TreeArgs::Cut cut = {-1, 0, 0, 0};
  for (int p0 = 0; p0 < a.pieces; p0 += 64) {
    const int p = p0 + lane;
    if (p < a.pieces) cut = a.cuts[p * a.kv_heads + h];
    uint64_t there = __ballot(p < a.pieces && cut.more >= 0);
    const int n = __popcll(there);
    if (rank >= n) {
      rank -= n;
      continue;
    }
    for (; rank > 0; --rank) there &= there - 1;
    const int from = __ffsll(static_cast<unsigned long long>(there)) - 1;
    piece = p0 + from;
    cut = {__builtin_amdgcn_readlane(cut.more, from), __builtin_amdgcn_readlane(cut.first_row, from),
           __builtin_amdgcn_readlane(cut.rows, from), __builtin_amdgcn_readlane(cut.start, from)};
    break;
  }
  if (piece < 0) return;
  const int first = piece * a.kv_heads + h;
  const int i0 = lane / kQuads, d = lane % kQuads * 4, n = cut.rows, parts = cut.more + 1;
  float m, l;
  f32x4 o;
  // Row i of the parts k0, k0 + step, ...: kFew / 2 of them under way together.
  auto gather = [&](int i, bool there, int k0, int step) {
    m = -INFINITY;
    l = 0.f;
    o = {0.f, 0.f, 0.f, 0.f};
    for (int k1 = k0; k1 < parts; k1 += step * (kFew / 2)) {
      float2 w[kFew / 2];
      f32x4 y[kFew / 2];
#pragma unroll
      for (int k = 0; k < kFew / 2; ++k) {
        const int part = k1 + step * k;
        const int64_t at = (static_cast<int64_t>(first + part * a.kv_heads) * 2 + (part == 0)) * ROWS + i;
        const bool in = there && part < parts;
        w[k] = in ? a.part_ml[at] : make_float2(-INFINITY, 0.f);
        if (in) y[k] = *reinterpret_cast<const f32x4 *>(a.part_o + at * D + d);
      }
#pragma unroll
      for (int k = 0; k < kFew / 2; ++k) {
        if (w[k].y == 0.f) continue;
        const float top = fmaxf(m, w[k].x), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(w[k].x - base);
        l = l * f + w[k].y * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f + y[k][e] * g;
        m = top;
      }
    }
  };
  auto write = [&](int i) {
    const float inv = l == 0.f ? 0.f : 1.f / l, base = m == -INFINITY ? 0.f : m;
    const int x = cut.first_row + i, t = cut.start + x / a.group, head = h * a.group + x % a.group;
    const O4 y = {M::from(o[0] * inv), M::from(o[1] * inv), M::from(o[2] * inv), M::from(o[3] * inv)};
    *reinterpret_cast<O4 *>(static_cast<typename T::S *>(a.o) + t * a.o_token + head * a.o_head + d) = y;
    if (a.lse && d == 0) a.lse[t * a.lse_token + head * a.lse_head] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.69314718056f;
  };
  if (parts <= kFew) {
    for (int i = (blockIdx.y * 4 + wave) * kStep + i0; i - i0 < n; i += gridDim.y * 4 * kStep) {
      const bool there = i0 < kStep && i < n;
      gather(i, there, 0, 1);
      if (there) write(i);
    }
    return;
  }
  for (int i1 = blockIdx.y * kStep; i1 < n; i1 += gridDim.y * kStep) {
    const int i = i1 + i0;
    const bool there = i0 < kStep && i < n;
    gather(i, there, wave, 4);
    __syncthreads();  // (of the last rows)
    sums[wave][lane] = o;
    if (there && d == 0) weights[wave][i0] = make_float2(m, l);
    __syncthreads();
    if (wave != 0 || !there) continue;
    m = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) m = fmaxf(m, weights[g][i0].x);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float2 w = weights[g][i0];
      if (w.y == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(w.x - base);
      l += f * w.y;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * sums[g][lane][e];
    }
    write(i);
  }
}

template <typename T, int D, int RW, int KW> void launch(const TreeArgs &a, const TreePlan &p, hipStream_t s) {
  using S = Shape<D, RW, KW>;
  const void *fn = reinterpret_cast<const void *>(attend_tree<T, D, RW, KW>);
  if (S::kBytes > 64 * 1024)
    hip_check(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, S::kBytes), "attend_tree shared memory");
  hipLaunchKernelGGL((attend_tree<T, D, RW, KW>), dim3(static_cast<uint32_t>(p.groups)), dim3(64 * S::kWaves), S::kBytes, s, a);
  hip_check(hipGetLastError(), "attend_tree launch");
  if (p.pieces == 1) return;  // nothing is cut
  hipLaunchKernelGGL((join_tree<T, D, S::kRows>), dim3(static_cast<uint32_t>(p.cuts), static_cast<uint32_t>(p.join_groups)), dim3(256),
                     0, s, a);
  hip_check(hipGetLastError(), "join_tree launch");
}

template <typename T, int D> void launch_rows(const TreeArgs &a, const TreePlan &p, hipStream_t s) {
  if (p.rows == 64) launch<T, D, 2, 2>(a, p, s);
  else if constexpr (D == 192) launch<T, D, 4, 1>(a, p, s);
  else if constexpr (D <= 128) {
    if (p.rows == 256) launch<T, D, 8, 1>(a, p, s);
    else launch<T, D, 4, D == 64 ? 1 : 2>(a, p, s);
  }
}

template <typename T> void launch_dim(const TreeArgs &a, int64_t dim, const TreePlan &p, hipStream_t s) {
  switch (dim) {
  case 64: launch_rows<T, 64>(a, p, s); break;
  case 96: launch_rows<T, 96>(a, p, s); break;
  case 128: launch_rows<T, 128>(a, p, s); break;
  case 192: launch_rows<T, 192>(a, p, s); break;
  default: launch_rows<T, 256>(a, p, s); break;
  }
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_tree_attention(const lmc_tensor *query, const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                                  const lmc_tensor *block_table, const lmc_tensor *seq_lens,
                                  const lmc_tensor *query_start_loc, const lmc_tensor *tree_mask, double scale,
                                  const lmc_tensor *output, const lmc_tensor *lse, const lmc_tensor *workspace,
                                  int64_t *workspace_bytes, int32_t kvcache_format, int32_t vllm_two_major, void *stream) {
  return guarded([&] {
    TreeArgs a;
    std::memset(&a, 0, sizeof(a));
    const PagedSizes n = paged_call(a, "tree_attention", query, vllm_kv_caches, n_caches, kvcache_format,
                                    vllm_two_major != 0, block_table, seq_lens, query_start_loc, scale, output, lse);
    const PagedKv &kv = n.kv;
    const lmc_tensor &tm = deref(tree_mask, "tree_mask");
    check_on(tm, "tree_mask", kv.device, LMC_I64);
    expect(tm.ndim == 2 && tm.sizes[0] == n.tokens, "tree_mask must be [tokens, words]");
    expect(tm.sizes[1] <= 1 || tm.strides[1] == 1, "tree_mask rows must be contiguous");
    expect(tm.strides[0] >= 0, "negative strides unsupported");
    expect(tm.sizes[1] <= (1 << 20), "tree_mask has more than 2^20 words a row");
    if (workspace_bytes) *workspace_bytes = 0;
    if (n.tokens == 0 || n.heads == 0 || n.requests == 0) return;
    const TreePlan p = make_plan(n.tokens, n.requests, kv.heads, n.group, kv.dim, n.keys);
    const int64_t parts = p.groups * 2 * p.rows;
    const int64_t bytes = parts * (kv.dim * 4 + 8) + p.groups * static_cast<int64_t>(sizeof(TreeArgs::Cut));
    // A launch has less than 2^32 threads along a dimension.
    expect(p.groups <= UINT32_MAX / 512, "too many heads");
    if (workspace_bytes) {
      *workspace_bytes = bytes;
      return;
    }
    // A tile that is not cut is written while others' queries are read.
    auto same = [](const lmc_tensor &x, const lmc_tensor &y) {
      if (x.data != y.data) return false;
      for (int i = 0; i < 3; ++i)
        if (x.sizes[i] > 1 && x.strides[i] != y.strides[i]) return false;
      return true;
    };
    expect(same(*output, *query) || !may_share(*output, *query), "output overlaps query and is not the same tensor");
    expect(!lse || !extents_meet(*lse, *query), "lse overlaps query");
    check_outputs(query, output, lse, workspace, bytes, kv.device, vllm_kv_caches, n_caches,
                  {query_start_loc, seq_lens, block_table, tree_mask});
    a.mask = static_cast<const int64_t *>(tm.data);
    a.mask_token = tm.strides[0];
    a.words = static_cast<int>(tm.sizes[1]);
    a.pieces = static_cast<int>(p.pieces);
    a.part_o = static_cast<float *>(workspace->data);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + parts * kv.dim);
    a.cuts = reinterpret_cast<TreeArgs::Cut *>(a.part_ml + parts);
    DeviceGuard guard(kv.device);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (kv.dtype == LMC_BF16) launch_dim<BF16>(a, kv.dim, p, s);
    else launch_dim<F16>(a, kv.dim, p, s);
  });
}
