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
// The tiles, their products and what is rounded: paged_attention.h.
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
// and 256 dims take accumulation registers too, a wave a SIMD.  33 to 43 scalar
// registers are kept in vector registers.
#include "paged_attention.h"

namespace lmc {

namespace {

// Keys of a part of a request's own ones where requests are many: 256 requests
// over 16384 shared and up to 1024 own keys take 151 us with 384, 156 with 256
// (more starts and ends) and 149 with 512, which takes 116 over 1024 shared keys
// against 112.  An equal share of all own keys for every wave, over the
// requests' borders, took as long (124 against 120 for the own keys alone) and
// cost small batches 2 of 12 us.
constexpr int kOwnChunk = 384;

struct AttnArgs : PagedArgs {
  const int32_t *shared;
  int shared_len;
  uint32_t shared_width;
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
      hide<1>(s, seen & r.visible(a, j0));
    }
    refer_to<T, D>(r, largest<1>(s, a.scale2));
    weigh<T, D>(r, s[0], p, a.scale2);
    if (more) wait_loads<2 * kPer>();
    else wait_loads<0>();
    if (cut && has_odd<T, D, 32>(v)) take_odd_out<T, D, 32, false>(r, v, seen & r.visible(a, j0));
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
    hide<2>(s, seen & r.visible(a, k0));
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
    if (cut && has_odd<T, D, 64>(v)) take_odd_out<T, D, 64, true>(r, v, seen & r.visible(a, j0));
    s16x8 vf[2][kPer];
#pragma unroll
    for (int t = 0; t < kPer; ++t) vf[0][t] = read_v(0, t);
    s[0] = next[0];
    s[1] = next[1];
    cut = least < min(j0 + 128, k1);
    if (cut || !keys.template all<64>(j0 + 64)) {
      seen = keys.template seen<64>(j0 + 64);
      hide<2>(s, seen & r.visible(a, j0 + 64));
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
    load_rows<T, D>(a, r, t, h * a.group + (t < 0 ? 0 : x % a.group));
    r.limit = t >= 0 && limit > 0 ? limit : INT32_MAX;
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
    load_rows<T, D>(a, r, t, head);
    r.limit = t >= 0 && limit > 0 ? limit : INT32_MAX;
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
    AttnArgs a;
    std::memset(&a, 0, sizeof(a));
    const lmc_tensor &sb = deref(shared_blocks, "shared_blocks");
    const PagedSizes n = paged_call(a, "shared_prefix_attention", query, vllm_kv_caches, n_caches, kvcache_format,
                                    vllm_two_major != 0, block_table, seq_lens, query_start_loc, scale, output, lse);
    const PagedKv &kv = n.kv;
    check_vector(sb, "shared_blocks", kv.device, LMC_I32);
    expect(shared_len >= 0 && shared_len <= kMaxKeys, "shared_len must be between 0 and 2^30");
    expect((shared_len + kv.block_size - 1) / kv.block_size <= sb.sizes[0], "shared_blocks has too few blocks for shared_len");
    if (workspace_bytes) *workspace_bytes = 0;
    if (n.tokens == 0 || n.heads == 0 || n.requests == 0) return;
    const Plan p = make_plan(n.tokens, n.requests, kv.heads, n.group, shared_len, n.keys);
    const int64_t parts = p.prefix_parts + p.own_parts, rows = n.tokens * n.heads;
    const int64_t bytes = parts * rows * (kv.dim * 4 + 8);
    // A launch has less than 2^32 threads along a dimension.
    const int64_t own_items = n.requests * kv.heads * p.own_tiles * p.own_parts, own_groups = (own_items + 31) / 32;
    const int64_t prefix_groups = (kv.heads * p.prefix_parts + 7) / 8 * p.prefix_tiles;
    expect((own_groups + prefix_groups) * 8 <= UINT32_MAX / 256, "too many rows");
    if (workspace_bytes) {
      *workspace_bytes = bytes;
      return;
    }
    // (output and lse may lie over query: parts are joined in a launch of their own)
    check_outputs(query, output, lse, workspace, bytes, kv.device, vllm_kv_caches, n_caches,
                  {query_start_loc, seq_lens, block_table, shared_blocks});
    a.shared = static_cast<const int32_t *>(sb.data);
    a.shared_len = static_cast<int>(shared_len);
    a.shared_width = static_cast<uint32_t>(sb.sizes[0]);
    a.max_keys = static_cast<int>(std::max(shared_len, n.keys));
    a.part_o = static_cast<float *>(workspace->data);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + parts * rows * kv.dim);
    a.prefix_parts = p.prefix_parts;
    a.own_parts = p.own_parts;
    a.prefix_tiles = p.prefix_tiles;
    a.prefix_chunk = p.prefix_chunk;
    a.own_tiles = p.own_tiles;
    a.own_want = p.own_want;
    a.own_items = static_cast<int>(own_items);
    a.prefix_groups = static_cast<int>(prefix_groups);
    DeviceGuard guard(kv.device);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t groups = static_cast<uint32_t>(own_groups + prefix_groups);
    if (kv.dtype == LMC_BF16) launch_dim<BF16>(a, kv.dim, p.wide, groups, s);
    else launch_dim<F16>(a, kv.dim, p.wide, groups, s);
  });
}
