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
// heads of the group, 128 of them or 256) against blocks of 64 of the
// request's keys.  The lengths are on the GPU, so the cut is made there: a KV
// head's tiles, one request's behind the other's, are one line of key blocks,
// and each of its workgroups takes an equal piece of it, wherever requests
// begin and end.  A tile that lies in one piece is written at once; one that is
// cut leaves sums (32 bits, with their maximum) for every piece, which a second
// launch joins.  Each workgroup has two places for sums: one for a tile that an
// earlier workgroup began, one for a tile that a later one ends.
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
  struct Cut { int request, tile, more; } *cuts;  // of the place "ended behind": the pieces that follow, or request -1
};

// Rows that see the context and the drafted tokens of their mask.
template <typename T, int D> struct TreeRows : RowSums<T, D> {
  int context;  // keys before the drafted tokens
  // Bit i: the row sees key j0 + i.
  __device__ __forceinline__ uint64_t visible(const PagedArgs &p, int j0) const {
    const TreeArgs &a = static_cast<const TreeArgs &>(p);
    const int d = j0 - context;
    if (d <= -64 || this->row < 0) return ~uint64_t(0);
    const int64_t *w = a.mask + static_cast<uint32_t>(this->row) / static_cast<uint32_t>(a.heads) * a.mask_token;
    auto word = [&](int i) { return i < a.words ? static_cast<uint64_t>(w[i]) : 0; };
    if (d < 0) return (~uint64_t(0) >> (64 + d)) | (word(0) << -d);
    const int i = d >> 6, s = d & 63;
    return s ? (word(i) >> s) | (word(i + 1) << (64 - s)) : word(i);
  }
};

// One request's part of the line.
struct Span {
  int start, n_rows, context, end, blocks;  // rows of a KV head; keys; blocks of keys of a tile
  int64_t units;
};

template <int ROWS> __device__ __forceinline__ Span span_of(const TreeArgs &a, int r) {
  Span s;
  const int start = a.starts[r], stop = a.starts[r + 1], seq = a.seq_lens[r];
  s.start = max(0, start);
  s.n_rows = max(0, min(a.n_tokens, stop) - s.start) * a.group;
  s.end = max(0, min(seq, a.max_keys));
  // (no mask reaches 2^29 tokens)
  s.context = static_cast<int>(max(static_cast<int64_t>(seq) - stop + start, -(int64_t(1) << 29)));
  // (rows without keys are written too)
  s.blocks = max(1, (s.end + 63) / 64);
  s.units = static_cast<int64_t>((s.n_rows + ROWS - 1) / ROWS) * s.blocks;
  return s;
}

// The request and the unit of it where a workgroup's piece begins.
struct Begin {
  int64_t total, unit;
  int r;
};

// All requests' units, summed by the workgroup: each thread has a run of them.
template <int ROWS, int THREADS> __device__ __forceinline__ Begin find_piece(const TreeArgs &a, int piece) {
  __shared__ int64_t sums[THREADS / 64];
  __shared__ int64_t found_unit;
  __shared__ int found_r;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (a.n_requests + THREADS - 1) / THREADS;
  const int r0 = min(a.n_requests, static_cast<int>(threadIdx.x) * per), r1 = min(a.n_requests, r0 + per);
  int64_t own = 0;
  for (int r = r0; r < r1; ++r) own += span_of<ROWS>(a, r).units;
  int64_t upto = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t below = __shfl_up(upto, d);
    if (lane >= d) upto += below;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) upto += sums[w];
    total += sums[w];
  }
  const int64_t first = (total + a.pieces - 1) / a.pieces * piece;
  if (first >= upto - own && first < upto) {
    int64_t at = upto - own;
    int r = r0;
    for (; r < r1 - 1; ++r) {
      const int64_t n = span_of<ROWS>(a, r).units;
      if (first < at + n) break;
      at += n;
    }
    found_r = r;
    found_unit = first - at;
  }
  __syncthreads();
  Begin b;
  b.total = total;
  b.r = __builtin_amdgcn_readfirstlane(found_r);
  b.unit = found_unit;
  return b;
}

// The sums of a wave's rows, divided, to the output.
template <typename T, int D> __device__ __forceinline__ void write_rows(const TreeArgs &a, const RowSums<T, D> &r) {
  using S = typename T::S;
  const int hb = (threadIdx.x & 63) >> 5;
  const float2 ls = both_halves(r.l);
  if (r.row < 0) return;
  const float l = ls.x + ls.y, inv = l == 0.f ? 0.f : 1.f / l;
  const uint32_t t = static_cast<uint32_t>(r.row) / static_cast<uint32_t>(a.heads), h = r.row - t * a.heads;
  S *o = static_cast<S *>(a.o) + t * a.o_token + h * a.o_head;
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      Pack<S, 4> y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y.v[e] = from_f32<T>(l == 0.f ? 0.f : r.o[x][4 * b + e] * inv);
      *reinterpret_cast<Pack<S, 4> *>(o + 32 * x + 8 * b + 4 * hb) = y;
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

template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, D > 128 ? 1 : 2) attend_tree(TreeArgs a) {
  constexpr int kRows = 32 * WAVES;
  extern __shared__ uint8_t lds[];
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = threadIdx.x & 31;
  const int h = blockIdx.x % a.kv_heads, piece = blockIdx.x / a.kv_heads;
  const Begin begin = find_piece<kRows, 64 * WAVES>(a, piece);
  const int64_t each = (begin.total + a.pieces - 1) / a.pieces;
  int64_t left = min(each, begin.total - each * piece), unit = begin.unit;
  TreeArgs::Cut cut = {-1, 0, 0};
  for (int r = begin.r; left > 0; ++r, unit = 0) {
    const Span s = span_of<kRows>(a, r);
    while (left > 0 && unit < s.units) {
      const int tile = static_cast<int>(unit / s.blocks), b0 = static_cast<int>(unit - static_cast<int64_t>(tile) * s.blocks);
      const int blocks = static_cast<int>(min(left, static_cast<int64_t>(s.blocks - b0)));
      const int x = tile * kRows + wave * 32 + n;
      const int t = x < s.n_rows ? s.start + x / a.group : -1;
      TreeRows<T, D> rows;
      rows.context = s.context;
      Keys keys{a, a.table + r * a.table_stride, a.width, b0 * 64, min(s.end, (b0 + blocks) * 64), b0 * 64, 32, h * a.k_head,
                h * a.v_head, a.block_size % 16 != 0};
      const int entry = keys.entry(0);
      load_rows<T, D>(a, rows, t, h * a.group + (t < 0 ? 0 : x % a.group));
      __syncthreads();  // the last tile's keys have been read
      if (keys.k0 < keys.k1) attend_wide<T, D, WAVES>(a, rows, keys, entry, s.context, at);
      if (blocks == s.blocks) {
        write_rows<T, D>(a, rows);
      } else {
        const bool ends = b0 + blocks < s.blocks && b0 == 0;
        write_part<T, D>(a, rows, (static_cast<int64_t>(blockIdx.x) * 2 + ends) * kRows + wave * 32);
        if (ends) cut = {r, tile, static_cast<int>((s.blocks - blocks + each - 1) / each)};
      }
      left -= blocks;
      unit += blocks;
    }
  }
  if (threadIdx.x == 0) a.cuts[blockIdx.x] = cut;
}

// Joins the pieces of the tile that a workgroup began and a later one ended:
// D / 4 lanes a row.
constexpr int kJoinRows = 32;

template <typename T, int D, int WAVES> __global__ void __launch_bounds__(256) join_tree(TreeArgs a) {
  constexpr int kRows = 32 * WAVES, kQuads = D / 4, kStep = 256 / kQuads;
  using S = typename T::S;
  const TreeArgs::Cut cut = a.cuts[blockIdx.x];
  if (cut.request < 0) return;
  const Span s = span_of<kRows>(a, cut.request);
  const int h = blockIdx.x % a.kv_heads;
  const int i0 = threadIdx.x / kQuads, d = threadIdx.x % kQuads * 4;
  if (i0 >= kStep) return;
  const int n = min(kRows, s.n_rows - cut.tile * kRows);
  for (int i = blockIdx.y * kJoinRows + i0; i < min(n, static_cast<int>(blockIdx.y + 1) * kJoinRows); i += kStep) {
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 <= cut.more; k0 += 4) {
      float2 w[4];
      f32x4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int part = k0 + k;
        const int64_t place = (static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(part) * a.kv_heads) * 2 + (part == 0);
        const bool there = part <= cut.more;
        w[k] = there ? a.part_ml[place * kRows + i] : make_float2(-INFINITY, 0.f);
        if (there) y[k] = *reinterpret_cast<const f32x4 *>(a.part_o + (place * kRows + i) * D + d);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (w[k].y == 0.f) continue;
        const float top = fmaxf(m, w[k].x), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(w[k].x - base);
        l = l * f + w[k].y * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f + y[k][e] * g;
        m = top;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int x = cut.tile * kRows + i, t = s.start + x / a.group, head = h * a.group + x % a.group;
    Pack<S, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = from_f32<T>(o[e] * inv);
    *reinterpret_cast<Pack<S, 4> *>(static_cast<S *>(a.o) + t * a.o_token + head * a.o_head + d) = y;
    if (a.lse && d == 0) a.lse[t * a.lse_token + head * a.lse_head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
  }
}

template <typename T, int D, int WAVES> void launch(const TreeArgs &a, hipStream_t s) {
  constexpr int kBytes = 2 * 2 * 64 * D * 2;  // two blocks of K and of V
  const void *fn = reinterpret_cast<const void *>(attend_tree<T, D, WAVES>);
  hip_check(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, kBytes), "attend_tree shared memory");
  const uint32_t groups = static_cast<uint32_t>(a.pieces) * a.kv_heads;
  hipLaunchKernelGGL((attend_tree<T, D, WAVES>), dim3(groups), dim3(64 * WAVES), kBytes, s, a);
  hip_check(hipGetLastError(), "attend_tree launch");
  hipLaunchKernelGGL((join_tree<T, D, WAVES>), dim3(groups, 32 * WAVES / kJoinRows), dim3(256), 0, s, a);
  hip_check(hipGetLastError(), "join_tree launch");
}

template <typename T> void launch_dim(const TreeArgs &a, int64_t dim, int waves, hipStream_t s) {
  switch (dim) {
  case 64: waves == 8 ? launch<T, 64, 8>(a, s) : launch<T, 64, 4>(a, s); break;
  case 96: waves == 8 ? launch<T, 96, 8>(a, s) : launch<T, 96, 4>(a, s); break;
  case 128: waves == 8 ? launch<T, 128, 8>(a, s) : launch<T, 128, 4>(a, s); break;
  case 192: launch<T, 192, 4>(a, s); break;
  default: launch<T, 256, 4>(a, s); break;
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
    // Rows of a request and KV head, about.
    const int64_t per = (n.tokens + n.requests - 1) / n.requests * n.group;
    const int waves = kv.dim <= 128 && per > 128 ? 8 : 4, rows = 32 * waves;
    // Workgroups that the 256 CUs hold at once.
    const int64_t places = kv.dim <= 128 && waves == 4 ? 512 : 256;
    const int64_t most = (n.tokens * n.group / rows + n.requests) * std::max<int64_t>(1, (n.keys + 63) / 64);
    a.pieces = static_cast<int>(std::min(most, std::max<int64_t>(1, places / kv.heads)));
    const int64_t groups = a.pieces * kv.heads, parts = groups * 2 * rows;
    const int64_t bytes = parts * (kv.dim * 4 + 8) + groups * static_cast<int64_t>(sizeof(TreeArgs::Cut));
    // A launch has less than 2^32 threads along a dimension.
    expect(groups <= UINT32_MAX / 512, "too many heads");
    if (workspace_bytes) {
      *workspace_bytes = bytes;
      return;
    }
    check_outputs(query, output, lse, workspace, bytes, kv.device, vllm_kv_caches, n_caches,
                  {query_start_loc, seq_lens, block_table, tree_mask});
    a.mask = static_cast<const int64_t *>(tm.data);
    a.mask_token = tm.strides[0];
    a.words = static_cast<int>(tm.sizes[1]);
    a.part_o = static_cast<float *>(workspace->data);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + parts * kv.dim);
    a.cuts = reinterpret_cast<TreeArgs::Cut *>(a.part_ml + parts);
    DeviceGuard guard(kv.device);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (kv.dtype == LMC_BF16) launch_dim<BF16>(a, kv.dim, waves, s);
    else launch_dim<F16>(a, kv.dim, waves, s);
  });
}
