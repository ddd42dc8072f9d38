// Pages of the paged caches copied, rows moved together, and pages given back,
// on MI355X (gfx950).
//
//   copy_kv_pages:  cache[l, p, dst] = cache[l, p, src]     for pairs (src, dst) of pages
//   compact_kv:     row(base_r + i) = row(base_r + keep[r, i])   for i < keep_lens[r]
//   release_pages:  pages ceil(keep / BS) <= j < ceil(held / BS) of each request lose a holder
//
// The first two in every layer l and plane p (K, V; the planes of an MLA
// layer), through a table of the layers' addresses.  Both are copies.  Pages go
// at the rate of the memory system: 256 of 128 tokens in 8 layers (8 heads of 128
// bf16 dims) 317 us in order (6.8 TB/s), 331 at random, 327 with a quarter of them
// read twice.  Rows at random do not: half of 8 contexts of 8000 tokens 264 to 286
// us, 4.1 to 4.5 TB/s (lists of one length 258, 4.6 TB/s; runs of adjacent rows
// 5.4 TB/s).  The accepted rows of 64 requests in 32 layers take 9.1 to 9.9 us.
//
// release_pages is latency, three launches: holders taken off with atomics, pages
// without one counted for each 1024, and those written to the list in ascending
// order, which does not depend on the order of the atomics.  64 requests' drafts
// among 20000 pages 8.8 to 10.5 us, 256 requests that end among 300000 12 us.
#include "serving.h"

#include <type_traits>
#include <vector>

namespace lmc {

namespace {

// A plane's bytes: row (page, token) has `heads` runs of `run` bytes.
struct PagePlane {
  int64_t offset;                 // from the layer's address
  int64_t page, token, head;
  int64_t heads, run;
  int tensor;                     // which of the layer's addresses
};

struct PageGeom {
  PagePlane plane[kMaxPlanes];
  int n_planes, n_tensors, device;
  int64_t pages, block_size;
  uint64_t align;                 // all addresses and steps, as bits
};

PageGeom page_geom(const lmc_tensor *caches, int n, int fmt, bool two_major, const char *op) {
  PageGeom g;
  std::memset(&g, 0, sizeof(g));
  if (fmt == LMC_FMT_MERGED_KV || fmt == LMC_FMT_SEPARATE_KV) {
    const PagedKv kv = paged_kv(caches, n, fmt, two_major, op);
    const int64_t run = kv.dim * dtype_size(kv.dtype);
    const bool merged = fmt == LMC_FMT_MERGED_KV;
    expect(k_and_v_apart(kv), "rows of the K and V caches overlap");
    g.plane[0] = {0, kv.k_page, kv.k_token, kv.k_head, kv.heads, run, 0};
    g.plane[1] = {merged ? kv.v - kv.k : 0, kv.v_page, kv.v_token, kv.v_head, kv.heads, run, merged ? 0 : 1};
    g.n_planes = 2;
    g.device = kv.device;
    g.pages = kv.pages;
    g.block_size = kv.block_size;
  } else {
    validate_vllm_caches(caches, n, fmt);
    expect(n <= kMaxPlanes, "a layer has at most ", kMaxPlanes, " caches");
    for (int i = 0; i < n; ++i) {
      const lmc_tensor &t = deref(&caches[i], "vllm_kv_caches");
      expect(t.ndim == 3 || t.ndim == 4, op, ": caches of this format are [pages, block, (heads,) dim]");
      expect(t.device >= 0, op, ": the paged caches are not on a GPU");
      expect(t.device == caches[0].device && t.sizes[0] == caches[0].sizes[0] && t.sizes[1] == caches[0].sizes[1],
             "a layer's caches differ in pages, block or device");
      for (int d = 0; d < t.ndim; ++d) expect(t.strides[d] >= 0, "negative strides unsupported");
      for (int k = 0; k < i; ++k) expect(!may_share(t, caches[k]), "a layer's caches overlap");
      const int64_t es = elem_size(t);
      expect(t.sizes[t.ndim - 1] <= 1 || t.strides[t.ndim - 1] == 1, "a cache row's head dims must be adjacent");
      expect(numel(t) > 0 || t.sizes[0] == 0, "the paged caches hold no rows");
      g.plane[i] = {0, t.strides[0] * es, t.strides[1] * es, t.ndim == 4 ? t.strides[2] * es : 0,
                    t.ndim == 4 ? t.sizes[2] : 1, t.sizes[t.ndim - 1] * es, i};
    }
    g.n_planes = n;
    g.device = caches[0].device;
    g.pages = caches[0].sizes[0];
    g.block_size = caches[0].sizes[1];
    expect(g.pages <= INT32_MAX && g.block_size <= INT32_MAX && g.pages * g.block_size <= static_cast<int64_t>(UINT32_MAX),
           "paged caches of more than 2^32 slots are not supported");
  }
  g.n_tensors = n;
  for (int i = 0; i < n; ++i) g.align |= reinterpret_cast<uintptr_t>(caches[i].data);
  for (int i = 0; i < g.n_planes; ++i) {
    PagePlane &p = g.plane[i];
    // (the stride of a dim of one entry says nothing)
    if (p.heads <= 1 || p.head == p.run) {
      p.run *= p.heads;
      p.heads = 1;
      p.head = 0;
    }
    if (g.block_size <= 1) p.token = 0;
    if (g.pages <= 1) p.page = 0;
    g.align |= p.offset | p.page | p.token | p.head | p.run;
    // Rows must be apart: what one row's copy writes is no other's.
    expect(rows_apart({g.pages, g.block_size, p.heads, p.run}, {p.page, p.token, p.head, 1}), "the paged caches have overlapping rows");
  }
  return g;
}

// [layers, caches of a layer] addresses.
int layers_of(const lmc_tensor &ptrs, const PageGeom &g) {
  check_on(ptrs, "layer_ptrs", g.device, LMC_I64);
  expect(ptrs.ndim == 2 && ptrs.sizes[1] == g.n_tensors, "layer_ptrs must be [layers, caches of a layer]");
  expect((ptrs.sizes[1] <= 1 || ptrs.strides[1] == 1) && (ptrs.sizes[0] <= 1 || ptrs.strides[0] == ptrs.sizes[1]),
         "layer_ptrs must be contiguous");
  expect(ptrs.sizes[0] <= 65535, "more than 65535 layers");
  return static_cast<int>(ptrs.sizes[0]);
}

// ---------------------------------------------------------------------------
// Pages copied
// ---------------------------------------------------------------------------

// A page of a plane as n1 x n0 runs of bytes.
struct CopyPlane {
  int64_t offset, page, s1, s0;
  uint32_t n0, pieces;            // runs in the inner dim; vectors of a run
  uint32_t vectors;               // of the page
  int tensor;
};

struct CopyArgs {
  CopyPlane plane[kMaxPlanes];
  const int64_t *ptrs;
  int n_tensors, n_planes;
  const void *pairs;
  int wide;                       // pairs are int64
  int64_t pair_stride;
  int64_t n_pages;
  uint32_t groups;                // workgroups of a page
};

// A vector a thread: what is under way together is other waves' (256 pages of 256
// KiB in 16 planes: 330 us; two vectors 368, four 400, eight 590).  Stores are
// written through: streaming ones take 344 us, 7.2 instead of 5.5 with 8 pages.
template <int VEC> __global__ void __launch_bounds__(256) copy_pages(CopyArgs a) {
  using V = typename VecOf<VEC>::T;
  const uint32_t pair = blockIdx.x / a.groups, x = (blockIdx.x - pair * a.groups) * 256 + threadIdx.x;
  const int p = blockIdx.y % a.n_planes, l = blockIdx.y / a.n_planes;
  int64_t src, dst;
  if (a.wide) {
    const int64_t *at = static_cast<const int64_t *>(a.pairs) + pair * a.pair_stride;
    src = at[0];
    dst = at[1];
  } else {
    const int32_t *at = static_cast<const int32_t *>(a.pairs) + pair * a.pair_stride;
    src = at[0];
    dst = at[1];
  }
  const CopyPlane &c = a.plane[p];
  uint8_t *base = reinterpret_cast<uint8_t *>(a.ptrs[l * a.n_tensors + c.tensor]) + c.offset;
  if (src < 0 || src >= a.n_pages || dst < 0 || dst >= a.n_pages || src == dst || x >= c.vectors) return;
  const uint32_t run = x / c.pieces, i1 = run / c.n0;
  const int64_t at = i1 * c.s1 + (run - i1 * c.n0) * c.s0 + (x - run * c.pieces) * static_cast<int64_t>(VEC);
  st<V, true>(reinterpret_cast<V *>(base + dst * c.page + at), ld<V, true>(reinterpret_cast<const V *>(base + src * c.page + at)));
}

// ---------------------------------------------------------------------------
// Rows moved together
// ---------------------------------------------------------------------------

struct MovePlane {
  int64_t offset, page, token, head;
  uint32_t pieces;                // vectors of a run
  uint32_t vectors;               // of a row
  int tensor;
};

struct MoveArgs {
  MovePlane plane[kMaxPlanes];
  const int64_t *ptrs;
  int n_tensors, n_planes, n_layers;
  const int32_t *table;
  int64_t table_stride;
  uint32_t width, block_size;
  int64_t n_pages;
  const int32_t *base_lens, *keep, *keep_lens;
  int64_t keep_stride;
  int most;                       // entries of a list
  int32_t *seq_lens;              // may be null
  int lanes;                      // threads of a row: a power of two, kLeastLanes to 256
};

// Rows of a thread in a step, with one step and with more: half of 8 contexts
// takes 267 us with 8, 304 with 4.
constexpr int kRowsOnce = 4, kRowsMore = 8;
constexpr int kBatch = 256;       // rows whose places are looked up together
constexpr int kLeastLanes = 8;    // of a row
// A step's rows are looked up: a batch holds whole steps.
static_assert(kBatch % (256 / kLeastLanes * kRowsOnce) == 0 && kBatch % (256 / kLeastLanes * kRowsMore) == 0, "");

// A workgroup moves a slice of one request's rows in one layer (in PL planes
// of one geometry), some rows at a time, in order: rows move down (keep[i] >= i),
// so what a step writes has been read by it or by an earlier one.  With MORE
// than one step, the next one's rows are loaded before this one's are written:
// they lie behind all that it writes.  A row's place takes a chain of two loads
// (list, table), so a thread each looks up 256 rows at once, into LDS.
template <int VEC, int PL, bool MORE> __global__ void __launch_bounds__(256) move_rows(MoveArgs a) {
  using V = typename VecOf<VEC>::T;
  using Held = std::conditional_t<(VEC < 4), uint32_t, V>;  // in a register
  constexpr int kUnroll = MORE ? kRowsMore : kRowsOnce;
  __shared__ int64_t from[MORE ? 2 : 1][kBatch], to[MORE ? 2 : 1][kBatch];  // bytes from the plane's first row; -1: stays
  const int groups = a.n_planes / PL, p = blockIdx.y % groups * PL, l = blockIdx.y / groups, r = blockIdx.z;
  const MovePlane &c = a.plane[p];
  const int32_t *keep = a.keep + r * a.keep_stride, *table = a.table + r * a.table_stride;
  const int first = a.most > 0 ? keep[min(static_cast<int>(threadIdx.x), a.most - 1)] : 0;  // (beside the lengths)
  const int64_t b = a.base_lens[r];
  const int n = min(max(a.keep_lens[r], 0), a.most);
  if (a.seq_lens && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    a.seq_lens[r] = static_cast<int32_t>(min(b + n, static_cast<int64_t>(INT32_MAX)));
  if (l >= a.n_layers) return;  // (a call without layers)
  uint8_t *base[PL];
#pragma unroll
  for (int q = 0; q < PL; ++q) base[q] = reinterpret_cast<uint8_t *>(a.ptrs[l * a.n_tensors + a.plane[p + q].tensor]) + a.plane[p + q].offset;
  // Where a position's row lies, or -1 where the caches have none.
  auto place = [&](int64_t pos) -> int64_t {
    if (pos < 0 || pos >= static_cast<int64_t>(a.width) * a.block_size) return -1;
    const uint32_t j = static_cast<uint32_t>(pos) / a.block_size;
    const int64_t page = table[j];
    if (page < 0 || page >= a.n_pages) return -1;
    return page * c.page + (static_cast<uint32_t>(pos) - j * a.block_size) * c.token;
  };
  auto look_up = [&](int batch, int k) {
    const int x = threadIdx.x, i = batch * kBatch + x;
    int64_t s = -1, d = -1;
    if (i < n && k != i) {
      s = place(b + k);
      d = place(b + i);
    }
    from[MORE ? batch & 1 : 0][x] = s;
    to[MORE ? batch & 1 : 0][x] = s < 0 ? -1 : d;
  };
  const int rows = 256 / a.lanes, own = threadIdx.x / a.lanes, step = rows * kUnroll;
  const uint32_t x = blockIdx.x * a.lanes + (threadIdx.x & (a.lanes - 1));
  const bool in = x < c.vectors;
  const int64_t column = (x / c.pieces) * c.head + (x % c.pieces) * static_cast<int64_t>(VEC);
  Held now[kUnroll][PL], next[kUnroll][PL];
  auto load = [&](int i0, Held (&v)[kUnroll][PL]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * rows + own;
      const int64_t d = in && i < n ? to[MORE ? i / kBatch & 1 : 0][i % kBatch] : -1, s = from[MORE ? i / kBatch & 1 : 0][i % kBatch];
#pragma unroll
      for (int q = 0; q < PL; ++q) {
        v[u][q] = Held{};
        if (d >= 0) v[u][q] = gload(reinterpret_cast<const V *>(base[q] + s + column));
      }
    }
  };
  auto store = [&](int i0, const Held (&v)[kUnroll][PL]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * rows + own;
      const int64_t d = in && i < n ? to[MORE ? i / kBatch & 1 : 0][i % kBatch] : -1;
#pragma unroll
      for (int q = 0; q < PL; ++q)
        if (d >= 0) gstore_nt(reinterpret_cast<V *>(base[q] + d + column), static_cast<V>(v[u][q]));
    }
  };
  // A step's rows have arrived, in every wave.
  auto arrive = [&](Held (&v)[kUnroll][PL]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int q = 0; q < PL; ++q) asm volatile("" : "+v"(v[u][q])::"memory");
    __syncthreads();
  };
  look_up(0, first);
  __syncthreads();
  load(0, now);
  if constexpr (!MORE) {
    arrive(now);
    store(0, now);
  } else {
    for (int i0 = 0; i0 < n; i0 += step) {
      // The batch behind this one, once every wave is done with the one before.
      if (i0 % kBatch == 0) {
        __syncthreads();
        const int ahead = i0 / kBatch + 1, i = ahead * kBatch + threadIdx.x;
        look_up(ahead, i < n ? keep[i] : 0);
        __syncthreads();
      }
      load(i0 + step, next);
      arrive(now);
      store(i0, now);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int q = 0; q < PL; ++q) now[u][q] = next[u][q];
    }
  }
}

template <int VEC> void launch_moves(const MoveArgs &a, int planes, bool more, dim3 grid, hipStream_t s) {
  if (planes == 2 && more) hipLaunchKernelGGL((move_rows<VEC, 2, true>), grid, dim3(256), 0, s, a);
  else if (planes == 2) hipLaunchKernelGGL((move_rows<VEC, 2, false>), grid, dim3(256), 0, s, a);
  else if (more) hipLaunchKernelGGL((move_rows<VEC, 1, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((move_rows<VEC, 1, false>), grid, dim3(256), 0, s, a);
  hip_check(hipGetLastError(), "move_rows launch");
}

// ---------------------------------------------------------------------------
// Pages given back
// ---------------------------------------------------------------------------

struct ReleaseArgs {
  const int32_t *table;
  int64_t table_stride;
  uint32_t width, block_size;
  const int32_t *held, *keep;
  int32_t *refs;
  int whole;                      // refs is on a 16-byte boundary
  int n_pages;
  int32_t *free_blocks;
  int64_t n_free;
  const int64_t *cursor;
  int64_t *next_cursor;
  int32_t *counts;                // pages given back of each run of kRun
  int runs;
};

constexpr int kRun = 1024;        // pages of a workgroup, four a thread

// A holder less for each page that a request gives back.
__global__ void __launch_bounds__(256) drop_holders(ReleaseArgs a) {
  const int r = blockIdx.x;
  auto pages_for = [&](int tokens) {
    const uint32_t n = static_cast<uint32_t>(max(0, tokens));
    return min(n / a.block_size + (n % a.block_size != 0), a.width);
  };
  const uint32_t first = pages_for(a.keep[r]), stop = pages_for(a.held[r]);
  for (uint32_t j = first + blockIdx.y * 256 + threadIdx.x; j < stop; j += gridDim.y * 256) {
    const int page = a.table[r * a.table_stride + j];
    if (page >= 0 && page < a.n_pages) atomicSub(a.refs + page, 1);
  }
}

// Which of the pages from p0 on (a multiple of 4) have no holder left.
__device__ __forceinline__ uint32_t without_holder(const ReleaseArgs &a, int p0) {
  uint32_t bits = 0;
  if (p0 + 4 <= a.n_pages && a.whole) {
    const int4 x = *reinterpret_cast<const int4 *>(a.refs + p0);
    bits = (x.x < 0) | (x.y < 0) << 1 | (x.z < 0) << 2 | (x.w < 0) << 3;
  } else {
    for (int i = 0; i < 4; ++i)
      if (p0 + i < a.n_pages && a.refs[p0 + i] < 0) bits |= 1u << i;
  }
  return bits;
}

// Those pages to the list from `at` on.
__device__ __forceinline__ void give_back(const ReleaseArgs &a, int p0, uint32_t bits, int64_t at) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(bits >> i & 1)) continue;
    a.refs[p0 + i] = 0;
    if (at >= 0 && at < a.n_free) a.free_blocks[at] = p0 + i;
    ++at;
  }
}

__device__ __forceinline__ int sum_of_wave(int n) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
  return n;
}

// The sum of the lanes up to this one.
__device__ __forceinline__ int sum_to_lane(int n) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(n, d);
    if ((threadIdx.x & 63) >= d) n += below;
  }
  return n;
}

__global__ void __launch_bounds__(256) count_free(ReleaseArgs a) {
  __shared__ int part[4];
  const int n = sum_of_wave(__popc(without_holder(a, blockIdx.x * kRun + threadIdx.x * 4)));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) a.counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

__global__ void __launch_bounds__(256) place_free(ReleaseArgs a) {
  __shared__ int part[3][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p0 = blockIdx.x * kRun + threadIdx.x * 4;
  // (places past the list's end were never handed out)
  const int64_t cursor = min(*a.cursor, a.n_free);
  const uint32_t bits = without_holder(a, p0);
  int before = 0, total = 0;
  for (int i = threadIdx.x; i < a.runs; i += 256) {
    const int n = a.counts[i];
    total += n;
    if (i < static_cast<int>(blockIdx.x)) before += n;
  }
  before = sum_of_wave(before);
  total = sum_of_wave(total);
  const int own = __popc(bits), upto = sum_to_lane(own);
  if (lane == 63) {
    part[0][wave] = upto;
    part[1][wave] = before;
    part[2][wave] = total;
  }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    before += part[1][w] + (w < wave ? part[0][w] : 0);
    total += part[2][w];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.next_cursor = cursor - total;
  give_back(a, p0, bits, cursor - total + before + upto - own);
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_check_layers_apart(const lmc_tensor *caches, int64_t n, int64_t *ranges, int64_t *n_ranges) {
  return guarded([&] {
    struct Cache {
      int64_t begin, end;
      int device;
      Layout layout;
    };
    std::vector<Cache> all;
    for (int64_t i = 0; i < n; ++i) {
      const lmc_tensor &t = deref(&caches[i], "caches");
      const int64_t begin = reinterpret_cast<int64_t>(t.data), bytes = extent_bytes(t);
      if (bytes > 0) all.push_back({begin, begin + bytes, t.device, layout_of(t)});
    }
    std::sort(all.begin(), all.end(), [](const Cache &a, const Cache &b) { return a.begin < b.begin; });
    for (size_t i = 0; i < all.size(); ++i)
      for (size_t k = i + 1; k < all.size() && all[k].begin < all[i].end; ++k)
        expect(all[i].device != all[k].device || apart(all[i].layout, all[k].layout, all[k].begin - all[i].begin),
               "two of the layers' caches overlap");
    if (!ranges) return;
    int64_t count = 0;
    for (const Cache &c : all) {
      if (count > 0 && c.begin <= ranges[2 * count - 1]) {
        ranges[2 * count - 1] = std::max(ranges[2 * count - 1], c.end);
        continue;
      }
      ranges[2 * count] = c.begin;
      ranges[2 * count + 1] = c.end;
      ++count;
    }
    *n_ranges = count;
  });
}

extern "C" int lmc_check_outside(const int64_t *ranges, int64_t n, const lmc_tensor *const *tensors, int32_t n_tensors) {
  return guarded([&] {
    for (int i = 0; i < n_tensors; ++i) {
      const int64_t bytes = tensors[i] ? extent_bytes(*tensors[i]) : 0;
      if (bytes == 0) continue;
      const int64_t from = reinterpret_cast<int64_t>(tensors[i]->data);
      int64_t lo = 0, hi = n;  // the first range that ends behind `from`
      while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (ranges[2 * mid + 1] > from) hi = mid;
        else lo = mid + 1;
      }
      expect(lo == n || ranges[2 * lo] >= from + bytes, "the call's tables or lists overlap the paged caches of a layer");
    }
  });
}

extern "C" int lmc_copy_kv_pages(const lmc_tensor *layer_ptrs, const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                                 const lmc_tensor *pages, int32_t kvcache_format, int32_t vllm_two_major, void *stream) {
  return guarded([&] {
    const PageGeom g = page_geom(vllm_kv_caches, n_caches, kvcache_format, vllm_two_major != 0, "copy_kv_pages");
    const lmc_tensor &lp = deref(layer_ptrs, "layer_ptrs");
    const lmc_tensor &pr = deref(pages, "pages");
    const int layers = layers_of(lp, g);
    check_on(pr, "pages", g.device, LMC_I32, LMC_I64);
    expect(pr.ndim == 2 && pr.sizes[1] == 2, "pages must be [pairs, 2]");
    expect(pr.strides[1] == 1, "a pair's two pages must be adjacent");
    expect(pr.strides[0] >= 0, "negative strides unsupported");
    expect(pr.sizes[0] <= INT32_MAX, "too many pairs");
    for (int i = 0; i < n_caches; ++i)
      expect(!extents_meet(pr, vllm_kv_caches[i]) && !extents_meet(lp, vllm_kv_caches[i]), "pages or layer_ptrs overlap the paged caches");
    if (pr.sizes[0] == 0 || layers == 0 || g.pages == 0) return;
    CopyArgs a;
    std::memset(&a, 0, sizeof(a));
    const int vec = vec_for(static_cast<int64_t>(g.align));
    int64_t most = 0;
    for (int i = 0; i < g.n_planes; ++i) {
      const PagePlane &p = g.plane[i];
      int64_t run = p.run, n[2] = {p.heads, g.block_size}, s[2] = {p.head, p.token};
      if (s[0] > s[1] && n[1] > 1) {
        std::swap(n[0], n[1]);
        std::swap(s[0], s[1]);
      }
      for (int d = 0; d < 2; ++d)
        if (n[0] == 1 || s[0] == run) {
          run *= n[0];
          n[0] = n[1];
          s[0] = s[1];
          n[1] = 1;
        }
      a.plane[i] = {p.offset, p.page, s[1], s[0], static_cast<uint32_t>(n[0]), static_cast<uint32_t>(run / vec),
                    static_cast<uint32_t>(run / vec * n[0] * n[1]), p.tensor};
      expect(run / vec * n[0] * n[1] < (int64_t(1) << 31), "pages of 2^31 elements or more");
      most = std::max(most, run / vec * n[0] * n[1]);
    }
    a.ptrs = static_cast<const int64_t *>(lp.data);
    a.n_tensors = g.n_tensors;
    a.n_planes = g.n_planes;
    a.pairs = pr.data;
    a.wide = pr.dtype == LMC_I64;
    a.pair_stride = pr.strides[0];
    a.n_pages = g.pages;
    a.groups = static_cast<uint32_t>((most + 255) / 256);
    expect(a.groups * pr.sizes[0] <= UINT32_MAX / 256 && layers * g.n_planes <= 65535, "too many pages");
    DeviceGuard guard(g.device);
    const dim3 grid(static_cast<uint32_t>(a.groups * pr.sizes[0]), static_cast<uint32_t>(layers * g.n_planes));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (vec) {
    case 16: hipLaunchKernelGGL(copy_pages<16>, grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL(copy_pages<8>, grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL(copy_pages<4>, grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL(copy_pages<2>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(copy_pages<1>, grid, dim3(256), 0, s, a); break;
    }
    hip_check(hipGetLastError(), "copy_pages launch");
  });
}

extern "C" int lmc_compact_kv(const lmc_tensor *layer_ptrs, const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                              const lmc_tensor *block_table, const lmc_tensor *base_lens, const lmc_tensor *keep,
                              const lmc_tensor *keep_lens, const lmc_tensor *seq_lens, int32_t kvcache_format,
                              int32_t vllm_two_major, void *stream) {
  return guarded([&] {
    const PageGeom g = page_geom(vllm_kv_caches, n_caches, kvcache_format, vllm_two_major != 0, "compact_kv");
    const lmc_tensor &lp = deref(layer_ptrs, "layer_ptrs");
    const lmc_tensor &bt = deref(block_table, "block_table");
    const lmc_tensor &bl = deref(base_lens, "base_lens");
    const lmc_tensor &kp = deref(keep, "keep");
    const lmc_tensor &kl = deref(keep_lens, "keep_lens");
    const int layers = layers_of(lp, g), dev = g.device;
    check_on(bt, "block_table", dev, LMC_I32);
    check_vector(bl, "base_lens", dev, LMC_I32);
    check_on(kp, "keep", dev, LMC_I32);
    check_vector(kl, "keep_lens", dev, LMC_I32);
    const int64_t R = bl.sizes[0];
    expect(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    expect(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    expect(kp.ndim == 2 && kp.sizes[0] == R, "keep must be [requests, rows]");
    expect(kp.sizes[1] <= 1 || kp.strides[1] == 1, "keep's lists must be contiguous");
    expect(kl.sizes[0] == R, "keep_lens must have one entry per request");
    expect(bt.strides[0] >= 0 && kp.strides[0] >= 0, "negative strides unsupported");
    expect(bt.sizes[1] == 0 || g.block_size <= INT32_MAX / bt.sizes[1], "a block_table row spans 2^31 positions or more");
    expect(kp.sizes[1] <= INT32_MAX / 2 && R <= 65535, "more than 65535 requests, or lists of more than 2^30 rows");
    if (seq_lens) {
      const lmc_tensor &sl = deref(seq_lens, "seq_lens");
      check_vector(sl, "seq_lens", dev, LMC_I32);
      expect(sl.sizes[0] == R, "seq_lens must have one entry per request");
      for (const lmc_tensor *in : {block_table, base_lens, keep, keep_lens, layer_ptrs})
        expect(!extents_meet(sl, *in), "seq_lens overlaps what it is computed from");
    }
    for (const lmc_tensor *x : {block_table, base_lens, keep, keep_lens, seq_lens, layer_ptrs})
      for (int i = 0; x && i < n_caches; ++i)
        expect(!extents_meet(*x, vllm_kv_caches[i]), "the tables or lists overlap the paged caches");
    if (R == 0 || (layers == 0 && !seq_lens)) return;
    MoveArgs a;
    std::memset(&a, 0, sizeof(a));
    const int vec = vec_for(static_cast<int64_t>(g.align));
    int64_t most = 0;
    for (int i = 0; i < g.n_planes; ++i) {
      const PagePlane &p = g.plane[i];
      const int64_t vectors = p.run / vec * p.heads;
      expect(vectors < (int64_t(1) << 30), "rows of 2^30 elements or more");
      a.plane[i] = {p.offset, p.page, p.token, p.head, static_cast<uint32_t>(p.run / vec), static_cast<uint32_t>(vectors), p.tensor};
      most = std::max(most, vectors);
    }
    a.ptrs = static_cast<const int64_t *>(lp.data);
    a.n_tensors = g.n_tensors;
    a.n_planes = g.n_planes;
    a.n_layers = layers;
    a.table = static_cast<const int32_t *>(bt.data);
    a.table_stride = bt.strides[0];
    a.width = static_cast<uint32_t>(bt.sizes[1]);
    a.block_size = static_cast<uint32_t>(g.block_size);
    a.n_pages = g.pages;
    a.base_lens = static_cast<const int32_t *>(bl.data);
    a.keep = static_cast<const int32_t *>(kp.data);
    a.keep_lens = static_cast<const int32_t *>(kl.data);
    a.keep_stride = kp.strides[0];
    a.most = static_cast<int>(kp.sizes[1]);
    a.seq_lens = seq_lens ? static_cast<int32_t *>(seq_lens->data) : nullptr;
    // K and V of one geometry go together.
    const MovePlane &k = a.plane[0], &v = a.plane[1];
    const int planes = g.n_planes == 2 && k.page == v.page && k.token == v.token && k.head == v.head && k.pieces == v.pieces &&
                               k.vectors == v.vectors ? 2 : 1;
    const int64_t groups = std::max(1, layers) * (g.n_planes / planes), items = R * groups;
    // Slices of a row for 1024 workgroups or more, but no narrower than that takes
    // (128 bytes at least: half of 8 contexts of 8000 tokens 276 us so; 64 requests
    // of 6 rows 10.6 us with whole rows, 13.7 with slices for 4096 workgroups).
    a.lanes = kLeastLanes;
    while (a.lanes < 256 && a.lanes < most && items * ((most + 2 * a.lanes - 1) / (2 * a.lanes)) >= 1024) a.lanes *= 2;
    const int64_t slices = (most + a.lanes - 1) / a.lanes;
    expect(groups <= 65535 && slices <= UINT32_MAX / 256, "too many layers");
    DeviceGuard guard(dev);
    const dim3 grid(static_cast<uint32_t>(slices), static_cast<uint32_t>(groups), static_cast<uint32_t>(R));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool more = a.most > 256 / a.lanes * kRowsOnce;
    switch (vec) {
    case 16: launch_moves<16>(a, planes, more, grid, s); break;
    case 8: launch_moves<8>(a, planes, more, grid, s); break;
    case 4: launch_moves<4>(a, planes, more, grid, s); break;
    case 2: launch_moves<2>(a, planes, more, grid, s); break;
    default: launch_moves<1>(a, planes, more, grid, s); break;
    }
  });
}

extern "C" int lmc_release_pages(const lmc_tensor *block_table, const lmc_tensor *held_lens, const lmc_tensor *keep_lens,
                                 int64_t block_size, const lmc_tensor *page_refs, const lmc_tensor *free_blocks,
                                 const lmc_tensor *free_cursor, const lmc_tensor *next_cursor,
                                 const lmc_tensor *workspace, int64_t *workspace_bytes, void *stream) {
  return guarded([&] {
    const lmc_tensor &bt = deref(block_table, "block_table");
    const lmc_tensor &hl = deref(held_lens, "held_lens");
    const lmc_tensor &kl = deref(keep_lens, "keep_lens");
    const lmc_tensor &pr = deref(page_refs, "page_refs");
    const lmc_tensor &fb = deref(free_blocks, "free_blocks");
    const lmc_tensor &fc = deref(free_cursor, "free_cursor");
    const lmc_tensor &nc = deref(next_cursor, "next_cursor");
    const int dev = pr.device;
    expect(dev >= 0, "page_refs is not on a GPU");
    check_vector(pr, "page_refs", dev, LMC_I32);
    check_on(bt, "block_table", dev, LMC_I32);
    check_vector(hl, "held_lens", dev, LMC_I32);
    check_vector(kl, "keep_lens", dev, LMC_I32);
    check_vector(fb, "free_blocks", dev, LMC_I32);
    check_vector(fc, "free_cursor", dev, LMC_I64);
    check_vector(nc, "next_cursor", dev, LMC_I64);
    const int64_t R = hl.sizes[0], P = pr.sizes[0];
    expect(kl.sizes[0] == R, "held_lens and keep_lens differ in length");
    expect(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    expect(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    expect(bt.strides[0] >= 0, "negative strides unsupported");
    expect(bt.sizes[1] <= INT32_MAX / 2 && R <= INT32_MAX / 256, "block_table is too large");
    expect(block_size > 0 && block_size < (int64_t(1) << 31), "block_size must be positive");
    expect(P <= INT32_MAX - 2 * kRun, "page_refs has too many entries");
    expect(fc.sizes[0] == 1, "free_cursor must have one entry");
    expect(nc.sizes[0] == 1, "next_cursor must have one entry");
    const int64_t runs = std::max<int64_t>(1, (P + kRun - 1) / kRun), bytes = runs * 4;
    if (workspace_bytes) {
      *workspace_bytes = bytes;
      return;
    }
    const lmc_tensor &ws = deref(workspace, "workspace");
    check_on(ws, "workspace", dev, LMC_U8);
    expect(ws.ndim == 1 && (ws.sizes[0] <= 1 || ws.strides[0] == 1) && ws.sizes[0] >= bytes &&
               reinterpret_cast<uintptr_t>(ws.data) % 4 == 0,
           "workspace must be 1-D, contiguous, on a 4-byte boundary and of at least ", bytes, " bytes");
    const lmc_tensor *outs[] = {page_refs, free_blocks, next_cursor, workspace};
    for (const lmc_tensor *out : outs) {
      for (const lmc_tensor *in : {block_table, held_lens, keep_lens, free_cursor})
        expect(!extents_meet(*out, *in), "an output overlaps what it is computed from");
    }
    for (int i = 0; i < 4; ++i)
      for (int k = 0; k < i; ++k) expect(!extents_meet(*outs[i], *outs[k]), "two outputs overlap");
    ReleaseArgs a;
    std::memset(&a, 0, sizeof(a));
    a.table = static_cast<const int32_t *>(bt.data);
    a.table_stride = bt.strides[0];
    a.width = static_cast<uint32_t>(bt.sizes[1]);
    a.block_size = static_cast<uint32_t>(block_size);
    a.held = static_cast<const int32_t *>(hl.data);
    a.keep = static_cast<const int32_t *>(kl.data);
    a.refs = static_cast<int32_t *>(pr.data);
    a.whole = reinterpret_cast<uintptr_t>(pr.data) % 16 == 0;
    a.n_pages = static_cast<int>(P);
    a.free_blocks = static_cast<int32_t *>(fb.data);
    a.n_free = fb.sizes[0];
    a.cursor = static_cast<const int64_t *>(fc.data);
    a.next_cursor = static_cast<int64_t *>(nc.data);
    a.counts = static_cast<int32_t *>(ws.data);
    a.runs = static_cast<int>(runs);
    DeviceGuard guard(dev);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t turns = static_cast<uint32_t>(std::min<int64_t>(16, (bt.sizes[1] + 255) / 256));
    if (R > 0 && turns > 0) hipLaunchKernelGGL(drop_holders, dim3(static_cast<uint32_t>(R), turns), dim3(256), 0, s, a);
    hip_check(hipGetLastError(), "drop_holders launch");
    hipLaunchKernelGGL(count_free, dim3(static_cast<uint32_t>(runs)), dim3(256), 0, s, a);
    hip_check(hipGetLastError(), "count_free launch");
    hipLaunchKernelGGL(place_free, dim3(static_cast<uint32_t>(runs)), dim3(256), 0, s, a);
    hip_check(hipGetLastError(), "place_free launch");
  });
}
