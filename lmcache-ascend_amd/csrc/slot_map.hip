// Block tables, slot mapping and positions of a batch from its request
// lengths, on MI355X (gfx950).
//
//   start_r = sum of query_lens before r          (query_start_loc)
//   pos(t)  = context_lens[r] + t - start_r       for start_r <= t < start_r + query_lens[r]
//   slot(t) = table[r, pos / BS] * BS + pos % BS  (-1 where there is no page)
//
// and, with a free list, table[r, j] = free[cursor + off_r + j - have_r] for
// the pages have_r = ceil(context / BS) <= j < need_r = ceil((context +
// query) / BS) that the new tokens open, off_r being the pages that earlier
// requests open.
//
// One launch.  The two prefix sums over the requests are small (8 to 16
// bytes a request, from L2), so every workgroup computes them for itself in
// LDS instead of waiting for another launch or workgroup; after that, tokens
// and new table entries are independent.  A token finds its request by
// bisection over the sums in LDS, between the requests of its wave's first
// and last token, so long prompts search once a wave.  A page that this call
// takes from the free list is read from the list, not from the table, which
// another workgroup is writing.
//
// A decode step's few tokens are latency: launch, lengths, pages, store.
// Requests of a few new tokens need no search, and their pages are loaded
// beside the sums.  64 requests of one token with a free list: 4.5 us (3.7 in
// a graph); 256 requests of up to 4096 tokens: 7.8 us.
#include "serving.h"

namespace lmc {

namespace {

// Two sums of 64 KiB each in the 160 KiB of LDS.
constexpr int kMaxRequests = 16384;
constexpr int kWaves = 16;  // of the largest workgroup

struct SlotMapArgs {
  const void *query_lens, *context_lens;
  int lens_i64;
  int n_requests;
  int32_t *table;
  int64_t table_stride;
  uint32_t width, block_size;
  int64_t *slots, *positions;  // positions may be null
  int64_t n_tokens;
  int32_t *starts, *seq_lens;  // either may be null
  int grow;                    // 0: the table is complete
  const int32_t *free_blocks;
  int64_t n_free;
  const int64_t *cursor;       // null: 0
  int64_t *next_cursor;        // may be null
  int token_blocks;            // workgroups of the tokens; those behind them complete the table
};

constexpr uint32_t kTop = 0x7fffffffu;

// Sums stop at 2^31 - 1: no output has a token there.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kTop); }

__device__ __forceinline__ int64_t len_at(const void *p, int i64, int r) {
  const int64_t v = i64 ? static_cast<const int64_t *>(p)[r] : static_cast<const int32_t *>(p)[r];
  return v < 0 ? 0 : v;
}

// The position of the i-th new token behind c tokens, 2^63 - 1 past that.
__device__ __forceinline__ int64_t position(int64_t c, uint32_t i) { return c > INT64_MAX - i ? INT64_MAX : c + i; }

// Pages that hold `tokens` tokens, at most the table's width.
__device__ __forceinline__ uint32_t pages_for(int64_t tokens, const SlotMapArgs &a) {
  const int64_t cap = static_cast<int64_t>(a.width) * a.block_size;  // < 2^31
  const uint32_t n = static_cast<uint32_t>(tokens < cap ? tokens : cap);
  return (n + a.block_size - 1) / a.block_size;
}

// The last r in [lo, hi] with sums[r] <= x (sums[lo] <= x).
__device__ __forceinline__ int find(const uint32_t *sums, int lo, int hi, uint32_t x) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Adds of the lanes below, in the wave's registers.
__device__ __forceinline__ uint32_t sums_to(uint32_t x) {
#define LMC_STEP(ctrl, rows) x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false))
  LMC_STEP(0x111, 0xf);  // 1, 2, 4 and 8 lanes down within 16
  LMC_STEP(0x112, 0xf);
  LMC_STEP(0x114, 0xf);
  LMC_STEP(0x118, 0xf);
  LMC_STEP(0x142, 0xa);  // the 16 lanes before, and the 32 before
  LMC_STEP(0x143, 0xc);
#undef LMC_STEP
  return x;
}

// Requests of at most this many new tokens are written by the thread that
// summed them up: no search, and the page is loaded beside the sums.
constexpr uint32_t kShort = 8;
constexpr int kUnroll = 4;  // tokens of a lane that are under way together

__global__ void __launch_bounds__(1024) slot_map(SlotMapArgs a) {
  extern __shared__ uint32_t lds[];
  const int R = a.n_requests, nt = blockDim.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const bool grow = a.grow != 0;
  uint32_t *sq = lds, *sb = lds + R + 1;  // sums before each request; sb only with a free list
  __shared__ uint32_t part[3][kWaves];
  uint32_t carry_q = 0, carry_b = 0, any_long = 0;
  const int64_t cursor = grow && a.cursor ? *a.cursor : 0;
  const int64_t cap = static_cast<int64_t>(a.width) * a.block_size;  // < 2^31
  auto free_at = [&](int64_t i) {
    i = static_cast<int64_t>(static_cast<uint64_t>(i) + static_cast<uint64_t>(cursor));  // (any cursor)
    return i >= 0 && i < a.n_free ? a.free_blocks[i] : -1;
  };
  auto write = [&](int64_t t, int64_t pos, uint32_t at, int32_t page) {
    a.slots[t] = page >= 0 ? static_cast<int64_t>(page) * a.block_size + at : -1;
    if (a.positions) a.positions[t] = pos;
  };
  for (int r0 = 0; r0 < R; r0 += nt) {
    const int r = r0 + tid;
    const bool mine = r < R && (r0 / nt) % a.token_blocks == static_cast<int>(blockIdx.x);
    uint32_t q = 0, b = 0, have = a.width;
    int64_t c = 0;
    int32_t page = -1;
    if (r < R) {
      const int64_t ql = len_at(a.query_lens, a.lens_i64, r);
      c = len_at(a.context_lens, a.lens_i64, r);
      q = static_cast<uint32_t>(ql < kTop ? ql : kTop);
      const int64_t end = c > INT64_MAX - ql ? INT64_MAX : c + ql;
      if (grow) {
        have = pages_for(c, a);
        b = pages_for(end, a) - have;
      }
      if (mine && q && q <= kShort && c < cap) {
        const uint32_t j = static_cast<uint32_t>(c) / a.block_size;
        if (j < have) page = a.table[r * a.table_stride + j];
      }
      if (blockIdx.x == 0 && a.seq_lens) a.seq_lens[r] = static_cast<int32_t>(end < kTop ? end : kTop);
    }
    const uint32_t iq = sums_to(q), ib = grow ? sums_to(b) : 0;
    // (not iq - q: the sum may have stopped at its top)
    uint32_t eq = __shfl_up(iq, 1), eb = __shfl_up(ib, 1);
    if (lane == 0) eq = eb = 0;
    const bool longer = __any(q > kShort);
    if (lane == 63) {
      part[0][wave] = iq;
      part[1][wave] = ib;
      part[2][wave] = longer;
    }
    __syncthreads();
    uint32_t bq = carry_q, bb = carry_b;
    for (int w = 0; w < nt / 64; ++w) {
      if (w < wave) {
        bq = add_sat(bq, part[0][w]);
        bb = add_sat(bb, part[1][w]);
      }
      carry_q = add_sat(carry_q, part[0][w]);
      carry_b = add_sat(carry_b, part[1][w]);
      any_long |= part[2][w];
    }
    const uint32_t start = add_sat(bq, eq), before_b = add_sat(bb, eb);
    if (r < R) {
      sq[r] = start;
      if (grow) sb[r] = before_b;
      if (blockIdx.x == 0 && a.starts) a.starts[r] = static_cast<int32_t>(start);
    }
    if (mine && q <= kShort) {
      for (uint32_t i = 0; i < q && start + i < a.n_tokens; ++i) {
        const int64_t pos = position(c, i);
        uint32_t at = 0;
        if (pos < cap) {
          const uint32_t p = static_cast<uint32_t>(pos), j = p / a.block_size;
          at = p - j * a.block_size;
          if (j >= have) page = free_at(static_cast<int64_t>(before_b) + (j - have));
          else if (i && at == 0) page = a.table[r * a.table_stride + j];
        } else {
          page = -1;
        }
        write(start + i, pos, at, page);
      }
    }
    __syncthreads();
  }
  if (tid == 0) {
    sq[R] = carry_q;
    if (grow) sb[R] = carry_b;
    if (blockIdx.x == 0) {
      if (a.starts) a.starts[R] = static_cast<int32_t>(carry_q);
      if (grow && a.next_cursor) *a.next_cursor = cursor + carry_b;
    }
  }
  __syncthreads();
  // New table entries, in workgroups of their own.
  if (static_cast<int>(blockIdx.x) >= a.token_blocks) {
    const int64_t step = static_cast<int64_t>(gridDim.x - a.token_blocks) * nt;
    for (int64_t u = static_cast<int64_t>(blockIdx.x - a.token_blocks) * nt + tid; u < carry_b; u += step) {
      const int32_t page = free_at(u);
      const int r = find(sb, 0, R - 1, static_cast<uint32_t>(u));
      const uint32_t j = pages_for(len_at(a.context_lens, a.lens_i64, r), a) + static_cast<uint32_t>(u - sb[r]);
      a.table[r * a.table_stride + j] = page;
    }
    return;
  }
  const int64_t step = static_cast<int64_t>(a.token_blocks) * nt;

  // Tokens of the longer requests, kUnroll times 64 of them a wave, and the
  // entries behind the last token.
  const int64_t total = carry_q;
  int64_t t0 = (static_cast<int64_t>(blockIdx.x) * nt + wave * 64) * kUnroll;
  if (!any_long) t0 += total / (step * kUnroll) * (step * kUnroll);
  for (; t0 < a.n_tokens; t0 += step * kUnroll) {
    int lo = 0, hi = 0;
    if (t0 < total && any_long) {
      lo = find(sq, 0, R - 1, static_cast<uint32_t>(t0));
      hi = find(sq, lo, R - 1, static_cast<uint32_t>(min(t0 + 64 * kUnroll, total) - 1));
    }
    int64_t pos[kUnroll];
    int r[kUnroll];
    int32_t page[kUnroll];
    uint32_t at[kUnroll];
    bool todo[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t t = t0 + 64 * u + lane;
      todo[u] = t < a.n_tokens && (t >= total || any_long);
      r[u] = -1;
      pos[u] = 0;
      if (todo[u] && t < total) {
        r[u] = find(sq, lo, hi, static_cast<uint32_t>(t));
        todo[u] = sq[r[u] + 1] - sq[r[u]] > kShort;
        if (todo[u]) pos[u] = len_at(a.context_lens, a.lens_i64, r[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      page[u] = -1;
      at[u] = 0;
      if (!todo[u] || r[u] < 0) continue;
      const uint32_t have = grow ? pages_for(pos[u], a) : a.width;
      pos[u] = position(pos[u], static_cast<uint32_t>(t0 + 64 * u + lane) - sq[r[u]]);
      if (pos[u] < cap) {
        const uint32_t p = static_cast<uint32_t>(pos[u]), j = p / a.block_size;
        at[u] = p - j * a.block_size;
        page[u] = j < have ? a.table[r[u] * a.table_stride + j] : free_at(static_cast<int64_t>(sb[r[u]]) + (j - have));
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (todo[u]) write(t0 + 64 * u + lane, pos[u], at[u], page[u]);
  }
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_build_slot_mapping(const lmc_tensor *query_lens, const lmc_tensor *context_lens,
                                      const lmc_tensor *block_table, int64_t block_size,
                                      const lmc_tensor *slot_mapping, const lmc_tensor *positions,
                                      const lmc_tensor *query_start_loc, const lmc_tensor *seq_lens,
                                      const lmc_tensor *free_blocks, const lmc_tensor *free_cursor,
                                      const lmc_tensor *next_cursor, void *stream) {
  return guarded([&] {
    const lmc_tensor &ql = deref(query_lens, "query_lens");
    const lmc_tensor &cl = deref(context_lens, "context_lens");
    const lmc_tensor &bt = deref(block_table, "block_table");
    const lmc_tensor &sm = deref(slot_mapping, "slot_mapping");
    const int dev = sm.device;
    expect(dev >= 0, "slot_mapping is not on a GPU");
    check_vector(sm, "slot_mapping", dev, LMC_I64);
    check_vector(ql, "query_lens", dev, LMC_I32, LMC_I64);
    check_vector(cl, "context_lens", dev, ql.dtype);
    check_on(bt, "block_table", dev, LMC_I32);
    const int64_t R = ql.sizes[0], N = sm.sizes[0];
    expect(cl.sizes[0] == R, "query_lens and context_lens differ in length");
    expect(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    expect(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    expect(R <= 1 || bt.strides[0] >= bt.sizes[1], "block_table rows overlap");
    expect(R <= kMaxRequests, "a call takes at most ", kMaxRequests, " requests");
    expect(block_size > 0 && block_size < (int64_t(1) << 31), "block_size must be positive");
    expect(bt.sizes[1] == 0 || block_size <= INT32_MAX / bt.sizes[1], "a block_table row spans 2^31 positions or more");
    expect(R * bt.sizes[1] <= INT32_MAX, "block_table has 2^31 entries or more");
    expect(N <= INT32_MAX - 65536, "slot_mapping has too many entries");
    SlotMapArgs a;
    std::memset(&a, 0, sizeof(a));
    a.query_lens = ql.data;
    a.context_lens = cl.data;
    a.lens_i64 = ql.dtype == LMC_I64;
    a.n_requests = static_cast<int>(R);
    a.table = static_cast<int32_t *>(bt.data);
    a.table_stride = bt.strides[0];
    a.width = static_cast<uint32_t>(bt.sizes[1]);
    a.block_size = static_cast<uint32_t>(block_size);
    a.slots = static_cast<int64_t *>(sm.data);
    a.n_tokens = N;
    if (positions) {
      const lmc_tensor &p = deref(positions, "positions");
      check_vector(p, "positions", dev, LMC_I64);
      expect(p.sizes[0] == N, "positions and slot_mapping differ in length");
      a.positions = static_cast<int64_t *>(p.data);
    }
    if (query_start_loc) {
      const lmc_tensor &q = deref(query_start_loc, "query_start_loc");
      check_vector(q, "query_start_loc", dev, LMC_I32);
      expect(q.sizes[0] == R + 1, "query_start_loc must have one entry per request and one more");
      a.starts = static_cast<int32_t *>(q.data);
    }
    if (seq_lens) {
      const lmc_tensor &q = deref(seq_lens, "seq_lens");
      check_vector(q, "seq_lens", dev, LMC_I32);
      expect(q.sizes[0] == R, "seq_lens must have one entry per request");
      a.seq_lens = static_cast<int32_t *>(q.data);
    }
    if (free_blocks) {
      const lmc_tensor &f = deref(free_blocks, "free_blocks");
      check_vector(f, "free_blocks", dev, LMC_I32);
      expect(!extents_meet(f, bt), "free_blocks overlaps block_table");
      a.grow = 1;
      a.free_blocks = static_cast<const int32_t *>(f.data);
      a.n_free = f.sizes[0];
    } else {
      expect(!free_cursor && !next_cursor, "free_cursor and next_cursor go with free_blocks");
    }
    if (free_cursor) {
      const lmc_tensor &c = deref(free_cursor, "free_cursor");
      check_vector(c, "free_cursor", dev, LMC_I64);
      expect(c.sizes[0] == 1, "free_cursor must have one entry");
      a.cursor = static_cast<const int64_t *>(c.data);
    }
    if (next_cursor) {
      const lmc_tensor &c = deref(next_cursor, "next_cursor");
      check_vector(c, "next_cursor", dev, LMC_I64);
      expect(c.sizes[0] == 1, "next_cursor must have one entry");
      expect(!free_cursor || !extents_meet(c, deref(free_cursor, "free_cursor")),
                  "next_cursor is free_cursor: workgroups read the one while the other is written");
      a.next_cursor = static_cast<int64_t *>(c.data);
    }
    // Every workgroup reads the lengths while the first ones write.
    for (const lmc_tensor *out : {slot_mapping, positions, query_start_loc, seq_lens, next_cursor, block_table})
      expect(!out || (!extents_meet(*out, ql) && !extents_meet(*out, cl)), "an output overlaps the lengths it is computed from");
    const lmc_tensor *grown = free_blocks ? block_table : nullptr;
    const lmc_tensor *outs[] = {slot_mapping, positions, query_start_loc, seq_lens, next_cursor, grown};
    for (const lmc_tensor *out : outs) {
      if (!out) continue;
      for (const lmc_tensor *in : {block_table, free_blocks, free_cursor})
        expect(!in || in == out || !extents_meet(*out, *in), "an output overlaps the table or the free list");
      for (const lmc_tensor *other : outs)
        expect(!other || other == out || !extents_meet(*out, *other), "two outputs overlap");
    }
    if (R == 0 && N == 0 && !a.starts && !a.next_cursor) return;
    DeviceGuard guard(dev);
    const int nt = R > 256 ? 1024 : 256;
    const int64_t blocks = std::min<int64_t>(std::max<int64_t>(1, (N + kUnroll * nt - 1) / (kUnroll * nt)), 1024);
    a.token_blocks = static_cast<int>(blocks);
    // About a new page a request and a block of new tokens.
    const int64_t pages = std::min(R * bt.sizes[1], R + N / block_size);
    const int64_t table_blocks = a.grow ? std::min<int64_t>(std::max<int64_t>(1, (pages + nt - 1) / nt), 256) : 0;
    const size_t shared = (a.grow ? 2 : 1) * (R + 1) * sizeof(uint32_t);
    if (shared > 48 * 1024)
      hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(slot_map), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(shared)),
                "slot_map shared memory");
    hipLaunchKernelGGL(slot_map, dim3(static_cast<uint32_t>(blocks + table_blocks)), dim3(nt), shared, static_cast<hipStream_t>(stream), a);
    hip_check(hipGetLastError(), "slot_map launch");
  });
}
