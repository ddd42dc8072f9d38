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
};

constexpr uint32_t kTop = 0x7fffffffu;

// Sums stop at 2^31 - 1: no output has a token there.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kTop); }

__device__ __forceinline__ int64_t len_at(const void *p, int i64, int r) {
  const int64_t v = i64 ? static_cast<const int64_t *>(p)[r] : static_cast<const int32_t *>(p)[r];
  return v < 0 ? 0 : v;
}

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

__global__ void __launch_bounds__(1024) slot_map(SlotMapArgs a) {
  extern __shared__ uint32_t lds[];
  const int R = a.n_requests, nt = blockDim.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const bool grow = a.grow != 0;
  uint32_t *sq = lds, *sb = lds + R + 1;  // sums before each request; sb only with a free list
  __shared__ uint32_t part[2][kWaves];
  uint32_t carry_q = 0, carry_b = 0;
  for (int r0 = 0; r0 < R; r0 += nt) {
    const int r = r0 + tid;
    uint32_t q = 0, b = 0;
    if (r < R) {
      const int64_t ql = len_at(a.query_lens, a.lens_i64, r), cl = len_at(a.context_lens, a.lens_i64, r);
      q = static_cast<uint32_t>(ql < kTop ? ql : kTop);
      const int64_t end = cl > INT64_MAX - ql ? INT64_MAX : cl + ql;
      if (grow) b = pages_for(end, a) - pages_for(cl, a);
      if (blockIdx.x == 0 && a.seq_lens) a.seq_lens[r] = static_cast<int32_t>(end < kTop ? end : kTop);
    }
    uint32_t iq = q, ib = b;  // inclusive sums of the wave
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t uq = __shfl_up(iq, d), ub = __shfl_up(ib, d);
      if (lane >= d) {
        iq = add_sat(iq, uq);
        ib = add_sat(ib, ub);
      }
    }
    // (not iq - q: the sum may have stopped at its top)
    uint32_t eq = __shfl_up(iq, 1), eb = __shfl_up(ib, 1);
    if (lane == 0) eq = eb = 0;
    if (lane == 63) {
      part[0][wave] = iq;
      part[1][wave] = ib;
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
    }
    if (r < R) {
      const uint32_t before_q = add_sat(bq, eq), before_b = add_sat(bb, eb);
      sq[r] = before_q;
      if (grow) sb[r] = before_b;
      if (blockIdx.x == 0 && a.starts) a.starts[r] = static_cast<int32_t>(before_q);
    }
    __syncthreads();
  }
  if (tid == 0) {
    sq[R] = carry_q;
    if (grow) sb[R] = carry_b;
    if (blockIdx.x == 0) {
      if (a.starts) a.starts[R] = static_cast<int32_t>(carry_q);
      if (grow && a.next_cursor) *a.next_cursor = (a.cursor ? *a.cursor : 0) + carry_b;
    }
  }
  __syncthreads();
  const int64_t cursor = grow && a.cursor ? *a.cursor : 0;
  auto free_at = [&](int64_t i) {
    i += cursor;
    return i >= 0 && i < a.n_free ? a.free_blocks[i] : -1;
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * nt;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * nt + tid;

  for (int64_t t = first; t < a.n_tokens; t += step) {
    int64_t pos = 0, slot = -1;
    if (t < carry_q) {
      // The wave's tokens t - lane .. t + 63 - lane lie between two requests.
      const uint32_t x = static_cast<uint32_t>(t), x0 = x - lane;
      const uint32_t x1 = static_cast<uint32_t>(min(static_cast<int64_t>(x0) + 63, static_cast<int64_t>(carry_q) - 1));
      const int lo = find(sq, 0, R - 1, __builtin_amdgcn_readfirstlane(x0));
      const int hi = find(sq, lo, R - 1, __builtin_amdgcn_readfirstlane(x1));
      const int r = find(sq, lo, hi, x);
      const int64_t c = len_at(a.context_lens, a.lens_i64, r);
      pos = c + (x - sq[r]);
      if (pos < static_cast<int64_t>(a.width) * a.block_size) {
        const uint32_t p = static_cast<uint32_t>(pos), j = p / a.block_size;
        const uint32_t have = grow ? pages_for(c, a) : a.width;
        const int32_t page = j < have ? a.table[r * a.table_stride + j] : free_at(static_cast<int64_t>(sb[r]) + (j - have));
        if (page >= 0) slot = static_cast<int64_t>(page) * a.block_size + (p - j * a.block_size);
      }
    }
    a.slots[t] = slot;
    if (a.positions) a.positions[t] = pos;
  }
  if (grow) {
    for (int64_t u = first; u < carry_b; u += step) {
      const int r = find(sb, 0, R - 1, static_cast<uint32_t>(u));
      const uint32_t j = pages_for(len_at(a.context_lens, a.lens_i64, r), a) + static_cast<uint32_t>(u - sb[r]);
      a.table[r * a.table_stride + j] = free_at(u);
    }
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
    check_value(dev >= 0, "slot_mapping is not on a GPU");
    check_vector(sm, "slot_mapping", dev, LMC_I64);
    check_vector(ql, "query_lens", dev, LMC_I32, LMC_I64);
    check_vector(cl, "context_lens", dev, ql.dtype);
    check_on(bt, "block_table", dev, LMC_I32);
    const int64_t R = ql.sizes[0], N = sm.sizes[0];
    check_value(cl.sizes[0] == R, "query_lens and context_lens differ in length");
    check_value(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    check_value(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    check_value(R <= 1 || bt.strides[0] >= bt.sizes[1], "block_table rows overlap");
    check_value(R <= kMaxRequests, "a call takes at most " + std::to_string(kMaxRequests) + " requests");
    check_value(block_size > 0 && block_size < (int64_t(1) << 31), "block_size must be positive");
    check_value(bt.sizes[1] == 0 || block_size <= INT32_MAX / bt.sizes[1], "a block_table row spans 2^31 positions or more");
    check_value(R * bt.sizes[1] <= INT32_MAX, "block_table has 2^31 entries or more");
    check_value(N <= INT32_MAX, "slot_mapping has 2^31 entries or more");
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
      check_value(p.sizes[0] == N, "positions and slot_mapping differ in length");
      a.positions = static_cast<int64_t *>(p.data);
    }
    if (query_start_loc) {
      const lmc_tensor &q = deref(query_start_loc, "query_start_loc");
      check_vector(q, "query_start_loc", dev, LMC_I32);
      check_value(q.sizes[0] == R + 1, "query_start_loc must have one entry per request and one more");
      a.starts = static_cast<int32_t *>(q.data);
    }
    if (seq_lens) {
      const lmc_tensor &q = deref(seq_lens, "seq_lens");
      check_vector(q, "seq_lens", dev, LMC_I32);
      check_value(q.sizes[0] == R, "seq_lens must have one entry per request");
      a.seq_lens = static_cast<int32_t *>(q.data);
    }
    if (free_blocks) {
      const lmc_tensor &f = deref(free_blocks, "free_blocks");
      check_vector(f, "free_blocks", dev, LMC_I32);
      check_value(!extents_meet(f, bt), "free_blocks overlaps block_table");
      a.grow = 1;
      a.free_blocks = static_cast<const int32_t *>(f.data);
      a.n_free = f.sizes[0];
    } else {
      check_value(!free_cursor && !next_cursor, "free_cursor and next_cursor go with free_blocks");
    }
    if (free_cursor) {
      const lmc_tensor &c = deref(free_cursor, "free_cursor");
      check_vector(c, "free_cursor", dev, LMC_I64);
      check_value(c.sizes[0] == 1, "free_cursor must have one entry");
      a.cursor = static_cast<const int64_t *>(c.data);
    }
    if (next_cursor) {
      const lmc_tensor &c = deref(next_cursor, "next_cursor");
      check_vector(c, "next_cursor", dev, LMC_I64);
      check_value(c.sizes[0] == 1, "next_cursor must have one entry");
      check_value(!free_cursor || !extents_meet(c, deref(free_cursor, "free_cursor")),
                  "next_cursor is free_cursor: workgroups read the one while the other is written");
      a.next_cursor = static_cast<int64_t *>(c.data);
    }
    // Every workgroup reads the lengths while the first ones write.
    for (const lmc_tensor *out : {slot_mapping, positions, query_start_loc, seq_lens, next_cursor, block_table})
      check_value(!out || (!extents_meet(*out, ql) && !extents_meet(*out, cl)), "an output overlaps the lengths it is computed from");
    if (R == 0 && N == 0 && !a.starts && !a.next_cursor) return;
    DeviceGuard guard(dev);
    const int nt = R > 256 ? 1024 : 256;
    const int64_t entries = std::max(N, a.grow ? R * bt.sizes[1] / 16 : int64_t(0));
    const int64_t blocks = std::min<int64_t>(std::max<int64_t>(1, (entries + 4 * nt - 1) / (4 * nt)), 1024);
    const size_t shared = (a.grow ? 2 : 1) * (R + 1) * sizeof(uint32_t);
    if (shared > 48 * 1024)
      hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(slot_map), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(shared)),
                "slot_map shared memory");
    hipLaunchKernelGGL(slot_map, dim3(static_cast<uint32_t>(blocks)), dim3(nt), shared, static_cast<hipStream_t>(stream), a);
    hip_check(hipGetLastError(), "slot_map launch");
  });
}
