// Masks and positions of trees of drafted tokens on MI355X (gfx950).
//
//   anc(i)  = {i} + anc(parent(i)) where 0 <= parent(i) < i, else {i}
//   mask(i) = the bits of anc(i),  position(i) = seq - q + |anc(i)| - 1
//
// for the i-th of a request's q drafted tokens, the last of its seq ones.
//
// A wave a request, 64 tokens at a time, a token a lane.  Within a block the
// ancestors are doubled in registers: a lane takes the bits of the lane it
// points at and points where that one does, so six steps close any chain.  The
// lowest bit is then the chain's first token in the block; its parent, if it
// has one, lies in an earlier block, whose row is complete in LDS.  Nothing of
// this takes longer than the loads: the call is latency (256 requests of up to 100
// tokens 3.6 us, 4 of 8 2.3; 4.4 with the call).
#include "serving.h"

namespace lmc {

namespace {

constexpr int kMaxWords = 16;  // rows of 1024 tokens, 128 of the 160 KiB of LDS

struct DraftArgs {
  const int32_t *parents, *starts, *seq_lens;
  int n_requests, n_tokens, words;
  int64_t *mask, *positions;  // positions may be null
  int64_t mask_token;
};

__global__ void __launch_bounds__(64) draft_tree(DraftArgs a) {
  extern __shared__ uint64_t rows[];  // [64 * words][words], with more than one word
  const int lane = threadIdx.x, W = a.words;
  if (static_cast<int>(blockIdx.x) >= a.n_requests) {
    // Rows behind the last request.
    const int step = 64 * (gridDim.x - a.n_requests);
    for (int64_t t = static_cast<int64_t>(max(0, a.starts[a.n_requests])) + (blockIdx.x - a.n_requests) * 64 + lane; t < a.n_tokens; t += step) {
      for (int w = 0; w < W; ++w) a.mask[t * a.mask_token + w] = 0;
      if (a.positions) a.positions[t] = 0;
    }
    return;
  }
  const int start = a.starts[blockIdx.x], stop = a.starts[blockIdx.x + 1];
  const int64_t first = static_cast<int64_t>(a.seq_lens[blockIdx.x]) - stop + start;
  const int q = min(stop, a.n_tokens) - max(start, 0);
  for (int b = 0; b * 64 < q; ++b) {
    const int i = b * 64 + lane, t = max(start, 0) + i;
    int parent = i < q ? a.parents[t] : -1;
    if (parent >= i || parent < 0) parent = -1;
    const bool fits = b < W;
    uint64_t bits = uint64_t(1) << lane;
    int up = fits && parent >= b * 64 ? parent - b * 64 : -1;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const int from = up < 0 ? lane : up;
      bits |= __shfl(bits, from);
      const int next = __shfl(up, from);
      up = up < 0 ? -1 : next;
    }
    const int top = __shfl(parent, __ffsll(static_cast<unsigned long long>(bits)) - 1);
    const int before = fits && top >= 0 && top < b * 64 ? top : -1;
    int count = fits ? __popcll(bits) : 1;
    if (i < q) {
      for (int w = 0; w < W; ++w) {
        uint64_t x = w == b ? bits : 0;
        if (w < b && before >= 0) x = rows[before * W + w];
        if (w < b) count += __popcll(x);
        a.mask[t * a.mask_token + w] = static_cast<int64_t>(x);
        if (W > 1 && fits) rows[i * W + w] = x;
      }
      if (a.positions) a.positions[t] = first + count - 1;
    }
    __syncthreads();
  }
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_build_draft_tree(const lmc_tensor *parents, const lmc_tensor *query_start_loc,
                                    const lmc_tensor *seq_lens, const lmc_tensor *tree_mask,
                                    const lmc_tensor *positions, void *stream) {
  return guarded([&] {
    const lmc_tensor &p = deref(parents, "parents");
    const lmc_tensor &qs = deref(query_start_loc, "query_start_loc");
    const lmc_tensor &sl = deref(seq_lens, "seq_lens");
    const lmc_tensor &tm = deref(tree_mask, "tree_mask");
    const int dev = tm.device;
    expect(dev >= 0, "tree_mask is not on a GPU");
    check_on(tm, "tree_mask", dev, LMC_I64);
    check_vector(p, "parents", dev, LMC_I32);
    check_vector(qs, "query_start_loc", dev, LMC_I32);
    check_vector(sl, "seq_lens", dev, LMC_I32);
    const int64_t T = p.sizes[0], R = sl.sizes[0];
    expect(qs.sizes[0] == R + 1, "query_start_loc must have one entry per request and one more");
    expect(tm.ndim == 2 && tm.sizes[0] == T, "tree_mask must be [tokens, words]");
    expect(tm.sizes[1] >= 1 && tm.sizes[1] <= kMaxWords, "tree_mask must have 1 to ", kMaxWords, " words a row");
    expect(tm.sizes[1] == 1 || tm.strides[1] == 1, "tree_mask rows must be contiguous");
    expect(T <= 1 || tm.strides[0] >= tm.sizes[1], "tree_mask has overlapping rows");
    expect(T < INT32_MAX - 65536 && R <= INT32_MAX / 4096, "too many tokens or requests");
    DraftArgs a;
    std::memset(&a, 0, sizeof(a));
    if (positions) {
      const lmc_tensor &x = deref(positions, "positions");
      check_vector(x, "positions", dev, LMC_I64);
      expect(x.sizes[0] == T, "positions and parents differ in length");
      expect(!may_share(x, tm), "positions and tree_mask overlap");
      a.positions = static_cast<int64_t *>(x.data);
    }
    for (const lmc_tensor *out : {tree_mask, positions})
      for (const lmc_tensor *in : {parents, query_start_loc, seq_lens})
        expect(!out || !extents_meet(*out, *in), "an output overlaps what it is computed from");
    if (T == 0) return;
    a.parents = static_cast<const int32_t *>(p.data);
    a.starts = static_cast<const int32_t *>(qs.data);
    a.seq_lens = static_cast<const int32_t *>(sl.data);
    a.n_requests = static_cast<int>(R);
    a.n_tokens = static_cast<int>(T);
    a.words = static_cast<int>(tm.sizes[1]);
    a.mask = static_cast<int64_t *>(tm.data);
    a.mask_token = tm.strides[0];
    DeviceGuard guard(dev);
    const int shared = a.words > 1 ? 64 * a.words * a.words * 8 : 0;
    if (shared > 64 * 1024)
      hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(draft_tree), hipFuncAttributeMaxDynamicSharedMemorySize, shared),
                "draft_tree shared memory");
    // (rows behind the last request are few)
    const uint32_t behind = static_cast<uint32_t>(std::min<int64_t>(64, (T + 255) / 256));
    hipLaunchKernelGGL(draft_tree, dim3(static_cast<uint32_t>(R) + behind), dim3(64), shared, static_cast<hipStream_t>(stream), a);
    hip_check(hipGetLastError(), "draft_tree launch");
  });
}
