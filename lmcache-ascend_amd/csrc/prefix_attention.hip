// Attention of a batch whose requests share a prefix, over paged K and V
// caches, on MI355X (gfx950).
//
//   o(t, h)   = sum_j softmax_j(scale q(t, h) . k(j)) v(j)
//   lse(t, h) = log sum_j exp(scale q(t, h) . k(j))
//
// over the keys j of token t's request up to the token's own position.  Keys
// before shared_len lie in the blocks of one list for the whole batch, the
// others in the request's row of the block table.
#include "rope_math.h"
#include "serving.h"

#include <cmath>

namespace lmc {

namespace {

struct AttnArgs {
  const void *q;
  int64_t q_token, q_head;  // elements
  void *o;
  int64_t o_token, o_head;
  float *lse;               // may be null
  int64_t lse_token, lse_head;
  PagedKv kv;
  const int32_t *shared;
  int64_t shared_len;
  const int32_t *table;
  int64_t table_stride;
  int64_t width;
  const int32_t *seq_lens, *starts;
  int n_requests;
  int64_t n_tokens;
  int heads, group;
  float scale;
};

// One wave per (token, query head): 64 keys a step, a lane a key for the
// scores and a lane a dim for the sums.
template <typename T> __global__ void __launch_bounds__(64) attend_rows(AttnArgs a) {
  using S = typename T::S;
  const int lane = threadIdx.x, h = blockIdx.y;
  const int64_t t = blockIdx.x;
  int r = 0;
  while (r < a.n_requests && !(t >= a.starts[r] && t < a.starts[r + 1])) ++r;
  if (r == a.n_requests) return;
  const int64_t keys = static_cast<int64_t>(a.seq_lens[r]) - a.starts[r + 1] + t + 1;
  const int D = static_cast<int>(a.kv.dim);
  const S *q = static_cast<const S *>(a.q) + t * a.q_token + h * a.q_head;
  const int64_t kh = h / a.group;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  auto page_of = [&](int64_t j) -> int64_t {
    const int64_t b = j / a.kv.block_size;
    if (j >= a.shared_len && b >= a.width) return -1;
    const int64_t p = j < a.shared_len ? a.shared[b] : a.table[r * a.table_stride + b];
    return p >= 0 && p < a.kv.pages ? p : -1;
  };
  for (int64_t j0 = 0; j0 < keys; j0 += 64) {
    const int64_t j = j0 + lane;
    const int64_t page = j < keys ? page_of(j) : -1, at = j % a.kv.block_size;
    float s = -INFINITY;
    if (page >= 0) {
      const S *k = reinterpret_cast<const S *>(a.kv.k + page * a.kv.k_page + at * a.kv.k_token + kh * a.kv.k_head);
      float x = 0.f;
      for (int d = 0; d < D; ++d) x += to_f32<T>(q[d]) * to_f32<T>(k[d]);
      s = x * a.scale;
    }
    float top = s;
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float m2 = fmaxf(m, top);
    const float base = m2 == -INFINITY ? 0.f : m2;
    const float p = page >= 0 ? expf(s - base) : 0.f;
    const float f = expf(m - base);
    float sum = p;
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    l = l * f + sum;
    m = m2;
    for (int c = 0; c < 4; ++c) o[c] *= f;
    for (int i = 0; i < 64; ++i) {
      const float pi = __shfl(p, i);
      const int64_t pg = __shfl(page, i);
      if (pg < 0) continue;
      const int64_t ai = (j0 + i) % a.kv.block_size;
      const S *v = reinterpret_cast<const S *>(a.kv.v + pg * a.kv.v_page + ai * a.kv.v_token + kh * a.kv.v_head);
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) o[c] += pi * to_f32<T>(v[lane + 64 * c]);
    }
  }
  S *out = static_cast<S *>(a.o) + t * a.o_token + h * a.o_head;
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < D) out[lane + 64 * c] = from_f32<T>(l == 0.f ? 0.f : o[c] / l);
  if (a.lse && lane == 0) a.lse[t * a.lse_token + h * a.lse_head] = m + logf(l);
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_shared_prefix_attention(const lmc_tensor *query, const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                                           const lmc_tensor *shared_blocks, int64_t shared_len,
                                           const lmc_tensor *block_table, const lmc_tensor *seq_lens,
                                           const lmc_tensor *query_start_loc, double scale, const lmc_tensor *output,
                                           const lmc_tensor *lse, int32_t kvcache_format, int32_t vllm_two_major,
                                           void *stream) {
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
    check_value(kv.dim == 64 || kv.dim == 96 || kv.dim == 128 || kv.dim == 192 || kv.dim == 256,
                "shared_prefix_attention takes heads of 64, 96, 128, 192 or 256 dims");
    check_value(q.ndim == 3 && o.ndim == 3, "query and output must be [tokens, heads, dim]");
    const int64_t T = q.sizes[0], R = sl.sizes[0], Hq = q.sizes[1];
    for (int i = 0; i < 3; ++i) {
      check_value(q.sizes[i] == o.sizes[i], "query and output differ in shape");
      check_value(q.strides[i] >= 0 && o.strides[i] >= 0, "negative strides unsupported");
    }
    check_value(q.sizes[2] == kv.dim, "query heads are not of the caches' dim");
    check_value(q.strides[2] == 1 && o.strides[2] == 1, "a head's dims must be adjacent");
    check_value(Hq % kv.heads == 0, "query heads are not a multiple of the caches' heads");
    check_value(qs.sizes[0] == R + 1, "query_start_loc must have one entry per request and one more");
    check_value(bt.ndim == 2 && bt.sizes[0] == R, "block_table must be [requests, pages]");
    check_value(bt.sizes[1] <= 1 || bt.strides[1] == 1, "block_table rows must be contiguous");
    check_value(shared_len >= 0 && shared_len <= INT32_MAX, "shared_len must be between 0 and 2^31 - 1");
    check_value((shared_len + kv.block_size - 1) / kv.block_size <= sb.sizes[0], "shared_blocks has too few blocks for shared_len");
    check_value(scale > 0 && std::isfinite(scale), "scale must be positive and finite");
    AttnArgs a;
    std::memset(&a, 0, sizeof(a));
    if (lse) {
      const lmc_tensor &e = deref(lse, "lse");
      check_on(e, "lse", dev, LMC_F32);
      check_value(e.ndim == 2 && e.sizes[0] == T && e.sizes[1] == Hq, "lse must be [tokens, heads]");
      a.lse = static_cast<float *>(e.data);
      a.lse_token = e.strides[0];
      a.lse_head = e.strides[1];
    }
    if (T == 0 || Hq == 0 || R == 0) return;
    a.q = q.data;
    a.q_token = q.strides[0];
    a.q_head = q.strides[1];
    a.o = o.data;
    a.o_token = o.strides[0];
    a.o_head = o.strides[1];
    a.kv = kv;
    a.shared = static_cast<const int32_t *>(sb.data);
    a.shared_len = shared_len;
    a.table = static_cast<const int32_t *>(bt.data);
    a.table_stride = bt.strides[0];
    a.width = bt.sizes[1];
    a.seq_lens = static_cast<const int32_t *>(sl.data);
    a.starts = static_cast<const int32_t *>(qs.data);
    a.n_requests = static_cast<int>(R);
    a.n_tokens = T;
    a.heads = static_cast<int>(Hq);
    a.group = static_cast<int>(Hq / kv.heads);
    a.scale = static_cast<float>(scale);
    DeviceGuard guard(dev);
    const dim3 grid(static_cast<uint32_t>(T), static_cast<uint32_t>(Hq));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (kv.dtype == LMC_BF16) hipLaunchKernelGGL(attend_rows<BF16>, grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL(attend_rows<F16>, grid, dim3(64), 0, s, a);
    hip_check(hipGetLastError(), "attend_rows launch");
  });
}
