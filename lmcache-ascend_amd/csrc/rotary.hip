// Rotary positions of queries and keys on MI355X (gfx950), forward and
// inverse, with the option of writing the rotated keys and the values to
// their paged caches.
//
//   (z1, z2) = (x1 c - x2 s, x2 c + x1 s),  (c, s) = scale * (cos, sin)(pos * inv_freq[i])
//
// for the pairs of dims [offset, offset + 2 n_freq) of each head (halves or
// interleaved); the other dims pass through.  The inverse takes -s: the
// transpose, which is the gradient of the rotation.
//
// No table: a table's row is as long as a key head and there are as many
// rows as the longest context has positions, while the angle costs a few
// 64-bit operations.  pos * inv_freq / 2 pi is formed in 64 bits and reduced
// to an eighth of a turn there, so far positions lose nothing, and cos and
// sin are polynomials of that rest in 32 bits (1.3e-7 relative).  A
// workgroup computes the pairs of its tokens once and all heads read them
// from LDS.  The key and value elements are widened to 32 bits, rotated, and
// rounded once.
//
// HBM-bound: each element is read and written once.  A lane moves VP pairs
// (two 16-byte accesses each way where the layout allows); 16384 tokens of 32
// query and 8 KV heads of 128 bf16 dims to their pages take 71 us, 5.6 TB/s.
// 64 tokens of 32 + 8 heads: 4 us, the call itself (2.8 in a graph).
#include "rope_math.h"
#include "serving.h"

#include <cmath>

namespace lmc {

namespace {

// cos and sin of 2 pi r for |r| <= 1/8, least-maximum fits in r * r (own
// fits: 5e-12 and 6e-11 before rounding).
__device__ __forceinline__ void sincos_eighth(float r, float &s, float &c) {
  const float u = r * r;
  s = r * (6.28318531f + u * (-41.3417022f + u * (81.6052047f + u * (-76.6978700f + u * 41.4729485f))));
  c = 1.0f + u * (-19.7392082f + u * (64.9393082f + u * (-85.4422989f + u * 59.2027969f)));
}

__device__ __forceinline__ void sincos_turn(int64_t pos, double inv_freq, float &s, float &c) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  const double t = static_cast<double>(pos) * (inv_freq * kInvTwoPi);
  const double part = t - rint(t);                       // [-1/2, 1/2]
  const double quarter = rint(part * 4.0);
  const float r = static_cast<float>(part - quarter * 0.25);
  float ps, pc;
  sincos_eighth(r, ps, pc);
  const int q = static_cast<int>(quarter) & 3;
  s = (q & 1) ? pc : ps;
  c = (q & 1) ? ps : pc;
  if (q & 2) s = -s;
  if (q == 1 || q == 2) c = -c;
}

// Rows of one tensor: heads of a token, and where they go.  Strides in elements.
struct Rows {
  const void *in;
  void *out;
  int64_t in_token, in_head, out_token, out_head;
  uint32_t units;   // per token
  uint32_t magic;   // ceil(2^32 / units per head): a division
  uint32_t per_head;
  int paged;        // out is a cache: rows at the token's slot
  uint32_t first_block, blocks;  // workgroups (y) that take these rows
};

struct RotaryArgs {
  const void *positions;
  int pos_i32;
  const double *inv_freq;
  int half, offset;
  float scale;
  int inverse;
  int64_t n_tokens;
  int tokens_per_block;
  uint32_t units;   // per token, all three
  Rows q, k, v;
  const int64_t *slots;
  int slots_i32;
  uint32_t block_size;
  int64_t num_slots;
  int64_t k_page, k_slot, v_page, v_slot;  // elements
};

constexpr int kThreads = 256;
constexpr int kMaxTokens = 2;  // per workgroup

// Rounded to the type once (by the conversion instructions).
template <typename KD> __device__ __forceinline__ typename KD::S rounded(float x);
template <> __device__ __forceinline__ uint16_t rounded<BF16>(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
template <> __device__ __forceinline__ uint16_t rounded<F16>(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
template <> __device__ __forceinline__ float rounded<F32>(float x) { return x; }

// VP pairs: a and b are their first and second halves, or 2 VP elements of
// interleaved pairs in order.
template <typename KD, bool NEOX, int VP>
__device__ __forceinline__ void turn(typename VecOf<VP * sizeof(typename KD::S)>::T &a,
                                     typename VecOf<VP * sizeof(typename KD::S)>::T &b, const float *c, const float *s) {
  using S = typename KD::S;
  using V = typename VecOf<VP * sizeof(S)>::T;
  using P = Pack<S, VP>;
  S in[2 * VP], out[2 * VP];
  P u = __builtin_bit_cast(P, a), v = __builtin_bit_cast(P, b);
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    in[i] = u.v[i];
    in[VP + i] = v.v[i];
  }
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    const int i1 = NEOX ? i : 2 * i, i2 = NEOX ? VP + i : 2 * i + 1;
    const float x1 = to_f32<KD>(in[i1]), x2 = to_f32<KD>(in[i2]);
    out[i1] = rounded<KD>(x1 * c[i] - x2 * s[i]);
    out[i2] = rounded<KD>(x2 * c[i] + x1 * s[i]);
  }
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    u.v[i] = out[i];
    v.v[i] = out[VP + i];
  }
  a = __builtin_bit_cast(V, u);
  b = __builtin_bit_cast(V, v);
}

// The units of one tensor's rows of this workgroup's tokens: TURN rotates the
// first of each head and copies the others, else all are copied.
template <typename KD, bool NEOX, int VP, bool STREAM, bool TURN>
__device__ __forceinline__ void rows_of(const RotaryArgs &a, const Rows &rows, int64_t t0, int nt, const float *cosv,
                                        const float *sinv, const int64_t *paged_row) {
  using S = typename KD::S;
  using V = typename VecOf<VP * sizeof(S)>::T;
  auto store = [&](S *to, V v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<V *>(to));
    else *reinterpret_cast<V *>(to) = v;
  };
  const uint32_t total = nt * rows.units, step = kThreads * rows.blocks, turned = TURN ? a.half / VP : 0;
  uint32_t x = (blockIdx.y - rows.first_block) * kThreads + threadIdx.x;
  if (x >= total) return;
  uint32_t t = x / rows.units, w = x - t * rows.units;
  for (; x < total; x += step) {
    const uint32_t h = rows.per_head == 1 ? w : __umulhi(w, rows.magic), u = w - h * rows.per_head;
    const int64_t at = rows.paged ? paged_row[t] : (t0 + t) * rows.out_token;
    const S *in = static_cast<const S *>(rows.in) + (t0 + t) * rows.in_token + h * rows.in_head;
    if (at >= 0) {
      S *out = static_cast<S *>(rows.out) + at + h * rows.out_head;
      if (u < turned) {
        const uint32_t i0 = u * VP;
        const uint32_t e1 = a.offset + (NEOX ? i0 : 2 * i0), e2 = e1 + (NEOX ? a.half : VP);
        V p = *reinterpret_cast<const V *>(in + e1), q = *reinterpret_cast<const V *>(in + e2);
        turn<KD, NEOX, VP>(p, q, cosv + t * a.half + i0, sinv + t * a.half + i0);
        store(out + e1, p);
        store(out + e2, q);
      } else {
        uint32_t e = (u - turned) * VP;
        if (TURN && e >= static_cast<uint32_t>(a.offset)) e += 2 * a.half;
        store(out + e, *reinterpret_cast<const V *>(in + e));
      }
    }
    w += step;
    while (w >= rows.units) {
      w -= rows.units;
      ++t;
    }
  }
}

template <typename KD, bool NEOX, int VP, bool STREAM>
__global__ void __launch_bounds__(kThreads) rotary_rows(RotaryArgs a) {
  extern __shared__ float cs[];  // cos [tokens][half], then sin
  __shared__ int64_t row_k[kMaxTokens], row_v[kMaxTokens];
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.n_tokens - t0));
  float *cosv = cs, *sinv = cs + a.tokens_per_block * a.half;
  for (int i = tid; i < nt * a.half; i += kThreads) {
    const int t = i / a.half, j = i - t * a.half;
    const int64_t pos = a.pos_i32 ? static_cast<const int32_t *>(a.positions)[t0 + t]
                                  : static_cast<const int64_t *>(a.positions)[t0 + t];
    float s, c;
    sincos_turn(pos, a.inv_freq[j], s, c);
    cosv[i] = c * a.scale;
    sinv[i] = (a.inverse ? -s : s) * a.scale;
  }
  if (a.slots && tid < nt) {
    const int64_t slot = a.slots_i32 ? reinterpret_cast<const int32_t *>(a.slots)[t0 + tid] : a.slots[t0 + tid];
    int64_t rk = -1, rv = -1;
    if (slot >= 0 && slot < a.num_slots) {
      const uint32_t x = static_cast<uint32_t>(slot), page = x / a.block_size, at = x - page * a.block_size;
      rk = page * a.k_page + at * a.k_slot;
      rv = page * a.v_page + at * a.v_slot;
    }
    row_k[tid] = rk;
    row_v[tid] = rv;
  }
  __syncthreads();
  // One tensor, or all of them where a workgroup has the tokens to itself.
  auto mine = [&](const Rows &rows) { return blockIdx.y - rows.first_block < rows.blocks; };
  if (mine(a.q)) rows_of<KD, NEOX, VP, STREAM, true>(a, a.q, t0, nt, cosv, sinv, nullptr);
  if (mine(a.k)) rows_of<KD, NEOX, VP, STREAM, true>(a, a.k, t0, nt, cosv, sinv, row_k);
  if (mine(a.v)) rows_of<KD, NEOX, VP, STREAM, false>(a, a.v, t0, nt, nullptr, nullptr, row_v);
}

template <typename KD, bool NEOX, int VP> void launch(RotaryArgs a, hipStream_t s) {
  const int64_t blocks = (a.n_tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  // Few tokens: a unit a lane, spread over workgroups, and the tensors apart
  // (a decode step is latency).  Many: all of a token's rows in one.
  uint32_t y = 0;
  for (Rows *r : {&a.q, &a.k, &a.v}) {
    const int64_t units = static_cast<int64_t>(a.tokens_per_block) * r->units;
    r->first_block = blocks >= 1024 ? 0 : y;
    r->blocks = static_cast<uint32_t>(blocks >= 1024 ? units > 0 : std::min<int64_t>((units + kThreads - 1) / kThreads, 1024 / blocks));
    y = std::max(y, r->first_block + r->blocks);
  }
  const size_t shared = static_cast<size_t>(a.tokens_per_block) * a.half * 2 * sizeof(float);
  // Streaming stores past 8 MiB: 8192 tokens of 40 heads take 28 us with them
  // and 38 without, a decode step's 48 tokens to their pages 4.6 and 3.4.
  const bool stream = a.n_tokens * a.units * VP * static_cast<int64_t>(sizeof(typename KD::S)) >= (int64_t(8) << 20);
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(y));
  if (stream) hipLaunchKernelGGL((rotary_rows<KD, NEOX, VP, true>), grid, dim3(kThreads), shared, s, a);
  else hipLaunchKernelGGL((rotary_rows<KD, NEOX, VP, false>), grid, dim3(kThreads), shared, s, a);
  hip_check(hipGetLastError(), "rotary_rows launch");
}

template <typename KD, bool NEOX> void launch_vp(const RotaryArgs &a, int vp, hipStream_t s) {
  switch (vp) {
  case 8:
    if constexpr (sizeof(typename KD::S) == 2) launch<KD, NEOX, 8>(a, s);
    break;
  case 4: launch<KD, NEOX, 4>(a, s); break;
  case 2: launch<KD, NEOX, 2>(a, s); break;
  default: launch<KD, NEOX, 1>(a, s); break;
  }
}

template <typename KD> void launch_style(const RotaryArgs &a, bool neox, int vp, hipStream_t s) {
  neox ? launch_vp<KD, true>(a, vp, s) : launch_vp<KD, false>(a, vp, s);
}

// One tensor's token and head strides: [T, heads * D] or [T, heads, D].
struct HeadView {
  const lmc_tensor *t = nullptr;
  int64_t token = 0, head = 0, heads = 0;
};

HeadView head_view(const lmc_tensor &t, const char *name, int64_t dim, int device, int32_t dtype) {
  check_on(t, name, device, dtype);
  HeadView v;
  v.t = &t;
  expect(t.ndim == 2 || t.ndim == 3, name, " must be [tokens, heads * head_size] or [tokens, heads, head_size]");
  for (int i = 0; i < t.ndim; ++i) expect(t.strides[i] >= 0, name, ": negative strides unsupported");
  expect(size(t, -1) <= 1 || stride(t, -1) == 1, name, ": a head's dims must be adjacent");
  v.token = t.strides[0];
  if (t.ndim == 2) {
    expect(t.sizes[1] % dim == 0, name, " width is not a multiple of head_size");
    v.heads = t.sizes[1] / dim;
    v.head = dim;
  } else {
    expect(t.sizes[2] == dim, name, " heads are not of head_size");
    v.heads = t.sizes[1];
    v.head = t.strides[1];
  }
  return v;
}

bool same_rows(const HeadView &a, const HeadView &b) {
  return a.t->data == b.t->data && a.heads == b.heads && (a.t->sizes[0] <= 1 || a.token == b.token) &&
         (a.heads <= 1 || a.head == b.head);
}

void rotary(const lmc_tensor *positions, const lmc_tensor *query, const lmc_tensor *key, const lmc_tensor *value,
            const lmc_tensor *caches, int n_caches, int fmt, bool two_major, const lmc_tensor *slot_mapping,
            int64_t head_size, const double *inv_freq, int64_t n_freq, double scale, bool neox, int64_t offset,
            bool inverse, const lmc_tensor *query_out, const lmc_tensor *key_out, bool paged, hipStream_t stream) {
  expect(query || key, "neither query nor key is given");
  const lmc_tensor &lead = deref(query ? query : key, query ? "query" : "key");
  const int dev = lead.device;
  expect(dev >= 0, "query and key must be on a GPU");
  if (lead.dtype != LMC_BF16 && lead.dtype != LMC_F16 && lead.dtype != LMC_F32)
    fail(LMC_ERR_VALUE, "rotary positions take bfloat16, float16 or float32 queries and keys only");
  expect(head_size > 0 && head_size <= 8192, "head_size must be between 1 and 8192");
  expect(inv_freq != nullptr && n_freq > 0, "inv_freq is empty");
  expect(offset >= 0 && n_freq <= head_size / 2 && offset <= head_size - 2 * n_freq,
              "the rotated dims [rotary_offset, rotary_offset + 2 * len(inv_freq)) do not lie in a head");
  expect(std::isfinite(static_cast<float>(scale)), "scale must be finite in 32 bits");
  const int64_t T = size(lead, 0), rot = 2 * n_freq, es = elem_size(lead);
  const lmc_tensor &pos = deref(positions, "positions");
  check_vector(pos, "positions", dev, LMC_I64, LMC_I32);
  expect(pos.sizes[0] == T, "positions must have one entry per token");

  RotaryArgs a;
  std::memset(&a, 0, sizeof(a));
  int64_t grain = 16;  // bytes every address and length is a multiple of
  auto need = [&](int64_t bytes) {
    while (bytes % grain) grain /= 2;
  };
  HeadView views[5];
  bool written[5];
  int n_views = 0;
  auto add = [&](Rows &rows, const lmc_tensor *in_t, const lmc_tensor *out_t, const char *name, const char *out_name,
                 int64_t dim, bool turn) {
    const HeadView in = head_view(deref(in_t, name), name, dim, dev, lead.dtype);
    expect(in.t->sizes[0] == T, name, " has another number of tokens than the call's other tensors");
    expect(in.heads * dim <= INT32_MAX / 4, name, " rows are too wide");
    const int at = n_views++;
    views[at] = in;
    written[at] = false;
    HeadView out = in;
    bool moved = paged && rows.paged;
    if (!moved && out_t) {
      out = head_view(deref(out_t, out_name), out_name, dim, dev, lead.dtype);
      expect(out.t->sizes[0] == T && out.heads == in.heads, out_name, " differs in shape from ", name);
      moved = !same_rows(in, out);
      if (moved) {
        views[n_views] = out;
        written[n_views++] = true;
      }
    }
    if (!moved) written[at] = true;
    if (!rows.paged)
      expect(rows_apart({T, out.heads, dim}, {out.token, out.head, 1}),
                  (moved ? out_name : name), " has overlapping rows");
    rows.in = in.t->data;
    rows.in_token = in.token;
    rows.in_head = in.head;
    need(reinterpret_cast<uintptr_t>(in.t->data));
    need(in.token * es);
    need(in.head * es);
    if (!rows.paged) {
      rows.out = out.t->data;
      rows.out_token = out.token;
      rows.out_head = out.head;
      need(reinterpret_cast<uintptr_t>(out.t->data));
      need(out.token * es);
      need(out.head * es);
    }
    need(dim * es);
    rows.per_head = static_cast<uint32_t>(!turn ? dim : moved ? n_freq + dim - rot : n_freq);  // elements or pairs
    rows.units = static_cast<uint32_t>(in.heads);                                              // heads, for now
    return in;
  };
  a.k.paged = a.v.paged = paged;
  if (query) add(a.q, query, query_out, "query", "query_out", head_size, true);
  else expect(!query_out, "query_out without query");
  PagedKv kv;
  if (paged) {
    kv = paged_kv(caches, n_caches, fmt, two_major, "rotary_embedding_to_paged");
    expect(kv.device == dev && kv.dtype == lead.dtype, "the paged caches differ in device or dtype from the rows");
    expect(rows_apart({kv.pages, kv.block_size, kv.heads, kv.dim * es}, {kv.k_page, kv.k_token, kv.k_head, 1}) &&
                    rows_apart({kv.pages, kv.block_size, kv.heads, kv.dim * es}, {kv.v_page, kv.v_token, kv.v_head, 1}),
                "the paged caches have overlapping rows");
    expect(k_and_v_apart(kv), "the K and V caches overlap");
    expect(kv.dim == head_size, "the paged caches' heads are not of head_size");
    const HeadView k = add(a.k, key, nullptr, "key", "", head_size, true);
    const HeadView v = add(a.v, value, nullptr, "value", "", head_size, false);
    expect(k.heads == kv.heads && v.heads == kv.heads, "the paged caches have another number of heads than key and value");
    for (int i = 0; i < n_views; ++i)
      for (int c = 0; c < n_caches; ++c)
        expect(!extents_meet(*views[i].t, caches[c]), "the paged caches overlap the call's rows");
    const lmc_tensor &sm = deref(slot_mapping, "slot_mapping");
    check_vector(sm, "slot_mapping", dev, LMC_I64, LMC_I32);
    expect(sm.sizes[0] == T, "slot_mapping must have one entry per token");
    a.slots = static_cast<const int64_t *>(sm.data);
    a.slots_i32 = sm.dtype == LMC_I32;
    a.block_size = static_cast<uint32_t>(kv.block_size);
    a.num_slots = kv.pages * kv.block_size;
    a.k.out = kv.k;
    a.v.out = kv.v;
    a.k.out_head = kv.k_head / es;
    a.v.out_head = kv.v_head / es;
    a.k_page = kv.k_page / es;
    a.k_slot = kv.k_token / es;
    a.v_page = kv.v_page / es;
    a.v_slot = kv.v_token / es;
    for (int64_t b : {static_cast<int64_t>(reinterpret_cast<uintptr_t>(kv.k)), static_cast<int64_t>(reinterpret_cast<uintptr_t>(kv.v)),
                      kv.k_page, kv.k_token, kv.k_head, kv.v_page, kv.v_token, kv.v_head})
      need(b);
  } else {
    if (key) add(a.k, key, key_out, "key", "key_out", head_size, true);
    else expect(!key_out, "key_out without key");
  }
  // What is written must not be read by another lane.
  for (int i = 0; i < n_views; ++i)
    for (int j = 0; j < i; ++j)
      expect(!(written[i] || written[j]) || !may_share(*views[i].t, *views[j].t), "two of query, key, value and the outputs overlap");
  // Nor may a workgroup write what others take their angles and slots from.
  lmc_tensor freq = pos;  // n_freq doubles: as wide as I64
  freq.data = const_cast<double *>(inv_freq);
  freq.dtype = LMC_I64;
  freq.sizes[0] = n_freq;
  freq.strides[0] = 1;
  for (const lmc_tensor *in : {positions, paged ? slot_mapping : positions, static_cast<const lmc_tensor *>(&freq)}) {
    for (int i = 0; i < n_views; ++i)
      expect(!written[i] || !extents_meet(*views[i].t, *in), "positions, slot_mapping or inv_freq overlap what the call writes");
    for (int c = 0; c < n_caches; ++c)
      expect(!extents_meet(caches[c], *in), "positions, slot_mapping or inv_freq overlap the paged caches");
  }
  if (T == 0) return;
  need(n_freq * es);
  need(offset * es);
  const int vp = static_cast<int>(std::max<int64_t>(1, grain / es));
  uint32_t units = 0;
  for (Rows *r : {&a.q, &a.k, &a.v}) {
    if (r->units == 0) continue;
    r->per_head /= vp;
    r->magic = static_cast<uint32_t>(((uint64_t(1) << 32) + r->per_head - 1) / r->per_head);
    expect(static_cast<uint64_t>(r->units) * r->per_head * r->per_head < (uint64_t(1) << 32), "rows are too wide");
    r->units *= r->per_head;
    units += r->units;
  }
  if (units == 0) return;
  a.units = units;
  a.positions = pos.data;
  a.pos_i32 = pos.dtype == LMC_I32;
  a.inv_freq = inv_freq;
  a.half = static_cast<int>(n_freq);
  a.offset = static_cast<int>(offset);
  a.scale = static_cast<float>(scale);
  a.inverse = inverse;
  a.n_tokens = T;
  // Two tokens share a workgroup once there are workgroups enough (their
  // angles then fill its lanes): 16384 tokens of 32 + 8 + 8 heads to their
  // pages take 73 us with two, 74 with one, 79 with four and 93 with eight.
  const int tb = T >= 2048 ? kMaxTokens : 1;
  a.tokens_per_block = tb;
  // A launch has less than 2^32 threads along a dimension.
  expect((T + tb - 1) / tb <= UINT32_MAX / kThreads, "too many tokens");
  expect(static_cast<int64_t>(tb) * units <= INT32_MAX, "rows are too wide");
  DeviceGuard guard(dev);
  switch (lead.dtype) {
  case LMC_BF16: launch_style<BF16>(a, neox, vp, stream); break;
  case LMC_F16: launch_style<F16>(a, neox, vp, stream); break;
  default: launch_style<F32>(a, neox, vp, stream); break;
  }
}

} // namespace

} // namespace lmc

using namespace lmc;

extern "C" int lmc_rotary_embedding(const lmc_tensor *positions, const lmc_tensor *query, const lmc_tensor *key,
                                    int64_t head_size, const double *inv_freq, int64_t n_freq, double scale,
                                    int32_t is_neox, int64_t rotary_offset, int32_t inverse,
                                    const lmc_tensor *query_out, const lmc_tensor *key_out, void *stream) {
  return guarded([&] {
    rotary(positions, query, key, nullptr, nullptr, 0, 0, false, nullptr, head_size, inv_freq, n_freq, scale,
           is_neox != 0, rotary_offset, inverse != 0, query_out, key_out, false, static_cast<hipStream_t>(stream));
  });
}

extern "C" int lmc_rotary_embedding_to_paged(const lmc_tensor *positions, const lmc_tensor *query,
                                             const lmc_tensor *key, const lmc_tensor *value,
                                             const lmc_tensor *vllm_kv_caches, int32_t n_caches,
                                             const lmc_tensor *slot_mapping, int64_t head_size, const double *inv_freq,
                                             int64_t n_freq, double scale, int32_t is_neox, int64_t rotary_offset,
                                             const lmc_tensor *query_out, int32_t kvcache_format,
                                             int32_t vllm_two_major, void *stream) {
  return guarded([&] {
    rotary(positions, query, key, value, vllm_kv_caches, n_caches, kvcache_format, vllm_two_major != 0, slot_mapping,
           head_size, inv_freq, n_freq, scale, is_neox != 0, rotary_offset, false, query_out, nullptr, true,
           static_cast<hipStream_t>(stream));
  });
}
