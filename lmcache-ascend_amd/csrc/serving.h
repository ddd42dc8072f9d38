// Argument checks shared by the serving operators (slot maps, rotary
// positions, shared-prefix attention): tensors of one GPU, and one layer's
// paged K and V caches with every stride taken from the tensors.
#pragma once

#include "kv_geom.h"

#include <functional>
#include <initializer_list>
#include <sstream>

namespace lmc {

// A failed check is LMC_ERR_VALUE; its message is put together only then.
template <typename... Parts> inline void expect(bool ok, const Parts &...parts) {
  if (__builtin_expect(ok, 1)) return;
  std::ostringstream text;
  (text << ... << parts);
  fail(LMC_ERR_VALUE, text.str());
}

// A device tensor of `device` with one of two dtypes.
inline void check_on(const lmc_tensor &t, const char *name, int device, int32_t dtype, int32_t or_dtype = -1) {
  if (t.device < 0 || t.device != device)
    fail(LMC_ERR_VALUE, std::string(name) + " is not on the GPU of the call's other tensors");
  if (t.dtype != dtype && t.dtype != or_dtype) fail(LMC_ERR_VALUE, std::string(name) + " has a dtype the call does not take");
}

// The same, 1-D with adjacent elements.
inline void check_vector(const lmc_tensor &t, const char *name, int device, int32_t dtype, int32_t or_dtype = -1) {
  check_on(t, name, device, dtype, or_dtype);
  if (t.ndim != 1 || (t.sizes[0] > 1 && t.strides[0] != 1))
    fail(LMC_ERR_VALUE, std::string(name) + " must be 1-D and contiguous");
}

// Whether the address ranges of two tensors meet.
inline bool extents_meet(const lmc_tensor &a, const lmc_tensor &b) {
  const int64_t na = extent_bytes(a), nb = extent_bytes(b);
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.data), pb = reinterpret_cast<uintptr_t>(b.data);
  return na > 0 && nb > 0 && pa < pb + nb && pb < pa + na;
}

// A strided layout of bytes: (stride, size) of each dim of more than one
// entry, strides descending, the element's bytes last.
struct Layout {
  std::pair<int64_t, int64_t> dims[LMC_MAX_DIMS + 1];
  int n = 0;
  bool empty = false;
  void dim(int64_t size, int64_t stride) {
    if (size == 0) empty = true;
    if (size > 1) dims[n++] = {stride, size};
  }
  void sort() { std::sort(dims, dims + n, std::greater<>()); }
};

inline Layout layout_of(const lmc_tensor &t) {
  Layout l;
  const int64_t es = elem_size(t);
  for (int i = 0; i < t.ndim; ++i) l.dim(t.sizes[i], t.strides[i] * es);
  l.dim(es, 1);
  l.sort();
  return l;
}

// Whether no byte of a's dims from i on is one of b's from j on, b beginning d
// bytes behind a.  Ranges that do not meet are apart; else, where both step
// by the same outermost stride, each pair of steps whose inner ranges meet has
// to be.  (A stride's two neighbours are the most that can; layouts that cross
// themselves or step differently count as not apart.)
inline bool apart(const Layout &a, const Layout &b, int64_t d, int i = 0, int j = 0) {
  auto extent = [](const Layout &l, int k) {
    int64_t n = 1;
    for (; k < l.n; ++k) n += (l.dims[k].second - 1) * l.dims[k].first;
    return n;
  };
  if (a.empty || b.empty || d >= extent(a, i) || -d >= extent(b, j)) return true;
  if (i == a.n || j == b.n || a.dims[i].first != b.dims[j].first || a.dims[i].first <= 0) return false;
  const int64_t s = a.dims[i].first, wide_a = extent(a, i + 1), wide_b = extent(b, j + 1);
  auto floor_by_s = [s](int64_t x) { return (x >= 0 ? x : x - s + 1) / s; };
  // b's entry n behind a's begins d + s n behind it: in (-wide_b, wide_a).
  const int64_t first = std::max(1 - a.dims[i].second, floor_by_s(-wide_b - d) + 1);
  const int64_t last = std::min(b.dims[j].second - 1, -floor_by_s(d - wide_a) - 1);
  if (last - first > 1) return false;
  for (int64_t n = first; n <= last; ++n)
    if (!apart(a, b, d + s * n, i + 1, j + 1)) return false;
  return true;
}

// Whether two tensors may share an element: column slices of one buffer, and
// rows of theirs in turn, are told apart.
inline bool may_share(const lmc_tensor &a, const lmc_tensor &b) {
  return extents_meet(a, b) &&
         !apart(layout_of(a), layout_of(b), reinterpret_cast<intptr_t>(b.data) - reinterpret_cast<intptr_t>(a.data));
}

// Whether no two elements of a strided layout are the same one: in order of
// stride, each dim steps over all of the dims below it.
inline bool rows_apart(std::initializer_list<int64_t> sizes, std::initializer_list<int64_t> strides) {
  std::pair<int64_t, int64_t> dims[LMC_MAX_DIMS];
  int n = 0;
  const int64_t *stride = strides.begin();
  for (const int64_t size : sizes) {
    if (size == 0) return true;
    if (size > 1) dims[n++] = {*stride, size};
    ++stride;
  }
  std::sort(dims, dims + n);
  int64_t span = 1;
  for (int i = 0; i < n; ++i) {
    if (dims[i].first < span) return false;
    span += dims[i].first * (dims[i].second - 1);
  }
  return true;
}

// One layer's caches: row (page, offset, head) of K is at
// k + page * k_page + offset * k_token + head * k_head (bytes).
struct PagedKv {
  uint8_t *k, *v;
  int64_t k_page, k_token, k_head;
  int64_t v_page, v_token, v_head;
  int64_t pages;
  int64_t block_size;
  int64_t heads, dim;
  int32_t dtype;
  int device;
};

// Whether no row of K is one of V's: the caches one behind the other, pages
// that hold K's part and V's beside each other, or rows dealt in turn.
inline bool k_and_v_apart(const PagedKv &g) {
  Layout k, v;
  auto add = [&](int64_t size, int64_t k_stride, int64_t v_stride) {
    k.dim(size, k_stride);
    v.dim(size, v_stride);
  };
  add(g.pages, g.k_page, g.v_page);
  add(g.block_size, g.k_token, g.v_token);
  add(g.heads, g.k_head, g.v_head);
  add(g.dim * dtype_size(g.dtype), 1, 1);
  k.sort();
  v.sort();
  return apart(k, v, g.v - g.k);
}

inline PagedKv paged_kv(const lmc_tensor *caches, int n, int fmt, bool two_major, const char *op) {
  validate_vllm_caches(caches, n, fmt);
  if (fmt != LMC_FMT_MERGED_KV && fmt != LMC_FMT_SEPARATE_KV)
    fail(LMC_ERR_VALUE, std::string(op) + " takes MERGED_KV or SEPARATE_KV caches");
  const lmc_tensor &k = deref(&caches[0], "vllm_kv_caches[0]");
  PagedKv g;
  g.dtype = k.dtype;
  g.device = k.device;
  expect(k.device >= 0, op, ": the paged caches are not on a GPU");
  const int64_t es = elem_size(k);
  g.k = static_cast<uint8_t *>(k.data);
  if (fmt == LMC_FMT_MERGED_KV) {
    // [2, pages, block, heads, dim] (two-major) or [pages, 2, block, heads, dim].
    expect(k.ndim == 5 && size(k, two_major ? 0 : 1) == 2, "a MERGED_KV cache is 5-D with K and V along its ",
           two_major ? "first" : "second", " dim");
    g.pages = size(k, two_major ? 1 : 0);
    g.k_page = g.v_page = stride(k, two_major ? 1 : 0) * es;
    g.v = g.k + stride(k, two_major ? 0 : 1) * es;
    g.v_token = stride(k, 2) * es;
    g.v_head = stride(k, 3) * es;
    expect(size(k, 4) <= 1 || stride(k, 4) == 1, "a cache row's head dims must be adjacent");
  } else {
    const lmc_tensor &v = deref(&caches[1], "vllm_kv_caches[1]");
    expect(k.ndim == 4, "SEPARATE_KV caches are [pages, block, heads, dim]");
    expect(v.device == k.device && v.dtype == k.dtype, "K and V caches differ in device or dtype");
    g.pages = size(k, 0);
    g.k_page = stride(k, 0) * es;
    g.v_page = stride(v, 0) * es;
    g.v = static_cast<uint8_t *>(v.data);
    g.v_token = stride(v, 1) * es;
    g.v_head = stride(v, 2) * es;
    expect(size(v, 3) <= 1 || stride(v, 3) == 1, "a cache row's head dims must be adjacent");
    expect(size(k, 3) <= 1 || stride(k, 3) == 1, "a cache row's head dims must be adjacent");
    for (int i = 0; i < v.ndim; ++i) expect(v.strides[i] >= 0, "negative strides unsupported");
  }
  g.block_size = size(k, -3);
  g.heads = size(k, -2);
  g.dim = size(k, -1);
  g.k_token = stride(k, -3) * es;
  g.k_head = stride(k, -2) * es;
  for (int i = 0; i < k.ndim; ++i) expect(k.strides[i] >= 0, "negative strides unsupported");
  expect(g.block_size > 0 && g.heads > 0 && g.dim > 0, "the paged caches hold no rows");
  // Page numbers and slots are split in 32 bits.
  expect(g.pages <= INT32_MAX && g.block_size <= INT32_MAX && g.pages * g.block_size <= static_cast<int64_t>(UINT32_MAX),
              "paged caches of more than 2^32 slots are not supported");
  return g;
}

} // namespace lmc
