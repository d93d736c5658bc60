// What the kernels of the 8-bit paged cache share: the pool's layout and a step's rows.
#pragma once

#include "common.cuh"

namespace gptoss {
namespace kv8 {

constexpr int kPage = GPTOSS_KV8_PAGE;
constexpr int kMaxTokens = 1 << 30; // rows of a call and tokens of a sequence: sums of two fit an int

// One layer of a pool.
struct Layer {
  int8_t *codes;
  float *scales;
  int n_pages, n_kv_heads;
  // Codes / scales of (page, head): D-wide rows, 64 for the keys, then 64 for the values.
  template <int D> __device__ __forceinline__ int8_t *block(int page, int head) const {
    return codes + ((size_t)page * n_kv_heads + head) * (2 * kPage * D);
  }
  __device__ __forceinline__ float *scale(int page, int head) const {
    return scales + ((size_t)page * n_kv_heads + head) * 2;
  }
  // A table entry that names no page of the pool reads as -1.
  __device__ __forceinline__ int checked(int page) const { return (unsigned)page < (unsigned)n_pages ? page : -1; }
};

// The rows of a step, sequence after sequence.
struct Rows {
  const int *row_start, *kv_len, *pages;
  int T, n_seqs, pages_stride, max_new;
  __device__ __forceinline__ int start(int s) const { return min(max(__ldg(row_start + s), 0), T); }
  struct Span {
    int row, q;  // first row, rows that are processed
    int pos;     // position of the first row (negative where kv_len is less than the rows)
  };
  __device__ __forceinline__ Span span(int s) const {
    const int r0 = start(s), n = max(start(s + 1) - r0, 0);
    return Span{r0, min(n, max_new), min(max(__ldg(kv_len + s), 0), kMaxTokens) - n};
  }
  // The last sequence s with first(s) <= u, where first(s) never falls as s grows and first(0) <= u.  By whole
  // warps, 32 places looked at per round: a search by halves is a chain of loads eight long at 200 sequences.
  template <typename F> __device__ __forceinline__ int find(int u, F first) const {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seqs;
    while (n > 1) {
      const int step = (n + 31) / 32, at = min(lane * step, n - 1);
      const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && first(lo + at) <= u);
      const int k = 31 - __clz(below | 1u);
      lo += k * step;
      n = min(step, n - k * step);
    }
    return lo;
  }
};

// Arguments that every call on a pool checks.
inline int check_pool(const gptoss_kv8_pool_t *p) {
  if (!p || p->n_layers <= 0 || p->n_pages <= 0 || p->n_kv_heads <= 0)
    return GPTOSS_ERR_BAD_ARG;
  if (p->head_dim != 64 && p->head_dim != 128)
    return GPTOSS_ERR_UNSUPPORTED;
  if (!p->codes || !p->scales || !aligned16(p->codes) || (reinterpret_cast<uintptr_t>(p->scales) & 7u))
    return GPTOSS_ERR_BAD_ARG;
  return GPTOSS_OK;
}
// Arguments that every call on a step's rows checks (T > 0).
inline int check_rows(const gptoss_kv8_pool_t *p, int layer, int T, const void *qkv, gptoss_dtype_t dtype,
                      long row_stride, int n_q_heads, int n_seqs, const int *row_start, const int *kv_len,
                      const int *pages, int pages_stride, int max_new) {
  if (layer < 0 || layer >= p->n_layers || n_q_heads < 0 || n_seqs <= 0 || pages_stride <= 0 || max_new <= 0 ||
      !valid_dtype(dtype) || row_stride < (long)(n_q_heads + 2l * p->n_kv_heads) * p->head_dim)
    return GPTOSS_ERR_BAD_ARG;
  if (T > kMaxTokens || n_seqs > kMaxTokens / 4 || pages_stride > kMaxTokens / kPage)
    return GPTOSS_ERR_UNSUPPORTED;
  if (!qkv || !row_start || !kv_len || !pages || (reinterpret_cast<uintptr_t>(qkv) & (dtype_size(dtype) - 1)))
    return GPTOSS_ERR_BAD_ARG;
  return GPTOSS_OK;
}
inline size_t layer_codes(const gptoss_kv8_pool_t *p) {
  return (size_t)p->n_pages * p->n_kv_heads * 2 * kPage * p->head_dim;
}
inline size_t layer_scales(const gptoss_kv8_pool_t *p) { return (size_t)p->n_pages * p->n_kv_heads * 2; }
inline Layer layer_of(const gptoss_kv8_pool_t *p, int layer) {
  return Layer{p->codes + (size_t)layer * layer_codes(p), p->scales + (size_t)layer * layer_scales(p), p->n_pages,
               p->n_kv_heads};
}

} // namespace kv8
} // namespace gptoss
