// Attention over the 8-bit paged cache (gptoss_kv8_attention).
#include "kv8.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One warp per (row, query head): the plainest form.  A lane takes every 32nd token for the
// scores, then D / 32 elements of the output.
template <typename QT, typename OT, int D>
__global__ void __launch_bounds__(128)
    attend_rows(Layer cache, const QT *__restrict__ qkv, long row_stride, int n_q_heads, Rows rows, float scale, int window,
                int n_first, const float *__restrict__ sinks, OT *__restrict__ out, long out_row_stride) {
  pdl_prologue();
  __shared__ float q_of[4][D], p_of[4][kPage];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y * 4 + warp, row = blockIdx.x;
  if (h >= n_q_heads)
    return;
  const int s = rows.find(row, [&](int i) { return rows.start(i); });
  const Rows::Span sp = rows.span(s);
  if (row < sp.row || row >= sp.row + sp.q)
    return;
  const int pos = sp.pos + row - sp.row, head = h / (n_q_heads / cache.n_kv_heads);
  bool bad = false, seen = false;
  for (int i = lane; i < D; i += 32) {
    const float q = load1(qkv + (size_t)row * row_stride + (size_t)h * D + i);
    bad = bad || !isfinite(q);
    q_of[warp][i] = isfinite(q) ? q * scale : 0.0f;
  }
  bad = __any_sync(0xffffffffu, bad);
  __syncwarp();
  float m = sinks ? sinks[h] : -INFINITY, l = m > -INFINITY ? 1.0f : 0.0f, acc[D / 32] = {};
  const int from = window > 0 ? pos - window + 1 : 0; // tokens >= from are in the window
  for (int p = 0; p < rows.pages_stride && p * kPage <= pos; p++) {
    if (p * kPage + kPage <= from && p * kPage >= n_first)
      continue;
    const int page = cache.checked(rows.pages[(size_t)s * rows.pages_stride + p]);
    if (page < 0)
      continue;
    const int8_t *codes = cache.block<D>(page, head);
    const float ks = cache.scale(page, head)[0], vs = cache.scale(page, head)[1];
    float z[2], top = m;
    for (int u = 0; u < 2; u++) {
      const int t = p * kPage + lane + 32 * u;
      z[u] = -INFINITY;
      if (t <= pos && (t >= from || t < n_first)) {
        float dot = 0.0f;
        for (int i = 0; i < D; i++)
          dot += q_of[warp][i] * codes[(lane + 32 * u) * D + i];
        z[u] = dot * ks;
        seen = true;
      }
      top = fmaxf(top, z[u]);
    }
    for (int o = 16; o > 0; o >>= 1)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY)
      continue;
    const float fade = expf(m - top);
    m = top;
    float sum = 0.0f;
    for (int u = 0; u < 2; u++) {
      const float w = expf(z[u] - m);
      sum += w;
      p_of[warp][lane + 32 * u] = w * vs;
    }
    l = l * fade + warp_sum(sum);
    __syncwarp();
    for (int i = 0; i < D / 32; i++) {
      float a = 0.0f;
      for (int t = 0; t < kPage; t++)
        a += p_of[warp][t] * codes[(kPage + t) * D + i * 32 + lane];
      acc[i] = acc[i] * fade + a;
    }
    __syncwarp();
  }
  bad = __any_sync(0xffffffffu, seen) && bad;
  for (int i = 0; i < D / 32; i++)
    store1(out + (size_t)row * out_row_stride + (size_t)h * D + i * 32 + lane, bad ? NAN : l > 0.0f ? acc[i] / l : 0.0f);
}

template <typename QT, typename OT>
void launch(cudaStream_t stream, int D, const Layer &cache, const void *qkv, long row_stride, int n_q_heads,
            const Rows &rows, float scale, int window, int n_first, const float *sinks, void *out, long out_row_stride) {
  auto kernel = D == 64 ? attend_rows<QT, OT, 64> : attend_rows<QT, OT, 128>;
  launch_kernel(kernel, dim3(rows.T, (n_q_heads + 3) / 4), dim3(128), 0, stream, cache, static_cast<const QT *>(qkv),
                row_stride, n_q_heads, rows, scale, window, n_first, sinks, static_cast<OT *>(out), out_row_stride);
}

} // namespace
} // namespace kv8
} // namespace gptoss

extern "C" size_t gptoss_kv8_attention_workspace(const gptoss_kv8_pool_t *pool, int T, int n_q_heads, int n_seqs,
                                                 int max_new) {
  using namespace gptoss;
  if (kv8::check_pool(pool) != GPTOSS_OK || T <= 0 || n_q_heads <= 0 || n_seqs <= 0 || max_new <= 0 ||
      n_q_heads % pool->n_kv_heads)
    return 0;
  return 16;
}

extern "C" int gptoss_kv8_attention(gptoss_stream_t stream, const gptoss_kv8_pool_t *pool, int layer, int T,
                                    const void *qkv, gptoss_dtype_t qkv_dtype, long row_stride, int n_q_heads, int n_seqs,
                                    const int *row_start, const int *kv_len, const int *pages, int pages_stride,
                                    int max_new, float scale, int window, int n_first, const float *sinks, void *out,
                                    gptoss_dtype_t out_dtype, long out_row_stride, void *workspace,
                                    size_t workspace_bytes, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (T < 0 || window < 0 || n_first < 0 || !valid_dtype(out_dtype))
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_pool(pool))
    return st;
  if (T == 0)
    return GPTOSS_OK;
  if (const int st = kv8::check_rows(pool, layer, T, qkv, qkv_dtype, row_stride, n_q_heads, n_seqs, row_start, kv_len,
                                     pages, pages_stride, max_new))
    return st;
  const int D = pool->head_dim;
  if (n_q_heads <= 0 || !out || out_row_stride < (long)n_q_heads * D ||
      (reinterpret_cast<uintptr_t>(out) & (dtype_size(out_dtype) - 1)))
    return GPTOSS_ERR_BAD_ARG;
  if (n_q_heads % pool->n_kv_heads != 0 || (n_q_heads + 3) / 4 > 65535)
    return GPTOSS_ERR_UNSUPPORTED;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < gptoss_kv8_attention_workspace(pool, T, n_q_heads, n_seqs, max_new))
    return GPTOSS_ERR_BAD_ARG;
  GPTOSS_SPAN(qkv, strided_bytes(T, row_stride, (long)(n_q_heads + 2l * pool->n_kv_heads) * D, dtype_size(qkv_dtype)));
  GPTOSS_SPAN(out, strided_bytes(T, out_row_stride, (long)n_q_heads * D, dtype_size(out_dtype)));
  GPTOSS_SPAN(pool->codes, kv8::layer_codes(pool) * pool->n_layers);
  GPTOSS_SPAN(pool->scales, kv8::layer_scales(pool) * pool->n_layers * 4);
  GPTOSS_SPAN(row_start, ((size_t)n_seqs + 1) * 4);
  GPTOSS_SPAN(kv_len, (size_t)n_seqs * 4);
  GPTOSS_SPAN(pages, (size_t)n_seqs * pages_stride * 4);
  GPTOSS_SPAN(sinks, (size_t)n_q_heads * 4);
  GPTOSS_SPAN(workspace, workspace_bytes);
  const kv8::Layer cache = kv8::layer_of(pool, layer);
  const kv8::Rows rows = {row_start, kv_len, pages, T, n_seqs, pages_stride, max_new > T ? T : max_new};
  window = window > kv8::kMaxTokens ? kv8::kMaxTokens : window;
  const cudaStream_t s = as_stream(stream);
#define GPTOSS_ATTEND(QT, OT)                                                                                          \
  kv8::launch<QT, OT>(s, D, cache, qkv, row_stride, n_q_heads, rows, scale, window, n_first, sinks, out, out_row_stride)
  if (qkv_dtype == GPTOSS_F32)
    out_dtype == GPTOSS_F32 ? GPTOSS_ATTEND(float, float) : GPTOSS_ATTEND(float, uint16_t);
  else
    out_dtype == GPTOSS_F32 ? GPTOSS_ATTEND(uint16_t, float) : GPTOSS_ATTEND(uint16_t, uint16_t);
#undef GPTOSS_ATTEND
  return launch_status();
}
