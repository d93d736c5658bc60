// What the two kernels of the attention over the 8-bit cache share: the call, what a row group looks at,
// reading queries and writing outputs.
#pragma once

#include "kv8_mma.cuh"

namespace gptoss {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;
// Value scales.  Codes are multiplied by their page's scale relative to a reference, the scale that most of the first 32
// pages are near: by 2^(kValueBits - 2 kNear) to 2^kValueBits, exact in fp16, for scales within 2^kNear of the reference.  Pages
// further away (far pages: one value 1000 times its neighbours', an infinity stored as the largest finite number) are left
// out there and summed by far_row, in fp32, row by row, and only then joined: what a row holds never depends on the
// size of what it does not see, or gives no weight.  (A reference that followed the largest page lost everything 2^29
// smaller, for all rows of a block; one per row would still lose it where the large code is not the row's to see.)
constexpr int kNear = 10, kValueBits = 5;
constexpr int kMaxTokenRows = 64; // (new tokens) x (query heads per key/value head) of one sequence: attend_tokens up to
                                  // here, attend_tiles above (24 sequences of 40 rows and 2000 tokens: 57 us here, 77
                                  // there; of 64 rows 84 and 86; 100 of 64 rows and 1000 tokens 211 and 145; one of 64
                                  // rows and 100000 tokens 101 and 136; heads of 128: 72 / 135, 81 / 118, 159 / 199, 125 / 172)

template <typename QT> struct Call {
  Layer cache;
  const QT *qkv;
  long row_stride;
  int group;
  Rows rows;
  float scale;
  int window, n_first;
  const float *sinks;
  void *out;
  long out_row_stride;
  unsigned *giveups;
  bool out_f32, q_vec, out_vec; // vec: rows may be read / written 4 elements at a time
};

// A head's sink logit in powers of two; an infinite one is brought to where differences are still numbers.  A NaN stays
// one: no maximum takes it, but the sum does.
template <typename QT> __device__ __forceinline__ float sink_of(const Call<QT> &a, int h) {
  const float z = __ldg(a.sinks + h) * kLog2e;
  return z > 3e38f ? 3e38f : z;
}

// Between two bounds; a NaN stays one.
__device__ __forceinline__ float at_most(float x, float top) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(top));
  return r;
}
__device__ __forceinline__ float at_least(float x, float bottom) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(bottom));
  return r;
}
// A row's and a page's scale together stay finite: in a page whose key scale is 2^122 for the sake of a token that is not
// seen the codes of the others are 0, and so are their scores.
constexpr float kMostFactor = 3e38f;

// The table columns a row group looks at: the first `head` ones, then those from `lo` on; n in all (at
// least one, so that every row is visited; what it must not see is masked).
struct Columns {
  int head, lo, n;
  __device__ __forceinline__ int at(int i) const { return i < head ? i : lo + i - head; }
};
__device__ __forceinline__ Columns columns(const Rows &rows, int window, int n_first, int min_pos, int max_pos) {
  const int last = min(max(max_pos, 0) / kPage, rows.pages_stride - 1);
  const int lo = window > 0 ? min(max(min_pos - window + 1, 0) / kPage, last) : 0;
  const int head = min((int)(((long)n_first + kPage - 1) / kPage), lo);
  return Columns{head, lo, head + last - lo + 1};
}

__device__ __forceinline__ bool is_far(int v_exp, int ref) { return v_exp != 0 && (unsigned)(v_exp - ref + kNear) > 2u * kNear; }
// The reference of up to 32 pages, whose value scales' exponents (0: none) the lanes have: the first's, unless most are
// far from it and fewer from the first of those, as when the first page holds one huge value.
__device__ __forceinline__ int pick_ref(int v_exp) {
  const unsigned valued = __ballot_sync(0xffffffffu, v_exp != 0);
  if (!valued)
    return 0;
  const int first = __shfl_sync(0xffffffffu, v_exp, __ffs(valued) - 1);
  const unsigned far = __ballot_sync(0xffffffffu, is_far(v_exp, first));
  if (2 * __popc(far) <= __popc(valued))
    return first;
  const int second = __shfl_sync(0xffffffffu, v_exp, __ffs(far) - 1);
  return __popc(__ballot_sync(0xffffffffu, is_far(v_exp, second))) < __popc(far) ? second : first;
}
// fp16 2^e and -1152 * 2^e, twice in a word, for the values of a page that is not far (e in [-15, 5]); zero for a page of
// zeros.
__device__ __forceinline__ void value_factor(int v_exp, int ref, uint32_t &mul, uint32_t &add) {
  const int e = v_exp - ref - kNear + kValueBits;
  const uint32_t m = e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << (e + 24), a = 0x8080u | (uint32_t)(e + 25) << 10;
  mul = v_exp ? m * 0x10001u : 0u, add = v_exp ? a * 0x10001u : 0u;
}
// The matrix units cut off what an addition to an fp32 sum leaves below its last bit; over the hundreds of additions of a
// long context results shrink by some 4e-6 (measured: 5000 tokens of a prompt, 16000 of single rows).  For fp32 rows their
// sums are therefore started afresh after this many additions and the partial sums added in ordinary fp32.
constexpr int kFold = 64;
// Where weighted values are added up before the division they are held in units of 2^kSumBits: a few thousand of 2^128.
constexpr int kSumBits = 16;
__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f); }

template <typename QT> __device__ __forceinline__ void load4(const QT *p, bool vec, float (&v)[4]) {
  if (vec) {
    if constexpr (sizeof(QT) == 4) {
      const float4 f = *reinterpret_cast<const float4 *>(p);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(p);
      v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      v[i] = load1(p + i);
  }
}
// Four elements of the output, from element `at` on.
template <typename QT> __device__ __forceinline__ void store4(const Call<QT> &a, size_t at, float4 v) {
  if (a.out_f32) {
    float *p = static_cast<float *>(a.out) + at;
    if (a.out_vec)
      *reinterpret_cast<float4 *>(p) = v;
    else
      p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
  } else {
    uint16_t *p = static_cast<uint16_t *>(a.out) + at;
    if (a.out_vec)
      *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    else
      store1(p, v.x), store1(p + 1, v.y), store1(p + 2, v.z), store1(p + 3, v.w);
  }
}

// What a row (query q at position pos) sees of the far pages among the columns [i0, i1), joined to what it saw of the
// others: `mean` (D values) and ml (maximum, sum of the weights), both in shared memory.  A page is `steps` steps, dealt in
// turn to n_refs warps; refs has the references they held pages against.  Plain fp32 by a whole warp, two tokens to a lane
// for the scores, then D / 32 elements: made for pages that hardly ever are.  One such page in each of 64 sequences of
// 8000 tokens: 0.12 -> 0.23 ms; in a prompt of 2048 tokens 0.10 -> 0.49.  A call of its own, so that it takes no registers
// from the kernels' loops.
template <int D, typename QT>
__device__ __noinline__ void far_row(const Call<QT> &a, int s, int head, Columns cols, int i0, int i1, const QT *q, int pos,
                                     const int *refs, int n_refs, int steps, float *mean, float2 *ml) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
  auto value = [](uint32_t w, int i) { // byte i of four biased codes: the lowest of 2^23 + code + 128
    return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | i)) - 8388736.0f;
  };
  float top = 0.0f;
  bool odd = false;
#pragma unroll
  for (int n = 0; n < N; n++) {
    const float x = load1(q + lane * N + n);
    odd = odd || !(fabsf(x) <= 3.402823466e38f);
    top = fmaxf(top, fabsf(x));
  }
  odd = __any_sync(0xffffffffu, odd);
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  const int up = odd || top == 0.0f ? 0 : max(min(127 - exponent_field(top), 126), -126); // largest |q| into [1, 2)
  const float lift = two_to(up), row_factor = odd ? NAN : a.scale * kLog2e * two_to(-up);
  float m = -INFINITY, l = 0.0f, o[N] = {};
  int page_of = -1, held = i0 - 32; // lane l has the page and scales of column held + l
  float2 scale_of = make_float2(0.0f, 0.0f);
  unsigned far = 0; // columns with a far page that are still to be done
#pragma unroll 1
  for (;;) {
    while (!far && held + 32 < i1) {
      held += 32;
      const int i = held + lane;
      page_of = i < i1 ? a.cache.checked(__ldg(table + cols.at(i))) : -1;
      bool any = false;
      if (page_of >= 0) {
        scale_of = *reinterpret_cast<const float2 *>(a.cache.scale(page_of, head));
        for (int step = 0; step < steps; step++)
          any = any || is_far(exponent_field(scale_of.y), refs[((i - i0) * steps + step) % n_refs]);
      }
      far = __ballot_sync(0xffffffffu, any);
    }
    if (!far)
      break;
    const int from = __ffs(far) - 1, i = held + from, page = __shfl_sync(0xffffffffu, page_of, from);
    far &= far - 1;
    const float key_scale = __shfl_sync(0xffffffffu, scale_of.x, from);
    const int v_exp = exponent_field(__shfl_sync(0xffffffffu, scale_of.y, from)), first = cols.at(i) * kPage;
    bool sees[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int t = lane + 32 * u, token = first + t;
      sees[u] = is_far(v_exp, refs[((i - i0) * steps + t * steps / kPage) % n_refs]) && token <= pos &&
                (a.window <= 0 || token > pos - a.window || token < a.n_first);
    }
    if (!__any_sync(0xffffffffu, sees[0] || sees[1]))
      continue;
    const int8_t *block = a.cache.template block<D>(page, head);
    float z[2][4] = {};
#pragma unroll 1
    for (int d = 0; d < D; d += 16) {
      const uint4 k[2] = {ld_plain(block + lane * D + d), ld_plain(block + (lane + 32) * D + d)};
      float x[4][4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        load4(q + d + 4 * e, a.q_vec, x[e]);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t w[4] = {biased(k[u].x), biased(k[u].y), biased(k[u].z), biased(k[u].w)};
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int b = 0; b < 4; b++)
            z[u][b] = fmaf(x[e][b] * lift, value(w[e], b), z[u][b]);
      }
    }
    const float factor = at_least(at_most(row_factor * key_scale, kMostFactor), -kMostFactor);
    float y[2], now = m, p[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      y[u] = sees[u] ? ((z[u][0] + z[u][1]) + (z[u][2] + z[u][3])) * factor : -INFINITY;
      now = fmaxf(now, y[u]);
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1)
      now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, x));
    const float base = now > -INFINITY ? now : 0.0f, fade = fast_exp2(m - base), unit = two_to(v_exp - 127 - kSumBits);
#pragma unroll
    for (int u = 0; u < 2; u++)
      p[u] = sees[u] ? fast_exp2(y[u] - base) : 0.0f;
    m = now, l = fmaf(l, fade, warp_sum(p[0] + p[1]));
    float page_sum[N] = {};
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll 1
      for (int t0 = 0; t0 < 32; t0 += 8) { // eight at a time, so that sums stay short
        float part[N] = {};
#pragma unroll
        for (int t = 0; t < 8; t++) {
          const int8_t *v = block + (kPage + 32 * u + t0 + t) * D + lane * N;
          const uint32_t w = biased(N == 2 ? *reinterpret_cast<const uint16_t *>(v) : *reinterpret_cast<const uint32_t *>(v));
          const float weight = __shfl_sync(0xffffffffu, p[u], t0 + t);
#pragma unroll
          for (int n = 0; n < N; n++)
            part[n] = fmaf(weight, value(w, n), part[n]);
        }
#pragma unroll
        for (int n = 0; n < N; n++)
          page_sum[n] += part[n];
      }
#pragma unroll
    for (int n = 0; n < N; n++)
      o[n] = fmaf(o[n], fade, page_sum[n] * unit);
  }
  if (l == 0.0f) // a NaN passes, here and below
    return;
  const float2 near = *ml;
  const float most = fmaxf(near.x, m), f = m > -INFINITY ? fast_exp2(m - most) : 1.0f;
  const float near_sum = near.y != 0.0f ? near.y * fast_exp2(near.x - most) : 0.0f, sum = near_sum + l * f;
#pragma unroll
  for (int n = 0; n < N; n++)
    mean[lane * N + n] = finite(fmaf(mean[lane * N + n], near_sum / sum, o[n] * (f / sum * (float)(1 << kSumBits))));
  __syncwarp();
  if (lane == 0)
    *ml = make_float2(most, sum);
  __syncwarp();
}

// Sequences of more than kMaxTokenRows rows (kv8_prompt.cu).
template <typename QT> void launch_tiles(cudaStream_t stream, const Call<QT> &a, int head_dim, void *workspace);
size_t tiles_workspace(long T, int group, int heads, int n_seqs, int head_dim);

} // namespace kv8
} // namespace gptoss
