// What the two kernels of the attention over the 8-bit cache share: the call, what a row group looks at,
// reading queries and writing outputs.
#pragma once

#include "kv8_mma.cuh"

namespace gptoss {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;
// Value scales.  Codes are multiplied by their page's scale relative to a reference, the scale of the first page that
// has one: by 2^(kValueBits - 2 kNear) to 2^kValueBits, exact in fp16, for scales within 2^kNear of the reference.  Pages
// further away (far pages: one value 1000 times its neighbours', an infinity stored as the largest finite number) are left
// out there and summed by far_pages, in fp32, row by row, and only then joined: what a row holds never depends on the
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
// fp16 2^e and -1152 * 2^e, twice in a word, for the values of a page that is not far (e in [-15, 5]); zero for a page of
// zeros.
__device__ __forceinline__ void value_factor(int v_exp, int ref, uint32_t &mul, uint32_t &add) {
  const int e = v_exp - ref - kNear + kValueBits;
  const uint32_t m = e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << 9, a = 0x8080u | (uint32_t)(e + 25) << 10;
  mul = v_exp ? m * 0x10001u : 0u, add = v_exp ? a * 0x10001u : 0u;
}
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

// What one row (query q at position pos) sees of the far pages among the columns [i0, i1): maximum, sum of the weights,
// and N of its elements from d0 on, in units of 2^kSumBits.  A page is `steps` steps, dealt in turn to n_refs warps; refs
// has the references they held pages against.  Plain fp32, eight tokens at a time: some ten times what a near page costs,
// for pages that hardly ever are.  A call of its own, so that it takes no registers from the kernels' loops (inlined,
// prompts ran 2-3 % longer).
template <int N> struct FarSum {
  float m, l, o[N];
};
template <int D, int N, typename QT>
__device__ __noinline__ FarSum<N> far_pages(const Call<QT> &a, int s, Columns cols, int i0, int i1, int head, const QT *q, int pos,
                                            int d0, const int *refs, int n_refs, int steps) {
  const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
  FarSum<N> f;
  f.m = -INFINITY, f.l = 0.0f;
#pragma unroll
  for (int n = 0; n < N; n++)
    f.o[n] = 0.0f;
  bool odd = false;
#pragma unroll 1
  for (int d = 0; d < D; d++)
    odd = odd || !(fabsf(load1(q + d)) <= 3.402823466e38f);
#pragma unroll 1
  for (int i = i0; i < i1; i++) {
    const int page = a.cache.checked(__ldg(table + cols.at(i)));
    if (page < 0)
      continue;
    const float *scale = a.cache.scale(page, head);
    const int v_exp = exponent_field(scale[1]);
    const int8_t *block = a.cache.template block<D>(page, head);
    const float factor = odd ? NAN : a.scale * kLog2e * scale[0], unit = two_to(v_exp - 127 - kSumBits);
#pragma unroll 1
    for (int t0 = 0; t0 < kPage; t0 += 8) {
      if (!is_far(v_exp, refs[((i - i0) * steps + t0 * steps / kPage) % n_refs]))
        continue;
      float z[8], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int token = cols.at(i) * kPage + t0 + u;
        z[u] = -INFINITY;
        if (token <= pos && (a.window <= 0 || token > pos - a.window || token < a.n_first)) {
          float part[4] = {};
#pragma unroll 1
          for (int d = 0; d < D; d += 4) {
            const char4 k = *reinterpret_cast<const char4 *>(block + (t0 + u) * D + d);
            float x[4];
            load4(q + d, a.q_vec, x);
#pragma unroll
            for (int e = 0; e < 4; e++)
              x[e] = at_least(at_most(x[e] * factor, kMostFactor), -kMostFactor);
            part[0] = fmaf(x[0], k.x, part[0]), part[1] = fmaf(x[1], k.y, part[1]);
            part[2] = fmaf(x[2], k.z, part[2]), part[3] = fmaf(x[3], k.w, part[3]);
          }
          z[u] = (part[0] + part[1]) + (part[2] + part[3]);
        }
        top = fmaxf(top, z[u]);
      }
      const float now = fmaxf(f.m, top), base = now > -INFINITY ? now : 0.0f, fade = fast_exp2(f.m - base);
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        z[u] = fast_exp2(z[u] - base);
        sum += z[u];
      }
      f.m = now, f.l = fmaf(f.l, fade, sum);
#pragma unroll
      for (int n = 0; n < N; n += 4) {
        float part[4] = {};
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const char4 v = *reinterpret_cast<const char4 *>(block + (kPage + t0 + u) * D + d0 + n);
          part[0] = fmaf(z[u], v.x, part[0]), part[1] = fmaf(z[u], v.y, part[1]);
          part[2] = fmaf(z[u], v.z, part[2]), part[3] = fmaf(z[u], v.w, part[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
          f.o[n + e] = fmaf(f.o[n + e], fade, part[e] * unit);
      }
    }
  }
  return f;
}

// Sequences of more than kMaxTokenRows rows (kv8_prompt.cu).
template <typename QT> void launch_tiles(cudaStream_t stream, const Call<QT> &a, int head_dim, void *workspace);
size_t tiles_workspace(long T, int group, int heads, int n_seqs, int head_dim);

} // namespace kv8
} // namespace gptoss
