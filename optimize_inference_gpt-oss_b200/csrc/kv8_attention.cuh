// What the two kernels of the attention over the 8-bit cache share: the call, what a row group looks at,
// reading queries and writing outputs.
#pragma once

#include "kv8_mma.cuh"

namespace gptoss {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kValueBits = 5;     // codes of the largest value scale met so far are held times 2^5
constexpr int kMaxTokenRows = 64; // (new tokens) x (query heads per key/value head) of one sequence: attend_tokens up to
                                  // here, attend_tiles above (24 sequences of 40 rows and 2000 tokens: 57 us here, 77
                                  // there; of 64 rows 84 and 86; 100 of 64 rows and 1000 tokens 211 and 145; one of 64
                                  // rows and 100000 tokens 101 and 136; heads of 128: 72 / 135, 81 / 118, 159 / 199, 125 / 172)

template <typename QT> struct Call {
  Layer cache;
  const QT *qkv;
  long row_stride;
  int n_q_heads, group;
  Rows rows;
  float scale;
  int window, n_first;
  const float *sinks;
  void *out;
  long out_row_stride;
  unsigned *giveups;
  bool out_f32, q_vec, out_vec; // vec: rows may be read / written 4 elements at a time
};

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

// fp16 2^e and -1152 * 2^e, twice in a word; e <= 5, zero below fp16's range.
__device__ __forceinline__ void value_factor(int e, uint32_t &mul, uint32_t &add) {
  const uint32_t m = e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
  const uint32_t a = e >= -24 ? 0x8080u | (uint32_t)(e + 25) << 10 : 0u;
  mul = m * 0x10001u, add = a * 0x10001u;
}

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

// Sequences of more than kMaxTokenRows rows (kv8_prompt.cu).
template <typename QT> void launch_tiles(cudaStream_t stream, const Call<QT> &a, int head_dim, void *workspace);
size_t tiles_workspace(long T, int group, int heads, int n_seqs, int head_dim);

} // namespace kv8
} // namespace gptoss
