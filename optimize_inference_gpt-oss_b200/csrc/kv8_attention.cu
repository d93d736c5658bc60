// Attention over the 8-bit paged cache (gptoss_kv8_attention) for few rows per sequence.
//
//     z_t = scale q . k_t,   out = sum_t 2^(z_t' - m) v_t / (sum_t 2^(z_t' - m) + 2^(sink' - m)),   ' = times log2(e)
//
// The rows of a sequence that share a key/value head (its new tokens x the query heads of the group)
// are the 16-row tiles of a matrix instruction; one pass over the pages with the running maximum and
// sum of each row.  What bounds it is the cache's bytes: at 16 rows or fewer a token costs one byte per
// element and some twelve instructions per 4 bytes.  So:
//   - a warp works alone on steps of CH tokens, its loads going from global memory straight into the
//     registers that feed the matrix instruction (the order of a head's elements within a product and
//     of a step's tokens is free, and is chosen so that a lane needs 16 or 8 consecutive bytes), the
//     next step's loads in flight while this one is computed; no shared memory, no barrier per step;
//   - codes become fp16 exactly (kv8_mma.cuh); key scales multiply the scores, value scales, powers
//     of two, multiply the codes relative to the largest met so far;
//   - queries are brought to fp16 range by a power of two per row; a bf16 row is then exact, an fp32 row
//     is two fp16 parts and two products, and so are its softmax weights, which is what keeps fp32's
//     accuracy on these tensor cores;
//   - the weights carry a factor 2^9, so that weights down to 2^-23 of the largest are normal fp16;
//   - work is cut into equal pieces of pages over all blocks whatever the lengths (a long sequence
//     beside short ones, one sequence alone); a sequence cut across blocks is joined by merge_pieces.
#include <algorithm>

#include "kv8_mma.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWeightBits = 9, kValueBits = 5;
constexpr int kTokenWarps = 4;
constexpr int kMaxTokenRows = 64; // (new tokens) x (query heads per key/value head) of one sequence
constexpr int kMinPages = 8;      // of a block's piece: below that joining costs more than it saves

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
  bool out_f32, q_vec, out_vec; // vec: rows may be read / written 4 elements at a time
};

// A block's piece of an item (sequence, head, row group) that other blocks have pieces of.
struct Pieces {
  int4 *first; // [grid] {sequence, head, row group, last block}: the item whose first piece this block has; sequence -1: none
  float *o;    // [grid][2][rows][D]
  float2 *ml;  // [grid][2][rows]
  static size_t bytes(int grid, int rows, int D) {
    return (size_t)grid * (16 + 2 * (size_t)rows * (D * 4 + 8));
  }
  static Pieces at(void *ws, int grid, int rows, int D) {
    int4 *f = static_cast<int4 *>(ws);
    float *o = reinterpret_cast<float *>(f + grid);
    return Pieces{f, o, reinterpret_cast<float2 *>(o + (size_t)grid * 2 * rows * D)};
  }
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

// Row n of an 8-token tile of scores is token n with its lowest bit flipped in every other pair: the
// four tokens that a lane multiplies values of then lie in different halves of a 128-byte line from
// its neighbours'.
__device__ __forceinline__ int token_of(int n) { return n ^ ((n >> 1) & 1); }

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

// A row's sum and maximum joined with its head's sink logit; what the row's values are to be divided by.
__device__ __forceinline__ void join_sink(const float *sinks, int h, float &m, float &l) {
  if (!sinks || l == 0.0f)
    return;
  const float z = fminf(__ldg(sinks + h) * kLog2e, 3e38f), top = fmaxf(m, z);
  l = l * fast_exp2(m - top) + fast_exp2(z - top);
  m = top;
}

template <typename QT, int D, int MT> struct TokenKernel {
  static constexpr bool kSplit = sizeof(QT) == 4;            // two fp16 parts
  static constexpr int CH = (D == 64 ? 64 : 32) / MT;        // tokens of a step
  static constexpr int kSteps = kPage / CH;                  // steps of a page
  static constexpr int NT = CH / 8, KK = CH / 16, KS = D / 16, DV = D / 8;
  static constexpr int kRows = 16 * MT;
  static constexpr int kPitch = D + 4;                       // floats of a row in shared memory
  static constexpr int kSmem = kTokenWarps * kRows * (kPitch * 4 + 8);
  using VWord = typename std::conditional<D == 64, uint2, uint4>::type;

  uint4 K[NT][D / 64];
  VWord V[KK][4];
  uint32_t q[MT][KS][4], q_rest[kSplit ? MT : 1][kSplit ? KS : 1][4];
  float row_factor[MT][2], m[MT][2], l[MT][2], o[MT][DV][4];
  int row_pos[MT][2]; // -1: no such row
  bool bad[MT][2];
  int value_exp;

  __device__ __forceinline__ void load_keys(const int8_t *block, int step) {
    const int lane = threadIdx.x & 31, n = token_of(lane >> 2), t = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < D / 64; j++)
        K[i][j] = ld_stream(block + (size_t)(step * CH + 8 * i + n) * D + j * 64 + t * 16);
  }
  __device__ __forceinline__ void load_values(const int8_t *block, int step) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int token = step * CH + 16 * kk + 8 * (c >> 1) + token_of(2 * t + (c & 1));
        const int8_t *p = block + (size_t)(kPage + token) * D + g * (D / 8);
        if constexpr (D == 64)
          asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(V[kk][c].x), "=r"(V[kk][c].y) : "l"(p));
        else
          V[kk][c] = ld_stream(p);
      }
  }

  // The group's queries as left operands; a row's elements in the order that K's lanes have them.
  __device__ __forceinline__ void load_queries(const Call<QT> &a, const Rows::Span &sp, int head, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, R = sp.q * a.group;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int r = row0 + 16 * mt + 8 * half + g;
        const bool is = r < R;
        const int token = is ? r / a.group : 0, h = head * a.group + (is ? r % a.group : 0);
        row_pos[mt][half] = is ? sp.pos + token : -1;
        const QT *p = a.qkv + (size_t)(sp.row + token) * a.row_stride + (size_t)h * D + 16 * t;
        float v[KS][4], top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < KS; j++) {
          load4(p + (j / 4) * 64 + (j % 4) * 4, a.q_vec, v[j]);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            v[j][e] = is ? v[j][e] : 0.0f;
            odd = odd || !(fabsf(v[j][e]) <= 3.402823466e38f);
            top = fmaxf(top, fabsf(v[j][e]));
          }
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
          odd = __shfl_xor_sync(0xffffffffu, (int)odd, s) || odd;
        }
        bad[mt][half] = odd;
        // largest |q| into [2^13, 2^14); rows too small for the exponent keep a factor of 2^126
        const int up = odd || top == 0.0f ? 0 : min(13 - (exponent_field(top) - 127), 126);
        const float f = two_to(max(up, -126)) * (a.scale < 0.0f ? -1.0f : 1.0f);
        row_factor[mt][half] = fabsf(a.scale) * kLog2e * two_to(-max(up, -126));
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float x = odd ? 0.0f : v[j][e] * f, y = odd ? 0.0f : v[j][e + 1] * f;
            const uint32_t w = pack_f16(x, y);
            q[mt][j][e + half] = w; // a0/a1: elements 0,1; a2/a3: elements 2,3
            if constexpr (kSplit)
              q_rest[mt][j][e + half] = pack_rest(w, x, y);
          }
      }
  }

  __device__ __forceinline__ void begin() {
    value_exp = 0;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        m[mt][half] = -INFINITY, l[mt][half] = 0.0f;
#pragma unroll
        for (int j = 0; j < DV; j++)
          o[mt][j][2 * half] = o[mt][j][2 * half + 1] = 0.0f;
      }
  }

  __device__ __forceinline__ void scores(float (&s)[MT][NT][4]) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
        s[mt][i][0] = s[mt][i][1] = s[mt][i][2] = s[mt][i][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; j++) {
        const uint4 w4 = K[i][j / 4];
        const uint32_t u = biased(j % 4 == 0 ? w4.x : j % 4 == 1 ? w4.y : j % 4 == 2 ? w4.z : w4.w);
        const uint32_t b0 = minus_1152(low_pair(u)), b1 = minus_1152(high_pair(u));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          mma_f16(s[mt][i], q[mt][j], b0, b1);
          if constexpr (kSplit)
            mma_f16(s[mt][i], q_rest[mt][j], b0, b1);
        }
      }
    }
  }

  // s becomes the weights of the step's tokens first_token ..
  __device__ __forceinline__ void weigh(float (&s)[MT][NT][4], float key_scale, int v_exp, bool masked, int first_token,
                                        int window, int n_first) {
    const int t = threadIdx.x & 3;
    bool moved = v_exp > value_exp;
    float fade[MT][2];
    const float beta = moved ? two_to(value_exp - v_exp) : 1.0f;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        uint32_t seen = 0xffffffffu;
        float top = -INFINITY;
        if (masked) {
          seen = 0;
          const int pos = row_pos[mt][half];
#pragma unroll
          for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int token = first_token + 8 * i + token_of(2 * t + e);
              const bool ok = token <= pos && (window <= 0 || token > pos - window || token < n_first);
              seen |= (uint32_t)ok << (2 * i + e);
              top = fmaxf(top, ok ? s[mt][i][2 * half + e] : -INFINITY);
            }
        } else {
#pragma unroll
          for (int i = 0; i < NT; i++)
            top = fmaxf(top, fmaxf(s[mt][i][2 * half], s[mt][i][2 * half + 1]));
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1)
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float f = row_factor[mt][half] * key_scale;
        const float now = top > -INFINITY ? fmaxf(m[mt][half], top * f) : m[mt][half];
        const float base = now > -INFINITY ? now : 0.0f;
        const float a = fast_exp2(m[mt][half] - base), off = (float)kWeightBits - base;
        m[mt][half] = now;
        moved = moved || a != 1.0f;
        fade[mt][half] = a * beta;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float p = fast_exp2(fmaf(s[mt][i][2 * half + e], f, off));
            if (masked)
              p = seen >> (2 * i + e) & 1 ? p : 0.0f;
            s[mt][i][2 * half + e] = p;
            sum += p;
          }
        l[mt][half] = l[mt][half] * a + sum;
      }
    value_exp = max(value_exp, v_exp);
    if (__any_sync(0xffffffffu, moved))
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int j = 0; j < DV; j++)
          o[mt][j][0] *= fade[mt][0], o[mt][j][1] *= fade[mt][0], o[mt][j][2] *= fade[mt][1], o[mt][j][3] *= fade[mt][1];
  }

  __device__ __forceinline__ void add_values(const float (&s)[MT][NT][4], int v_exp) {
    uint32_t mul, add;
    value_factor(v_exp == 0 ? -99 : v_exp - value_exp + kValueBits, mul, add);
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      uint32_t p[MT][4], rest[kSplit ? MT : 1][4];
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int r = 0; r < 4; r++) { // a0, a1: rows g, g + 8 of the first tile; a2, a3: of the second
          const float x = s[mt][2 * kk + (r >> 1)][2 * (r & 1)], y = s[mt][2 * kk + (r >> 1)][2 * (r & 1) + 1];
          p[mt][r] = pack_f16(x, y);
          if constexpr (kSplit)
            rest[mt][r] = pack_rest(p[mt][r], x, y);
        }
#pragma unroll
      for (int w = 0; w < D / 32; w++) { // words of 4 elements
        uint32_t c[4];
#pragma unroll
        for (int x = 0; x < 4; x++)
          c[x] = biased(word(V[kk][x], w));
#pragma unroll
        for (int hi = 0; hi < 2; hi++) {
          const uint32_t a = __byte_perm(c[0], c[1], hi ? 0x7362 : 0x5140), b = __byte_perm(c[2], c[3], hi ? 0x7362 : 0x5140);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t b0 = scaled_pair(e ? high_pair(a) : low_pair(a), mul, add);
            const uint32_t b1 = scaled_pair(e ? high_pair(b) : low_pair(b), mul, add);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
              mma_f16(o[mt][4 * w + 2 * hi + e], p[mt], b0, b1);
              if constexpr (kSplit)
                mma_f16(o[mt][4 * w + 2 * hi + e], rest[mt], b0, b1);
            }
          }
        }
      }
    }
  }
  static __device__ __forceinline__ uint32_t word(uint2 v, int w) { return w ? v.y : v.x; }
  static __device__ __forceinline__ uint32_t word(uint4 v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

  // The columns [i0, i1) of an item, steps dealt to the block's warps in turn.
  __device__ __forceinline__ void run(const Call<QT> &a, int s, int head, const Columns &cols, int i0, int i1, int min_pos,
                                      int max_pos) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int end = i1 * kSteps;
    const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
    int page_of = -1, held = i0 * kSteps + warp; // lane l has the page of step held + 4 l
    float2 scale_of = make_float2(0.0f, 0.0f);
    auto fetch = [&]() {
      const int j = held + kTokenWarps * lane;
      page_of = j < end ? a.cache.checked(__ldg(table + cols.at(j / kSteps))) : -1;
      if (page_of >= 0)
        scale_of = *reinterpret_cast<const float2 *>(a.cache.scale(page_of, head));
    };
    begin();
    int j = held;
    if (j >= end)
      return;
    fetch();
    int page = __shfl_sync(0xffffffffu, page_of, 0), at = 0;
    float ks = __shfl_sync(0xffffffffu, scale_of.x, 0), vs = __shfl_sync(0xffffffffu, scale_of.y, 0);
    if (page >= 0) {
      load_keys(a.cache.template block<D>(page, head), j % kSteps);
      load_values(a.cache.template block<D>(page, head), j % kSteps);
    }
    for (; j < end; j += kTokenWarps) {
      if (++at == 32) {
        held += 32 * kTokenWarps, at = 0;
        fetch();
      }
      const int next = __shfl_sync(0xffffffffu, page_of, at), next_step = (j + kTokenWarps) % kSteps;
      const float next_ks = __shfl_sync(0xffffffffu, scale_of.x, at), next_vs = __shfl_sync(0xffffffffu, scale_of.y, at);
      const int8_t *next_block = a.cache.template block<D>(max(next, 0), head);
      float w[MT][NT][4];
      if (page >= 0)
        scores(w);
      if (next >= 0)
        load_keys(next_block, next_step);
      if (page >= 0) {
        const int token = cols.at(j / kSteps) * kPage + (j % kSteps) * CH, v_exp = exponent_field(vs);
        const bool all = token + CH - 1 <= min_pos && (a.window <= 0 || token > max_pos - a.window || token + CH <= a.n_first);
        weigh(w, ks, v_exp, !all, token, a.window, a.n_first);
        add_values(w, v_exp);
      }
      if (next >= 0)
        load_values(next_block, next_step);
      page = next, ks = next_ks, vs = next_vs;
    }
  }

  // The warps' results joined: into the output, or into a piece for merge_pieces.  Whole block.
  __device__ __forceinline__ void finish(const Call<QT> &a, const Rows::Span &sp, int head, int row0, float *piece_o,
                                         float2 *piece_ml) {
    extern __shared__ float4 smem4[];
    float *so = reinterpret_cast<float *>(smem4);
    float2 *sml = reinterpret_cast<float2 *>(so + kTokenWarps * kRows * kPitch);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const float unit = two_to(value_exp - 127 - kValueBits);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        float sum = l[mt][half];
#pragma unroll
        for (int x = 1; x < 4; x <<= 1)
          sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int r = 16 * mt + 8 * half + g;
        if (t == 0)
          sml[warp * kRows + r] = make_float2(m[mt][half], bad[mt][half] && sum > 0.0f ? NAN : sum * two_to(-kWeightBits));
        const float inverse = sum > 0.0f ? 1.0f / sum : 0.0f;
        float *row = so + (warp * kRows + r) * kPitch;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int j = 0; j < DV; j += 4)
            *reinterpret_cast<float4 *>(row + (2 * t + n) * DV + j) =
                make_float4(o[mt][j][2 * half + n] * inverse * unit, o[mt][j + 1][2 * half + n] * inverse * unit,
                            o[mt][j + 2][2 * half + n] * inverse * unit, o[mt][j + 3][2 * half + n] * inverse * unit);
      }
    __syncthreads();
    const int R = min(sp.q * a.group - row0, kRows);
    for (int i = threadIdx.x; i < R * (D / 4); i += kTokenWarps * 32) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kTokenWarps; w++)
        top = fmaxf(top, sml[w * kRows + r].x);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kTokenWarps; w++) {
        const float2 ml = sml[w * kRows + r];
        if (ml.y == 0.0f)
          continue;
        const float part = ml.y * fast_exp2(ml.x - top);
        const float4 x = *reinterpret_cast<const float4 *>(so + (w * kRows + r) * kPitch + d);
        sum += part;
        acc.x += part * x.x, acc.y += part * x.y, acc.z += part * x.z, acc.w += part * x.w;
      }
      const int h = head * a.group + (row0 + r) % a.group;
      if (!piece_o)
        join_sink(a.sinks, h, top, sum);
      // the weights above are relative to the warps' maximum, the sum now perhaps to the sink's
      float f = sum != 0.0f ? 1.0f / sum : 0.0f;
      if (!piece_o && a.sinks && sum != 0.0f) {
        float before = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTokenWarps; w++)
          before = fmaxf(before, sml[w * kRows + r].x);
        f *= fast_exp2(before - top);
      }
      acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
      if (piece_o) {
        *reinterpret_cast<float4 *>(piece_o + (size_t)r * D + d) = acc;
        if (d == 0)
          piece_ml[r] = make_float2(top, sum);
      } else {
        const int row = sp.row + (row0 + r) / a.group;
        store4(a, (size_t)row * a.out_row_stride + (size_t)h * D + d, acc);
      }
    }
    __syncthreads(); // the arrays may be used for the next item
  }

  __device__ __forceinline__ void item(const Call<QT> &a, const Rows::Span &sp, int s, int head, int rg, const Columns &cols,
                                       int i0, int i1, int min_pos, int max_pos, float *piece_o, float2 *piece_ml) {
    load_queries(a, sp, head, rg * kRows);
    run(a, s, head, cols, i0, i1, min_pos, max_pos);
    finish(a, sp, head, rg * kRows, piece_o, piece_ml);
  }
};

struct GroupRange { // positions of a row group
  int lo, hi;
};
__device__ __forceinline__ GroupRange group_range(const Rows::Span &sp, int group, int rg, int rows) {
  return GroupRange{sp.pos + rg * rows / group, sp.pos + min(sp.q * group - 1, rg * rows + rows - 1) / group};
}

// WHOLE: a block per (sequence, head, row group), for calls whose items are all short.  Otherwise all
// items' columns, in order, in equal pieces.
template <typename QT, int D, int MT, bool WHOLE>
__global__ void __launch_bounds__(kTokenWarps * 32, (D == 64 && MT == 1 ? 3 : 2))
    attend_tokens(Call<QT> a, int groups, Pieces pieces) {
  using K = TokenKernel<QT, D, MT>;
  pdl_prologue();
  K k;
  const int heads = a.cache.n_kv_heads;
  auto n_groups = [&](const Rows::Span &sp) {
    const long R = (long)sp.q * a.group;
    return R > kMaxTokenRows ? 0 : (int)(R + K::kRows - 1) / K::kRows;
  };
  if constexpr (WHOLE) {
    const int rg = blockIdx.x % groups, rest = blockIdx.x / groups, head = rest % heads, s = rest / heads;
    const Rows::Span sp = a.rows.span(s);
    if (rg >= n_groups(sp))
      return;
    const GroupRange gr = group_range(sp, a.group, rg, K::kRows);
    const Columns cols = columns(a.rows, a.window, a.n_first, gr.lo, gr.hi);
    k.item(a, sp, s, head, rg, cols, 0, cols.n, gr.lo, gr.hi, nullptr, nullptr);
  } else {
    // columns of a sequence and one head
    auto cost = [&](const Rows::Span &sp) {
      int n = 0;
      for (int rg = 0; rg < n_groups(sp); rg++) {
        const GroupRange gr = group_range(sp, a.group, rg, K::kRows);
        n += columns(a.rows, a.window, a.n_first, gr.lo, gr.hi).n;
      }
      return n;
    };
    __shared__ long warp_sum_of[kTokenWarps];
    __shared__ long found_base;
    __shared__ int found_seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_seqs = a.rows.n_seqs;
    const int chunk = (n_seqs + blockDim.x - 1) / blockDim.x;
    const int s0 = min((int)threadIdx.x * chunk, n_seqs), s1 = min(s0 + chunk, n_seqs);
    long mine = 0;
    for (int s = s0; s < s1; s++)
      mine += cost(a.rows.span(s));
    long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o)
        x += y;
    }
    if (lane == 31)
      warp_sum_of[warp] = x;
    if (threadIdx.x == 0)
      found_seq = n_seqs;
    __syncthreads();
    long total = 0, before = x - mine;
#pragma unroll
    for (int w = 0; w < kTokenWarps; w++) {
      before += w < warp ? warp_sum_of[w] : 0;
      total += warp_sum_of[w];
    }
    total *= heads, before *= heads;
    const long per = max((total + gridDim.x - 1) / gridDim.x, (long)kMinPages);
    long w = blockIdx.x * per;
    const long w_end = min(total, w + per);
    if (w < w_end && before <= w && w < before + mine * heads) {
      long base = before;
      for (int s = s0; s < s1; s++) {
        const long n = (long)cost(a.rows.span(s)) * heads;
        if (w < base + n) {
          found_seq = s, found_base = base;
          break;
        }
        base += n;
      }
    }
    __syncthreads();
    int4 first = make_int4(-1, 0, 0, 0);
    if (w < w_end) {
      int s = found_seq;
      long base = found_base;
      for (; s < n_seqs && w < w_end; s++) {
        const Rows::Span sp = a.rows.span(s);
        const int n = cost(sp), groups_here = n_groups(sp);
        if (n == 0)
          continue;
        while (w < w_end && w < base + (long)n * heads) {
          const int head = (int)((w - base) / n);
          long item0 = base + (long)head * n;
          for (int rg = 0; rg < groups_here && w < w_end; rg++) {
            const GroupRange gr = group_range(sp, a.group, rg, K::kRows);
            const Columns cols = columns(a.rows, a.window, a.n_first, gr.lo, gr.hi);
            const long item1 = item0 + cols.n;
            if (w < item1) {
              const int i0 = (int)(w - item0), i1 = (int)(min(item1, w_end) - item0);
              const bool whole = i0 == 0 && i1 == cols.n;
              const size_t slot = (size_t)blockIdx.x * 2 + (i0 == 0);
              k.item(a, sp, s, head, rg, cols, i0, i1, gr.lo, gr.hi, whole ? nullptr : pieces.o + slot * K::kRows * D,
                     whole ? nullptr : pieces.ml + slot * K::kRows);
              if (i0 == 0 && !whole)
                first = make_int4(s, head, rg, (int)((item1 - 1) / per));
              w = item0 + i1;
            }
            item0 = item1;
          }
        }
        base += (long)n * heads;
      }
    }
    if (threadIdx.x == 0)
      pieces.first[blockIdx.x] = first;
  }
}

// One item that was cut: block blockIdx.x has its first piece, the blocks after it the others.
template <typename QT, int D, int MT>
__global__ void __launch_bounds__(128) merge_pieces(Call<QT> a, Pieces pieces) {
  constexpr int kRows = 16 * MT;
  pdl_prologue();
  const int4 it = pieces.first[blockIdx.x];
  if (it.x < 0)
    return;
  const Rows::Span sp = a.rows.span(it.x);
  const int R = min(sp.q * a.group - it.z * kRows, kRows);
  const int i = blockIdx.y * 128 + threadIdx.x, r = i / (D / 4), d = (i % (D / 4)) * 4;
  if (r >= R)
    return;
  auto slot = [&](int b) { return ((size_t)b * 2 + (b == (int)blockIdx.x)) * kRows + r; };
  float top = -INFINITY, sum = 0.0f;
  for (int b = blockIdx.x; b <= it.w; b++)
    top = fmaxf(top, pieces.ml[slot(b)].x);
  const int row = it.z * kRows + r, h = it.y * a.group + row % a.group;
  if (a.sinks)
    top = fmaxf(top, fminf(__ldg(a.sinks + h) * kLog2e, 3e38f));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int b = blockIdx.x; b <= it.w; b++) {
    const float2 ml = pieces.ml[slot(b)];
    const float4 x = *reinterpret_cast<const float4 *>(pieces.o + slot(b) * D + d);
    const float part = ml.y != 0.0f ? ml.y * fast_exp2(ml.x - top) : 0.0f;
    sum += part;
    acc.x += part * x.x, acc.y += part * x.y, acc.z += part * x.z, acc.w += part * x.w;
  }
  if (sum != 0.0f && a.sinks)
    sum += fast_exp2(fminf(__ldg(a.sinks + h) * kLog2e, 3e38f) - top);
  const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
  store4(a, (size_t)(sp.row + row / a.group) * a.out_row_stride + (size_t)h * D + d,
         make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

// One warp per (row, query head): the plainest form.  A lane takes every 32nd token for the
// scores, then D / 32 elements of the output.
template <typename QT, int D>
__global__ void __launch_bounds__(128)
    attend_rows(Call<QT> a) {
  pdl_prologue();
  const Layer &cache = a.cache;
  const Rows &rows = a.rows;
  const int n_q_heads = a.n_q_heads, window = a.window, n_first = a.n_first;
  const float *sinks = a.sinks;
  const float scale = a.scale;
  __shared__ float q_of[4][D], p_of[4][kPage];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y * 4 + warp, row = blockIdx.x;
  if (h >= n_q_heads)
    return;
  const int s = rows.find(row, [&](int i) { return rows.start(i); });
  const Rows::Span sp = rows.span(s);
  if (row < sp.row || row >= sp.row + sp.q || (long)sp.q * (n_q_heads / cache.n_kv_heads) <= kMaxTokenRows)
    return;
  const int pos = sp.pos + row - sp.row, head = h / (n_q_heads / cache.n_kv_heads);
  bool bad = false, seen = false;
  for (int i = lane; i < D; i += 32) {
    const float q = load1(a.qkv + (size_t)row * a.row_stride + (size_t)h * D + i);
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
  for (int i = 0; i < D / 32; i++) {
    const size_t at = (size_t)row * a.out_row_stride + (size_t)h * D + i * 32 + lane;
    const float v = bad ? NAN : l > 0.0f ? acc[i] / l : 0.0f;
    if (a.out_f32)
      static_cast<float *>(a.out)[at] = v;
    else
      store1(static_cast<uint16_t *>(a.out) + at, v);
  }
}

constexpr int kMostBlocksPerSm = 4;

// Blocks of attend_tokens on the current device; the workspace is laid out for this many.
template <typename QT, int D, int MT> int token_grid() {
  const int per_sm = blocks_per_sm_smem(attend_tokens<QT, D, MT, false>, kTokenWarps * 32, TokenKernel<QT, D, MT>::kSmem);
  return sm_count() * std::min(std::max(per_sm, 1), kMostBlocksPerSm);
}
template <typename QT, int D, int MT>
void launch_tokens(cudaStream_t stream, const Call<QT> &a, void *workspace) {
  using K = TokenKernel<QT, D, MT>;
  const int heads = a.cache.n_kv_heads;
  const long most_rows = std::min((long)a.rows.max_new * a.group, (long)kMaxTokenRows);
  const int groups = (int)((most_rows + K::kRows - 1) / K::kRows);
  const long items = (long)a.rows.n_seqs * heads * groups;
  // columns of an item at most: the window and what its rows span, the first tokens, the table
  const long most = std::min(a.window > 0 ? ((long)a.window + a.rows.max_new) / kPage + 2 + ((long)a.n_first + kPage - 1) / kPage
                                          : (long)a.rows.pages_stride,
                             (long)a.rows.pages_stride);
  const dim3 block(kTokenWarps * 32);
  if (most <= 2 * kMinPages && items <= 0x7fffffff) {
    blocks_per_sm_smem(attend_tokens<QT, D, MT, true>, kTokenWarps * 32, K::kSmem);
    launch_kernel(attend_tokens<QT, D, MT, true>, dim3((unsigned)items), block, K::kSmem, stream, a, groups, Pieces{});
    return;
  }
  const int grid = (int)std::min((long)token_grid<QT, D, MT>(), items * most);
  const Pieces pieces = Pieces::at(workspace, grid, K::kRows, D);
  launch_kernel(attend_tokens<QT, D, MT, false>, dim3(grid), block, K::kSmem, stream, a, groups, pieces);
  const PdlScope chained(GPTOSS_PDL);
  launch_kernel(merge_pieces<QT, D, MT>, dim3(grid, K::kRows * D / 4 / 128), dim3(128), 0, stream, a, pieces);
}

template <typename QT, int D> void launch(cudaStream_t stream, const Call<QT> &a, void *workspace) {
  if ((long)a.rows.max_new * a.group <= 16)
    launch_tokens<QT, D, 1>(stream, a, workspace);
  else
    launch_tokens<QT, D, 2>(stream, a, workspace);
  if ((long)a.rows.max_new * a.group > kMaxTokenRows)
    launch_kernel(attend_rows<QT, D>, dim3(a.rows.T, (a.n_q_heads + 3) / 4), dim3(128), 0, stream, a);
}

template <typename QT>
void launch(cudaStream_t stream, int D, const Layer &cache, const void *qkv, long row_stride, int n_q_heads,
            const Rows &rows, float scale, int window, int n_first, const float *sinks, void *out, gptoss_dtype_t out_dtype,
            long out_row_stride, void *workspace) {
  const size_t q4 = 4 * sizeof(QT), out4 = 4 * dtype_size(out_dtype);
  const Call<QT> a = {cache, static_cast<const QT *>(qkv), row_stride, n_q_heads, n_q_heads / cache.n_kv_heads, rows, scale,
                      window, n_first, sinks, out, out_row_stride, out_dtype == GPTOSS_F32,
                      (reinterpret_cast<uintptr_t>(qkv) & (q4 - 1)) == 0 && row_stride % 4 == 0,
                      (reinterpret_cast<uintptr_t>(out) & (out4 - 1)) == 0 && out_row_stride % 4 == 0};
  if (!a.q_vec || !a.out_vec)
    note_generic_launch();
  D == 64 ? launch<QT, 64>(stream, a, workspace) : launch<QT, 128>(stream, a, workspace);
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
  return kv8::Pieces::bytes(sm_count() * kv8::kMostBlocksPerSm, 32, pool->head_dim);
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
  (qkv_dtype == GPTOSS_F32 ? kv8::launch<float> : kv8::launch<uint16_t>)(
      as_stream(stream), D, cache, qkv, row_stride, n_q_heads, rows, scale, window, n_first, sinks, out, out_dtype,
      out_row_stride, workspace);
  return launch_status();
}
