// Attention over the 8-bit paged cache (gptoss_kv8_attention) for few rows per sequence.
//
//     z_t = scale q . k_t,   out = sum_t 2^(z_t' - m) v_t / (sum_t 2^(z_t' - m) + 2^(sink' - m)),   ' = times log2(e)
//
// The rows of a sequence that share a key/value head (its new tokens x the query heads of the group)
// are the 8-wide side of a matrix instruction; one pass over the pages with the running maximum and
// sum of each row.  What bounds it is the cache's bytes, and the instructions that make fp16 of them (ten
// for eight codes).  So:
//   - a warp works alone on steps of CH tokens: one lane asks the copy engine for the keys and the values of
//     the steps to come (cp.async.bulk, 2-4 KB each, a page's keys or values of a head being consecutive) into
//     the warp's own 16 KB ring, each part with its own barrier, so that 12 to 16 KB per warp are in flight
//     at any time and the block meets only at the end;
//   - the order of a head's elements within a product and of a step's tokens is free, and is chosen so
//     that a lane needs 16 or 8 consecutive bytes of a token;
//   - codes become fp16 exactly (kv8_mma.cuh); key scales multiply the scores, value scales, powers
//     of two, multiply the codes relative to a reference of the warp (kv8_attention.cuh, also on pages far from it);
//   - queries are brought to fp16 range by a power of two per row; a bf16 row is then exact, an fp32 row
//     is two fp16 parts and two products, and so are its softmax weights, and its sums are folded (kFold), which is what
//     keeps fp32's accuracy on these tensor cores;
//   - the weights carry a factor 2^9, so that weights down to 2^-23 of the largest are normal fp16;
//   - work is cut into equal pieces of pages over all blocks whatever the lengths (a long sequence
//     beside short ones, one sequence alone); a sequence cut across blocks is joined by merge_pieces.
// Measured: 64 sequences, 8000 tokens on average, 8 heads of 64: 0.57 GB in 107 us with the join, 0.81 of a copy's
// rate.  One sequence of 131072 tokens, heads of 128: 0.27 GB in 68 us, of which 3 us finding the pieces, 5 us
// joining.  Some 700 instructions per page and warp at 2 per clock and SM: the next bound is issue, not memory.
// Most forms for 32 rows, fp32 rows or 128-wide heads need more registers than there are and spill (-Xptxas -v: up to
// 200 bytes of stores per thread for bf16 rows, 830 for 32 fp32 rows of 128).
#include <algorithm>

#include "kv8_attention.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr int kWeightBits = 9;
constexpr int kTokenWarps = 4;
constexpr int kMinPages = 8;      // of a block's piece: below that joining costs more than it saves
// What starting and ending an item costs a block, in pages (some 3 us where a page takes 0.6): without it a
// block that got many short sequences ran 130 us where the others took 90.
constexpr int kItemPages = 5;

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

// Row n of an 8-token tile of scores holds this token of the tile (the lowest bit flipped in every
// other pair): neighbouring rows and the rows of a quad's lanes then fall into both halves of the 128
// bytes that shared memory's banks repeat over.
__device__ __forceinline__ int token_of(int n) { return n ^ ((n >> 1) & 1); }

// Scores and outputs are kept transposed (tokens x rows, elements x rows): the 8-wide side of the
// matrix instruction is the rows', so that 8 rows (a group of 8 query heads and one token) waste nothing.
template <typename QT, int D, int RB, bool WHOLE> struct TokenKernel {
  static constexpr bool kSplit = sizeof(QT) == 4;                     // two fp16 parts
  static constexpr int CH = (D == 64 ? 64 : 32) / (RB == 4 ? 2 : 1);  // tokens of a step
  static constexpr int kSteps = kPage / CH;                           // steps of a page
  static constexpr int TT = CH / 16, KS = D / 16, DT = D / 16;        // 16-token tiles, products of a score, 16-element tiles
  static constexpr int kRows = 8 * RB;
  static constexpr int kPitch = D + 4; // floats of a row in shared memory
  static constexpr int kPart = CH * D;              // bytes of a step's keys, and of its values
  // Steps' keys (and values) in a warp's ring.  Short items have hardly more than one step per warp: half the
  // ring, and four blocks on an SM instead of three.
  static constexpr int kDepth = (WHOLE ? 4096 : 8192) / kPart;
  static constexpr int kResult = kRows * (kPitch * 4 + 8); // a warp's results, which lie where its ring was
  static constexpr int kRing = 2 * kDepth * kPart > kResult ? 2 * kDepth * kPart : kResult; // 8 or 16 KB per warp
  static constexpr int kSmem = kTokenWarps * (kRing + 2 * kDepth * 8 + kDepth * 16 + 4);
  static constexpr bool kFolds = kSplit && !WHOLE;
  static constexpr int kFoldSteps = kFold / (2 * TT), kFolded = kFolds ? (4 * DT + 2) * RB : 1;
  using VWord = typename std::conditional<D == 64, uint2, uint4>::type;

  uint32_t q[RB][KS][2], q_rest[kSplit ? RB : 1][kSplit ? KS : 1][2];
  float row_factor[RB][2], m[RB][2], l[RB][2], o[RB][DT][4]; // of rows 2t, 2t + 1 of each 8
  int row_pos[RB][2];                                        // -1: no such row
  int ref;             // exponent of the value scale that this warp's outputs are relative to; 0: no page has had one yet
  bool met_far;        // pages far from it were left out
  uint32_t ring, bars; // this warp's, as shared-space addresses
  int4 *slots;         // what a part is: page, step, scales
  int done;            // parts used so far, over all items
  int since;           // steps since outputs were last folded; negative: they never were
  bool lost;           // a copy did not arrive in time

  __device__ __forceinline__ void setup() {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5;
    ring = smem_u32(smem) + warp * kRing;
    bars = smem_u32(smem) + kTokenWarps * kRing + warp * 2 * kDepth * 8;
    slots = reinterpret_cast<int4 *>(smem + kTokenWarps * (kRing + 2 * kDepth * 8)) + warp * kDepth;
    done = 0, lost = false;
    if ((threadIdx.x & 31) == 0) {
      for (int i = 0; i < 2 * kDepth; i++)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + i * 8) : "memory");
      mbar_init_fence();
    }
    __syncwarp();
  }

  // The group's queries as right operands (lane: row g), a row's elements in the order that K's lanes
  // have them; then what a lane keeps of the rows it has scores of (2t, 2t + 1).
  __device__ __forceinline__ void load_queries(const Call<QT> &a, const Rows::Span &sp, int head, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, R = sp.q * a.group;
#pragma unroll
    for (int b = 0; b < RB; b++) {
      const int r = row0 + 8 * b + g;
      const bool is = r < R;
      const int token = is ? r / a.group : 0, h = head * a.group + (is ? r % a.group : 0);
      const QT *p = a.qkv + (size_t)(sp.row + token) * a.row_stride + (size_t)h * D + 16 * t;
      float v[KS][4], top = 0.0f;
      bool odd = false;
#pragma unroll
      for (int j = 0; j < KS; j++)
        load4(p + (j / 4) * 64 + (j % 4) * 4, a.q_vec, v[j]);
#pragma unroll
      for (int j = 0; j < KS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          odd = odd || !(fabsf(v[j][e]) <= 3.402823466e38f);
          top = fmaxf(top, fabsf(v[j][e]));
        }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        odd = __shfl_xor_sync(0xffffffffu, (int)odd, x) || odd;
      }
      // largest |q| into [2^13, 2^14); rows too small for the exponent keep a factor of 2^126
      const int up = odd || top == 0.0f ? 0 : max(min(13 - (exponent_field(top) - 127), 126), -126);
      const float f = odd || !is ? 0.0f : two_to(up) * (a.scale < 0.0f ? -1.0f : 1.0f);
#pragma unroll
      for (int j = 0; j < KS; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float x = odd || !is ? 0.0f : v[j][2 * e] * f, y = odd || !is ? 0.0f : v[j][2 * e + 1] * f;
          q[b][j][e] = pack_f16(x, y);
          if constexpr (kSplit)
            q_rest[b][j][e] = pack_rest(q[b][j][e], x, y);
        }
      const float factor = odd ? NAN : fabsf(a.scale) * kLog2e * two_to(-up);
      const int pos = is ? sp.pos + token : -1;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        row_factor[b][e] = __shfl_sync(0xffffffffu, factor, (2 * t + e) * 4);
        row_pos[b][e] = __shfl_sync(0xffffffffu, pos, (2 * t + e) * 4);
      }
    }
  }

  __device__ __forceinline__ void begin() {
    ref = 0, met_far = false, since = -kFoldSteps;
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        m[b][e] = -INFINITY, l[b][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < DT; j++)
          o[b][j][e] = o[b][j][2 + e] = 0.0f;
      }
  }

  // Outputs so far to (or, at the end, from) this thread's memory, where they are relative to the rows' maxima of then.
  template <bool BACK> __device__ __forceinline__ void fold(volatile float (&kept)[kFolded], bool first) {
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        volatile float *at = kept + (2 * b + e) * (2 * DT + 1);
        const float then = first ? -INFINITY : at[2 * DT], f = then > -INFINITY ? fast_exp2(then - m[b][e]) : 0.0f;
#pragma unroll
        for (int j = 0; j < DT; j++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            float &x = o[b][j][2 * half + e];
            const float sum = first ? x : fmaf(at[2 * j + half], f, x);
            if (!BACK)
              at[2 * j + half] = sum;
            x = BACK ? sum : 0.0f;
          }
        if (!BACK)
          at[2 * DT] = m[b][e];
      }
  }

  __device__ __forceinline__ void scores(float (&s)[RB][TT][4], uint32_t keys) {
    const int lane = threadIdx.x & 31;
    keys += token_of(lane >> 2) * D + (lane & 3) * 16;
#pragma unroll
    for (int i = 0; i < TT; i++) {
      uint4 K[2][D / 64]; // tokens g and g + 8 of the tile
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int j = 0; j < D / 64; j++)
          K[half][j] = lds16(keys + (16 * i + 8 * half) * D + j * 64);
#pragma unroll
      for (int b = 0; b < RB; b++)
        s[b][i][0] = s[b][i][1] = s[b][i][2] = s[b][i][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; j++) {
        const uint32_t u = biased(word(K[0][j / 4], j % 4)), v = biased(word(K[1][j / 4], j % 4));
        const uint32_t k[4] = {minus_1152(low_pair(u)), minus_1152(low_pair(v)), minus_1152(high_pair(u)),
                               minus_1152(high_pair(v))};
#pragma unroll
        for (int b = 0; b < RB; b++) {
          mma_f16(s[b][i], k, q[b][j][0], q[b][j][1]);
          if constexpr (kSplit)
            mma_f16(s[b][i], k, q_rest[b][j][0], q_rest[b][j][1]);
        }
      }
    }
  }

  // s becomes the weights of the step's tokens first_token ..
  template <bool MASKED>
  __device__ __forceinline__ void weigh(float (&s)[RB][TT][4], float key_scale, int first_token, int window, int n_first) {
    const int first = first_token + token_of((threadIdx.x & 31) >> 2); // tile i's rows g, g + 8: tokens first + 16 i, + 8
    bool moved = false;
    float fade[RB][2];
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        uint32_t seen = 0;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < TT; i++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            if constexpr (MASKED) {
              const int token = first + 16 * i + 8 * half, pos = row_pos[b][e];
              const bool ok = token <= pos && (window <= 0 || token > pos - window || token < n_first);
              seen |= (uint32_t)ok << (2 * i + half);
              top = fmaxf(top, ok ? s[b][i][2 * half + e] : -INFINITY);
            } else {
              top = fmaxf(top, s[b][i][2 * half + e]);
            }
          }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float f = at_most(row_factor[b][e] * key_scale, kMostFactor);
        const float now = top > -INFINITY ? fmaxf(m[b][e], top * f) : m[b][e];
        const float base = now > -INFINITY ? now : 0.0f;
        const float a = fast_exp2(m[b][e] - base), off = (float)kWeightBits - base;
        m[b][e] = now;
        moved = moved || a != 1.0f;
        fade[b][e] = a;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < TT; i++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            float p = fast_exp2(fmaf(s[b][i][2 * half + e], f, off));
            if constexpr (MASKED)
              p = seen >> (2 * i + half) & 1 ? p : 0.0f;
            s[b][i][2 * half + e] = p;
            sum += p;
          }
        l[b][e] = fmaf(l[b][e], a, sum);
      }
    if (__any_sync(0xffffffffu, moved))
#pragma unroll
      for (int b = 0; b < RB; b++)
#pragma unroll
        for (int j = 0; j < DT; j++)
          o[b][j][0] *= fade[b][0], o[b][j][1] *= fade[b][1], o[b][j][2] *= fade[b][0], o[b][j][3] *= fade[b][1];
  }

  __device__ __forceinline__ void add_values(const float (&s)[RB][TT][4], int v_exp, uint32_t values) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    const uint32_t even = values + token_of(2 * t) * D + (lane >> 2) * (D / 8), odd = values + token_of(2 * t + 1) * D + (lane >> 2) * (D / 8);
    uint32_t mul, add;
    value_factor(v_exp, ref, mul, add);
#pragma unroll
    for (int i = 0; i < TT; i++) {
      uint32_t p[RB][2], rest[kSplit ? RB : 1][2];
#pragma unroll
      for (int b = 0; b < RB; b++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint32_t w = pack_f16(s[b][i][2 * half], s[b][i][2 * half + 1]);
          p[b][half] = transposed(w);
          if constexpr (kSplit)
            rest[b][half] = transposed(pack_rest(w, s[b][i][2 * half], s[b][i][2 * half + 1]));
        }
      VWord V[4]; // of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of the tile
#pragma unroll
      for (int c = 0; c < 4; c++)
        load_word(V[c], (c & 1 ? odd : even) + (16 * i + 8 * (c >> 1)) * D);
#pragma unroll
      for (int w = 0; w < D / 32; w++) { // words of 4 elements: two 16-element tiles' rows g and g + 8
        uint32_t c[4];
#pragma unroll
        for (int x = 0; x < 4; x++)
          c[x] = biased(word(V[x], w));
#pragma unroll
        for (int hi = 0; hi < 2; hi++) {
          const uint32_t x = __byte_perm(c[0], c[1], hi ? 0x7362 : 0x5140), y = __byte_perm(c[2], c[3], hi ? 0x7362 : 0x5140);
          const uint32_t v[4] = {scaled_pair(low_pair(x), mul, add), scaled_pair(high_pair(x), mul, add),
                                 scaled_pair(low_pair(y), mul, add), scaled_pair(high_pair(y), mul, add)};
#pragma unroll
          for (int b = 0; b < RB; b++) {
            mma_f16(o[b][2 * w + hi], v, p[b][0], p[b][1]);
            if constexpr (kSplit)
              mma_f16(o[b][2 * w + hi], v, rest[b][0], rest[b][1]);
          }
        }
      }
    }
  }
  static __device__ __forceinline__ void load_word(uint4 &v, uint32_t a) { v = lds16(a); }
  static __device__ __forceinline__ void load_word(uint2 &v, uint32_t a) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  }
  static __device__ __forceinline__ uint32_t word(uint2 v, int w) { return w ? v.y : v.x; }
  static __device__ __forceinline__ uint32_t word(uint4 v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

  // Part p of the warp's sequence of keys (kind 0) or values (kind 1): where it lies, its barrier.
  __device__ __forceinline__ uint32_t part_at(int p, int kind) const { return ring + (2 * (p % kDepth) + kind) * kPart; }
  __device__ __forceinline__ uint32_t bar_at(int p, int kind) const { return bars + (2 * (p % kDepth) + kind) * 8; }
  // One lane asks the copy engine for a part; its barrier completes when the bytes are there.
  __device__ __forceinline__ void start(int p, int kind, const int8_t *block, int step) const {
    const uint32_t bar = bar_at(p, kind);
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kPart) : "memory");
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(part_at(p, kind)),
                 "l"(block + (size_t)(kind * kPage + step * CH) * D), "r"(kPart), "r"(bar)
                 : "memory");
  }
  // One answer for the warp: where the wait runs out, lanes that had seen the barrier complete must not go on alone to
  // what the whole warp does next.
  __device__ __forceinline__ bool arrived(int p, int kind) const {
    return __all_sync(0xffffffffu, mbar_wait_at(bar_at(p, kind), p / kDepth & 1));
  }

  // The columns [i0, i1) of an item, steps dealt to the block's warps in turn.
  __device__ __forceinline__ void run(const Call<QT> &a, const Rows::Span &sp, int s, int head, int row0, const Columns &cols,
                                      int i0, int i1, int min_pos, int max_pos, volatile float (&kept)[kFolded]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j0 = i0 * kSteps + warp, end = i1 * kSteps;
    const int steps = j0 < end && !lost ? (end - j0 + kTokenWarps - 1) / kTokenWarps : 0;
    const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
    int page_of = -1, held = -32, ahead = 0; // lane l has the page and scales of step held + l; steps before `ahead` are asked for
    float2 scale_of = make_float2(0.0f, 0.0f);
    int asked = done; // parts
    auto ask_keys = [&](bool values_too) { // of the next step that has a page
      for (; ahead < steps; ahead = held + 32) {
        if (ahead >= held + 32) {
          held += 32;
          const int j = j0 + kTokenWarps * (held + lane);
          page_of = j < end ? a.cache.checked(__ldg(table + cols.at(j / kSteps))) : -1;
          if (page_of >= 0)
            scale_of = *reinterpret_cast<const float2 *>(a.cache.scale(page_of, head));
        }
        const unsigned there = __ballot_sync(0xffffffffu, page_of >= 0) >> (ahead - held);
        if (there) {
          ahead += __ffs(there) - 1;
          const int page = __shfl_sync(0xffffffffu, page_of, ahead - held);
          const int step = j0 + kTokenWarps * ahead;
          const int8_t *block = a.cache.template block<D>(page, head);
          if (lane == 0) { // the copies first: they need the page alone, and its scales may still be on their way
            start(asked, 0, block, step % kSteps);
            if (values_too)
              start(asked, 1, block, step % kSteps);
          }
          const float ks = __shfl_sync(0xffffffffu, scale_of.x, ahead - held), vs = __shfl_sync(0xffffffffu, scale_of.y, ahead - held);
          if (lane == 0)
            slots[asked % kDepth] = make_int4(page, step, __float_as_int(ks), __float_as_int(vs));
          asked++, ahead++;
          return;
        }
      }
    };
    auto ask_values = [&](int p) {
      if (p < asked && lane == 0) {
        const int4 it = slots[p % kDepth];
        start(p, 1, a.cache.template block<D>(it.x, head), it.y % kSteps);
      }
    };
    begin();
#pragma unroll 1
    for (int d = 0; d < kDepth; d++)
      ask_keys(true);
    load_queries(a, sp, head, row0); // while the first parts are on their way
#pragma unroll 1
    for (; done < asked; done++) {
      __syncwarp();
      const int4 it = slots[done % kDepth];
      if (!arrived(done, 0)) {
        lost = true;
        break;
      }
      float w[RB][TT][4];
      const int v_exp = exponent_field(__int_as_float(it.w));
      if (ref == 0) {
        ref = pick_ref(page_of >= 0 ? exponent_field(scale_of.y) : 0);
        ref = ref ? ref : v_exp; // where the lanes are on to pages without a scale
      }
      if (is_far(v_exp, ref)) { // left to finish: its parts are given back as they are
        met_far = true;
        if (!arrived(done, 1)) {
          lost = true;
          break;
        }
        __syncwarp();
        ask_keys(true);
        continue;
      }
      scores(w, part_at(done, 0));
      __syncwarp(); // every lane has read the keys and the slot
      ask_keys(false);
      const int token = cols.at(it.y / kSteps) * kPage + (it.y % kSteps) * CH;
      if (token + CH - 1 <= min_pos && (a.window <= 0 || token > max_pos - a.window || token + CH <= a.n_first))
        weigh<false>(w, __int_as_float(it.z), token, a.window, a.n_first);
      else
        weigh<true>(w, __int_as_float(it.z), token, a.window, a.n_first);
      if (!arrived(done, 1)) {
        lost = true;
        break;
      }
      add_values(w, v_exp, part_at(done, 1));
      if constexpr (kFolds)
        if (++since == 0 || since == kFoldSteps)
          fold<false>(kept, since == 0), since = 0;
      __syncwarp();
      ask_values(done + kDepth);
    }
    if (lost && done < asked) { // counted; what is still on its way is waited for (again with a limit) before the block ends
      if (lane == 0 && a.giveups)
        atomicAdd(a.giveups, 1u);
      for (int p = done; p < asked; p++)
        arrived(p, 0), arrived(p, 1);
      done = asked;
    }
    if constexpr (kFolds)
      if (since >= 0)
        fold<true>(kept, false);
  }

  // The warps' results, and the far pages of columns [i0, i1), joined: into the output, or into a piece for
  // merge_pieces.  Whole block.
  __device__ __forceinline__ void finish(const Call<QT> &a, const Rows::Span &sp, int s, int head, int row0, const Columns &cols,
                                         int i0, int i1, float *piece_o, float2 *piece_ml) {
    extern __shared__ __align__(16) uint8_t smem[];
    auto so = [&](int w, int r) { return reinterpret_cast<float *>(smem + w * kRing) + r * kPitch; };
    auto sml = [&](int w) { return reinterpret_cast<float2 *>(smem + w * kRing + kRows * kPitch * 4); };
    int *const refs = reinterpret_cast<int *>(smem + kTokenWarps * (kRing + 2 * kDepth * 8 + kDepth * 16)); // the warps'
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const float unit = two_to(ref - 127);
    if (lane == 0)
      refs[warp] = ref;
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = l[b][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int r = 8 * b + 2 * t + e;
        if (g == 0)
          sml(warp)[r] = make_float2(m[b][e], sum * two_to(-kWeightBits));
        const float f = sum > 0.0f ? (float)(1 << (kNear - kValueBits)) / sum : 0.0f;
        float *row = so(warp, r) + g * (D / 8);
        auto mean = [&](float x) { return finite(x * f * unit); }; // 64 x 2^122 is not; a NaN shows by its sum
#pragma unroll
        for (int j = 0; j < DT; j += 2)
          *reinterpret_cast<float4 *>(row + 2 * j) =
              make_float4(mean(o[b][j][e]), mean(o[b][j][2 + e]), mean(o[b][j + 1][e]), mean(o[b][j + 1][2 + e]));
      }
    const int R = min(sp.q * a.group - row0, kRows);
    if (__syncthreads_or(met_far)) { // a row's far pages go to the result of the warp that sums them
      for (int r = warp; r < R; r += kTokenWarps) {
        const int token = (row0 + r) / a.group;
        const QT *row = a.qkv + (size_t)(sp.row + token) * a.row_stride + (size_t)(head * a.group + (row0 + r) % a.group) * D;
        far_row<D>(a, s, head, cols, i0, i1, row, sp.pos + token, refs, kTokenWarps, kSteps, so(warp, r), sml(warp) + r);
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < R * (D / 4); i += kTokenWarps * 32) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4, h = head * a.group + (row0 + r) % a.group;
      const bool sink = !piece_o && a.sinks;
      const float z = sink ? sink_of(a, h) : -INFINITY;
      float2 ml[kTokenWarps];
      float top = z, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kTokenWarps; w++) {
        ml[w] = sml(w)[r];
        top = fmaxf(top, ml[w].x);
      }
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kTokenWarps; w++) {
        const float part = ml[w].y != 0.0f ? ml[w].y * fast_exp2(ml[w].x - top) : 0.0f; // a NaN passes
        const float4 x = *reinterpret_cast<const float4 *>(so(w, r) + d);
        const float of = part * two_to(-kSumBits);
        sum += part;
        acc.x += of * x.x, acc.y += of * x.y, acc.z += of * x.z, acc.w += of * x.w;
      }
      if (sink && sum != 0.0f)
        sum += fast_exp2(z - top);
      const float f = sum != 0.0f ? (float)(1 << kSumBits) / sum : 0.0f;
      acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
      if (piece_o) {
        *reinterpret_cast<float4 *>(piece_o + (size_t)r * D + d) =
            make_float4(finite(acc.x), finite(acc.y), finite(acc.z), finite(acc.w));
        if (d == 0)
          piece_ml[r] = make_float2(top, sum);
      } else {
        const int row = sp.row + (row0 + r) / a.group;
        store4(a, (size_t)row * a.out_row_stride + (size_t)h * D + d, acc);
      }
    }
    fence_async_smem();
    __syncthreads(); // the rings may be written by the copy engine again
  }

  __device__ __forceinline__ void item(const Call<QT> &a, const Rows::Span &sp, int s, int head, int rg, const Columns &cols,
                                       int i0, int i1, int min_pos, int max_pos, float *piece_o, float2 *piece_ml) {
    volatile float kept[kFolded]; // volatile: in memory, the registers are full
    run(a, sp, s, head, rg * kRows, cols, i0, i1, min_pos, max_pos, kept);
    finish(a, sp, s, head, rg * kRows, cols, i0, i1, piece_o, piece_ml);
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
template <typename QT, int D, int RB, bool WHOLE>
__global__ void __launch_bounds__(kTokenWarps * 32, RB <= 2 ? (WHOLE && D == 64 && RB == 1 ? 4 : 3) : 2)
    attend_tokens(const __grid_constant__ Call<QT> a, int above, int upto, int groups, Pieces pieces) { // sequences of above < rows <= upto
  using K = TokenKernel<QT, D, RB, WHOLE>;
  pdl_prologue();
  K k;
  k.setup();
  const int heads = a.cache.n_kv_heads;
  auto n_groups = [&](const Rows::Span &sp) {
    const long R = (long)sp.q * a.group;
    return R > upto || R <= above ? 0 : (int)(R + K::kRows - 1) / K::kRows;
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
    // work of a sequence and one head: its items' columns and kItemPages for each item
    auto cost = [&](const Rows::Span &sp) {
      int n = 0;
      for (int rg = 0; rg < n_groups(sp); rg++) {
        const GroupRange gr = group_range(sp, a.group, rg, K::kRows);
        n += columns(a.rows, a.window, a.n_first, gr.lo, gr.hi).n + kItemPages;
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
            const long item1 = item0 + kItemPages + cols.n; // its columns are the last part of [item0, item1)
            if (w < item1) {
              const int i0 = max((int)(w - item0) - kItemPages, 0), i1 = (int)(min(item1, w_end) - item0) - kItemPages;
              if (i0 < i1) {
                const bool whole = i0 == 0 && i1 == cols.n;
                const size_t slot = (size_t)blockIdx.x * 2 + (i0 == 0);
                k.item(a, sp, s, head, rg, cols, i0, i1, gr.lo, gr.hi, whole ? nullptr : pieces.o + slot * K::kRows * D,
                       whole ? nullptr : pieces.ml + slot * K::kRows);
                if (i0 == 0 && !whole)
                  first = make_int4(s, head, rg, (int)((item1 - 1) / per));
              }
              w = min(item1, w_end);
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

// One item that was cut: block blockIdx.x has its first piece, the blocks after it the others.  Threads
// share 8 rows' elements four at a time, and the pieces among themselves where that leaves threads over (one
// long sequence may have fifty).
constexpr int kMergeThreads = 512;
template <typename QT, int D, int RB> __global__ void __launch_bounds__(kMergeThreads) merge_pieces(Call<QT> a, Pieces pieces) {
  constexpr int kRows = 8 * RB, D4 = D / 4;
  __shared__ float4 part_of[kMergeThreads];
  __shared__ float sum_of[kMergeThreads];
  pdl_prologue();
  const int4 it = pieces.first[blockIdx.x];
  if (it.x < 0)
    return;
  const Rows::Span sp = a.rows.span(it.x);
  const int row0 = blockIdx.y * 8, R = min(min(sp.q * a.group - it.z * kRows, kRows) - row0, 8);
  if (R <= 0)
    return;
  const int n = R * D4, slices = kMergeThreads / n, slice = threadIdx.x / n, i = threadIdx.x % n;
  const int r = row0 + i / D4, d = (i % D4) * 4;
  const int row = it.z * kRows + r, h = it.y * a.group + row % a.group;
  auto slot = [&](int b) { return ((size_t)b * 2 + (b == (int)blockIdx.x)) * kRows + r; };
  const float z = a.sinks ? sink_of(a, h) : -INFINITY;
  float top = z, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int b = blockIdx.x; b <= it.w; b++)
    top = fmaxf(top, pieces.ml[slot(b)].x);
  if (slice < slices)
#pragma unroll 8
    for (int b = blockIdx.x + slice; b <= it.w; b += slices) {
      const float2 ml = pieces.ml[slot(b)];
      const float4 x = *reinterpret_cast<const float4 *>(pieces.o + slot(b) * D + d);
      const float part = ml.y != 0.0f ? ml.y * fast_exp2(ml.x - top) : 0.0f, of = part * two_to(-kSumBits);
      sum += part;
      acc.x += of * x.x, acc.y += of * x.y, acc.z += of * x.z, acc.w += of * x.w;
    }
  part_of[threadIdx.x] = acc, sum_of[threadIdx.x] = sum;
  __syncthreads();
  if (slice != 0)
    return;
  for (int k = 1; k < slices; k++) {
    const float4 x = part_of[k * n + i];
    sum += sum_of[k * n + i];
    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
  }
  if (sum != 0.0f && a.sinks)
    sum += fast_exp2(z - top);
  const float f = sum != 0.0f ? (float)(1 << kSumBits) / sum : 0.0f;
  store4(a, (size_t)(sp.row + row / a.group) * a.out_row_stride + (size_t)h * D + d,
         make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

constexpr int kMostBlocksPerSm = 4;

// Blocks of attend_tokens on the current device; the workspace is laid out for this many.
template <typename QT, int D, int RB> int token_grid() {
  const int per_sm = blocks_per_sm_smem(attend_tokens<QT, D, RB, false>, kTokenWarps * 32, TokenKernel<QT, D, RB, false>::kSmem);
  return sm_count() * std::min(std::max(per_sm, 1), kMostBlocksPerSm);
}
template <typename QT, int D, int RB>
void launch_tokens(cudaStream_t stream, const Call<QT> &a, int above, int upto, void *workspace) {
  using K = TokenKernel<QT, D, RB, false>;
  const int heads = a.cache.n_kv_heads;
  const long most_rows = std::min((long)a.rows.max_new * a.group, (long)upto);
  const int groups = (int)((most_rows + K::kRows - 1) / K::kRows);
  const long items = (long)a.rows.n_seqs * heads * groups;
  // columns of an item at most: the window and what its rows span, the first tokens, the table
  const long most = std::min(a.window > 0 ? ((long)a.window + a.rows.max_new) / kPage + 2 + ((long)a.n_first + kPage - 1) / kPage
                                          : (long)a.rows.pages_stride,
                             (long)a.rows.pages_stride);
  const dim3 block(kTokenWarps * 32);
  if (most <= 2 * kMinPages && items <= 0x7fffffff) {
    constexpr int kSmem = TokenKernel<QT, D, RB, true>::kSmem;
    (void)blocks_per_sm_smem(attend_tokens<QT, D, RB, true>, kTokenWarps * 32, kSmem);
    launch_kernel(attend_tokens<QT, D, RB, true>, dim3((unsigned)items), block, kSmem, stream, a, above, upto, groups, Pieces{});
    return;
  }
  const int grid = (int)std::min((long)token_grid<QT, D, RB>(), items * most);
  const Pieces pieces = Pieces::at(workspace, grid, K::kRows, D);
  launch_kernel(attend_tokens<QT, D, RB, false>, dim3(grid), block, K::kSmem, stream, a, above, upto, groups, pieces);
  const PdlScope chained(GPTOSS_PDL);
  launch_kernel(merge_pieces<QT, D, RB>, dim3(grid, RB), dim3(kMergeThreads), 0, stream, a, pieces);
}

// One launch after the other on the same workspace: each has joined its pieces before the next begins.
template <typename QT, int D> void launch(cudaStream_t stream, const Call<QT> &a, void *workspace) {
  const long rows = (long)a.rows.max_new * a.group;
  if (rows <= 8)
    launch_tokens<QT, D, 1>(stream, a, 0, 8, workspace);
  else if (rows <= 16)
    launch_tokens<QT, D, 2>(stream, a, 0, 16, workspace);
  else {
    // Sequences may be of very different row counts: single tokens among chunks of prompts.  Those get the kernel for
    // 8 rows (64 sequences over 0.57 GB, one with 512 rows and the others with one: 294 us instead of 435; a batch that has
    // none such pays 4 us for asking), unless the sizes say that all have the same.
    const bool mixed = a.group <= 8 && (long)a.rows.n_seqs * a.rows.max_new > a.rows.T;
    if (mixed)
      launch_tokens<QT, D, 1>(stream, a, 0, 8, workspace);
    launch_tokens<QT, D, 4>(stream, a, mixed ? 8 : 0, kMaxTokenRows, workspace);
  }
  if (rows > kMaxTokenRows)
    launch_tiles(stream, a, D, workspace);
}

template <typename QT>
void launch(cudaStream_t stream, int D, const Layer &cache, const void *qkv, long row_stride, int n_q_heads,
            const Rows &rows, float scale, int window, int n_first, const float *sinks, void *out, gptoss_dtype_t out_dtype,
            long out_row_stride, void *workspace) {
  const size_t q4 = 4 * sizeof(QT), out4 = 4 * dtype_size(out_dtype);
  const Call<QT> a = {cache, static_cast<const QT *>(qkv), row_stride, n_q_heads / cache.n_kv_heads, rows, scale, window,
                      n_first, sinks, out, out_row_stride, wait_giveups_word(), out_dtype == GPTOSS_F32,
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
  if (kv8::check_pool(pool) != GPTOSS_OK || T <= 0 || T > kv8::kMaxTokens || n_q_heads <= 0 || n_seqs <= 0 ||
      n_seqs > kv8::kMaxTokens / 4 || max_new <= 0 || n_q_heads % pool->n_kv_heads)
    return 0;
  const int group = n_q_heads / pool->n_kv_heads;
  const size_t pieces = kv8::Pieces::bytes(sm_count() * kv8::kMostBlocksPerSm, 32, pool->head_dim);
  const bool tiles = (long)std::min(max_new, T) * group > kv8::kMaxTokenRows;
  return std::max(pieces, tiles ? kv8::tiles_workspace(T, group, pool->n_kv_heads, n_seqs, pool->head_dim) : 0);
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
  if (n_q_heads % pool->n_kv_heads != 0)
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
