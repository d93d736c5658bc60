// Attention over the 8-bit paged cache for many rows per sequence (prompts, chunks of prompts), on the
// fifth-generation tensor cores.
//
// The mathematics is that of kv8_attention.cu.  A block takes 256 rows (new tokens x query heads) of one
// sequence and key/value head as two tiles of 128, and goes over the pages they see, a page's 64 tokens at a
// time:
//     S = Q K^T   128 x 64, queries and keys from shared memory, sums in tensor memory
//     P = 2^(S f - m)  by one thread per row, written back over S as fp16
//     O += P V    128 x D, P from tensor memory, values from shared memory
// What bounds it at D = 64 is the exponential (16 per clock and SM: 512 clocks for a 128 x 64 tile against some
// 320 of matrix instructions), so everything else is kept off those warps and overlapped:
//   - warps 0-3 and 4-7: softmax of tile 0 and 1.  A row's running maximum is raised only when the new one is
//     2^8 above it, so that O is rescaled a few times per row and not once per page;
//   - warps 8-11: codes (brought by the copy engine into a ring of raw pages) to fp16 in the 128-byte swizzled
//     form the matrix instruction reads; once for both tiles;
//   - warp 12: one thread issues the matrix instructions.  Scores have two buffers per tile, so the next page's
//     are ready when a softmax warp comes for them.
// Queries, codes and weights are represented as in kv8_attention.cu: fp16, exact for codes and bf16 rows; fp32 rows
// and their weights in two parts with two products.
// Every wait is bounded: one that runs out is counted, tells the block's other roles, and the block frees its
// tensor memory and ends.
#include <type_traits>

#include "kv8_attention.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr int kTile = 128, kTiles = 2, kTileThreads = 416;
constexpr int kTileBits = 7, kRise = 8; // weights are at most 2^(kTileBits + kRise) < 65504
constexpr int kMeta = 16;

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Registers a thread of this warpgroup may use from here on.  The block starts with 13 x 32 x 128; the converting warps go
// down to 72 (128 threads) before the softmax warps' 152 (256) are granted: 9216 + 38912, and 4096 of the issuing
// warp, are 52224 of 53248.
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
// One arrival for a warp, after all its lanes.
__device__ __forceinline__ void arrive_warp(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Shared-memory operand in the 128-byte swizzle: rows of 128 bytes in groups of 8 (1024 bytes).  For keys and
// queries a row is 64 elements of one token and `other` is unused; for values, read across (a row is one step of
// the product's inner index), `other` is the distance of the next 64 elements.  The low word alone has addresses:
// operands are moved on by adding bytes / 16 to it.
__device__ __forceinline__ uint32_t operand_low(uint32_t address, uint32_t other) { return (address >> 4 & 0x3fff) | other >> 4 << 16; }
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
// fp16 x fp16 -> fp32, 128 x n; `across`: the right operand as values lie.
__host__ __device__ constexpr uint32_t shape_of(int n, bool across) {
  return 1u << 4 | (across ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kTile >> 4) << 24;
}
// Issued by the lane that has `leader` set.  The whole warp comes here, so that operands stay in uniform
// registers: with one lane in a branch of its own, moving them there took 2400 clocks per page.
__device__ __forceinline__ void mma_smem(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add, uint32_t leader) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
               "r"(a), "r"(b), "r"(shape), "r"(add), "r"(leader), "r"(kOperandHigh)
               : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add, uint32_t leader) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "mov.b64 b, {%2, %6};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
               "r"(a), "r"(b), "r"(shape), "r"(add), "r"(leader), "r"(kOperandHigh)
               : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t leader) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
               "r"(leader)
               : "memory");
}
__device__ __forceinline__ uint32_t elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
#define GPTOSS_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define GPTOSS_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of the calling warp's 32 lanes; the values are there after tmem_loaded.
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *x) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
               "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : GPTOSS_R8(x, 0), GPTOSS_R8(x, 8), GPTOSS_R8(x, 16), GPTOSS_R8(x, 24)
               : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t *x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
               "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
               GPTOSS_W8(x, 0), GPTOSS_W8(x, 8), GPTOSS_W8(x, 16), GPTOSS_W8(x, 24)
               : "memory");
}
#undef GPTOSS_R8
#undef GPTOSS_W8
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename QT, int D> struct TileKernel {
  static constexpr bool kSplit = sizeof(QT) == 4;
  static constexpr int kKeyStages = D == 64 ? 4 : kSplit ? 2 : 3, kValueStages = kKeyStages, kRawStages = D == 64 ? 4 : kSplit ? 2 : 3;
  static constexpr int kQueryBytes = kTile * D * 2;                    // of a tile and part
  static constexpr int kPageBytes = kPage * D * 2;                     // a page's keys or values as fp16
  static constexpr int kRawBytes = 2 * kPage * D;                      // a page's codes, keys then values
  static constexpr int kQueries = 0, kKeys = kQueries + kTiles * (kSplit ? 2 : 1) * kQueryBytes;
  static constexpr int kValues = kKeys + kKeyStages * kPageBytes, kRaw = kValues + kValueStages * kPageBytes;
  static constexpr int kMetaAt = kRaw + kRawStages * kRawBytes, kBars = kMetaAt + kMeta * 16;
  // barriers
  static constexpr int kQueryFull = 0, kScoreFull = 1 /* tile, buffer */, kWeightFull = kScoreFull + 4 /* tile, buffer */,
                       kOutDone = kWeightFull + 4 /* tile */, kKeyFull = kOutDone + 2, kKeyFree = kKeyFull + kKeyStages,
                       kValueFull = kKeyFree + kKeyStages, kValueFree = kValueFull + kValueStages,
                       kRawFull = kValueFree + kValueStages, kRawFree = kRawFull + kRawStages, kDrained = kRawFree + kRawStages,
                       kBarCount = kDrained + 1;
  static constexpr int kTmemAt = kBars + kBarCount * 8, kStopAt = kTmemAt + 4;
  static constexpr int kSmem = kStopAt + 4 + 1024; // the base is brought to 1024 bytes, the swizzle's period
  static_assert(kSmem <= 232448, "shared memory of a block");

  uint32_t base;
  volatile int *stop;
  unsigned *giveups;

  __device__ __forceinline__ uint32_t bar(int i) const { return base + kBars + i * 8; }
  // False: the block is to end (this wait ran out, or another role's did).
  __device__ __forceinline__ bool wait(int i, uint32_t parity) const {
    if (mbar_try_at(bar(i), parity))
      return true;
    const long long t0 = clock64();
    while (!mbar_try_at(bar(i), parity)) {
      if (*stop)
        return false;
      if (clock64() - t0 > kWaitCycles) {
        *stop = 1;
        if (giveups)
          atomicAdd(giveups, 1u);
        return false;
      }
    }
    return true;
  }

  // The same by a whole warp, with one answer: a warp stays together also when it ends early.
  __device__ __forceinline__ bool wait_warp(int i, uint32_t parity) const { return __all_sync(0xffffffffu, wait(i, parity)); }

  // 16-byte piece c of row r in the swizzled form; rows of 64 elements, `rows` of them per part.
  static __device__ __forceinline__ uint32_t swizzled(int r, int c, int rows) {
    return (uint32_t)(c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }
  static __device__ __forceinline__ void store16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
  }
};

struct Meta { // of a page: its first token (-1: there are no more), key scale, the exponent values are relative to
  int token;
  float key_scale;
  int value_exp, unused;
};

template <typename QT, int D>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tiles(Call<QT> a) {
  using K = TileKernel<QT, D>;
  constexpr bool kSplit = K::kSplit;
  extern __shared__ uint8_t raw_smem[];
  pdl_prologue();
  // the unit: 256 rows of a sequence and head; the last ones, which see most, first
  const int heads = a.cache.n_kv_heads, head = blockIdx.x % heads, unit = (int)(gridDim.x / heads) - 1 - (int)(blockIdx.x / heads);
  auto unit0 = [&](int s) { return (int)((long)a.rows.start(s) * a.group / (kTile * kTiles)) + s; };
  const int s = a.rows.find(unit, unit0);
  const Rows::Span sp = a.rows.span(s);
  const long R = (long)sp.q * a.group, row0 = (long)(unit - unit0(s)) * kTile * kTiles;
  if (unit < unit0(s) || R <= kMaxTokenRows || row0 >= R)
    return;
  const int tiles = R - row0 > kTile ? 2 : 1;
  auto pos_of = [&](long row) { return sp.pos + (int)(min(row, R - 1) / a.group); };
  const Columns cols = columns(a.rows, a.window, a.n_first, pos_of(row0), pos_of(row0 + kTile * kTiles - 1));

  K k;
  k.base = (smem_u32(raw_smem) + 1023) & ~1023u;
  uint8_t *const smem = raw_smem + (k.base - smem_u32(raw_smem));
  k.stop = reinterpret_cast<volatile int *>(smem + K::kStopAt);
  k.giveups = a.giveups;
  Meta *const meta = reinterpret_cast<Meta *>(smem + K::kMetaAt);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31; // the same for all lanes, and known to be
  if (threadIdx.x == 0) {
    auto init = [&](int first, int n, int arrivals) {
      for (int i = first; i < first + n; i++)
        mbar_init(smem + K::kBars + i * 8, arrivals);
    };
    init(K::kQueryFull, 1, 4 * tiles);
    init(K::kScoreFull, 4, 1);
    init(K::kWeightFull, 4, 4);
    init(K::kOutDone, 2, 1);
    init(K::kKeyFull, K::kKeyStages, 4);
    init(K::kKeyFree, K::kKeyStages, 1);
    init(K::kValueFull, K::kValueStages, 4);
    init(K::kValueFree, K::kValueStages, 1);
    init(K::kRawFull, K::kRawStages, 1);
    init(K::kRawFree, K::kRawStages, 4);
    init(K::kDrained, 1, 1);
    *k.stop = 0;
    mbar_init_fence();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(k.base + K::kTmemAt) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + K::kTmemAt);
  auto scores_at = [&](int tile, int j) { return tmem + (tile * 2 + (j & 1)) * 64; };
  auto out_at = [&](int tile) { return tmem + 256 + tile * D; };

  if (warp < 8) {
    // ---- softmax: a thread per row ----------------------------------------------------
    more_registers<152>();
    const int tile = warp >> 2, r = threadIdx.x & (kTile - 1);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21; // this warp's 32 lanes of tensor memory
    if (tile < tiles) {
      const long row = row0 + tile * kTile + r;
      const bool is = row < R;
      const int token = is ? (int)(row / a.group) : 0, h = head * a.group + (is ? (int)(row % a.group) : 0);
      const int pos = is ? sp.pos + token : -1;
      const int min_pos = pos_of(row0 + tile * kTile), max_pos = pos_of(row0 + tile * kTile + kTile - 1);
      float row_factor;
      {
        const QT *p = a.qkv + (size_t)(sp.row + token) * a.row_stride + (size_t)h * D;
        float top = 0.0f;
        bool odd = false;
#pragma unroll 16
        for (int c = 0; c < D; c += 4) {
          float v[4];
          load4(p + c, a.q_vec, v);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            odd = odd || !(fabsf(v[e]) <= 3.402823466e38f);
            top = fmaxf(top, fabsf(v[e]));
          }
        }
        // largest |q| into [2^13, 2^14), as in kv8_attention.cu
        const int up = odd || top == 0.0f ? 0 : max(min(13 - (exponent_field(top) - 127), 126), -126);
        const float f = two_to(up) * (a.scale < 0.0f ? -1.0f : 1.0f);
        row_factor = odd ? NAN : fabsf(a.scale) * kLog2e * two_to(-up);
        const uint32_t to = k.base + K::kQueries + tile * (kSplit ? 2 : 1) * K::kQueryBytes;
#pragma unroll 2
        for (int c = 0; c < D / 8; c++) {
          uint32_t w[4], rest[4];
#pragma unroll
          for (int half = 0; half < 2; half++) {
            float v[4];
            load4(p + 8 * c + 4 * half, a.q_vec, v);
#pragma unroll
            for (int e = 0; e < 4; e++)
              v[e] = odd || !is ? 0.0f : v[e] * f;
#pragma unroll
            for (int e = 0; e < 2; e++) {
              w[2 * half + e] = pack_f16(v[2 * e], v[2 * e + 1]);
              rest[2 * half + e] = pack_rest(w[2 * half + e], v[2 * e], v[2 * e + 1]);
            }
          }
          K::store16(to + K::swizzled(r, c, kTile), w[0], w[1], w[2], w[3]);
          if constexpr (kSplit)
            K::store16(to + K::kQueryBytes + K::swizzled(r, c, kTile), rest[0], rest[1], rest[2], rest[3]);
        }
        fence_async_smem();
        arrive_warp(k.bar(K::kQueryFull));
      }
      float m = -INFINITY, l = 0.0f;
      int value_exp = 0, j = 0;
      // Scores of page j to weights; false: the block is to end.
      auto step = [&](auto masked, const Meta &it, int j) {
        constexpr bool kMasked = decltype(masked)::value;
        uint32_t x[64];
        tmem_load32(scores_at(tile, j) + lanes, x);
        tmem_load32(scores_at(tile, j) + lanes + 32, x + 32);
        tmem_loaded();
        uint32_t seen[2] = {0, 0};
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}; // four chains, so that none waits for itself
        if constexpr (kMasked) {
          const int hi = pos - it.token, lo = a.window > 0 ? pos - a.window - it.token : -1, first = a.n_first - it.token;
#pragma unroll
          for (int c = 0; c < kPage; c++) {
            const bool sees = c <= hi && (c > lo || c < first);
            seen[c >> 5] |= (uint32_t)sees << (c & 31);
            tops[c & 3] = fmaxf(tops[c & 3], sees ? __uint_as_float(x[c]) : -INFINITY);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kPage; c += 8)
#pragma unroll
            for (int e = 0; e < 4; e++)
              tops[e] = fmaxf(tops[e], fmaxf(__uint_as_float(x[c + e]), __uint_as_float(x[c + 4 + e])));
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float f = row_factor * it.key_scale;
        const float now = top > -INFINITY ? fmaxf(m, top * f) : m;
        if (__any_sync(0xffffffffu, now > m + kRise || it.value_exp != value_exp)) {
          const float fade = now > -INFINITY ? fast_exp2(m - now) : 1.0f;
          const float factor = fade * two_to(value_exp - it.value_exp);
          m = now;
          l *= fade;
          value_exp = it.value_exp;
          if (j > 0) {
            if (!k.wait_warp(K::kOutDone + tile, (j - 1) & 1))
              return false;
            tc_after_sync();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_load32(out_at(tile) + lanes + c, o);
              tmem_loaded();
#pragma unroll
              for (int e = 0; e < 32; e++)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              tmem_store32(out_at(tile) + lanes + c, o);
            }
          }
        }
        const float off = (float)kTileBits - (m > -INFINITY ? m : 0.0f);
        uint32_t w[32];
        float2 sums[4] = {};
#pragma unroll
        for (int c = 0; c < kPage; c += 2) {
          const float2 z = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), make_float2(f, f), make_float2(off, off));
          float2 p = make_float2(fast_exp2(z.x), fast_exp2(z.y));
          if constexpr (kMasked) {
            p.x = seen[c >> 5] >> (c & 31) & 1 ? p.x : 0.0f;
            p.y = seen[c >> 5] >> ((c & 31) + 1) & 1 ? p.y : 0.0f;
          }
          sums[c / 2 & 3] = add2(sums[c / 2 & 3], p);
          w[c / 2] = pack_f16(p.x, p.y);
          if constexpr (kSplit)
            x[c / 2] = pack_rest(w[c / 2], p.x, p.y); // x[c / 2] has been read
        }
        const float2 sum = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
        l += sum.x + sum.y;
        tmem_store32(scores_at(tile, j) + lanes, w);
        if constexpr (kSplit)
          tmem_store32(scores_at(tile, j) + lanes + 32, x);
        return true;
      };
      bool ok = true;
      for (;; j++) {
        if (!(ok = k.wait_warp(K::kScoreFull + tile * 2 + (j & 1), j >> 1 & 1)))
          break;
        tc_after_sync();
        const Meta it = meta[j % kMeta];
        if (it.token < 0)
          break;
        const bool all = it.token + kPage - 1 <= min_pos &&
                         (a.window <= 0 || it.token > max_pos - a.window || it.token + kPage <= a.n_first);
        ok = all ? step(std::false_type{}, it, j) : step(std::true_type{}, it, j);
        if (!ok)
          break;
        tmem_stored();
        tc_before_sync();
        arrive_warp(k.bar(K::kWeightFull + tile * 2 + (j & 1)));
      }
      if (ok && j > 0)
        ok = k.wait_warp(K::kOutDone + tile, (j - 1) & 1);
      if (ok) {
        tc_after_sync();
        float f = 0.0f;
        if (l != 0.0f) { // a NaN passes
          const float z = a.sinks ? fminf(__ldg(a.sinks + h) * kLog2e, 3e38f) : -INFINITY, top = fmaxf(m, z);
          const float fade = m > -INFINITY ? fast_exp2(m - top) : 1.0f;
          const float all = l * fade + (a.sinks ? fast_exp2(z - top + (float)kTileBits) : 0.0f);
          f = fade * two_to(value_exp - 127 - kValueBits) / all;
        }
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (j > 0) {
            tmem_load32(out_at(tile) + lanes + c, o);
            tmem_loaded();
          }
          if (is)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float v[4];
#pragma unroll
              for (int i = 0; i < 4; i++)
                v[i] = l != 0.0f ? __uint_as_float(o[e + i]) * f : 0.0f;
              store4(a, (size_t)(sp.row + token) * a.out_row_stride + (size_t)h * D + c + e, make_float4(v[0], v[1], v[2], v[3]));
            }
        }
      }
    }
  } else if (warp < 12) {
    // ---- codes to fp16 ------------------------------------------------------------------
    fewer_registers<72>();
    const int t = threadIdx.x - 256, token = t >> 1, half = t & 1; // half of a token's codes
    const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
    int page_of = -1, held = -32, ahead = 0, asked = 0, value_exp = 0;
    float2 scale_of = make_float2(0.0f, 0.0f);
    // Every warp goes over the table the same way; thread 0 alone asks for the bytes.  Per stage in flight:
    int ring_token[K::kRawStages];
    float2 ring_scale[K::kRawStages];
    auto ask = [&](int stage) { // the next column that has a page into `stage`; token -1: there is none
      ring_token[stage] = -1;
      for (; ahead < cols.n; ahead = held + 32) {
        if (ahead >= held + 32) {
          held += 32;
          page_of = held + lane < cols.n ? a.cache.checked(__ldg(table + cols.at(held + lane))) : -1;
          if (page_of >= 0)
            scale_of = *reinterpret_cast<const float2 *>(a.cache.scale(page_of, head));
        }
        const unsigned there = __ballot_sync(0xffffffffu, page_of >= 0) >> (ahead - held);
        if (there) {
          ahead += __ffs(there) - 1;
          const int page = __shfl_sync(0xffffffffu, page_of, ahead - held);
          ring_token[stage] = cols.at(ahead) * kPage;
          ring_scale[stage].x = __shfl_sync(0xffffffffu, scale_of.x, ahead - held);
          ring_scale[stage].y = __shfl_sync(0xffffffffu, scale_of.y, ahead - held);
          if (t == 0) {
            const uint32_t b = k.bar(K::kRawFull + stage);
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(K::kRawBytes) : "memory");
            asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             k.base + K::kRaw + stage * K::kRawBytes),
                         "l"(a.cache.template block<D>(page, head)), "r"(K::kRawBytes), "r"(b)
                         : "memory");
          }
          ahead++, asked++;
          return;
        }
      }
    };
    auto convert = [&](uint32_t from, uint32_t to, uint32_t mul, uint32_t add) { // this thread's half token
#pragma unroll
      for (int i = 0; i < D / 32; i++) { // 16 codes: two 16-byte pieces
        const uint4 w = lds16(from + token * D + half * (D / 2) + i * 16);
        const uint32_t u[4] = {biased(w.x), biased(w.y), biased(w.z), biased(w.w)};
#pragma unroll
        for (int e = 0; e < 2; e++)
          K::store16(to + K::swizzled(token, half * (D / 16) + i * 2 + e, kPage), scaled_pair(low_pair(u[2 * e]), mul, add),
                     scaled_pair(high_pair(u[2 * e]), mul, add), scaled_pair(low_pair(u[2 * e + 1]), mul, add),
                     scaled_pair(high_pair(u[2 * e + 1]), mul, add));
      }
    };
#pragma unroll
    for (int i = 0; i < K::kRawStages; i++)
      ask(i);
    int used = 0;
    bool ok = true, more = true;
    while (ok && more) {
#pragma unroll
      for (int raw = 0; raw < K::kRawStages; raw++) { // j = used, its raw stage known at compile time
        if (!ok || !more)
          break;
        const int j = used;
        const int ks = j % K::kKeyStages, vs = j % K::kValueStages;
        more = ring_token[raw] >= 0;
        if (j >= K::kKeyStages && !(ok = k.wait_warp(K::kKeyFree + ks, (j / K::kKeyStages - 1) & 1)))
          break;
        const int v_exp = exponent_field(ring_scale[raw].y);
        if (more)
          value_exp = max(value_exp, v_exp);
        if (t == 0)
          meta[j % kMeta] = Meta{ring_token[raw], ring_scale[raw].x, value_exp, 0};
        const uint32_t from = k.base + K::kRaw + raw * K::kRawBytes;
        if (more) {
          if (!(ok = k.wait_warp(K::kRawFull + raw, j / K::kRawStages & 1)))
            break;
          convert(from, k.base + K::kKeys + ks * K::kPageBytes, 0x3c003c00u, 0xe480e480u); // times 1, minus 1152
        }
        fence_async_smem();
        arrive_warp(k.bar(K::kKeyFull + ks));
        if (!more)
          break;
        if (j >= K::kValueStages && !(ok = k.wait_warp(K::kValueFree + vs, (j / K::kValueStages - 1) & 1)))
          break;
        uint32_t mul, add;
        value_factor(v_exp == 0 ? -99 : v_exp - value_exp + kValueBits, mul, add);
        convert(from + kPage * D, k.base + K::kValues + vs * K::kPageBytes, mul, add);
        fence_async_smem();
        arrive_warp(k.bar(K::kValueFull + vs));
        arrive_warp(k.bar(K::kRawFree + raw)); // this thread has read the raw stage
        used++;
        if (warp == 8 && !(ok = k.wait_warp(K::kRawFree + raw, j / K::kRawStages & 1)))
          break;
        ask(raw);
      }
    }
    if (t == 0 && !ok) // what is still on its way is waited for, with a limit of its own
      for (int p = used; p < asked; p++)
        mbar_wait_at(k.bar(K::kRawFull + p % K::kRawStages), p / K::kRawStages & 1);
  } else {
    // ---- matrix instructions --------------------------------------------------------------
    constexpr uint32_t kScoreShape = shape_of(kPage, false), kOutShape = shape_of(D, true);
    const uint32_t leader = elected();
    const uint32_t queries = operand_low(k.base + K::kQueries, 16), keys0 = operand_low(k.base + K::kKeys, 16),
                   values0 = operand_low(k.base + K::kValues, kPage * 128);
    bool ok = k.wait_warp(K::kQueryFull, 0), more = true;
    int n = 0, key_stage = 0, value_stage = 0; // pages whose scores have been asked for; where the next ones lie
    uint32_t key_turn = 0, value_turn = 0;
    // The scores of page n for `tile`; the page's keys are waited for with tile 0.
    auto next_scores = [&](int tile) {
      if (!more)
        return;
      if (tile == 0) {
        if (!(ok = k.wait_warp(K::kKeyFull + key_stage, key_turn)))
          return;
        tc_after_sync();
      }
      const bool real = meta[n % kMeta].token >= 0;
      if (real) {
        const uint32_t q = queries + tile * ((kSplit ? 2 : 1) * K::kQueryBytes / 16), keys = keys0 + key_stage * (K::kPageBytes / 16);
#pragma unroll
        for (int part = 0; part < (kSplit ? 2 : 1); part++)
#pragma unroll
          for (int i = 0; i < D / 16; i++)
            mma_smem(scores_at(tile, n), q + (part * K::kQueryBytes + (i / 4) * kTile * 128 + (i % 4) * 32) / 16,
                     keys + ((i / 4) * kPage * 128 + (i % 4) * 32) / 16, kScoreShape, part + i > 0, leader);
      }
      tc_commit(k.bar(K::kScoreFull + tile * 2 + (n & 1)), leader); // also for the end of the pages
      if (tile == tiles - 1) {
        if (real) {
          tc_commit(k.bar(K::kKeyFree + key_stage), leader);
          n++;
          if (++key_stage == K::kKeyStages)
            key_stage = 0, key_turn ^= 1;
        }
        more = real;
      }
    };
    for (int i = 0; i < 2 && ok; i++)
      for (int tile = 0; tile < tiles && ok; tile++)
        next_scores(tile);
    for (int j = 0; ok && j < n; j++) {
      for (int tile = 0; tile < tiles && ok; tile++) {
        if (!(ok = k.wait_warp(K::kWeightFull + tile * 2 + (j & 1), j >> 1 & 1)))
          break;
        if (tile == 0 && !(ok = k.wait_warp(K::kValueFull + value_stage, value_turn)))
          break;
        tc_after_sync();
        const uint32_t values = values0 + value_stage * (K::kPageBytes / 16);
#pragma unroll
        for (int part = 0; part < (kSplit ? 2 : 1); part++)
#pragma unroll
          for (int i = 0; i < kPage / 16; i++)
            mma_tmem(out_at(tile), scores_at(tile, j) + part * 32 + i * 8, values + i * (2048 / 16), kOutShape, j + part + i > 0,
                     leader);
        tc_commit(k.bar(K::kOutDone + tile), leader);
        if (tile == tiles - 1)
          tc_commit(k.bar(K::kValueFree + value_stage), leader);
        next_scores(tile);
      }
      if (++value_stage == K::kValueStages)
        value_stage = 0, value_turn ^= 1;
    }
    if (!ok) { // matrix instructions still running are waited for, with a limit, before their memory is given back
      tc_commit(k.bar(K::kDrained), leader);
      mbar_wait_at(k.bar(K::kDrained), 0);
    }
  }
  __syncwarp();
  tc_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <typename QT, int D> void launch_d(cudaStream_t stream, const Call<QT> &a) {
  const long units = (long)a.rows.T * a.group / (kTile * kTiles) + a.rows.n_seqs;
  (void)blocks_per_sm_smem(attend_tiles<QT, D>, kTileThreads, TileKernel<QT, D>::kSmem);
  launch_kernel(attend_tiles<QT, D>, dim3((unsigned)(units * a.cache.n_kv_heads)), dim3(kTileThreads), TileKernel<QT, D>::kSmem,
                stream, a);
}

} // namespace

template <typename QT> void launch_tiles(cudaStream_t stream, const Call<QT> &a, int head_dim) {
  head_dim == 64 ? launch_d<QT, 64>(stream, a) : launch_d<QT, 128>(stream, a);
}
template void launch_tiles<float>(cudaStream_t, const Call<float> &, int);
template void launch_tiles<uint16_t>(cudaStream_t, const Call<uint16_t> &, int);

} // namespace kv8
} // namespace gptoss
