// Attention over the 8-bit paged cache for many rows per sequence (prompts, chunks of prompts), on the
// fifth-generation tensor cores.
//
// The mathematics is that of kv8_attention.cu.  A block takes 512 rows (new tokens x query heads) of one
// sequence and key/value head as four tiles of 128 (256 as two: fp32 rows, 128-wide heads, few rows), and goes over
// the pages they see, a page's 64 tokens at a time:
//     S = Q K^T   128 x 64, queries and keys from shared memory, sums in tensor memory
//     P = 2^(S f - m)  by one thread per row, written back over S as fp16
//     O += P V    128 x D, P from tensor memory, values from shared memory
// What would bound it at D = 64 is the exponential (16 per clock and SM: 512 clocks for a 128 x 64 tile against some
// 320 of matrix instructions); what does is how far the steps of a tile, which wait for each other (scores,
// weights, product), are covered by those of the others: 810 clocks per tile and page with four tiles, 1230 with two.
// An 8192-token prompt of 64 heads takes 0.78 ms, 0.70 PFLOP/s.  (Two tiles keep all they need in registers; four, at 80,
// do not: -Xptxas -v shows 108 bytes of spill stores and 216 of loads per thread.)  So:
//   - four warps per tile: softmax.  A row's running maximum is raised only when the new one is 2^8 above it, so
//     that O is rescaled a few times per row and not once per page;
//   - four warps: codes (brought by the copy engine into a ring of raw pages) to fp16 in the 128-byte swizzled
//     form the matrix instruction reads, once for all tiles; two warps for the keys and two for the values, since
//     what a page costs them is mostly waiting (barriers, the fence before the matrix unit may read);
//   - one warp: one of its threads issues the matrix instructions.  With two tiles scores have two buffers each, so
//     that the next page's are ready when a softmax warp comes for them; with four there is room for one;
//   - where there are few units (a chunk of some rows against a long context) their columns are shared out over more
//     blocks and joined by merge_parts.
// Queries, codes and weights are represented as in kv8_attention.cu: fp16, exact for codes and bf16 rows; fp32 rows
// and their weights in two parts with two products, and O folded into the softmax threads' memory every kFoldPages pages.
// Value scales are relative to one reference per block; far pages (kv8_attention.cuh) are left out of the loop and
// added by finish_far.
// Every wait is bounded: one that runs out is counted, tells the block's other roles, and the block frees its
// tensor memory and ends.
#include <algorithm>

#include "kv8_attention.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr int kTile = 128;
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
// Registers a thread of this warpgroup may use from here on (the split, TileKernel, stays within what the block
// was launched with).
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One arrival for a warp, after all its lanes.
__device__ __forceinline__ void arrive_warp(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    arrive(bar);
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
// Four steps of 16 along the inner index, issued by one lane.  The whole warp comes here and elects it: operands
// stay in uniform registers (with one lane in a branch of its own, moving them there took longer than the products).
__device__ __forceinline__ void mma4_smem(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
  asm volatile("{\n\t.reg .pred p, q, t;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\telect.sync _|q, 0xffffffff;\n\t"
               "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
               "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
               "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
               "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
               "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t}" ::"r"(d),
               "r"(a), "r"(b), "r"(shape), "r"(add), "r"(kOperandHigh)
               : "memory");
}
// `half`: columns from the first two steps' left operand to the others'.
template <int half>
__device__ __forceinline__ void mma4_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
  asm volatile("{\n\t.reg .pred p, q, t;\n\t.reg .b64 b;\n\t.reg .b32 x, y;\n\telect.sync _|q, 0xffffffff;\n\t"
               "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
               "mov.b64 b, {%2, %5};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
               "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 128;\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, t;\n\t"
               "add.u32 x, %1, %6;\n\tadd.u32 y, %2, 256;\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, t;\n\t"
               "add.u32 x, %1, %7;\n\tadd.u32 y, %2, 384;\n\tmov.b64 b, {y, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, t;\n\t}" ::"r"(d),
               "r"(a), "r"(b), "r"(shape), "r"(add), "r"(kOperandHigh), "n"(half), "n"(half + 8)
               : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
               : "memory");
}
#define GPTOSS_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define GPTOSS_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of the calling warp's 32 lanes; the values are there after tmem_loaded.  Arrays of another size than the
// columns moved do not compile.
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t (&x)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
               "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : GPTOSS_R8(x, 0), GPTOSS_R8(x, 8), GPTOSS_R8(x, 16), GPTOSS_R8(x, 24)
               : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&x)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
               "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
               GPTOSS_W8(x, 0), GPTOSS_W8(x, 8), GPTOSS_W8(x, 16), GPTOSS_W8(x, 24)
               : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&x)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : GPTOSS_R8(x, 0), GPTOSS_R8(x, 8)
               : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&x)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
               GPTOSS_W8(x, 0), GPTOSS_W8(x, 8)
               : "memory");
}
#undef GPTOSS_R8
#undef GPTOSS_W8
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename QT, int D, int TILES> struct TileKernel {
  static constexpr bool kSplit = sizeof(QT) == 4;
  static constexpr int kFoldPages = kSplit ? kFold / (2 * kPage / 16) : 1 << 30; // products of this page start O afresh
  static constexpr int kBuffers = TILES == 2 ? 2 : 1;                  // of scores, per tile
  static constexpr int kConverters = 4 * TILES, kIssuer = kConverters + 4, kThreads = 32 * (kIssuer + 1);
  static constexpr int kRowsOfBlock = kTile * TILES;
  // A thread's registers: at launch (65536 over the warps rounded up to whole groups of four), and of the
  // softmax and converting warps afterwards; the issuing warp keeps what it has.
  static constexpr int kLaunchRegisters = TILES == 2 ? 128 : 80, kSoftmaxRegisters = TILES == 2 ? 152 : 88,
                       kConverterRegisters = TILES == 2 ? 72 : 48;
  static_assert(128 * TILES * kSoftmaxRegisters + 128 * kConverterRegisters + 32 * kLaunchRegisters <= kThreads * kLaunchRegisters,
                "setmaxnreg.inc would wait for good");
  static_assert(TILES * (64 * kBuffers + D) <= 512, "tensor memory");
  static constexpr int kKeyStages = D == 64 ? 4 : kSplit ? 2 : 3, kValueStages = kKeyStages, kRawStages = D == 64 ? 4 : kSplit ? 2 : 3;
  static constexpr int kQueryBytes = kTile * D * 2;                    // of a tile and part
  static constexpr int kPageBytes = kPage * D * 2;                     // a page's keys or values as fp16
  static constexpr int kRawBytes = 2 * kPage * D;                      // a page's codes, keys then values
  static constexpr int kQueries = 0, kKeys = kQueries + TILES * (kSplit ? 2 : 1) * kQueryBytes;
  static constexpr int kValues = kKeys + kKeyStages * kPageBytes, kRaw = kValues + kValueStages * kPageBytes;
  static constexpr int kMetaAt = kRaw + kRawStages * kRawBytes, kBars = kMetaAt + kMeta * 16;
  // barriers
  static constexpr int kQueryFull = 0, kScoreFull = 1 /* tile, buffer */, kWeightFull = kScoreFull + TILES * kBuffers /* tile, buffer */,
                       kOutDone = kWeightFull + TILES * kBuffers /* tile */, kKeyFull = kOutDone + TILES, kKeyFree = kKeyFull + kKeyStages,
                       kValueFull = kKeyFree + kKeyStages, kValueFree = kValueFull + kValueStages,
                       kRawFull = kValueFree + kValueStages, kRawFree = kRawFull + kRawStages, kDrained = kRawFree + kRawStages,
                       kBarCount = kDrained + 1;
  static constexpr int kTmemAt = kBars + kBarCount * 8, kStopAt = kTmemAt + 4, kFarAt = kStopAt + 4; // the second: far pages, their reference
  static_assert(kRowsOfBlock * (D * 4 + 8) <= kMetaAt, "means of a block that has far pages");
  static constexpr int kSmem = kFarAt + 8 + 1024; // the base is brought to 1024 bytes, the swizzle's period
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

struct Meta { // of a page: its first token, key scale; behind the last (token -1) the value reference, and if there are far pages
  int token;
  float key_scale;
  int ref, far;
};

// The `rows` rows of a sequence and head that a block works on, and the table columns they look at.  Units are
// numbered over the sequences: s has those from unit0(s) on.
struct Unit {
  Rows::Span sp;
  int s, head;
  long row0, R; // first row, rows of the sequence
  Columns cols;
  template <typename QT> __device__ __forceinline__ bool find(const Call<QT> &a, int unit, int head_, int rows) {
    auto unit0 = [&](int i) { return (int)((long)a.rows.start(i) * a.group / rows) + i; };
    head = head_;
    s = a.rows.find(unit, unit0);
    sp = a.rows.span(s);
    R = (long)sp.q * a.group, row0 = (long)(unit - unit0(s)) * rows;
    if (unit < unit0(s) || R <= kMaxTokenRows || row0 >= R)
      return false;
    cols = columns(a.rows, a.window, a.n_first, pos_of(a, row0), pos_of(a, row0 + rows - 1));
    return true;
  }
  template <typename QT> __device__ __forceinline__ int pos_of(const Call<QT> &a, long row) const {
    return sp.pos + (int)(min(row, R - 1) / a.group);
  }
  // Columns of one of `splits` parts.
  __device__ __forceinline__ int column(int split, int splits) const { return (int)((long)cols.n * split / splits); }
};

// What the blocks of a unit whose columns are shared out leave for merge_parts: a row's values over its sum, and its
// maximum and sum.
struct Parts {
  int splits;
  float *o;   // [block][rows][D]
  float2 *ml; // [block][rows]
  static size_t bytes(long blocks, int rows, int D) { return (size_t)blocks * rows * (D * 4 + 8); }
};

// The unit and the part of its columns that this block works on; false where there is nothing to do.  The last units of a
// sequence, which see most, first.
struct Work {
  Unit u;
  int split, col0, col1;
  template <typename QT> __device__ __forceinline__ bool find(const Call<QT> &a, const Parts &parts, int rows) {
    const int heads = a.cache.n_kv_heads, index = blockIdx.x / parts.splits;
    split = blockIdx.x % parts.splits;
    if (!u.find(a, (int)(gridDim.x / parts.splits / heads) - 1 - index / heads, index % heads, rows))
      return false;
    col0 = u.column(split, parts.splits), col1 = u.column(split + 1, parts.splits);
    return col0 < col1;
  }
};

// The end of a block that has met far pages, by its softmax warps: one per row adds them to the row's mean, which lies in
// shared memory, and writes it.  What it needs is found again: nothing is held over the pages for its sake.
template <typename QT, int D, int TILES> __device__ __noinline__ void finish_far(const Call<QT> &a, const Parts &parts, uint8_t *smem, int warps) {
  using K = TileKernel<QT, D, TILES>;
  constexpr int N = D / 32;
  Work w = {};
  (void)w.find(a, parts, K::kRowsOfBlock);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = (int)min(w.u.R - w.u.row0, (long)K::kRowsOfBlock);
  const int *ref = reinterpret_cast<const int *>(smem + K::kFarAt) + 1;
#pragma unroll 1
  for (int r = warp; r < rows; r += warps) {
    float *mean = reinterpret_cast<float *>(smem) + r * D;
    float2 *ml = reinterpret_cast<float2 *>(smem + K::kRowsOfBlock * D * 4) + r;
    const int token = (int)((w.u.row0 + r) / a.group), h = w.u.head * a.group + (int)((w.u.row0 + r) % a.group);
    far_row<D>(a, w.u.s, w.u.head, w.u.cols, w.col0, w.col1, a.qkv + (size_t)(w.u.sp.row + token) * a.row_stride + (size_t)h * D,
               w.u.sp.pos + token, ref, 1, 1, mean, ml);
    const float2 x = *ml;
    const size_t part = (size_t)blockIdx.x * K::kRowsOfBlock + r;
    float f = x.y != 0.0f ? 1.0f : 0.0f; // a NaN passes
    if (parts.splits > 1) {
      if (lane == 0)
        parts.ml[part] = x;
    } else if (f != 0.0f) {
      const float z = a.sinks ? sink_of(a, h) : -INFINITY, top = fmaxf(x.x, z), sum = x.y * (x.x > -INFINITY ? fast_exp2(x.x - top) : 1.0f);
      f = sum / (sum + fast_exp2(z - top));
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
      const float v = f != 0.0f ? mean[lane * N + n] * f : 0.0f;
      const size_t at = (size_t)(w.u.sp.row + token) * a.out_row_stride + (size_t)h * D + lane * N + n;
      if (parts.splits > 1)
        parts.o[part * D + lane * N + n] = v;
      else if (a.out_f32)
        static_cast<float *>(a.out)[at] = v;
      else
        store1(static_cast<uint16_t *>(a.out) + at, v);
    }
  }
}

template <typename QT, int D, int TILES>
__global__ void __launch_bounds__(32 * (4 * TILES + 5), 1) attend_tiles(const __grid_constant__ Call<QT> a, const __grid_constant__ Parts parts) {
  using K = TileKernel<QT, D, TILES>;
  constexpr bool kSplit = K::kSplit;
  constexpr int kBuffers = K::kBuffers, kLeader = 32 * K::kConverters; // kLeader: the thread that asks for pages
  extern __shared__ uint8_t raw_smem[];
  pdl_prologue();
  Work work = {};
  if (!work.find(a, parts, K::kRowsOfBlock))
    return;
  const Unit &u = work.u;
  const int s = u.s, head = u.head, col0 = work.col0, col1 = work.col1;
  const Rows::Span sp = u.sp;
  const long R = u.R, row0 = u.row0;
  const Columns cols = u.cols;
  const int tiles = (int)min((R - row0 + kTile - 1) / kTile, (long)TILES);

  K k;
  k.base = (smem_u32(raw_smem) + 1023) & ~1023u;
  uint8_t *const smem = raw_smem + (k.base - smem_u32(raw_smem));
  k.stop = reinterpret_cast<volatile int *>(smem + K::kStopAt);
  k.giveups = a.giveups;
  Meta *const meta = reinterpret_cast<Meta *>(smem + K::kMetaAt);
  volatile int *const far_block = reinterpret_cast<volatile int *>(smem + K::kFarAt); // 1: there are far pages; their reference
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31; // the same for all lanes, and known to be
  if (threadIdx.x == 0) {
    auto init = [&](int first, int n, int arrivals) {
      for (int i = first; i < first + n; i++)
        mbar_init(smem + K::kBars + i * 8, arrivals);
    };
    init(K::kQueryFull, 1, 4 * tiles);
    init(K::kScoreFull, TILES * kBuffers, 1);
    init(K::kWeightFull, TILES * kBuffers, 4);
    init(K::kOutDone, TILES, 1);
    init(K::kKeyFull, K::kKeyStages, 2);
    init(K::kKeyFree, K::kKeyStages, 1);
    init(K::kValueFull, K::kValueStages, 2);
    init(K::kValueFree, K::kValueStages, 1);
    init(K::kRawFull, K::kRawStages, 1);
    init(K::kRawFree, K::kRawStages, 4);
    init(K::kDrained, 1, 1);
    *k.stop = 0, *far_block = 0;
    mbar_init_fence();
  }
  if (warp == K::kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(k.base + K::kTmemAt) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + K::kTmemAt);
  auto scores_at = [&](int tile, int j) { return tmem + (tile * kBuffers + j % kBuffers) * 64; };
  auto out_at = [&](int tile) { return tmem + 64 * TILES * kBuffers + tile * D; };
  auto buffer = [&](int tile, int j) { return tile * kBuffers + j % kBuffers; };
  auto phase = [&](int j) { return (uint32_t)(j / kBuffers & 1); };

  if (warp < K::kConverters) {
    // ---- softmax: a thread per row ----------------------------------------------------
    more_registers<K::kSoftmaxRegisters>();
    const int tile = warp >> 2, r = threadIdx.x & (kTile - 1);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21; // this warp's 32 lanes of tensor memory
    if (tile < tiles) {
      const long row = row0 + tile * kTile + r;
      const bool is = row < R;
      const int token = is ? (int)(row / a.group) : 0, h = head * a.group + (is ? (int)(row % a.group) : 0);
      const int pos = is ? sp.pos + token : -1;
      const int min_pos = u.pos_of(a, row0 + tile * kTile), max_pos = u.pos_of(a, row0 + tile * kTile + kTile - 1);
      // The warp's 32 queries, D / 8 lanes to a row and 8 elements to a lane, so that loads are of whole lines (a
      // thread per row took 6 us for them); then each lane keeps the factor of its own row.
      float row_factor = 0.0f;
      {
        constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes, kAhead = 4;
        const int piece = lane % kLanes, sub = lane / kLanes;
        const uint32_t to = k.base + K::kQueries + tile * (kSplit ? 2 : 1) * K::kQueryBytes;
        const long first = row0 + tile * kTile + (warp & 3) * 32;
#pragma unroll 1
        for (int i0 = 0; i0 < kLanes; i0 += kAhead) {
          float v[kAhead][8];
#pragma unroll
          for (int n = 0; n < kAhead; n++) {
            const long at = min(first + (i0 + n) * kRowsAtOnce + sub, R - 1);
            const QT *p = a.qkv + (size_t)(sp.row + (int)(at / a.group)) * a.row_stride +
                          (size_t)(head * a.group + (int)(at % a.group)) * D + piece * 8;
            float lo[4], hi[4];
            load4(p, a.q_vec, lo);
            load4(p + 4, a.q_vec, hi);
#pragma unroll
            for (int e = 0; e < 4; e++)
              v[n][e] = lo[e], v[n][4 + e] = hi[e];
          }
#pragma unroll
          for (int n = 0; n < kAhead; n++) {
            const int i = i0 + n, row_here = i * kRowsAtOnce + sub; // of the warp's 32
            float top = 0.0f;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              odd = odd || !(fabsf(v[n][e]) <= 3.402823466e38f);
              top = fmaxf(top, fabsf(v[n][e]));
            }
#pragma unroll
            for (int x = 1; x < kLanes; x <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              odd = __shfl_xor_sync(0xffffffffu, (int)odd, x) || odd;
            }
            const bool real = first + row_here < R;
            // largest |q| into [2^13, 2^14), as in kv8_attention.cu
            const int up = odd || !real || top == 0.0f ? 0 : max(min(13 - (exponent_field(top) - 127), 126), -126);
            const float f = two_to(up) * (a.scale < 0.0f ? -1.0f : 1.0f);
            const float factor = odd && real ? NAN : fabsf(a.scale) * kLog2e * two_to(-up);
            uint32_t w[4], rest[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float x = odd || !real ? 0.0f : v[n][2 * e] * f, y = odd || !real ? 0.0f : v[n][2 * e + 1] * f;
              w[e] = pack_f16(x, y);
              rest[e] = pack_rest(w[e], x, y);
            }
            const int r_here = (warp & 3) * 32 + row_here;
            K::store16(to + K::swizzled(r_here, piece, kTile), w[0], w[1], w[2], w[3]);
            if constexpr (kSplit)
              K::store16(to + K::kQueryBytes + K::swizzled(r_here, piece, kTile), rest[0], rest[1], rest[2], rest[3]);
            const float mine = __shfl_sync(0xffffffffu, factor, lane % kRowsAtOnce * kLanes);
            if (lane / kRowsAtOnce == i)
              row_factor = mine;
          }
        }
        fence_async_smem();
        arrive_warp(k.bar(K::kQueryFull));
      }
      float m = -INFINITY, l = 0.0f;
      float kept[kSplit ? D : 1], m_kept = -INFINITY; // O of the pages before the last fold, relative to the maximum of then
      int j = 0, ref = 0;
      bool far = false;
      // What this thread's row does not see of a page gets a score below all others.  Only pages at the edge of
      // what a tile sees come here, and the step itself has one form: with the masks in it, it ran 13 % longer
      // over the pages that need none.
      auto mask = [&](const Meta &it, int j) {
        const int hi = pos - it.token, lo = a.window > 0 ? pos - a.window - it.token : -1, first = a.n_first - it.token;
        auto ones = [](int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }; // columns below n
#pragma unroll 1
        for (int c0 = 0; c0 < kPage; c0 += 32) {
          const uint32_t sees = ones(hi + 1 - c0) & (~ones(lo + 1 - c0) | ones(first - c0));
          uint32_t x[32];
          tmem_load32(scores_at(tile, j) + lanes + c0, x);
          tmem_loaded();
#pragma unroll
          for (int c = 0; c < 32; c++)
            x[c] = sees & 1u << c ? x[c] : __float_as_uint(-3e38f);
          tmem_store32(scores_at(tile, j) + lanes + c0, x);
        }
        tmem_stored();
      };
      // Scores of page j to weights; false: the block is to end.
      auto step = [&](const Meta &it, int j) {
        // All 64 scores in registers where there is room (two tiles); else half by half, and the first half again for the
        // weights, which lie where their own half's scores were.
        constexpr int kHalves = TILES == 2 ? 2 : 1, kHeld = 32 * kHalves; // in registers
        uint32_t x[kHalves][32];
#pragma unroll
        for (int i = 0; i < kHalves; i++)
          tmem_load32(scores_at(tile, j) + lanes + 32 * i, x[i]);
        tmem_loaded();
        float tops[4] = {-3e38f, -3e38f, -3e38f, -3e38f}; // four chains, so that none waits for itself
#pragma unroll
        for (int c0 = 0; c0 < kPage; c0 += kHeld) {
          if (c0 > 0) {
            tmem_load32(scores_at(tile, j) + lanes + 32, x[0]);
            tmem_loaded();
          }
#pragma unroll
          for (int c = 0; c < kHeld; c += 8)
#pragma unroll
            for (int e = 0; e < 4; e++)
              tops[e] = fmaxf(tops[e], fmaxf(__uint_as_float(x[c / 32][c % 32 + e]), __uint_as_float(x[c / 32][c % 32 + 4 + e])));
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool any = top > -2e38f; // real scores are below 2^28
        // A factor that is not 0, so that what is masked stays below; 2^-100 of a score is as good as 0.
        const float f = any ? at_least(at_most(row_factor * it.key_scale, kMostFactor), 0x1p-100f) : 1.0f;
        const float now = any ? fmaxf(m, top * f) : m;
        const bool moved = __any_sync(0xffffffffu, now > m + kRise), fold = kSplit && j > 0 && j % K::kFoldPages == 0;
        if (moved || fold) {
          const float fade = moved && now > -INFINITY ? fast_exp2(m - now) : 1.0f;
          m = moved ? now : m;
          l *= fade;
          if (j > 0) {
            if (!k.wait_warp(K::kOutDone + tile, (j - 1) & 1))
              return false;
            tc_after_sync();
            const float then = m_kept > -INFINITY ? fast_exp2(m_kept - m) : 0.0f;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_load16(out_at(tile) + lanes + c, o);
              tmem_loaded();
#pragma unroll
              for (int e = 0; e < 16; e++)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
              if constexpr (kSplit)
                if (fold) {
#pragma unroll
                  for (int e = 0; e < 16; e++)
                    kept[c + e] = j == K::kFoldPages ? __uint_as_float(o[e]) : fmaf(kept[c + e], then, __uint_as_float(o[e]));
                  continue; // the next product overwrites O
                }
              tmem_store16(out_at(tile) + lanes + c, o);
            }
            m_kept = fold ? m : m_kept;
          }
        }
        const float off = (float)kTileBits - (m > -INFINITY ? m : 0.0f);
        uint32_t w[kHeld / 2];
        float2 sums[4] = {};
#pragma unroll
        for (int h0 = 0; h0 < kPage; h0 += kHeld) {
          const int c0 = kHeld == 64 ? 0 : kHeld - h0; // the half that is still in registers first
          if (h0 > 0) {
            tmem_load32(scores_at(tile, j) + lanes + c0, x[0]);
            tmem_loaded();
          }
#pragma unroll
          for (int c = 0; c < kHeld; c += 2) {
            const float2 z = fma2(make_float2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])),
                                  make_float2(f, f), make_float2(off, off));
            float2 p = make_float2(fast_exp2(z.x), fast_exp2(z.y));
            sums[c / 2 & 3] = add2(sums[c / 2 & 3], p);
            w[c / 2] = pack_f16(p.x, p.y);
            if constexpr (kSplit)
              x[0][c / 2] = pack_rest(w[c / 2], p.x, p.y); // x[0][c / 2] has been read
          }
          if constexpr (kHeld == 64)
            tmem_store32(scores_at(tile, j) + lanes, w);
          else
            tmem_store16(scores_at(tile, j) + lanes + c0, w);
        }
        const float2 sum = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
        l += sum.x + sum.y;
        if constexpr (kSplit)
          tmem_store32(scores_at(tile, j) + lanes + 32, x[0]);
        return true;
      };
      bool ok = true;
      for (;; j++) {
        if (!(ok = k.wait_warp(K::kScoreFull + buffer(tile, j), phase(j))))
          break;
        tc_after_sync();
        const Meta it = meta[j % kMeta];
        if (it.token < 0) {
          ref = it.ref, far = it.far;
          break;
        }
        const bool all = it.token + kPage - 1 <= min_pos &&
                         (a.window <= 0 || it.token > max_pos - a.window || it.token + kPage <= a.n_first);
        if (!all)
          mask(it, j);
        if (!(ok = step(it, j)))
          break;
        tmem_stored();
        tc_before_sync();
        arrive_warp(k.bar(K::kWeightFull + buffer(tile, j)));
      }
      if (ok && j > 0)
        ok = k.wait_warp(K::kOutDone + tile, (j - 1) & 1);
      if (ok) {
        tc_after_sync();
        const bool apart = parts.splits > 1;
        // 16 elements of O from c on, those folded before included.
        auto load_out = [&](int c, uint32_t (&o)[16]) {
          if (j > 0) {
            tmem_load16(out_at(tile) + lanes + c, o);
            tmem_loaded();
          }
          if constexpr (kSplit)
            if (j > K::kFoldPages) {
              const float then = m_kept > -INFINITY ? fast_exp2(m_kept - m) : 0.0f;
#pragma unroll
              for (int e = 0; e < 16; e++)
                o[e] = __float_as_uint(fmaf(kept[c + e], then, __uint_as_float(o[e])));
            }
        };
        const float z = !apart && !far && a.sinks ? sink_of(a, h) : -INFINITY, unit = two_to(ref - 127);
        float f = 0.0f;
        if (l != 0.0f) { // a NaN passes
          const float top = fmaxf(m, z), fade = (m > -INFINITY ? fast_exp2(m - top) : 1.0f) * two_to(-kTileBits);
          f = fade * (float)(1 << (kNear - kValueBits)) / (l * fade + fast_exp2(z - top));
        }
        const size_t part = (size_t)blockIdx.x * K::kRowsOfBlock + tile * kTile + r;
        if (apart && is)
          parts.ml[part] = make_float2(m, l * two_to(-kTileBits));
        if (far) { // means to shared memory (once no tile's products read there), for the whole block to go on from
          for (int i = 0; i < tiles && ok && j > 0; i++)
            ok = k.wait_warp(K::kOutDone + i, (j - 1) & 1);
          if (ok) {
            tc_after_sync();
            float *mean = reinterpret_cast<float *>(smem) + (tile * kTile + r) * D;
            reinterpret_cast<float2 *>(smem + K::kRowsOfBlock * D * 4)[tile * kTile + r] = make_float2(m, l * two_to(-kTileBits));
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              load_out(c, o);
#pragma unroll
              for (int e = 0; e < 16; e++)
                mean[c + e] = l != 0.0f ? finite(__uint_as_float(o[e]) * f * unit) : 0.0f;
            }
          }
        } else {
          // Where the row goes; then 32 elements at a time through the warp's part of the queries' memory (all products
          // are done), so that stores are of whole sectors.
          const unsigned long long place =
              !is ? ~0ull : apart ? part * D : (unsigned long long)(sp.row + token) * a.out_row_stride + (unsigned long long)h * D;
          const uint32_t stage = k.base + K::kQueries + tile * (kSplit ? 2 : 1) * K::kQueryBytes + (warp & 3) * 4096;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
#pragma unroll
            for (int half = 0; half < 32; half += 16) {
              uint32_t o[16];
              load_out(c + half, o);
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                  v[i] = l != 0.0f ? __float_as_uint(__uint_as_float(o[e + i]) * f * unit) : 0u;
                K::store16(stage + lane * 128 + (((half + e) / 4 ^ (lane & 7)) << 4), v[0], v[1], v[2], v[3]);
              }
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int row_here = i * 4 + (lane >> 3), piece = lane & 7;
              const unsigned long long to = __shfl_sync(0xffffffffu, place, row_here) + c + piece * 4;
              const bool there = __shfl_sync(0xffffffffu, (int)is, row_here);
              const uint4 v = lds16(stage + row_here * 128 + ((piece ^ (row_here & 7)) << 4));
              const float4 v4 = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
              if (there && apart)
                *reinterpret_cast<float4 *>(parts.o + to) = v4;
              else if (there)
                store4(a, to, v4);
            }
            __syncwarp();
          }
        }
      }
      // All softmax warps that have rows, also those that gave up; the others cannot take the call with the registers left.
      asm volatile("bar.sync 1, %0;" ::"r"(128 * tiles) : "memory");
      if (*far_block && !*k.stop)
        finish_far<QT, D, TILES>(a, parts, smem, 4 * tiles);
    }
  } else if (warp < K::kIssuer) {
    // ---- codes to fp16: two warps the keys, two the values, a token per thread ----
    fewer_registers<K::kConverterRegisters>();
    const int t = threadIdx.x & 63;
    const bool values = warp >= K::kConverters + 2;
    const int *table = a.rows.pages + (size_t)s * a.rows.pages_stride;
    int page_of = -1, held = col0 - 32, asked = 0, ref = 0; // ref: exponent of the value scale that outputs are relative to
    bool any_far = false;
    unsigned there = 0; // of the columns held .. held + 31: those with a page, not a far one, that is still to be asked for
    float2 scale_of = make_float2(0.0f, 0.0f);
    // Every warp goes over the table the same way; one thread asks for the bytes.  Per raw stage:
    int ring_token[K::kRawStages];
    float2 ring_scale[K::kRawStages];
    auto ask = [&](int stage) { // the next column that has a page into `stage`; token -1: there is none
      ring_token[stage] = -1;
      while (!there && held + 32 < col1) {
        held += 32;
        page_of = held + lane < col1 ? a.cache.checked(__ldg(table + cols.at(held + lane))) : -1;
        if (page_of >= 0)
          scale_of = *reinterpret_cast<const float2 *>(a.cache.scale(page_of, head));
        const int v_exp = page_of >= 0 ? exponent_field(scale_of.y) : 0;
        if (ref == 0)
          ref = pick_ref(v_exp);
        const unsigned far = __ballot_sync(0xffffffffu, is_far(v_exp, ref));
        any_far = any_far || far;
        there = __ballot_sync(0xffffffffu, page_of >= 0) & ~far;
      }
      if (!there)
        return;
      const int from = __ffs(there) - 1, page = __shfl_sync(0xffffffffu, page_of, from);
      there &= there - 1;
      ring_token[stage] = cols.at(held + from) * kPage;
      ring_scale[stage].x = __shfl_sync(0xffffffffu, scale_of.x, from);
      ring_scale[stage].y = __shfl_sync(0xffffffffu, scale_of.y, from);
      if (threadIdx.x == kLeader) {
        const uint32_t b = k.bar(K::kRawFull + stage);
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(K::kRawBytes) : "memory");
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         k.base + K::kRaw + stage * K::kRawBytes),
                     "l"(a.cache.template block<D>(page, head)), "r"(K::kRawBytes), "r"(b)
                     : "memory");
      }
      asked++;
    };
    // The order in which a thread takes its token's pieces: such that 8 neighbouring threads' reads (rows of D
    // bytes) and swizzled writes (rows of 128) both fall into different banks; x -> 0, 2, 3, 1 and its xor with x
    // are both permutations.
    const int turn_of = (0x78 >> (t & 6) & 3) | (D == 128 ? (t & 1) << 2 : 0);
    auto convert = [&](uint32_t from, uint32_t to, uint32_t mul, uint32_t add) { // this thread's token
#pragma unroll
      for (int n = 0; n < D / 16; n++) { // 16 codes: two 16-byte pieces
        const int i = n ^ turn_of;
        const uint4 w = lds16(from + t * D + i * 16);
        const uint32_t u[4] = {biased(w.x), biased(w.y), biased(w.z), biased(w.w)};
#pragma unroll
        for (int e = 0; e < 2; e++)
          K::store16(to + K::swizzled(t, i * 2 + e, kPage), scaled_pair(low_pair(u[2 * e]), mul, add),
                     scaled_pair(high_pair(u[2 * e]), mul, add), scaled_pair(low_pair(u[2 * e + 1]), mul, add),
                     scaled_pair(high_pair(u[2 * e + 1]), mul, add));
      }
    };
#pragma unroll
    for (int i = 0; i < K::kRawStages; i++)
      ask(i);
    int used = 0;
    bool ok = true, more = true;
    static_assert(K::kKeyStages == K::kRawStages && K::kValueStages == K::kRawStages, "one stage number for all rings");
    while (ok && more) {
#pragma unroll
      for (int stage = 0; stage < K::kRawStages; stage++) { // of page `used`, known at compile time
        if (!ok || !more)
          break;
        const int j = used;
        const uint32_t turn = j / K::kRawStages & 1;
        more = ring_token[stage] >= 0;
        if (values && !more)
          break;
        if (j >= K::kRawStages && !(ok = k.wait_warp((values ? K::kValueFree : K::kKeyFree) + stage, turn ^ 1)))
          break;
        if (threadIdx.x == kLeader && !more && any_far) // behind the last page all columns have been looked at
          far_block[0] = 1, far_block[1] = ref;
        if (threadIdx.x == kLeader)
          meta[j % kMeta] = Meta{ring_token[stage], ring_scale[stage].x, ref, any_far};
        if (more) {
          if (!(ok = k.wait_warp(K::kRawFull + stage, turn)))
            break;
          uint32_t mul = 0x3c003c00u, add = 0xe480e480u; // times 1, minus 1152
          if (values)
            value_factor(exponent_field(ring_scale[stage].y), ref, mul, add);
          convert(k.base + K::kRaw + stage * K::kRawBytes + (values ? kPage * D : 0),
                  k.base + (values ? K::kValues : K::kKeys) + stage * K::kPageBytes, mul, add);
        }
        fence_async_smem();
        arrive_warp(k.bar((values ? K::kValueFull : K::kKeyFull) + stage));
        if (!more)
          break;
        if (lane == 0)
          arrive(k.bar(K::kRawFree + stage)); // this warp has read its part of the raw page
        used++;
        // the stage of the page before, which the other warps have most likely read too, gets the next page
        const int before = (stage + K::kRawStages - 1) % K::kRawStages;
        if (j > 0) {
          if (warp == K::kConverters && !(ok = k.wait_warp(K::kRawFree + before, (j - 1) / K::kRawStages & 1)))
            break;
          ask(before);
        }
      }
    }
    if (threadIdx.x == kLeader && !ok) // what is still on its way is waited for, with a limit of its own
      for (int p = used > 0 ? used - 1 : 0; p < asked; p++)
        mbar_wait_at(k.bar(K::kRawFull + p % K::kRawStages), p / K::kRawStages & 1);
  } else {
    // ---- matrix instructions --------------------------------------------------------------
    constexpr uint32_t kScoreShape = shape_of(kPage, false), kOutShape = shape_of(D, true);
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
          for (int i = 0; i < D / 64; i++)
            mma4_smem(scores_at(tile, n), q + (part * K::kQueryBytes + i * kTile * 128) / 16, keys + i * (kPage * 128 / 16),
                      kScoreShape, part + i > 0);
      }
      tc_commit(k.bar(K::kScoreFull + buffer(tile, n))); // also for the end of the pages
      if (tile == tiles - 1) {
        if (real) {
          tc_commit(k.bar(K::kKeyFree + key_stage));
          n++;
          if (++key_stage == K::kKeyStages)
            key_stage = 0, key_turn ^= 1;
        }
        more = real;
      }
    };
    for (int i = 0; i < kBuffers && ok; i++)
      for (int tile = 0; tile < tiles && ok; tile++)
        next_scores(tile);
    for (int j = 0; ok && j < n; j++) {
      for (int tile = 0; tile < tiles && ok; tile++) {
        if (!(ok = k.wait_warp(K::kWeightFull + buffer(tile, j), phase(j))))
          break;
        if (tile == 0 && !(ok = k.wait_warp(K::kValueFull + value_stage, value_turn)))
          break;
        tc_after_sync();
        const uint32_t values = values0 + value_stage * (K::kPageBytes / 16);
#pragma unroll
        for (int part = 0; part < (kSplit ? 2 : 1); part++)
          mma4_tmem<TILES == 2 ? 16 : 32>(out_at(tile), scores_at(tile, j) + part * 32, values, kOutShape, j % K::kFoldPages + part > 0);
        tc_commit(k.bar(K::kOutDone + tile));
        if (tile == tiles - 1)
          tc_commit(k.bar(K::kValueFree + value_stage));
        next_scores(tile);
      }
      if (++value_stage == K::kValueStages)
        value_stage = 0, value_turn ^= 1;
    }
    if (!ok) { // matrix instructions still running are waited for, with a limit, before their memory is given back
      tc_commit(k.bar(K::kDrained));
      mbar_wait_at(k.bar(K::kDrained), 0);
    }
  }
  __syncwarp();
  tc_before_sync();
  __syncthreads();
  if (warp == K::kIssuer) {
    tc_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// The parts of a unit joined, four elements per thread.
template <typename QT, int D> __global__ void __launch_bounds__(256) merge_parts(Call<QT> a, Parts parts, int rows) {
  constexpr int D4 = D / 4, kRowsHere = 256 / D4;
  pdl_prologue();
  const int heads = a.cache.n_kv_heads, index = blockIdx.x;
  const long r = blockIdx.y * kRowsHere + threadIdx.x / D4;
  Unit u = {};
  if (!u.find(a, (int)(gridDim.x / heads) - 1 - index / heads, index % heads, rows) || u.row0 + r >= u.R)
    return;
  const int d = threadIdx.x % D4 * 4, h = u.head * a.group + (int)((u.row0 + r) % a.group);
  const float z = a.sinks ? sink_of(a, h) : -INFINITY;
  auto at = [&](int split) { return ((size_t)index * parts.splits + split) * rows + r; };
  float top = z, sum = 0.0f;
#pragma unroll 8
  for (int i = 0; i < parts.splits; i++)
    if (u.column(i, parts.splits) < u.column(i + 1, parts.splits))
      top = fmaxf(top, parts.ml[at(i)].x);
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < parts.splits; i++)
    if (u.column(i, parts.splits) < u.column(i + 1, parts.splits)) {
      const float2 ml = parts.ml[at(i)];
      const float4 x = *reinterpret_cast<const float4 *>(parts.o + at(i) * D + d);
      const float part = ml.y != 0.0f ? ml.y * fast_exp2(ml.x - top) : 0.0f, of = part * two_to(-kSumBits); // a NaN passes
      sum += part;
      acc.x += of * x.x, acc.y += of * x.y, acc.z += of * x.z, acc.w += of * x.w;
    }
  if (sum != 0.0f && a.sinks)
    sum += fast_exp2(z - top);
  const float f = sum != 0.0f ? (float)(1 << kSumBits) / sum : 0.0f;
  store4(a, (size_t)(u.sp.row + (u.row0 + r) / a.group) * a.out_row_stride + (size_t)h * D + d,
         make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

long units_of(long T, int group, int n_seqs, int tiles) { return T * group / (kTile * tiles) + n_seqs; }
// Parts that a unit's columns are cut into where there are few units: about two blocks per SM, counting the units
// that the call's sizes allow for (the true number may be half).
int splits_for(long blocks) { return (int)std::min(32l, std::max(1l, 2l * sm_count() / std::max(blocks, 1l))); }

template <typename QT, int D, int TILES>
void launch_with(cudaStream_t stream, const Call<QT> &a, long units, int splits, void *workspace) {
  using K = TileKernel<QT, D, TILES>;
  const long blocks = units * a.cache.n_kv_heads;
  Parts parts = {splits, static_cast<float *>(workspace), nullptr};
  parts.ml = reinterpret_cast<float2 *>(parts.o + (size_t)blocks * splits * K::kRowsOfBlock * D);
  (void)blocks_per_sm_smem(attend_tiles<QT, D, TILES>, K::kThreads, K::kSmem);
  launch_kernel(attend_tiles<QT, D, TILES>, dim3((unsigned)(blocks * splits)), dim3(K::kThreads), K::kSmem, stream, a, parts);
  if (splits > 1) {
    const PdlScope chained(GPTOSS_PDL);
    launch_kernel(merge_parts<QT, D>, dim3((unsigned)blocks, K::kRowsOfBlock / (1024 / D)), dim3(256), 0, stream, a, parts,
                  (int)K::kRowsOfBlock);
  }
}

} // namespace

size_t tiles_workspace(long T, int group, int heads, int n_seqs, int head_dim) {
  const long blocks = units_of(T, group, n_seqs, 2) * heads;
  const int splits = splits_for(blocks);
  return splits > 1 ? Parts::bytes(blocks * splits, 2 * kTile, head_dim) : 0;
}

template <typename QT> void launch_tiles(cudaStream_t stream, const Call<QT> &a, int head_dim, void *workspace) {
  const long two = units_of(a.rows.T, a.group, a.rows.n_seqs, 2), four = units_of(a.rows.T, a.group, a.rows.n_seqs, 4);
  const int splits = std::min(splits_for(two * a.cache.n_kv_heads), std::max(1, a.rows.pages_stride / 4));
  if (head_dim == 128) {
    launch_with<QT, 128, 2>(stream, a, two, splits, workspace);
    return;
  }
  // Four tiles fit tensor memory at 64 elements and bf16 rows (one part of weights).  Where they would leave SMs
  // without a block, two: one prompt, 64 and 8 heads, two tiles against four: 700 tokens (80 by the condition below)
  // 27 / 32 us, 1000 (120) 37 / 39, 1300 (160) 58 / 50, 4000 (496) 291 / 221; five chunks (144) 167 / 132.
  if constexpr (sizeof(QT) == 2)
    if ((four - a.rows.n_seqs) * a.cache.n_kv_heads >= sm_count() * 7 / 8) {
      launch_with<QT, 64, 4>(stream, a, four, 1, workspace);
      return;
    }
  launch_with<QT, 64, 2>(stream, a, two, splits, workspace);
}
template void launch_tiles<float>(cudaStream_t, const Call<float> &, int, void *);
template void launch_tiles<uint16_t>(cudaStream_t, const Call<uint16_t> &, int, void *);

} // namespace kv8
} // namespace gptoss
