// Pages of the 8-bit cache: release, reserve, fork, compact, copy.
//
// The tables are a few thousand integers and the answers depend on order (the lowest free page
// goes to the first request), so each call's decisions are taken by ONE block of 1024 threads with
// scans, and what is heavy -- the pages' bytes -- is moved by a second launch over the whole GPU,
// from a list that the first one left in the workspace.  Nothing comes back to the host.
//
// Copies: 16 KB pieces of (pair, layer), 256 threads with four 16-byte loads each in flight and
// six blocks per SM (96 KB in flight per SM), which is what a plain copy needs to run at the
// memory's speed; the same launch first brings the tables in line with the plan.
// Decisions: bound by latency.  The reference counts are looked through 8192 at a time, eight
// independent coalesced loads per thread, ranks from warp ballots; a search for free pages stops as
// soon as it has enough.
// Measured, 200 sequences, 3900 pages of 64 KB in 8 layers: release 4 us, forks 10 us and 12 us for 60 copies, reserve
// 10 us, compaction 7 us and 172 us for 1.0 GB of moves (6.1 TB/s, 0.93 of a copy's rate).
#include <limits.h>

#include <algorithm>

#include "kv8.cuh"

namespace gptoss {
namespace kv8 {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kUnroll = 8;

// What a call keeps between its two launches.
struct Scratch {
  int *count; // pairs in the list
  int *src, *dst; // [n_pages]
  int *mark, *a, *b; // [n_seqs]
  static size_t bytes(int n_pages, int n_seqs) { return (16 + 2 * (size_t)n_pages + 3 * (size_t)n_seqs) * 4; }
  static Scratch at(void *ws, int n_pages, int n_seqs) {
    int *p = static_cast<int *>(ws);
    int *lists = p + 16, *seqs = lists + 2 * (size_t)n_pages;
    return Scratch{p, lists, lists + n_pages, seqs, seqs + n_seqs, seqs + 2 * (size_t)n_seqs};
  }
};

struct Table {
  int *kv_len, *pages, *refs;
  int n_seqs, stride, n_pages;
  __device__ __forceinline__ bool has(int s) const { return (unsigned)s < (unsigned)n_seqs; }
  __device__ __forceinline__ int *row(int s) const { return pages + (size_t)s * stride; }
  __device__ __forceinline__ bool is_page(int p) const { return (unsigned)p < (unsigned)n_pages; }
};

// Exclusive scan of v over the block; total in every thread.
__device__ __forceinline__ int block_scan(int v, int *total) {
  __shared__ int warp_sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o)
      x += y;
  }
  if (lane == 31)
    warp_sums[warp] = x;
  __syncthreads();
  const int w = warp_sums[lane];
  int y = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o)
      y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  const int before = __shfl_sync(0xffffffffu, y - w, warp);
  __syncthreads(); // warp_sums may be used again
  return before + x - v;
}

// Calls take(page, rank, refs) for every page in [from, to) whose reference count pred accepts, rank
// counting them in order, until `want` of them are found; returns how many there were (at most
// `want`, or as many as the tile that reached it had).  Whole block.
template <typename Pred, typename Take>
__device__ int for_pages(const int *refs, int from, int to, int want, Pred pred, Take take) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int found = 0;
  for (long tile = from; tile < to && found < want; tile += kThreads * kUnroll) {
    const long first = tile + warp * (32 * kUnroll) + lane;
    int r[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; i++)
      r[i] = first + 32 * i < to ? refs[first + 32 * i] : 0;
    unsigned hit[kUnroll];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kUnroll; i++) {
      hit[i] = __ballot_sync(0xffffffffu, first + 32 * i < to && pred(r[i]));
      mine += __popc(hit[i]);
    }
    int total;
    int rank = found + __shfl_sync(0xffffffffu, block_scan(lane == 0 ? mine : 0, &total), 0);
#pragma unroll
    for (int i = 0; i < kUnroll; i++) {
      if (hit[i] >> lane & 1)
        take((int)first + 32 * i, rank + __popc(hit[i] & ((1u << lane) - 1)), r[i]);
      rank += __popc(hit[i]);
    }
    found += total;
  }
  return found;
}

// The `want` lowest free pages into list; returns how many there are, at most `want`.  Whole block.
__device__ int lowest_free(const Table &t, int want, int *list) {
  const int found = for_pages(
      t.refs, 0, t.n_pages, want, [](int r) { return r == 0; },
      [&](int page, int rank, int) {
        if (rank < want)
          list[rank] = page;
      });
  __syncthreads();
  return min(found, want);
}

// ---- release --------------------------------------------------------------------------

__global__ void __launch_bounds__(256) release_pages(Table t, int n, const int *__restrict__ seqs, int window, int n_first) {
  pdl_prologue();
  const long all = (long)n * t.stride;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
    const int s = seqs[i / t.stride], j = (int)(i % t.stride);
    if (!t.has(s))
      continue;
    if (window > 0) {
      // the next token's position is at least kv_len, and it sees t > position - window
      const long last = (long)j * kPage + kPage - 1;
      if (last > (long)t.kv_len[s] - window || (long)j * kPage < n_first)
        continue;
    }
    // an exchange, so that a sequence listed twice gives up each page once
    if (t.row(s)[j] != -1) {
      const int page = atomicExch(t.row(s) + j, -1);
      if (t.is_page(page))
        atomicSub(t.refs + page, 1);
    }
    if (window <= 0 && j == 0)
      t.kv_len[s] = 0;
  }
}

// ---- reserve --------------------------------------------------------------------------

// A sequence whose next token belongs on a page that it has begun and that is not there any more.  It gets none: the
// tokens before would come back with what a free page holds, another sequence's.
__device__ __forceinline__ bool lost_its_page(const Table &t, int s, long len) {
  return len % kPage != 0 && !t.is_page(t.row(s)[len / kPage]);
}

// Requests 1024 at a time: columns [lo, hi) of a sequence's row that are to have pages, flattened so
// that the threads share the columns of one long request as well as those of many short ones.
template <typename Column>
__device__ void for_columns(const Table &t, int n, const int *seqs, const int *new_len, const int *mark, Column column) {
  __shared__ int first[kThreads + 1], low[kThreads], of[kThreads];
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + threadIdx.x;
    int lo = 0, hi = 0, s = -1;
    if (i < n) {
      s = seqs[i];
      if (t.has(s) && mark[s] == i) {
        const long len = max(t.kv_len[s], 0), want = new_len[i];
        if (want <= (long)t.stride * kPage && want > len && !lost_its_page(t, s, len))
          lo = (int)((len + kPage - 1) / kPage), hi = (int)((want + kPage - 1) / kPage);
      }
    }
    int total;
    first[threadIdx.x] = block_scan(hi - lo, &total);
    low[threadIdx.x] = lo, of[threadIdx.x] = s;
    if (threadIdx.x == 0)
      first[kThreads] = total;
    __syncthreads();
    for (int c0 = 0; c0 < total; c0 += kThreads) {
      const int c = c0 + threadIdx.x;
      int k = 0;
      bool open = false;
      int *entry = nullptr;
      if (c < total) {
        int up = kThreads; // the last k with first[k] <= c
        while (up - k > 1) {
          const int mid = (k + up) >> 1;
          if (first[mid] <= c)
            k = mid;
          else
            up = mid;
        }
        entry = t.row(of[k]) + low[k] + (c - first[k]);
        open = !t.is_page(*entry);
      }
      column(base + k, entry, open, c < total && c == first[k], c < total && c + 1 == first[k + 1]);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads)
    reserve_pages(Table t, int n, const int *__restrict__ seqs, const int *__restrict__ new_len, int *served, Scratch ws) {
  pdl_prologue();
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (t.has(seqs[i]))
      ws.mark[seqs[i]] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (t.has(seqs[i]))
      atomicMin(ws.mark + seqs[i], i);
  for (int i = threadIdx.x; i < n; i += kThreads)
    ws.a[i] = ws.b[i] = 0; // pages asked for up to and with request i, and before it
  __syncthreads();
  int want = 0;
  for_columns(t, n, seqs, new_len, ws.mark, [&](int i, int *, bool open, bool first, bool last) {
    int total;
    const int rank = want + block_scan(open, &total);
    if (first)
      ws.b[i] = rank;
    if (last)
      ws.a[i] = rank + open;
    want += total;
  });
  const int found = lowest_free(t, want, ws.src);
  int given = 0;
  for_columns(t, n, seqs, new_len, ws.mark, [&](int i, int *entry, bool open, bool, bool) {
    int total;
    const int rank = given + block_scan(open, &total);
    if (open && ws.a[i] <= found) {
      *entry = ws.src[rank];
      t.refs[ws.src[rank]] = 1;
    }
    given += total;
  });
  if (served)
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int s = seqs[i];
      const long len = t.has(s) ? max(t.kv_len[s], 0) : 0;
      served[i] = t.has(s) && ws.mark[s] == i && new_len[i] <= (long)t.stride * kPage &&
                  (ws.a[i] <= found || ws.a[i] == ws.b[i]) && (new_len[i] <= len || !lost_its_page(t, s, len));
    }
}

// ---- fork -----------------------------------------------------------------------------

__global__ void __launch_bounds__(kThreads)
    plan_forks(Table t, int n, const int *__restrict__ parents, const int *__restrict__ children, int *served, Scratch ws) {
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    if (t.has(parents[i]))
      ws.mark[parents[i]] = INT_MAX;
    if (t.has(children[i]))
      ws.mark[children[i]] = INT_MAX;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (t.has(children[i]))
      atomicMin(ws.mark + children[i], i);
  __syncthreads();
  // a: 0 refused, 1 shares full pages only, 2 also copies a last page
  for (int i = warp; i < n; i += kWarps) {
    const int p = parents[i], c = children[i];
    bool ok = t.has(p) && t.has(c) && ws.mark[c] == i && ws.mark[p] == INT_MAX;
    int len = 0;
    if (ok) {
      len = t.kv_len[p];
      ok = t.kv_len[c] == 0 && len >= 0 && len <= (long)t.stride * kPage;
    }
    if (ok)
      for (int j = lane; j < t.stride; j += 32)
        ok = ok && !t.is_page(t.row(c)[j]);
    ok = __all_sync(0xffffffffu, ok);
    if (lane == 0)
      ws.a[i] = !ok ? 0 : len % kPage && t.is_page(t.row(p)[len / kPage]) ? 2 : 1;
  }
  __syncthreads();
  int want = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + threadIdx.x, copies = i < n && ws.a[i] == 2;
    int total;
    const int rank = block_scan(copies, &total);
    if (i < n)
      ws.b[i] = copies ? want + rank : -1;
    want += total;
  }
  const int found = lowest_free(t, want, ws.dst);
  // From here on src/dst hold one pair per fork that copies, in rank order, and b tells its rank.
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int rank = ws.b[i];
    if (rank >= found)
      ws.a[i] = 0;
    else if (rank >= 0)
      ws.src[rank] = t.row(parents[i])[t.kv_len[parents[i]] / kPage];
    if (served)
      served[i] = ws.a[i] != 0;
  }
  if (threadIdx.x == 0)
    *ws.count = found;
}

// The children's rows, a warp per fork.
struct WriteForks {
  Table t;
  int n;
  const int *parents, *children;
  Scratch ws;
  __device__ __forceinline__ void operator()() const {
    const int lane = threadIdx.x & 31;
    for (int i = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < n; i += (gridDim.x * blockDim.x) >> 5) {
      if (ws.a[i] == 0)
        continue;
      const int p = parents[i], c = children[i], len = t.kv_len[p], full = len / kPage;
      for (int j = lane; j < full; j += 32) {
        const int page = t.row(p)[j];
        if (t.is_page(page)) {
          t.row(c)[j] = page;
          atomicAdd(t.refs + page, 1);
        }
      }
      if (lane == 0) {
        t.kv_len[c] = len;
        if (ws.a[i] == 2) {
          const int page = ws.dst[ws.b[i]];
          t.row(c)[full] = page;
          t.refs[page] = 1;
        }
      }
    }
  }
};

// ---- compact --------------------------------------------------------------------------

__global__ void __launch_bounds__(kThreads) plan_compaction(Table t, int *remap, int *n_live_out, Scratch ws) {
  pdl_prologue();
  auto live = [](int r) { return r != 0; };
  const int n_live = for_pages(t.refs, 0, t.n_pages, INT_MAX, live, [&](int, int, int) {});
  const int holes = for_pages(
      t.refs, 0, n_live, INT_MAX, [](int r) { return r == 0; }, [&](int page, int rank, int) { ws.dst[rank] = page; });
  for_pages(t.refs, n_live, t.n_pages, holes, live, [&](int page, int rank, int) { ws.src[rank] = page; });
  for (int i = threadIdx.x; i < t.n_pages; i += kThreads)
    remap[i] = i < n_live && t.refs[i] != 0 ? i : -1;
  __syncthreads();
  for (int k = threadIdx.x; k < holes; k += kThreads) {
    const int from = ws.src[k], to = ws.dst[k];
    remap[from] = to;
    t.refs[to] = t.refs[from];
    t.refs[from] = 0;
  }
  if (threadIdx.x == 0)
    *n_live_out = n_live, *ws.count = holes;
}

struct RenumberTables {
  Table t;
  const int *remap;
  __device__ __forceinline__ void operator()() const {
    const long all = (long)t.n_seqs * t.stride;
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
      const int page = t.pages[i];
      if (t.is_page(page))
        t.pages[i] = remap[page];
    }
  }
};
struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};

// ---- the pages' bytes -------------------------------------------------------------------

constexpr int kPiece = 16384;

struct Pool {
  int8_t *codes;
  float *scales;
  long page_bytes; // codes of one page of one layer
  int page_scales, n_layers, n_pages;
};

// What a plan changes in the tables (`first`), then pairs (src[i], dst[i]), i < *count (or n where count is NULL),
// in every layer.  The two do not meet: the pairs come from the plan's list alone.
template <typename First>
__global__ void __launch_bounds__(256, 6)
    copy_pairs(First first, Pool pool, int n, const int *count, const int *__restrict__ src, const int *__restrict__ dst) {
  pdl_prologue();
  first();
  if (count)
    n = *count;
  const long pieces = (pool.page_bytes + kPiece - 1) / kPiece, all = (long)n * pool.n_layers * pieces;
  for (long w = blockIdx.x; w < all; w += gridDim.x) {
    const long piece = w % pieces, rest = w / pieces;
    const int layer = (int)(rest % pool.n_layers), i = (int)(rest / pool.n_layers);
    const int from = src[i], to = dst[i];
    if ((unsigned)from >= (unsigned)pool.n_pages || (unsigned)to >= (unsigned)pool.n_pages || from == to)
      continue;
    const size_t a = (size_t)layer * pool.n_pages + from, b = (size_t)layer * pool.n_pages + to;
    const int8_t *x = pool.codes + a * pool.page_bytes + piece * kPiece;
    int8_t *y = pool.codes + b * pool.page_bytes + piece * kPiece;
    const int left = (int)min((long)kPiece, pool.page_bytes - piece * kPiece);
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if ((int)(threadIdx.x + 256 * j) * 16 < left)
        v[j] = ld_stream(x + (threadIdx.x + 256 * j) * 16);
#pragma unroll
    for (int j = 0; j < 4; j++)
      if ((int)(threadIdx.x + 256 * j) * 16 < left)
        st_stream(y + (threadIdx.x + 256 * j) * 16, v[j]);
    if (piece == 0)
      for (int j = threadIdx.x; j < pool.page_scales; j += 256)
        pool.scales[b * pool.page_scales + j] = pool.scales[a * pool.page_scales + j];
  }
}

// first_blocks: blocks that `first` has work for.
template <typename First>
void launch_copies(cudaStream_t stream, First first, long first_blocks, const gptoss_kv8_pool_t *p, int n_most, const int *count,
                   const int *src, const int *dst) {
  const Pool pool = {p->codes, p->scales, (long)p->n_kv_heads * 2 * kPage * p->head_dim, p->n_kv_heads * 2, p->n_layers,
                     p->n_pages};
  const long all = (long)n_most * p->n_layers * ((pool.page_bytes + kPiece - 1) / kPiece);
  launch_kernel(copy_pairs<First>, dim3(row_grid(std::max(all, first_blocks), 6)), dim3(256), 0, stream, first, pool, n_most, count,
                src, dst);
}

int check_table(int n_seqs, const int *pages, int pages_stride, int n_pages, const int *refs) {
  if (n_seqs <= 0 || pages_stride <= 0 || n_pages <= 0 || !pages || !refs)
    return GPTOSS_ERR_BAD_ARG;
  if (n_seqs > kMaxTokens / 4 || pages_stride > kMaxTokens / kPage || n_pages > kMaxTokens)
    return GPTOSS_ERR_UNSUPPORTED;
  GPTOSS_SPAN(pages, (size_t)n_seqs * pages_stride * 4);
  GPTOSS_SPAN(refs, (size_t)n_pages * 4);
  return GPTOSS_OK;
}
int check_workspace(const void *ws, size_t bytes, int n_pages, int n_seqs) {
  if (!ws || !aligned16(ws) || bytes < Scratch::bytes(n_pages, n_seqs))
    return GPTOSS_ERR_BAD_ARG;
  GPTOSS_SPAN(ws, bytes);
  return GPTOSS_OK;
}
// A second launch of the same call need not be flushed to before it is set up.
struct Chained : PdlScope {
  Chained() : PdlScope(GPTOSS_PDL) {}
};

} // namespace
} // namespace kv8
} // namespace gptoss

extern "C" size_t gptoss_kv8_pages_workspace(int n_pages, int n_seqs) {
  return n_pages <= 0 || n_seqs <= 0 ? 0 : gptoss::kv8::Scratch::bytes(n_pages, n_seqs);
}

extern "C" int gptoss_kv8_release(gptoss_stream_t stream, int n, const int *seqs, int n_seqs, int *kv_len, int *pages,
                                  int pages_stride, int n_pages, int *refs, int window, int n_first, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (n < 0 || window < 0 || n_first < 0)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_table(n_seqs, pages, pages_stride, n_pages, refs))
    return st;
  if (n == 0)
    return GPTOSS_OK;
  if (!seqs || !kv_len)
    return GPTOSS_ERR_BAD_ARG;
  GPTOSS_SPAN(seqs, (size_t)n * 4);
  GPTOSS_SPAN(kv_len, (size_t)n_seqs * 4);
  const kv8::Table t = {kv_len, pages, refs, n_seqs, pages_stride, n_pages};
  const int grid = row_grid(((long)n * pages_stride + 255) / 256, 8);
  launch_kernel(kv8::release_pages, dim3(grid), dim3(256), 0, as_stream(stream), t, n, seqs, window, n_first);
  return launch_status();
}

extern "C" int gptoss_kv8_reserve(gptoss_stream_t stream, int n, const int *seqs, const int *new_len, int n_seqs,
                                  const int *kv_len, int *pages, int pages_stride, int n_pages, int *refs, int *served,
                                  void *workspace, size_t workspace_bytes, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (n < 0 || n > n_seqs)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_table(n_seqs, pages, pages_stride, n_pages, refs))
    return st;
  if ((long)n * pages_stride > kv8::kMaxTokens) // columns are numbered in 32 bits
    return GPTOSS_ERR_UNSUPPORTED;
  if (n == 0)
    return GPTOSS_OK;
  if (!seqs || !new_len || !kv_len)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_workspace(workspace, workspace_bytes, n_pages, n_seqs))
    return st;
  GPTOSS_SPAN(seqs, (size_t)n * 4);
  GPTOSS_SPAN(new_len, (size_t)n * 4);
  GPTOSS_SPAN(kv_len, (size_t)n_seqs * 4);
  GPTOSS_SPAN(served, (size_t)n * 4);
  const kv8::Table t = {const_cast<int *>(kv_len), pages, refs, n_seqs, pages_stride, n_pages};
  launch_kernel(kv8::reserve_pages, dim3(1), dim3(kv8::kThreads), 0, as_stream(stream), t, n, seqs, new_len, served,
                kv8::Scratch::at(workspace, n_pages, n_seqs));
  return launch_status();
}

extern "C" int gptoss_kv8_fork(gptoss_stream_t stream, const gptoss_kv8_pool_t *pool, int n, const int *parents,
                               const int *children, int n_seqs, int *kv_len, int *pages, int pages_stride, int *refs,
                               int *served, void *workspace, size_t workspace_bytes, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (n < 0 || n > n_seqs)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_pool(pool))
    return st;
  if (const int st = kv8::check_table(n_seqs, pages, pages_stride, pool->n_pages, refs))
    return st;
  if (n == 0)
    return GPTOSS_OK;
  if (!parents || !children || !kv_len)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_workspace(workspace, workspace_bytes, pool->n_pages, n_seqs))
    return st;
  GPTOSS_SPAN(parents, (size_t)n * 4);
  GPTOSS_SPAN(children, (size_t)n * 4);
  GPTOSS_SPAN(kv_len, (size_t)n_seqs * 4);
  GPTOSS_SPAN(served, (size_t)n * 4);
  GPTOSS_SPAN(pool->codes, kv8::layer_codes(pool) * pool->n_layers);
  GPTOSS_SPAN(pool->scales, kv8::layer_scales(pool) * pool->n_layers * 4);
  const kv8::Table t = {kv_len, pages, refs, n_seqs, pages_stride, pool->n_pages};
  const kv8::Scratch ws = kv8::Scratch::at(workspace, pool->n_pages, n_seqs);
  launch_kernel(kv8::plan_forks, dim3(1), dim3(kv8::kThreads), 0, as_stream(stream), t, n, parents, children, served, ws);
  const kv8::Chained chained;
  kv8::launch_copies(as_stream(stream), kv8::WriteForks{t, n, parents, children, ws}, (n + 7) / 8, pool, n, ws.count, ws.src, ws.dst);
  return launch_status();
}

extern "C" int gptoss_kv8_compact(gptoss_stream_t stream, const gptoss_kv8_pool_t *pool, int n_seqs, int *pages,
                                  int pages_stride, int *refs, int *remap, int *n_live_out, void *workspace,
                                  size_t workspace_bytes, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (const int st = kv8::check_pool(pool))
    return st;
  if (const int st = kv8::check_table(n_seqs, pages, pages_stride, pool->n_pages, refs))
    return st;
  if (!remap || !n_live_out)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_workspace(workspace, workspace_bytes, pool->n_pages, n_seqs))
    return st;
  GPTOSS_SPAN(remap, (size_t)pool->n_pages * 4);
  GPTOSS_SPAN(n_live_out, 4);
  GPTOSS_SPAN(pool->codes, kv8::layer_codes(pool) * pool->n_layers);
  GPTOSS_SPAN(pool->scales, kv8::layer_scales(pool) * pool->n_layers * 4);
  const kv8::Table t = {nullptr, pages, refs, n_seqs, pages_stride, pool->n_pages};
  const kv8::Scratch ws = kv8::Scratch::at(workspace, pool->n_pages, n_seqs);
  launch_kernel(kv8::plan_compaction, dim3(1), dim3(kv8::kThreads), 0, as_stream(stream), t, remap, n_live_out, ws);
  const kv8::Chained chained;
  // at most half of the pages can move: as many as there are holes below, and live pages above
  kv8::launch_copies(as_stream(stream), kv8::RenumberTables{t, remap}, ((long)n_seqs * pages_stride + 255) / 256, pool,
                     pool->n_pages / 2, ws.count, ws.src, ws.dst);
  return launch_status();
}

extern "C" int gptoss_kv8_copy_pages(gptoss_stream_t stream, const gptoss_kv8_pool_t *pool, int n, const int *src,
                                     const int *dst, unsigned flags) {
  using namespace gptoss;
  const PdlScope pdl(flags);
  if (n < 0)
    return GPTOSS_ERR_BAD_ARG;
  if (const int st = kv8::check_pool(pool))
    return st;
  if (n == 0)
    return GPTOSS_OK;
  if (!src || !dst)
    return GPTOSS_ERR_BAD_ARG;
  GPTOSS_SPAN(src, (size_t)n * 4);
  GPTOSS_SPAN(dst, (size_t)n * 4);
  GPTOSS_SPAN(pool->codes, kv8::layer_codes(pool) * pool->n_layers);
  GPTOSS_SPAN(pool->scales, kv8::layer_scales(pool) * pool->n_layers * 4);
  kv8::launch_copies(as_stream(stream), kv8::Nothing{}, 0, pool, n, nullptr, src, dst);
  return launch_status();
}
