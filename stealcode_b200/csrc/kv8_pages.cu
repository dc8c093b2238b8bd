// kv8_pages.cu -- page bookkeeping of the paged 8-bit cache, on the device:
// taking pages for new tokens (reserve), sharing a sequence's past with
// others (fork), giving pages back (release, slide) and moving the pages in
// use to the lowest ids (compact).
//
// refs[page] counts the table entries that name a page; a page is free when
// it is 0.  The result never depends on the order in which threads run: the
// r-th page that a call needs, in the order of the call's sequences, is the
// r-th lowest free id, and counts change by integer atomics only.
//
// The plans run in one thread-block cluster: its blocks count their share of
// refs, exchange the counts through distributed shared memory, and know from
// them the rank of every free page, in one launch.  A call that cannot be
// served (too few free pages, a table row too short, a sequence named twice
// or outside the cache) changes nothing and sets a bit of the cache's status
// word; while a bit is set, reserve, fork, compact and append do nothing, so
// a step queued behind a failed one cannot write over a page.  release and
// slide always run: giving pages back is how a caller recovers.
//
// Measured: reserving 256 prompts in a pool of 87 k pages 15 us (a chain of
// cluster barriers and table loads), release and slide 4.6 us each; forking
// 256 hypotheses over 24 layers 131 us, of them 117 for 684 MB of page copies
// (5.9 TB/s); moving half of 24 layers' pages 302 us for 1.7 GB (5.7 TB/s).
#include <atomic>

#include <cooperative_groups.h>

#include "kv8.cuh"
#include "sc_kernels.cuh"

namespace cg = cooperative_groups;

namespace sc {
namespace kv8 {

constexpr int kPlanCtas = 8;       // portable cluster size
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

// Workspace (int32 words): header, then one array each.
struct PageWs {
  int32_t *head;   // [0] pages to copy, [1] live pages
  int32_t *src, *dst, *used;  // [n_pages] copies: from, to, tokens
  int32_t *map;    // [n_pages] free pages by rank, or a moved page's new id
  int32_t *off, *len;  // [n_seqs]
  int32_t *rows;   // [n_seqs][max_pages] staged table rows
};
constexpr int kHeadWords = 64;

__host__ __device__ static inline PageWs page_ws(void *p, int64_t n_pages, int64_t n_seqs) {
  PageWs w;
  w.head = (int32_t *)p;
  w.src = w.head + kHeadWords;
  w.dst = w.src + n_pages;
  w.used = w.dst + n_pages;
  w.map = w.used + n_pages;
  w.off = w.map + n_pages;
  w.len = w.off + n_seqs;
  w.rows = w.len + n_seqs;
  return w;
}

size_t page_ws_bytes(int64_t n_pages, int64_t n_seqs, int64_t max_pages) {
  return 4 * (size_t)(kHeadWords + 4 * n_pages + 2 * n_seqs + n_seqs * max_pages);
}

__device__ __forceinline__ int pages_for(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// Exclusive sum of v over the block; *total gets the sum.  All threads call.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous use of warp_sums is over
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kPlanWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[kPlanWarps - 1];
  return (warp ? warp_sums[warp - 1] : 0) + x - v;
}

struct PlanShared {
  int sums[32];
  int mine[2];   // this block's counts, read by the others
  int flag;
};

// True if the cache's status word was set before this kernel: block 0's
// reading counts for the whole cluster, so its blocks leave together.
__device__ __forceinline__ bool stopped(cg::cluster_group cl, PlanShared &sh, const uint32_t *status) {
  if (threadIdx.x == 0) sh.flag = *status != 0;
  cl.sync();
  const bool stop = *cl.map_shared_rank(&sh.flag, 0) != 0;
  if (stop) cl.sync();  // block 0's shared memory is read until here
  return stop;
}

// Sum of a count over the cluster and over the blocks before this one.
__device__ __forceinline__ void cluster_scan(cg::cluster_group cl, int *slot, int *before, int *all) {
  cl.sync();
  int b = 0, t = 0;
  const int me = (int)cl.block_rank();
  for (int r = 0; r < kPlanCtas; r++) {
    const int v = *cl.map_shared_rank(slot, r);
    if (r < me) b += v;
    t += v;
  }
  *before = b;
  *all = t;
}

// This block's share of the pages: [lo, hi), a multiple of 4 wide.
__device__ __forceinline__ void page_share(int n_pages, int rank, int *lo, int *hi) {
  const int64_t per = ((int64_t)n_pages + kPlanCtas * 4 - 1) / (kPlanCtas * 4) * 4;
  const int64_t a = per * rank, b = a + per;
  *lo = (int)(a < n_pages ? a : n_pages);
  *hi = (int)(b < n_pages ? b : n_pages);
}

// Bit e: page p0 + e (of 4, from a multiple of 4) is free and below hi.
__device__ __forceinline__ unsigned free_bits(const int32_t *refs, int p0, int hi) {
  if (p0 >= hi) return 0;
  if (p0 + 4 > hi) {
    unsigned b = 0;
    for (int e = 0; p0 + e < hi; e++) b |= (refs[p0 + e] == 0 ? 1u : 0u) << e;
    return b;
  }
  const int4 r = *(const int4 *)(refs + p0);
  return (r.x == 0 ? 1u : 0u) | (r.y == 0 ? 2u : 0u) | (r.z == 0 ? 4u : 0u) | (r.w == 0 ? 8u : 0u);
}

// Writes the lowest `need` free pages, ascending, to list (if there are that
// many); returns the number of free pages of the pool.  All blocks call; the
// list is complete after the caller's next cluster sync.
__device__ int list_free(cg::cluster_group cl, PlanShared &sh, const int32_t *refs, int n_pages, int need,
                         int32_t *list) {
  constexpr int kStrip = 4 * kPlanThreads;
  int lo, hi;
  page_share(n_pages, (int)cl.block_rank(), &lo, &hi);
  int n = 0;
#pragma unroll 4
  for (int p = lo + 4 * (int)threadIdx.x; p < hi; p += kStrip) n += __popc(free_bits(refs, p, hi));
  int total, before, all;
  block_scan(n, sh.sums, &total);
  if (threadIdx.x == 0) sh.mine[0] = total;
  cluster_scan(cl, &sh.mine[0], &before, &all);
  if (all >= need) {
    for (int p0 = lo; p0 < hi && before < need; p0 += kStrip) {
      const int p = p0 + 4 * (int)threadIdx.x;
      unsigned f = free_bits(refs, p, hi);
      int r = before + block_scan(__popc(f), sh.sums, &total);
      for (; f && r < need; f &= f - 1, r++) list[r] = p + __ffs(f) - 1;
      before += total;
    }
  }
  return all;
}

// True if every id lies in the cache and none is named twice; each block
// finds out by itself, with a bit for each sequence in shared memory.
__device__ bool check_unique(const int32_t *seqs, int m, int n_seqs) {
  extern __shared__ uint32_t named[];
  if (!seqs) return m <= n_seqs;
  for (int i = (int)threadIdx.x; i < (n_seqs + 31) / 32; i += kPlanThreads) named[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = (int)threadIdx.x; i < m; i += kPlanThreads) {
    const unsigned s = (unsigned)seqs[i];
    bad |= s >= (unsigned)n_seqs || (atomicOr(&named[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1u;
  }
  return !__syncthreads_or(bad);
}

// ---- reserve -------------------------------------------------------------------

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    reserve_kernel(const PageArgs p, const int32_t *seqs, const int32_t *counts, int m) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ PlanShared sh;
  const PageWs w = page_ws(p.ws, p.n_pages, p.n_seqs);
  if (stopped(cl, sh, p.status)) return;
  uint32_t fail = check_unique(seqs, m, p.n_seqs) ? 0u : (uint32_t)kBadSeq;
  // pages each sequence needs, and where its pages start in the list
  int64_t need = 0;
  int wide = 0, negative = 0;
  for (int i0 = 0; !fail && i0 < m; i0 += kPlanThreads) {
    const int i = i0 + (int)threadIdx.x;
    int n = 0;
    if (i < m) {
      const int s = seqs ? seqs[i] : i;
      const int64_t len = p.length[s], end = len + counts[i];
      if (counts[i] < 0) negative = 1;
      else if (end > (int64_t)p.max_pages * p.page || end > INT32_MAX) wide = 1;
      else n = pages_for(end, p.page) - pages_for(len, p.page);
    }
    int total;
    const int at = block_scan(n, sh.sums, &total);
    if (cl.block_rank() == 0 && i < m) w.off[i] = (int)(need + at);
    need += total;
  }
  if (__syncthreads_or(wide)) fail |= kFullTable;
  if (__syncthreads_or(negative)) fail |= kBadSeq;
  if (!fail) {
    const int want = need > p.n_pages ? INT32_MAX : (int)need;
    if (list_free(cl, sh, p.refs, p.n_pages, want, w.map) < want) fail |= kFullPool;
  }
  cl.sync();
  if (fail) {
    if (cl.block_rank() == 0 && threadIdx.x == 0) atomicOr(p.status, fail);
    return;
  }
  const int warp = (int)(cl.block_rank() * kPlanWarps + (threadIdx.x >> 5)), lane = (int)threadIdx.x & 31;
  for (int i = warp; i < m; i += kPlanCtas * kPlanWarps) {
    const int s = seqs ? seqs[i] : i;
    const int64_t len = p.length[s], end = len + counts[i];
    const int have = pages_for(len, p.page), n = pages_for(end, p.page) - have;
    const int off = __ldcg(&w.off[i]);
    int32_t *row = p.table + (int64_t)s * p.max_pages + have;
    for (int j0 = lane; j0 < n; j0 += 256) {
      int pid[8];
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (j0 + 32 * e < n) pid[e] = __ldcg(&w.map[off + j0 + 32 * e]);
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (j0 + 32 * e < n) {
          row[j0 + 32 * e] = pid[e];
          p.refs[pid[e]] = 1;
        }
    }
    __syncwarp();
    if (lane == 0) p.length[s] = (int)end;
  }
}

// ---- fork ----------------------------------------------------------------------

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    fork_kernel(const PageArgs p, const int32_t *parents, const int32_t *children, int m) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ PlanShared sh;
  const PageWs w = page_ws(p.ws, p.n_pages, p.n_seqs);
  const bool first = cl.block_rank() == 0 && threadIdx.x == 0;
  if (first) w.head[0] = 0;
  if (stopped(cl, sh, p.status)) return;
  uint32_t fail = check_unique(children, m, p.n_seqs) ? 0u : (uint32_t)kBadSeq;
  int bad = 0;
  for (int i = (int)threadIdx.x; i < m; i += kPlanThreads) bad |= (unsigned)parents[i] >= (unsigned)p.n_seqs;
  if (__syncthreads_or(bad)) fail |= kBadSeq;
  // a child other than its parent gets a copy of the parent's last page, if
  // that is partly filled
  int need = 0;
  for (int i0 = 0; !fail && i0 < m; i0 += kPlanThreads) {
    const int i = i0 + (int)threadIdx.x;
    int fresh = 0, len = 0, last = -1;
    if (i < m) {
      const int par = parents[i];
      len = p.length[par];
      if (len < 0) len = 0;
      if (len > 0 && len % p.page != 0 && par != children[i]) {
        const int j = len / p.page;
        last = j < p.max_pages ? p.table[(int64_t)par * p.max_pages + j] : -1;
        fresh = (unsigned)last < (unsigned)p.n_pages;
      }
    }
    int total;
    const int r = need + block_scan(fresh, sh.sums, &total);
    if (cl.block_rank() == 0 && i < m) {
      w.len[i] = len;
      w.off[i] = fresh ? r : -1;
      if (fresh && r < p.n_pages) {
        w.src[r] = last;
        w.used[r] = len % p.page;
      }
    }
    need += total;
  }
  if (!fail && list_free(cl, sh, p.refs, p.n_pages, need, w.dst) < need) fail |= kFullPool;
  cl.sync();
  if (first) w.head[0] = fail ? 0 : need;
  if (fail) {
    if (first) atomicOr(p.status, fail);
    return;
  }
  // stage the parents' rows: a parent may be some other pair's child
  const int warp = (int)(cl.block_rank() * kPlanWarps + (threadIdx.x >> 5)), lane = (int)threadIdx.x & 31;
  for (int i = warp; i < m; i += kPlanCtas * kPlanWarps) {
    const int len = __ldcg(&w.len[i]), np = min(pages_for(len, p.page), p.max_pages);
    const int off = __ldcg(&w.off[i]);
    const int32_t *row = p.table + (int64_t)parents[i] * p.max_pages;
    for (int j = lane; j < np; j += 32)
      w.rows[(int64_t)i * p.max_pages + j] = off >= 0 && j == np - 1 ? __ldcg(&w.dst[off]) : row[j];
  }
  cl.sync();
  for (int i = warp; i < m; i += kPlanCtas * kPlanWarps) {
    const int len = __ldcg(&w.len[i]), np = min(pages_for(len, p.page), p.max_pages);
    const int s = children[i];
    const int was = min(pages_for(max(p.length[s], 0), p.page), p.max_pages);
    int32_t *row = p.table + (int64_t)s * p.max_pages;
    for (int j = lane; j < max(np, was); j += 32) {
      const int old = row[j], now = j < np ? __ldcg(&w.rows[(int64_t)i * p.max_pages + j]) : -1;
      if (old == now) continue;
      if ((unsigned)old < (unsigned)p.n_pages) atomicSub(&p.refs[old], 1);
      if ((unsigned)now < (unsigned)p.n_pages) atomicAdd(&p.refs[now], 1);
      row[j] = now;
    }
    __syncwarp();
    if (lane == 0) p.length[s] = len;
  }
}

// ---- compact -------------------------------------------------------------------

// The r-th live page at or above the number of live pages moves into the
// r-th free page below it.
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    compact_kernel(const PageArgs p) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ PlanShared sh;
  const PageWs w = page_ws(p.ws, p.n_pages, p.n_seqs);
  const bool first = cl.block_rank() == 0 && threadIdx.x == 0;
  if (first) w.head[0] = 0;
  if (stopped(cl, sh, p.status)) return;
  int lo, hi, total, live, before_from, before_to, moves, holes;
  page_share(p.n_pages, (int)cl.block_rank(), &lo, &hi);
  int n = 0;
  for (int q = lo + (int)threadIdx.x; q < hi; q += kPlanThreads) n += p.refs[q] > 0;
  block_scan(n, sh.sums, &total);
  if (threadIdx.x == 0) sh.mine[0] = total;
  cluster_scan(cl, &sh.mine[0], &before_from, &live);
  int from = 0, to = 0;
  for (int q = lo + (int)threadIdx.x; q < hi; q += kPlanThreads) {
    const bool used = p.refs[q] > 0;
    from += used && q >= live;
    to += !used && q < live;
  }
  cl.sync();  // mine[0] has been read by every block
  block_scan(from, sh.sums, &total);
  if (threadIdx.x == 0) sh.mine[0] = total;
  block_scan(to, sh.sums, &total);
  if (threadIdx.x == 0) sh.mine[1] = total;
  cluster_scan(cl, &sh.mine[0], &before_from, &moves);
  cluster_scan(cl, &sh.mine[1], &before_to, &holes);  // as many as moves
  for (int q0 = lo; q0 < hi; q0 += kPlanThreads) {
    const int q = q0 + (int)threadIdx.x;
    const bool in = q < hi, used = in && p.refs[q] > 0;
    const bool f = used && q >= live, t = in && !used && q < live;
    const int rf = before_from + block_scan(f, sh.sums, &total);
    before_from += total;
    const int rt = before_to + block_scan(t, sh.sums, &total);
    before_to += total;
    if (f) w.src[rf] = q;
    if (t) w.dst[rt] = q;
  }
  cl.sync();
  if (first) {
    w.head[0] = moves;
    w.head[1] = live;
  }
  for (int r = (int)(cl.block_rank() * kPlanThreads + threadIdx.x); r < moves; r += kPlanCtas * kPlanThreads) {
    const int a = __ldcg(&w.src[r]), b = __ldcg(&w.dst[r]);
    w.map[a] = b;
    w.used[r] = p.page;
    p.refs[b] = p.refs[a];
    p.refs[a] = 0;
  }
}

// ---- copying pages ---------------------------------------------------------------

// Copies the listed pages' first used[r] tokens, of every layer and head, K
// and V.  A block takes one page of one layer, a warp one head of its K or V,
// whose tokens are contiguous: eight 16-byte loads a lane before their stores
// (4 KB a warp in flight).  With `remap` the table's entries follow the moved
// pages.
__global__ void __launch_bounds__(256) copy_pages_kernel(const PageArgs p, int remap) {
  const PageWs w = page_ws(p.ws, p.n_pages, p.n_seqs);
  const int n = w.head[0];
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int per = p.page / p.block;
  const int64_t all = (int64_t)n * p.n_layers;
  for (int64_t at = blockIdx.x; at < all; at += gridDim.x) {
    const int64_t r = at / p.n_layers, l = at - r * p.n_layers;
    const int used = w.used[r], words = used * (p.head_dim / 16), nb = (used + p.block - 1) / p.block;
    const int64_t a0 = (l * p.n_pages + w.src[r]) * p.kv, b0 = (l * p.n_pages + w.dst[r]) * p.kv;
    for (int u = warp; u < 2 * p.kv; u += 8) {
      const bool z = u >= p.kv;
      const int64_t a = a0 + (z ? u - p.kv : u), b = b0 + (z ? u - p.kv : u);
      int8_t *c = z ? p.v : p.k;
      const uint4 *from = (const uint4 *)(c + a * p.page * p.head_dim);
      uint4 *to = (uint4 *)(c + b * p.page * p.head_dim);
      for (int x0 = lane; x0 < words; x0 += 256) {
        uint4 q[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (x0 + 32 * i < words) q[i] = __ldcs(from + x0 + 32 * i);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (x0 + 32 * i < words) __stcs(to + x0 + 32 * i, q[i]);
      }
      float *s = z ? p.vs : p.ks;
      for (int x = lane; x < nb; x += 32) s[b * per + x] = s[a * per + x];
    }
  }
  if (remap && n > 0) {
    const int live = w.head[1];
    const int64_t entries = (int64_t)p.n_seqs * p.max_pages, threads = (int64_t)gridDim.x * blockDim.x;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += threads) {
      const int pid = p.table[e];
      if (pid >= live && pid < p.n_pages) p.table[e] = w.map[pid];
    }
  }
}

// ---- release, slide ----------------------------------------------------------------

// One block per sequence.  An entry is taken by an exchange, so a sequence
// that is named twice gives its pages back once.
__global__ void __launch_bounds__(128) release_kernel(const PageArgs p, const int32_t *seqs) {
  const int s = seqs ? seqs[blockIdx.x] : (int)blockIdx.x;
  if ((unsigned)s >= (unsigned)p.n_seqs) {
    if (threadIdx.x == 0) atomicOr(p.status, kBadSeq);
    return;
  }
  int32_t *row = p.table + (int64_t)s * p.max_pages;
  const int np = min(pages_for(max(p.length[s], 0), p.page), p.max_pages);
  for (int j = (int)threadIdx.x; j < np; j += 128) {
    const int old = atomicExch(&row[j], -1);
    if ((unsigned)old < (unsigned)p.n_pages) atomicSub(&p.refs[old], 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) p.length[s] = 0;
}

// Gives back the pages that lie wholly behind the first `sinks` tokens and
// wholly before the window of every query at or after the last token.
__global__ void __launch_bounds__(128) slide_kernel(const PageArgs p, const int32_t *seqs, int window, int sinks) {
  const int s = seqs ? seqs[blockIdx.x] : (int)blockIdx.x;
  if ((unsigned)s >= (unsigned)p.n_seqs) {
    if (threadIdx.x == 0) atomicOr(p.status, kBadSeq);
    return;
  }
  int32_t *row = p.table + (int64_t)s * p.max_pages;
  const int end = min(max(p.length[s] - window, 0) / p.page, p.max_pages);
  for (int j = (int)(((int64_t)sinks + p.page - 1) / p.page) + (int)threadIdx.x; j < end; j += 128) {
    const int old = atomicExch(&row[j], -1);
    if ((unsigned)old < (unsigned)p.n_pages) atomicSub(&p.refs[old], 1);
  }
}

// ---- launches ----------------------------------------------------------------------

// Shared memory of a plan: one bit for each sequence.
static size_t named_bytes(const PageArgs &a) { return (size_t)ceil_div(a.n_seqs, 32) * 4; }

int reserve(const PageArgs &a, const int32_t *seqs, const int32_t *counts, int m, cudaStream_t st) {
  static std::atomic<size_t> limit[64];
  const int rc = raise_smem_limit((const void *)reserve_kernel, named_bytes(a), limit);
  if (rc) return rc;
  reserve_kernel<<<kPlanCtas, kPlanThreads, named_bytes(a), st>>>(a, seqs, counts, m);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

static int copy_pages(const PageArgs &a, int remap, int sm_count, cudaStream_t st) {
  copy_pages_kernel<<<sm_count * 4, 256, 0, st>>>(a, remap);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

int fork(const PageArgs &a, const int32_t *parents, const int32_t *children, int m, int sm_count, cudaStream_t st) {
  static std::atomic<size_t> limit[64];
  const int rc = raise_smem_limit((const void *)fork_kernel, named_bytes(a), limit);
  if (rc) return rc;
  fork_kernel<<<kPlanCtas, kPlanThreads, named_bytes(a), st>>>(a, parents, children, m);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return copy_pages(a, 0, sm_count, st);
}

int compact(const PageArgs &a, int sm_count, cudaStream_t st) {
  compact_kernel<<<kPlanCtas, kPlanThreads, 0, st>>>(a);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return copy_pages(a, 1, sm_count, st);
}

int release(const PageArgs &a, const int32_t *seqs, int m, cudaStream_t st) {
  release_kernel<<<m, 128, 0, st>>>(a, seqs);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

int slide(const PageArgs &a, const int32_t *seqs, int m, int window, int sinks, cudaStream_t st) {
  slide_kernel<<<m, 128, 0, st>>>(a, seqs, window, sinks);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

}  // namespace kv8
}  // namespace sc
