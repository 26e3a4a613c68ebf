// Pages, slots, positions and tree masks of one serving step, from the requests' lengths.
//
// (The reference keeps one contiguous cache for one sequence, LK/main.swift:176-182; paging is
// this library's own.)  Per request b with have_b pages, ctx_b cached and q_b new tokens:
//   need_b = max(0, ceil((ctx_b + q_b) / 16) - have_b)        pages to take from the free stack
//   off_b  = need_0 + ... + need_(b-1)
//   page j of the new ones = stack[top - 1 - off_b - j],  top = free pages + released pages
// and q_b < 0 releases the request's pages onto the stack first.  Everything after the three
// prefix sums is independent per request or per token.
//
// What bounds it: latency (a few hundred KB at most; a 32-request step reads and writes 24 KB).
// So it is ONE launch, and the prefix sums are not a pass of their own: every CTA of one cluster
// runs them over all requests (16 bytes each, from L2), keeps the results in shared memory and
// then works on its share of pages and tokens.  The cluster barrier orders the released pages'
// writes before the reads that hand them out again, and every read of the inputs before the
// first write of an output, so n_pages / n_free may be updated in place.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b2d {

namespace plan {

constexpr int kThreads = 512;
constexpr int kMaxBatch = 8192;     // shared memory: 16 bytes per request
constexpr int kMaxWords = 8;        // mask words per row: trees of up to 256 nodes
constexpr int kMaxTokens = 1 << 24;
constexpr int kMaxBlocks = 1 << 17;  // 8192 requests * 2^17 pages stay below 2^31

struct Params {
  const int* ctx_lens;
  const int* q_lens;
  const int* parents;
  int* table;
  int max_blocks;
  const int* n_pages;
  int* stack;
  int stack_cap;
  const int* n_free;
  int batch, max_tokens, words;
  int* cu_q;
  long long* slots;
  int* positions;
  uint32_t* mask;
  int* status;
  int* n_pages_out;
  int* n_free_out;
};

// Inclusive prefix sum over the CTA's threads of two 64-bit values; totals to tot[2].
__device__ __forceinline__ void scan2(unsigned long long& a, unsigned long long& b,
                                      unsigned long long* sm, unsigned long long* tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = kThreads / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, a, o);
    const unsigned long long y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    sm[2 * warp] = a;
    sm[2 * warp + 1] = b;
  }
  __syncthreads();
  unsigned long long pa = 0, pb = 0, ta = 0, tb = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const unsigned long long x = sm[2 * w], y = sm[2 * w + 1];
    if (w < warp) {
      pa += x;
      pb += y;
    }
    ta += x;
    tb += y;
  }
  a += pa;
  b += pb;
  tot[0] = ta;
  tot[1] = tb;
  __syncthreads();  // sm is written again by the next call
}

// Ancestor masks and positions of one request's tree, by one warp: 32 nodes at a time, each node
// following its parent pointer, doubling the path among the 32 and taking the finished result of
// an earlier group from the output.  A parent that is not an earlier node counts as the root (-1).
__device__ void tree_rows(const Params& p, int row0, int n, int ctx) {
  const int lane = threadIdx.x & 31;
  for (int c0 = 0; c0 < n; c0 += 32) {
    const int i = c0 + lane;
    uint32_t m[kMaxWords];
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) m[w] = (i < n && (i >> 5) == w) ? 1u << lane : 0u;
    int par = i < n ? p.parents[row0 + i] : -1;
    if (par >= i) par = -1;
    int depth = 0;
    // a path of up to 32 nodes of this group ends after 5 doublings; one more round takes the
    // ancestor of an earlier group
    for (int it = 0; it < 7 && __any_sync(0xffffffffu, par >= 0); ++it) {
      if (par >= 0 && par < c0) {
#pragma unroll
        for (int w = 0; w < kMaxWords; ++w)
          if (w < p.words) m[w] |= p.mask[(size_t)(row0 + par) * p.words + w];
        depth += p.positions[row0 + par] - ctx + 1;
        par = -1;
      }
      const int src = par >= 0 ? par - c0 : lane;
      const int d2 = __shfl_sync(0xffffffffu, depth, src);
      const int p2 = __shfl_sync(0xffffffffu, par, src);
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w)
        if (w < p.words) {
          const uint32_t m2 = __shfl_sync(0xffffffffu, m[w], src);
          if (par >= 0) m[w] |= m2;
        }
      if (par >= 0) {
        depth += d2 + 1;
        par = p2;
      }
    }
    if (i < n) {
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w)
        if (w < p.words) p.mask[(size_t)(row0 + i) * p.words + w] = m[w];
      p.positions[row0 + i] = ctx + depth;
    }
    __syncwarp();  // the next group reads this one's rows
  }
}

// Per request, in shared memory: first row, cached tokens, owned pages, and the offset of its new
// pages in the stack's order (kRefused where it gets none and its slots are -1).
struct Req {
  int row, ctx, have, off;
};
constexpr int kRefused = -1;

template <bool TREE>
__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t sm_raw[];
  Req* req = reinterpret_cast<Req*>(sm_raw);  // [batch], then row of the end
  __shared__ unsigned long long sm_scan[2 * (kThreads / 32)];
  __shared__ int sm_given;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31;
  const int gwarp = rank * (kThreads / 32) + (tid >> 5), nwarps = ranks * (kThreads / 32);
  const int n_free = min(max(*p.n_free, 0), p.stack_cap);
  if (tid == 0) sm_given = 0;

  // ---- prefix sums over the requests: rows; pages needed and released
  unsigned long long rows = 0, pages = 0;  // pages: needed in the low 32 bits, released above
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int ctx = 0, q = 0, have = 0;
    if (b < p.batch) {
      ctx = p.ctx_lens[b];
      q = p.q_lens[b];
      have = min(max(p.n_pages[b], 0), p.max_blocks);
    }
    unsigned long long add = q > 0 ? q : 0, none = 0, tot[2];
    const unsigned long long mine = add;
    scan2(add, none, sm_scan, tot);
    const unsigned long long end = rows + add;
    rows += tot[0];
    int why = B2D_PLAN_OK;
    const long long blocks = ((long long)ctx + (long long)mine + 15) / 16;
    if (q >= 0) {
      if (end > (unsigned long long)p.max_tokens) why = B2D_PLAN_ROWS;
      else if (ctx < 0 || blocks > p.max_blocks) why = B2D_PLAN_TABLE;
      else if (TREE && q > 32 * p.words) why = B2D_PLAN_TREE;
    }
    const unsigned need = (q >= 0 && why == B2D_PLAN_OK && blocks > have) ? (unsigned)(blocks - have) : 0;
    const unsigned back = q < 0 ? have : 0;
    unsigned long long pg = ((unsigned long long)back << 32) | need;
    none = 0;
    scan2(pg, none, sm_scan, tot);
    if (b < p.batch) {
      const unsigned long long at = pages + pg;  // inclusive
      Req r;
      r.row = (int)min(end - mine, (unsigned long long)p.max_tokens);
      r.ctx = ctx;
      // an ended request's released pages start at off; its have is negative
      r.have = q < 0 ? -1 - have : have;
      r.off = q < 0 ? (int)((unsigned)(at >> 32) - back)
                    : (why == B2D_PLAN_OK ? (int)((unsigned)at - need) : -1 - why);
      req[b] = r;
    }
    pages += tot[0];
  }
  const int total = (int)min(rows, (unsigned long long)p.max_tokens);
  if (tid == 0) req[p.batch].row = total;
  __syncthreads();
  const long long back_all = (long long)(pages >> 32);
  const int top = (int)min((long long)n_free + back_all, (long long)p.stack_cap);

  // ---- released pages onto the stack: a warp of every CTA per ended request, so that a long
  // request's pages are moved by all of them (40 requests of 1024 pages: 30 us with one warp each)
  for (int b = tid >> 5; b < p.batch; b += kThreads / 32) {
    const Req r = req[b];
    if (r.have >= 0) continue;
    const int n = -1 - r.have;
#pragma unroll 4
    for (int j = rank * 32 + lane; j < n; j += ranks * 32) {
      const long long at = (long long)n_free + r.off + j;
      if (at < p.stack_cap) p.stack[at] = p.table[(size_t)b * p.max_blocks + j];
    }
  }
  cluster.sync();  // inputs read everywhere; released pages visible to the whole cluster

  // ---- per request: grant, new table entries, outputs
  for (int b = tid; b < p.batch; b += kThreads) {
    Req r = req[b];
    int st = B2D_PLAN_OK, own = 0;
    if (r.have >= 0) {
      own = r.have;
      if (r.off < 0) {
        st = -1 - r.off;
        r.off = kRefused;
      } else {
        const int n = req[b + 1].row - r.row;
        const int need = max((r.ctx + n + 15) / 16 - r.have, 0);
        if (need > 0 && (long long)r.off + need > top) {
          st = B2D_PLAN_PAGES;
          r.off = kRefused;
        } else {
          own += need;
          if (need) atomicAdd(&sm_given, need);
        }
      }
      req[b].off = r.off;
    }
    if (rank == 0) {
      p.cu_q[b] = r.row;
      p.status[b] = st;
      p.n_pages_out[b] = own;
    }
  }
  __syncthreads();
  if (rank == 0 && tid == 0) {
    p.cu_q[p.batch] = total;
    *p.n_free_out = top - sm_given;
  }
  for (int b = tid >> 5; b < p.batch; b += kThreads / 32) {
    const Req r = req[b];
    if (r.have < 0) continue;
    if (r.off == kRefused) {
      // entries that an earlier owner of the row left behind are not this request's: its rows would
      // attend to them
      if (r.ctx < 0) continue;
      const long long blocks = ((long long)r.ctx + (req[b + 1].row - r.row) + 15) / 16;
      const int end = (int)min(blocks, (long long)p.max_blocks);
      for (int j = r.have + rank * 32 + lane; j < end; j += ranks * 32) p.table[(size_t)b * p.max_blocks + j] = -1;
      continue;
    }
    const int need = (r.ctx + req[b + 1].row - r.row + 15) / 16 - r.have;
#pragma unroll 4
    for (int j = rank * 32 + lane; j < need; j += ranks * 32)
      p.table[(size_t)b * p.max_blocks + r.have + j] = __ldcg(p.stack + top - 1 - r.off - j);
  }

  // ---- per token: slot and position
  for (int t = rank * kThreads + tid; t < total; t += ranks * kThreads) {
    int lo = 0, hi = p.batch;  // the last request whose first row is <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (req[mid].row <= t) lo = mid;
      else hi = mid;
    }
    const Req r = req[lo];
    const int at = (int)((unsigned)r.ctx + (unsigned)(t - r.row));
    long long slot = -1;
    if (r.off != kRefused) {
      const int pg = at >> 4;
      const int id = pg < r.have ? p.table[(size_t)lo * p.max_blocks + pg]
                                 : __ldcg(p.stack + top - 1 - r.off - (pg - r.have));
      if (id >= 0) slot = (long long)id * 16 + (at & 15);
    }
    p.slots[t] = slot;
    if (!TREE) p.positions[t] = at;
  }
  if constexpr (TREE) {
    for (int b = gwarp; b < p.batch; b += nwarps) {
      const Req r = req[b];
      const int n = req[b + 1].row - r.row;
      if (n <= 32 * p.words) {
        tree_rows(p, r.row, n, r.ctx);
      } else {  // refused: the rows exist, without ancestors
        for (int i = lane; i < n; i += 32) {
          p.positions[r.row + i] = r.ctx + i;
          for (int w = 0; w < p.words; ++w) p.mask[(size_t)(r.row + i) * p.words + w] = 0u;
        }
      }
    }
  }
}

}  // namespace plan

int paged_plan(const int* ctx_lens, const int* q_lens, const int* parents, int* block_table,
               int max_blocks, const int* n_pages, int* free_pages, int free_capacity,
               const int* n_free, int batch, int max_tokens, int mask_words, int* cu_q,
               long long* slots, int* positions, uint32_t* mask, int* status, int* n_pages_out,
               int* n_free_out, cudaStream_t stream) {
  if (!ctx_lens || !q_lens || !block_table || !n_pages || !free_pages || !n_free || !cu_q ||
      !slots || !positions || !status || !n_pages_out || !n_free_out)
    return B2D_ERR_NULL;
  if (parents && !mask) return B2D_ERR_NULL;
  if (batch <= 0 || batch > plan::kMaxBatch || max_tokens <= 0 || max_tokens > plan::kMaxTokens ||
      max_blocks <= 0 || max_blocks > plan::kMaxBlocks || free_capacity <= 0)
    return B2D_ERR_SHAPE;
  if (parents ? (mask_words <= 0 || mask_words > plan::kMaxWords) : mask_words != 0)
    return B2D_ERR_SHAPE;
  const plan::Params p = {ctx_lens, q_lens,    parents,       block_table, max_blocks,  n_pages,
                          free_pages, free_capacity, n_free,  batch,       max_tokens,  mask_words,
                          cu_q,     slots,     positions,     mask,        status,      n_pages_out,
                          n_free_out};
  const size_t smem = (size_t)(batch + 1) * sizeof(plan::Req);
  auto kern = parents ? plan::paged_plan_kernel<true> : plan::paged_plan_kernel<false>;
  static std::atomic<unsigned long long> done[2];
  B2D_TRY(allow_smem(kern, (plan::kMaxBatch + 1) * (int)sizeof(plan::Req), done[parents != nullptr]));
  cudaError_t e;
  {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(8);
    cfg.blockDim = dim3(plan::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 8;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, p);
  }
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return B2D_ERR_CUDA;
  }
  count_launch();
  return B2D_OK;
}

}  // namespace b2d
