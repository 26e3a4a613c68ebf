// Log probabilities of given tokens, entropy and top alternatives of rows of logits, in one read.
//
// (The reference samples greedily from the logits, LK/kernels.metal:310-345, and never forms
// probabilities; this is the scoring half next to argmax.)  With m the row's maximum:
//   s = sum_i e^(x_i - m),  u = sum_i (x_i - m) e^(x_i - m)
//   logprob(t) = x_t - m - ln s,   entropy = ln s - u / s
// both online: when a thread's maximum grows from m to m', s <- s e^(m-m'), and u likewise with
// (m - m') s added to it.  Work is done in units of log2 (z = x * L - M with L = fp32(log2 e) and
// M an fp32 number near max * L); the result is exact in M, and the relative error of L (1e-8)
// is a relative error of the results.  z of the maximum itself is what rounding max * L left over,
// up to half a step of M, so this form serves |max| < 2^24 only, where that is below 1; other rows
// are summed again as x - max (2^z of a rounding error beyond 128 is infinite: |max| >= 1.5e9).
//
// Top k without a second pass over the row: every thread remembers its own largest value and the
// vector it came from (one compare per vector of the main loop).  The k-th largest of the maxima
// of 64 groups of threads bounds the k-th largest element from below, so all of the top k lie in
// the few threads (about 64 ln(64 / (64 - k)) of them) whose maximum reaches the bound: only their
// vectors are read again, from L2, and the elements that reach the bound are ranked exactly.
// Keys are (value, index) pairs in one 64-bit number that are never equal, so ties go to the
// lowest index, and equal values everywhere (an untrained model, a row of -inf) do not swamp the
// candidates.  (Sorting all thread maxima for the tightest bound cost more than it saved: 9 us of
// a CTA's time were spent after the main loop.)
//
// What bounds it: memory (one read of the logits).
#include <cooperative_groups.h>

#include "common.cuh"

namespace b2d {

namespace lp {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxK = 32;
constexpr int kBatch = 2;  // vectors in flight per thread (four CTAs per SM)
constexpr int kGroup = kThreads / 64;  // threads per group of the bound
constexpr int kCand = 1024;  // candidates ranked at once; more of them take the slow way
constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.693147180559945309417;
// Values below -2^24 count as -2^24 in the sums: a thread that has seen nothing above it (tokens
// banned with any constant) then has a reference without a rounding error, and 0 * inf stays out of
// u.  Their weight is zero either way in a row whose maximum is kReach or more above the floor;
// lower rows are summed again.  A power of two, so that kFloor * kLog2e is exact and a vector of
// nothing else has z = 0.
constexpr float kFloor = -16777216.f;
constexpr float kReach = 256.f;  // e^-256 is nothing in fp32

struct Params {
  const void* x;
  long long ld;
  int V, rows;
  const int* n_rows;
  const int* targets;
  int n_targets;
  int k;
  float* logprobs;
  float* entropy;
  int* top_ids;
  float* top_lp;
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Larger key = larger value, then lower index.  NaN sorts below -inf; -0 equals +0.
__device__ __forceinline__ unsigned long long key_of(float v, unsigned idx) {
  v += 0.0f;
  uint32_t b = __float_as_uint(v);
  b = v != v ? 1u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
  return ((unsigned long long)b << 32) | (uint32_t)~idx;
}

__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return b == 1u ? __uint_as_float(0x7fffffffu) : __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

template <bool F16>
struct Row {  // one row of logits in 16-byte vectors; vector 0 may start before the row
  static constexpr int VEC = F16 ? 8 : 4;
  const void* x;
  int V, shift, nv;  // shift: elements of vector 0 that lie before the row
  __device__ Row(const Params& p, int row) {
    constexpr int E = F16 ? 2 : 4;
    const char* r = static_cast<const char*>(p.x) + (long long)row * p.ld * E;
    shift = (int)((reinterpret_cast<uintptr_t>(r) & 15) / E);
    x = r;
    V = p.V;
    nv = (V + shift + VEC - 1) / VEC;
  }
  __device__ float at(int i) const {
    if constexpr (F16) return h2f(static_cast<const uint16_t*>(x)[i]);
    else return static_cast<const float*>(x)[i];
  }
  // whole vectors are [full0, full1); at most one before and one behind them is partly outside
  __device__ int full0() const { return shift > 0; }
  __device__ int full1() const { return (V + shift) / VEC; }
  __device__ int first(int v) const { return v * VEC - shift; }  // element of vector v's start
  __device__ uint4 raw(int v) const {                            // a whole vector
    uint4 u;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
        : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
        : "l"(static_cast<const char*>(x) + (long long)first(v) * (F16 ? 2 : 4)));
    return u;
  }
  __device__ static void unpack(uint4 u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (F16) {
        const float2 t = h2f2(w[e]);
        f[2 * e] = t.x;
        f[2 * e + 1] = t.y;
      } else {
        f[e] = __uint_as_float(w[e]);
      }
    }
  }
  // any vector; elements outside the row are not read and come back as -inf
  __device__ void vec(int v, float* f) const {
    if (v >= full0() && v < full1()) {
      unpack(raw(v), f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = first(v) + e;
        f[e] = (i >= 0 && i < V) ? at(i) : -INFINITY;
      }
    }
  }
};

// Running statistics of a set of elements: M (log2 units), s, u as above.
struct Stat {
  float M, s, u;
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float M = fmaxf(a.M, b.M);
  // an empty set has M = -inf, s = u = 0
  const float da = a.M == -INFINITY ? 0.f : a.M - M, db = b.M == -INFINITY ? 0.f : b.M - M;
  const float ea = ex2(da), eb = ex2(db);
  // (z shifted by d) * e^..: u moves by d * s
  return Stat{M, a.s * ea + b.s * eb, (a.u + da * a.s) * ea + (b.u + db * b.s) * eb};
}
__device__ __forceinline__ Stat warp_join(Stat a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.M = __shfl_xor_sync(0xffffffffu, a.M, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
    a = join(a, b);
  }
  return a;
}

// How many of the warp's keys (the lane's: `other`, number `j`) come before `key`, number `c`.
__device__ __forceinline__ int rank_of(unsigned long long key, int c, unsigned long long other, int j) {
  return __popc(__ballot_sync(0xffffffffu, other > key || (other == key && j < c)));
}

// This CTA runs / every CTA of the cluster runs (their shared memory may be written).
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Largest value of the CTA's threads, NaN if any is.
__device__ __forceinline__ float block_max_nan(float v, float* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v = max_nan(v, sm[w]);
  return v;
}

template <bool F16>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const Params p) {
  constexpr int VEC = Row<F16>::VEC;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int row = blockIdx.x / ranks;
  if (p.n_rows && row >= *p.n_rows) return;  // the whole cluster: outputs left as they are
  __shared__ Stat w_stat[kWarps];
  __shared__ unsigned long long g_tau, g_keys[64];  // largest key of each group of threads
  __shared__ unsigned long long cand[kCand];
  __shared__ unsigned short owners[kThreads];
  __shared__ float w_f[kWarps];
  __shared__ int n_owners, n_cand;
  __shared__ unsigned long long best;
  // rank 0's copies of every rank's results
  __shared__ Stat r_stat[8];
  __shared__ unsigned long long r_keys[8 * kMaxK];  // k per rank
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive();
  const Row<F16> r(p, row);
  const int stride = ranks * kThreads, v0 = rank * kThreads + tid;

  // ---- one pass: statistics, and this thread's largest element and where it is
  Stat st = {-INFINITY, 0.f, 0.f};
  float mx = -INFINITY;
  int mv = -1;
  auto take = [&](int v, const float* f) {
    float vm = f[0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) vm = fmaxf(vm, f[e]);
    if (vm > mx || mv < 0) {
      mx = vm;
      mv = v;
    }
    const float M = fmaxf(st.M, fmaxf(vm, kFloor) * kLog2e);
    const float d = st.M == -INFINITY ? 0.f : st.M - M;
    const float c = ex2(d);
    st.u = fmaf(d, st.s, st.u) * c;
    st.s *= c;
    st.M = M;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float z = fmaf(max_nan(f[e], kFloor), kLog2e, -M);
      const float w = ex2(z);
      st.s += w;
      st.u = fmaf(z, w, st.u);
    }
  };
  const int f0 = r.full0(), f1 = r.full1();
  for (int v = v0; v < r.nv; v += kBatch * stride) {
    uint4 raw[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int vj = v + j * stride;
      if (vj >= f0 && vj < f1) raw[j] = r.raw(vj);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int vj = v + j * stride;
      if (vj >= r.nv) break;
      float f[VEC];
      if (vj >= f0 && vj < f1) r.unpack(raw[j], f);
      else r.vec(vj, f);
      take(vj, f);
    }
  }
  const Stat own = warp_join(st);
  if (lane == 0) w_stat[warp] = own;

  // ---- this CTA's top k
  if (p.k > 0) {
    // (value, last index of its vector): not above the key of the element it stands for
    const unsigned long long mine =
        mv < 0 ? 0ull : key_of(mx, (unsigned)(r.first(mv) + VEC - 1));
    unsigned long long gk = mine;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) {
      const unsigned long long w = __shfl_xor_sync(0xffffffffu, gk, o);
      gk = gk > w ? gk : w;
    }
    if (tid % kGroup == 0) g_keys[tid / kGroup] = gk;
    if (tid == 0) n_owners = n_cand = 0;
    __syncthreads();
    // the k-th largest of the 64 (equal ones, all of them empty groups, in order): a key's rank is a
    // count of ballots, a few keys per warp
    const unsigned long long ga = g_keys[lane], gb = g_keys[lane + 32];
#pragma unroll
    for (int j = warp; j < 64; j += kWarps)
      if (rank_of(g_keys[j], j, ga, lane) + rank_of(g_keys[j], j, gb, lane + 32) == p.k - 1) g_tau = g_keys[j];
    __syncthreads();
    const unsigned long long tau = g_tau;
    const float tau_v = key_value(tau);
    bool odd = false;  // a NaN (or a maximum past 1.5e9): the thread maxima may say nothing
    for (int w = 0; w < kWarps; ++w) odd |= w_stat[w].s != w_stat[w].s;
    // threads that may hold an element at or above tau
    if (mv >= 0 && key_of(mx, (unsigned)max(r.first(mv), 0)) >= tau)
      owners[atomicAdd(&n_owners, 1)] = (unsigned short)tid;
    __syncthreads();
    for (int o = odd ? n_owners : warp; o < n_owners; o += kWarps) {
      for (int v = rank * kThreads + owners[o] + lane * stride; v < r.nv; v += 32 * stride) {
        float f[VEC];
        r.vec(v, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int i = r.first(v) + e;
          if (f[e] < tau_v || i < 0 || i >= r.V) continue;
          const unsigned long long key = key_of(f[e], (unsigned)i);
          if (key >= tau) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) cand[at] = key;
          }
        }
      }
    }
    __syncthreads();
    const int n = n_cand;
    cluster_wait();  // rank 0 runs
    unsigned long long* out = cluster.map_shared_rank(&r_keys[rank * p.k], 0);
    if (n <= kCand && !odd) {
      for (int c = warp; c < n; c += kWarps) {
        const unsigned long long key = cand[c];
        int above = 0;
        for (int j0 = 0; j0 < n; j0 += 32) above += rank_of(key, c, j0 + lane < n ? cand[j0 + lane] : 0ull, j0 + lane);
        if (lane == 0 && above < p.k) out[above] = key;
      }
      for (int j = n + tid; j < p.k; j += kThreads) out[j] = 0ull;
    } else {  // many elements above the bound (rare): the next largest key, k times
      unsigned long long last = ~0ull;
      for (int j = 0; j < p.k; ++j) {
        if (tid == 0) best = 0ull;
        __syncthreads();
        unsigned long long b = 0ull;
        for (int v = v0; v < r.nv; v += stride) {
          float f[VEC];
          r.vec(v, f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int i = r.first(v) + e;
            if (i < 0 || i >= r.V) continue;
            const unsigned long long key = key_of(f[e], (unsigned)i);
            if (key < last && key > b) b = key;
          }
        }
        atomicMax(&best, b);
        __syncthreads();
        last = best;
        if (tid == 0) out[j] = last;
        __syncthreads();
      }
    }
  } else {
    cluster_wait();
    __syncthreads();
  }
  // ---- join the cluster's CTAs in rank 0
  if (warp == 0) {
    Stat t = lane < kWarps ? w_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    t = warp_join(t);
    if (lane == 0) *cluster.map_shared_rank(&r_stat[rank], 0) = t;
  }
  cluster.sync();
  if (rank != 0) return;
  Stat t = r_stat[0];
  for (int j = 1; j < ranks; ++j) t = join(t, r_stat[j]);
  // Rows whose maximum is not within (-2^24 + 256, 2^24), all of them -inf included: the plain
  // two-step form x - max, over the whole row by this CTA.  (Their sums may be infinite or NaN here.)
  float base = 0.f;
  const bool far = !(t.M > (kFloor + kReach) * kLog2e && t.M < -kFloor * kLog2e);
  if (far) {
    float m = -INFINITY;
    for (int v = tid; v < r.nv; v += kThreads) {
      float f[VEC];
      r.vec(v, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = max_nan(m, f[e]);
    }
    base = block_max_nan(m, w_f);
    t = Stat{0.f, 0.f, 0.f};
    for (int v = tid; v < r.nv; v += kThreads) {
      float f[VEC];
      r.vec(v, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = max_nan((f[e] - base) * kLog2e, kFloor);
        const float w = ex2(z);
        t.s += w;
        t.u = fmaf(z, w, t.u);
      }
    }
    t = warp_join(t);
    __syncthreads();
    if (lane == 0) w_stat[warp] = t;
    __syncthreads();
    t = w_stat[0];
    for (int w = 1; w < kWarps; ++w) t = join(t, w_stat[w]);
    if (base == -INFINITY) t = Stat{0.f, 1.f, 0.f};  // nothing but -inf: no choice, entropy 0
  }
  // log2 of the row's sum, in log2 units of x * L (of (x - base) * L in a far row)
  __shared__ double row_lz;
  if (tid == 0) {
    row_lz = (double)t.M + log2((double)t.s);
    if (p.entropy) p.entropy[row] = (float)((row_lz - (double)t.M - (double)t.u / (double)t.s) * kLn2);
  }
  __syncthreads();
  const double lz = row_lz;
  auto lp_of = [&](float x) -> float {
    if (far && base == -INFINITY) return x;
    const double d = far ? (double)x - (double)base : (double)x;
    return (float)((d * (double)kLog2e - lz) * kLn2);
  };
  for (int j = tid; j < p.n_targets; j += kThreads) {
    const int id = p.targets[(long long)row * p.n_targets + j];
    p.logprobs[(long long)row * p.n_targets + j] =
        id >= 0 && id < r.V ? lp_of(r.at(id)) : (t.s == t.s ? -INFINITY : t.s);
  }
  // the top of the ranks' tops, one entry per warp at a time (one rank's are in order already)
  const int nk = ranks * p.k;
  unsigned long long mine[8];
  if (ranks > 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) mine[j] = j * 32 + lane < nk ? r_keys[j * 32 + lane] : 0ull;
  for (int c = warp; c < nk; c += kWarps) {
    const unsigned long long key = r_keys[c];
    int above = c;
    if (ranks > 1) {
      above = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j * 32 < nk) above += rank_of(key, c, mine[j], j * 32 + lane);
    }
    if (lane == 0 && above < p.k) {
      p.top_ids[(long long)row * p.k + above] = (int)~(uint32_t)(key & 0xffffffffull);
      p.top_lp[(long long)row * p.k + above] = lp_of(key_value(key));
    }
  }
}

}  // namespace lp

// CTAs (one cluster) per row: several while they fill half of the machine or less.  More, to even
// out the last wave of CTAs, cost more than they gave: each pays for its own selection (2048 rows of
// 128256 fp32 logits 216 us with two, 193 with one).
static int logprob_ranks(int rows, int V, bool f16) {
  int c = 1;
  const int vecs = (V + (f16 ? 7 : 3)) / (f16 ? 8 : 4);
  while (c < 8 && (long long)rows * c < 2 * num_sms() && vecs > c * lp::kThreads) c *= 2;
  return c;
}

int token_logprobs(const void* logits, int dtype, long long ld, int V, int rows, const int* n_rows,
                   const int* targets, int n_targets, int top_k, float* logprobs, float* entropy,
                   int* top_ids, float* top_logprobs, cudaStream_t stream) {
  if (!logits || (n_targets > 0 && (!targets || !logprobs)) || (top_k > 0 && (!top_ids || !top_logprobs)))
    return B2D_ERR_NULL;
  if (dtype != B2D_F32 && dtype != B2D_F16) return B2D_ERR_UNSUPPORTED;
  if (rows <= 0 || rows > (1 << 27) || V <= 0 || V > (1 << 30) || ld < V || n_targets < 0 || top_k < 0 ||
      top_k > lp::kMaxK || top_k > V)
    return B2D_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == B2D_F16 ? 2 : 4)) return B2D_ERR_ALIGN;
  const lp::Params p = {logits, ld,       V,       rows,    n_rows, targets,
                        n_targets, top_k, logprobs, entropy, top_ids, top_logprobs};
  const int ranks = logprob_ranks(rows, V, dtype == B2D_F16);
  auto kern = dtype == B2D_F16 ? lp::token_logprobs_kernel<true> : lp::token_logprobs_kernel<false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ranks);
  cfg.blockDim = dim3(lp::kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return B2D_ERR_CUDA;
  }
  count_launch();
  return B2D_OK;
}

}  // namespace b2d
