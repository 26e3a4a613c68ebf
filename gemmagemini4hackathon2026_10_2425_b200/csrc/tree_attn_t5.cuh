// Tree attention on the 5th-generation tensor cores: the kernel of tree_attn.cu's entry point for
// head_dim 64 and 128 (that file holds the formulas and the one for head_dim 256).
//
// A unit of work is one M tile of query rows (row m = t * G + g) of one KV head of one sequence,
// a step of it 128 keys (256 in the key-split form below).  All units' steps form one line, cut
// into equal parts for one persistent CTA per SM: a ragged batch is balanced to a step, a long
// sequence is split over many CTAs and short ones share one, whatever the lengths are (the host
// knows their bounds only).  A CTA's part holds whole units and at most two incomplete ones,
// whose states (max, sum, unnormalized output) go to the workspace, 2 places per CTA; a second
// kernel joins them.
//
// Inside a CTA two warpgroups run the softmax of one 128 x 128 score tile each while the tensor
// cores work for the other: S = Q K^T (operands in shared memory, K from TMA page loads) lands in
// TMEM, a thread owns one row of it (no shuffles), writes P as fp16 over its S, and O += P V reads
// P from TMEM and V as it lies in the page (a transposed B operand).  Two forms:
//   MT2: the warpgroups hold different row tiles (256 rows a unit) and share each K/V tile;
//   key split: they hold the same 128 rows and take alternate key tiles; their two states meet
//   through TMEM at the end of the unit.
// Roles: warps 0-7 softmax (warp w reads TMEM lanes 32 (w % 4) ..), warp 8 TMA, warps 9 and 10
// issue the MMAs of one warpgroup each.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time (its
// weights are then up to 256 and still exact to 2^-11 in fp16), which after the first tiles of a
// unit is almost never; the sum and the weights always use the same reference, so nothing is lost.
//
// Included by tree_attn.cu, whose Params, Span and row helpers it uses.
#pragma once

namespace b2d {
namespace tree {

namespace t5 {

constexpr int kKeys = 128;
constexpr int kSoftmax = 256;               // threads of the two warpgroups
constexpr int kThreads = kSoftmax + 128;    // + TMA warp, two MMA warps, one idle
// Registers: a softmax thread holds a row of 128 scores.  384 threads launch with 168 each
// (64512); the split 256 * 216 + 128 * 72 uses the same number.
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
constexpr int kMaxBatch = 1024;             // prefix sums in shared memory
constexpr float kSlack = 8.f;               // log2 of the growth that O is rescaled for

template <int HD, bool MT2, bool X2>
struct Cfg {
  static constexpr int BOXES = HD / 64;
  static constexpr int TILE = kKeys * HD * 2;
  static constexpr int ROWS = MT2 ? 256 : 128;     // rows of a unit
  static constexpr int PLANES = MT2 || X2 ? 2 : 1;  // 128-row fp16 planes of Q
  static constexpr int SK = HD == 64 ? 4 : (PLANES == 2 ? 2 : 3);
  static constexpr int SV = HD == 64 ? 4 : 2;
  static constexpr int OFF_K = PLANES * TILE;  // a Q plane is as large as a tile
  static constexpr int OFF_V = OFF_K + SK * TILE;
  static constexpr int OFF_MISC = OFF_V + SV * TILE;
};

struct Misc {
  float2 ml[2][128];            // key split: the warpgroups' (reference, sum) per row
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2], pv_done[2], q_full[2];
  unsigned bad[2][4];           // non-finite V rows of the tile at hand
  unsigned miss[4];             // pages of a V stage's tile that do not exist
  uint32_t tmem;
  int failed;
  int prefix[kMaxBatch + 1];    // first step of each sequence
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// 128-byte swizzled operands.  K-major (Q, K): 8-row groups 1024 bytes apart.  MN-major (V, whose
// rows are the reduction): 8-row groups 1024 bytes apart, 64-column blocks `block` bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t block) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(block >> 4) << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
// kind::f16, D fp32, A and B fp16, M = 128; bit 16: B is MN-major.
constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id) {  // accumulates
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id));
}

// The part of one unit that a CTA works on.
struct Piece {
  Span s;
  int b, kvh, m0;
  int t0, nt;      // first key tile of the piece (of the unit's), number of them
  bool whole;      // the whole unit
  int slot;        // place in the workspace, if not
};

// Steps of one unit of sequence b, row tile mt.
template <int ROWS, int PER>
__device__ __forceinline__ int unit_steps(const Params& p, int b, int mt, int G, Span& s) {
  if (!span_of(p, b, mt * ROWS, mt * ROWS + ROWS, G, kKeys, s)) return 0;
  return max(1, (s.hi - s.lo + kKeys * PER - 1) / (kKeys * PER));
}

// Prefix sums of the sequences' steps into prefix[0 .. batch]; all threads of the CTA.
template <int ROWS, int PER>
__device__ void steps_prefix(const Params& p, int G, int* prefix, int threads) {
  __shared__ int carry, wsum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int b0 = 0; b0 < p.batch; b0 += threads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.batch) {
      Span s;
      for (int mt = 0; mt < p.m_tiles; ++mt) {
        const int u = unit_steps<ROWS, PER>(p, b, mt, G, s);
        if (u == 0) break;
        n += u;
      }
      n *= p.n_kv;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < warp; ++w) base += wsum[w];
    if (b < p.batch) prefix[b + 1] = base + x;
    __syncthreads();
    if (tid == threads - 1) carry = base + x;
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
}

// CTA cta's part of the line of W steps.
__device__ __forceinline__ int part_begin(int W, int cta, int ctas) { return (int)((long long)W * cta / ctas); }

// Walks the pieces of steps [x, end) of the line.
template <int ROWS, int PER>
struct Walk {
  int x, end, b;
  bool first;
  __device__ bool next(const Params& p, const int* prefix, int G, int cta, Piece& pc) {
    if (x >= end) return false;
    if (first) {  // the sequence that holds step x
      int lo = 0, hi = p.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= x) lo = mid;
        else hi = mid;
      }
      b = lo;
    }
    while (prefix[b + 1] <= x) ++b;
    int at = x - prefix[b], mt = 0, n;
    for (;; ++mt) {
      n = unit_steps<ROWS, PER>(p, b, mt, G, pc.s);
      if (at < n * p.n_kv) break;
      at -= n * p.n_kv;
    }
    pc.b = b;
    pc.m0 = mt * ROWS;
    pc.kvh = at / n;
    const int s0 = at % n, s1 = min(n, s0 + (end - x));
    const int tiles = (pc.s.hi - pc.s.lo + kKeys - 1) / kKeys;
    pc.t0 = s0 * PER;
    pc.nt = max(0, min(s1 * PER, tiles) - pc.t0);
    pc.whole = s0 == 0 && s1 == n;
    pc.slot = 2 * cta + (first ? 0 : 1);
    x += s1 - s0;
    first = false;
    return true;
  }
};

// q . k of a row's head and the key at place j, in fp32, from global memory.
template <int HD>
__device__ __forceinline__ float dot_place(const Params& p, const Span& s, int b, int kvh, int t, int head, int j) {
  const int id = p.block_table[(long long)b * p.max_blocks + j / 16];
  const uint16_t* k = p.k_pages + (((long long)id * p.n_kv + kvh) * 16 + j % 16) * HD;
  return dot_row<HD>(p, s.row0 + t, head, [&](int d) { return h2f(k[d]); });
}

// O += w v_j for the warp's rows, v_j from global memory; w = 0 adds nothing.
template <int HD>
__device__ __forceinline__ void add_place(const Params& p, int b, int kvh, int j, float w, uint32_t o_col) {
  const int id = p.block_table[(long long)b * p.max_blocks + j / 16];
  const uint16_t* v = p.v_pages + (((long long)id * p.n_kv + kvh) * 16 + j % 16) * HD;
#pragma unroll 1
  for (int c = 0; c < HD; c += 32) {
    uint32_t o[32];
    tmem_ld32(o_col + c, o);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (w != 0.f) o[e] = __float_as_uint(fmaf(w, h2f(v[c + e]), __uint_as_float(o[e])));
    tmem_st32(o_col + c, o);
  }
  tmem_wait_st();
}

// Bits of the places k0 .. k0 + 31 that row t (of the sequence's own rows, at position pos) sees,
// but for pages that do not exist.
__device__ __forceinline__ unsigned range_bits(int k0, int lo, int hi) {  // places [lo, hi)
  const int a = max(lo - k0, 0), b = min(hi - k0, 32);
  if (a >= b) return 0u;
  return (b == 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u);
}
__device__ unsigned see_bits(const Params& p, const Span& s, int t, int pos, int k0) {
  const int low = p.window > 0 ? pos - p.window + 1 : 0;
  unsigned v = range_bits(k0, low, s.ctx);
  if (!p.mask) return v | range_bits(k0, max(s.ctx, low), s.ctx + t + 1);
  if (k0 + 32 <= s.ctx) return v;
  const uint32_t* w = p.mask + (long long)(s.row0 + t) * p.words;
  const int o = k0 - s.ctx;  // own row of the first place (may be negative)
  const int wi = o >> 5, sh = o & 31;
  const unsigned a = wi >= 0 && wi < p.words ? w[wi] : 0u, c = wi + 1 >= 0 && wi + 1 < p.words ? w[wi + 1] : 0u;
  unsigned own = sh ? (a >> sh) | (c << (32 - sh)) : a;
  own &= range_bits(k0, s.ctx, s.hi);
  if (p.window > 0)
    for (unsigned m = own; m; m &= m - 1) {
      const int k = __ffs(m) - 1;
      if (row_position(p, s, k0 + k - s.ctx) < low) own &= ~(1u << k);
    }
  return v | own;
}

template <int HD, bool MT2, bool X2>
__global__ void __launch_bounds__(kThreads, 1) tree_attn_t5_kernel(const __grid_constant__ Params p) {
  using C = Cfg<HD, MT2, X2>;
  constexpr int PER = MT2 ? 1 : 2;  // key tiles per step
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
  Misc& mi = *reinterpret_cast<Misc*>(sm + C::OFF_MISC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.n_heads / p.n_kv;

  if (tid == 0) {
    for (int i = 0; i < C::SK; ++i) {
      mbar_init(&mi.k_full[i], 1);
      mbar_init(&mi.k_empty[i], MT2 ? 2 : 1);
    }
    for (int i = 0; i < C::SV; ++i) {
      mbar_init(&mi.v_full[i], 1);
      mbar_init(&mi.v_empty[i], MT2 ? 2 : 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&mi.s_full[g], 1);
      mbar_init(&mi.p_full[g], 128);
      mbar_init(&mi.pv_done[g], 1);
      mbar_init(&mi.q_full[g], MT2 ? 128 : 256);
      for (int w = 0; w < 4; ++w) mi.bad[g][w] = 0u;
    }
    mi.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&mi.tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  steps_prefix<C::ROWS, PER>(p, G, mi.prefix, kThreads);
  fence_after();
  const uint32_t tmem = mi.tmem;
  const int W = mi.prefix[p.batch];
  Walk<C::ROWS, PER> walk;
  walk.x = part_begin(W, blockIdx.x, gridDim.x);
  walk.end = part_begin(W, blockIdx.x + 1, gridDim.x);
  walk.b = 0;
  walk.first = true;
  Piece pc;
  bool dead = false;
  int kc = 0, vc = 0;  // tiles through the rings so far (every role counts them alike)
  auto wait = [&](uint64_t* bar, uint32_t phase) {
    // after a wait that gave up nobody waits any more, but every role runs to its end
    if (!dead && !mbar_wait(bar, phase, &g_error, 1)) {
      dead = true;
      mi.failed = 1;
    }
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 8) {
      // ---------------- TMA: page loads, lane = page of the tile ----------------
      while (!dead && walk.next(p, mi.prefix, G, blockIdx.x, pc)) {
        const int* bt = p.block_table + (long long)pc.b * p.max_blocks;
        int page0 = pc.s.lo / 16 + pc.t0 * (kKeys / 16);
        auto page_id = [&](int tile) {
          const int pg = page0 + tile * (kKeys / 16) + lane;
          const int id = (lane < kKeys / 16 && tile < pc.nt && pg < p.max_blocks && pg * 16 < pc.s.hi) ? bt[pg] : -1;
          return id >= 0 && id < p.n_blocks ? id : -1;
        };
        int id = page_id(0);
        for (int i = 0; i < pc.nt && !dead; ++i, ++kc, ++vc) {
          const int ahead = page_id(i + 1);
          const unsigned have = __ballot_sync(0xffffffffu, id >= 0) & 0xffu;
          const int row = (id * p.n_kv + pc.kvh) * 16;
          const uint32_t bytes = __popc(have) * 16 * HD * 2;
          const int ks = kc % C::SK, vs = vc % C::SV;
          if (kc >= C::SK) wait(&mi.k_empty[ks], (kc / C::SK - 1) & 1);
          dead = __any_sync(0xffffffffu, dead);
          if (dead) break;
          if (lane == 0) {
            if (bytes) mbar_expect_tx(&mi.k_full[ks], bytes);
            else mbar_arrive(&mi.k_full[ks]);
          }
          __syncwarp();
          if (id >= 0)
  #pragma unroll
            for (int bx = 0; bx < C::BOXES; ++bx)
              tma_load_2d(sm + C::OFF_K + ks * C::TILE + bx * kKeys * 128 + lane * 2048, &p.tmK, bx * 64, row,
                          &mi.k_full[ks]);
          if (vc >= C::SV) wait(&mi.v_empty[vs], (vc / C::SV - 1) & 1);
          dead = __any_sync(0xffffffffu, dead);
          if (dead) {
            ++kc;  // the K tile is in flight
            break;
          }
          if (lane == 0) {
            mi.miss[vs] = ~have & 0xffu;
            if (bytes) mbar_expect_tx(&mi.v_full[vs], bytes);
            else mbar_arrive(&mi.v_full[vs]);
          }
          __syncwarp();
          if (id >= 0)
  #pragma unroll
            for (int bx = 0; bx < C::BOXES; ++bx)
              tma_load_2d(sm + C::OFF_V + vs * C::TILE + bx * kKeys * 128 + lane * 2048, &p.tmV, bx * 64, row,
                          &mi.v_full[vs]);
          id = ahead;
        }
      }
    } else if (warp < 11) {
      // ---------------- MMA: one warp per warpgroup, one lane of it ----------------
      const int g = warp - 9;
      if (lane == 0) {
        const uint32_t s_col = tmem + g * 128, o_col = tmem + 256 + g * HD;
        const uint32_t q = smem_u32(sm) + (MT2 ? g * C::TILE : 0);
        int np = 0, nq = 0;  // PV products issued, pieces with tiles of this warpgroup
        while (walk.next(p, mi.prefix, G, blockIdx.x, pc)) {
          auto qk = [&](int i) {  // S = Q K^T of tile i of the piece
            const int c = kc + i, ks = c % C::SK;
            wait(&mi.k_full[ks], (c / C::SK) & 1);
            fence_after();
            const uint32_t k = smem_u32(sm) + C::OFF_K + ks * C::TILE;
  #pragma unroll
            for (int pl = 0; pl < (X2 ? 2 : 1); ++pl)
  #pragma unroll
              for (int e = 0; e < HD / 16; ++e) {
                const uint32_t o = (e >> 2) * kKeys * 128 + (e & 3) * 32;
                mma_ss(s_col, desc_k(q + pl * C::TILE + o), desc_k(k + o), idesc(kKeys, false), pl > 0 || e > 0);
              }
            commit(&mi.s_full[g]);
            commit(&mi.k_empty[ks]);
          };
          constexpr int STEP = MT2 ? 1 : 2;
          const int i0 = MT2 ? 0 : g;
          if (i0 < pc.nt) {
            wait(&mi.q_full[g], nq & 1);
            ++nq;
            fence_after();
            qk(i0);
          }
          for (int i = i0; i < pc.nt; i += STEP) {
            const int c = vc + i, vs = c % C::SV;
            wait(&mi.v_full[vs], (c / C::SV) & 1);
            wait(&mi.p_full[g], np & 1);
            fence_after();
            const uint32_t v = smem_u32(sm) + C::OFF_V + vs * C::TILE;
  #pragma unroll
            for (int pl = 0; pl < (X2 ? 2 : 1); ++pl)
  #pragma unroll
              for (int e = 0; e < kKeys / 16; ++e)
                mma_ts(o_col, s_col + pl * 64 + e * 8, desc_mn(v + e * 2048, kKeys * 128), idesc(HD, true));
            commit(&mi.pv_done[g]);
            commit(&mi.v_empty[vs]);
            if (i + STEP < pc.nt) {
              // the next scores overwrite the P this product reads
              wait(&mi.pv_done[g], np & 1);
              fence_after();
              qk(i + STEP);
            }
            ++np;
          }
          kc += pc.nt;
          vc += pc.nt;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------- softmax: one thread per row ----------------
    const int g = warp >> 2, r = tid & 127;          // warpgroup, row of its 128-row tile
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane of the warp's first row
    const uint32_t s_col = tmem + lanes + g * 128, o_col = tmem + lanes + 256 + g * HD;
    int ns = 0;  // score tiles of this warpgroup so far
    while (walk.next(p, mi.prefix, G, blockIdx.x, pc)) {
      const Span& s = pc.s;
      const int m = pc.m0 + (MT2 ? g * 128 : 0) + r, t = m / G, head = pc.kvh * G + m % G;
      const bool live = t < s.T;
      const int pos = live ? row_position(p, s, t) : s.ctx;
      const bool warp_live = __any_sync(0xffffffffu, live);
      // Q rows into shared memory: MT2, own tile; key split, half of the one tile each
      for (int x = (MT2 ? r : tid); x < 128 * (HD / 8); x += MT2 ? 128 : 256) {
        const int rr = x / (HD / 8), ch = x % (HD / 8);
        const int mm = pc.m0 + (MT2 ? g * 128 : 0) + rr, tt = mm / G;
        uint4 h = make_uint4(0u, 0u, 0u, 0u), l = h;
        if (tt < s.T) q_chunk(p, s.row0 + tt, pc.kvh * G + mm % G, HD, ch, h, l);
        uint8_t* dst = sm + (MT2 ? g * C::TILE : 0) + sw(rr, ch, 128);
        *reinterpret_cast<uint4*>(dst) = h;
        if (X2) *reinterpret_cast<uint4*>(dst + C::TILE) = l;
      }
      fence_async();
      if constexpr (MT2) {
        mbar_arrive(&mi.q_full[g]);
      } else {  // an MMA warp hears of the pieces that have a tile for it
        mbar_arrive(&mi.q_full[0]);
        if (pc.nt > 1) mbar_arrive(&mi.q_full[1]);
      }
      {  // O starts at zero: every product adds to it
        uint32_t z[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) z[e] = 0u;
#pragma unroll
        for (int c = 0; c < HD; c += 32) tmem_st32(o_col + c, z);
        tmem_wait_st();
      }
      float ref = -INFINITY, sum = 0.f;

      for (int i = MT2 ? 0 : g; i < pc.nt; i += PER) {
        const int c = vc + i, vs = c % C::SV, j0 = s.lo + (pc.t0 + i) * kKeys;
        wait(&mi.v_full[vs], (c / C::SV) & 1);
        const unsigned miss = mi.miss[vs];
        const bool whole = miss == 0 && j0 + kKeys <= s.ctx && (p.window == 0 || j0 > s.pmax - p.window);
        unsigned bad[4] = {0u, 0u, 0u, 0u};
        if (!whole) {
          // zero the V rows past the end or without a page, find and zero non-finite ones; MT2
          // shares the tile, and the two warpgroups do half each
          uint8_t* V = sm + C::OFF_V + vs * C::TILE;
          const int id = MT2 ? 3 : 1 + g, n = MT2 ? 256 : 128, me = MT2 ? tid : r;
          unsigned* flags = mi.bad[MT2 ? 0 : g];
          for (int x = me; x < kKeys * (HD / 8); x += n) {
            const int rr = x / (HD / 8), ch = x % (HD / 8);
            uint4* v = reinterpret_cast<uint4*>(V + sw(rr, ch, kKeys));
            if (j0 + rr >= s.hi || ((miss >> (rr >> 4)) & 1)) {
              *v = make_uint4(0u, 0u, 0u, 0u);
            } else if (nonfinite(*v)) {
              atomicOr(&flags[rr >> 5], 1u << (rr & 31));
            }
          }
          fence_async();
          bar_sync(id, n);
#pragma unroll
          for (int w = 0; w < 4; ++w) bad[w] = *reinterpret_cast<volatile unsigned*>(&flags[w]);
          if (bad[0] | bad[1] | bad[2] | bad[3]) {
            for (int x = me; x < kKeys * (HD / 8); x += n) {
              const int rr = x / (HD / 8), ch = x % (HD / 8);
              if ((bad[rr >> 5] >> (rr & 31)) & 1)
                *reinterpret_cast<uint4*>(V + sw(rr, ch, kKeys)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async();
            bar_sync(id, n);
            if (me < 4) flags[me] = 0u;
            bar_sync(id, n);
          }
        }
        wait(&mi.s_full[g], ns & 1);
        ++ns;
        fence_after();
        if (warp_live) {
          float x[kKeys];
#pragma unroll
          for (int e = 0; e < kKeys; e += 32) tmem_ld32(s_col + e, reinterpret_cast<uint32_t*>(x) + e);
          tmem_wait_ld();
          if (!whole) {  // places the row does not see, whatever they hold
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              unsigned see = live ? see_bits(p, s, t, pos, j0 + 32 * w) : 0u;
              if ((miss >> (2 * w)) & 1) see &= 0xffff0000u;
              if ((miss >> (2 * w + 1)) & 1) see &= 0x0000ffffu;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((see >> e) & 1u)) x[32 * w + e] = -INFINITY;
            }
          }
          if constexpr (X2) {
            // hi + lo parts make NaN of an infinite k where the product itself is fine
            float any = 0.f;
#pragma unroll
            for (int e = 0; e < kKeys; ++e) any += x[e];
            if (any != any && live) {
#pragma unroll 1
              for (int k = 0; k < kKeys; ++k) {
                float v = 0.f;
#pragma unroll
                for (int e = 0; e < kKeys; ++e) take_if(v, x[e], e, k);
                if (v == v) continue;
                v = dot_place<HD>(p, s, pc.b, pc.kvh, t, head, j0 + k);
#pragma unroll
                for (int e = 0; e < kKeys; ++e) take_if(x[e], v, e, k);
              }
            }
          }
          float mx = x[0];
#pragma unroll
          for (int e = 1; e < kKeys; ++e) mx = fmaxf(mx, x[e]);
          mx *= p.scale_log2;
          const bool grow = mx > ref + kSlack || (ref == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float to = grow ? mx : ref;
            const float corr = to == -INFINITY ? 1.f : ex2(ref - to);
            ref = to;
            sum *= corr;
            if (i >= PER) {  // O holds something; this tile's scores being there, its product is done
#pragma unroll
              for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_col + c0, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                tmem_st32(o_col + c0, o);
              }
            }
          }
          const float base = ref == -INFINITY ? 0.f : ref;  // nothing seen yet: weights 2^-inf
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int e = 0; e < kKeys; e += 2) {
            x[e] = ex2(fmaf(x[e], p.scale_log2, -base));
            x[e + 1] = ex2(fmaf(x[e + 1], p.scale_log2, -base));
            s0 += x[e];
            s1 += x[e + 1];
          }
          sum += s0 + s1;
          // weights as fp16 over the scores: relative 2^-11, the output's own rounding; with X2
          // their remainders behind them
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = pack2(x[64 * h + 2 * e], x[64 * h + 2 * e + 1]);
            tmem_st32(s_col + 32 * h, w);
            if constexpr (X2) {
#pragma unroll
              for (int e = 0; e < 32; ++e) w[e] = pack2_rest(x[64 * h + 2 * e], x[64 * h + 2 * e + 1], w[e]);
              tmem_st32(s_col + 64 + 32 * h, w);
            }
          }
          if (bad[0] | bad[1] | bad[2] | bad[3]) {  // non-finite V rows: the rows that see them alone
            tmem_wait_st();
#pragma unroll 1
            for (int k = 0; k < kKeys; ++k) {
              if (!((bad[k >> 5] >> (k & 31)) & 1u)) continue;
              float w = 0.f;
#pragma unroll
              for (int e = 0; e < kKeys; ++e) take_if(w, x[e], e, k);
              add_place<HD>(p, pc.b, pc.kvh, j0 + k, w, o_col);
            }
          }
          tmem_wait_st();
        }
        fence_before();
        mbar_arrive(&mi.p_full[g]);
      }
      kc += pc.nt;
      vc += pc.nt;

      // ---- the unit's (or piece's) result
      const bool any_tile = (MT2 ? 0 : g) < pc.nt;
      if (any_tile) wait(&mi.pv_done[g], (ns - 1) & 1);
      fence_after();
      float w0 = 1.f, w1 = 0.f;  // weights of this warpgroup's O and of the other one's
      if constexpr (!MT2) {
        mi.ml[g][r] = make_float2(ref, sum);
        fence_before();
        bar_sync(4, 256);
        fence_after();
        const float2 a = mi.ml[0][r], b = mi.ml[1][r];
        ref = fmaxf(a.x, b.x);
        const float base = ref == -INFINITY ? 0.f : ref;
        w0 = ex2(a.x - base);
        w1 = ex2(b.x - base);
        sum = a.y * w0 + b.y * w1;
      }
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // no place seen: zeros
      if (warp_live) {
        constexpr int COLS = MT2 ? HD : HD / 2;  // key split: each warpgroup finishes half of the columns
        const int c0 = MT2 ? 0 : g * COLS;
        const uint32_t col = MT2 ? o_col : tmem + lanes + 256 + c0;
        float* part = p.part_o + ((long long)pc.slot * C::ROWS + (m - pc.m0)) * HD + c0;
#pragma unroll 1
        for (int cc = 0; cc < COLS; cc += 32) {
          float o[32];
          tmem_ld32(col + cc, reinterpret_cast<uint32_t*>(o));
          if constexpr (!MT2) {
            float o1[32];
            tmem_ld32(col + HD + cc, reinterpret_cast<uint32_t*>(o1));
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(w0, o[e], w1 * o1[e]);
          } else {
            tmem_wait_ld();
          }
          if (!live) continue;
          if (pc.whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            store_row32(p, (long long)(s.row0 + t) * p.ldout + (long long)head * HD + c0 + cc, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + cc + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (!pc.whole && live && (MT2 || g == 0))
          *reinterpret_cast<float2*>(p.part_ml + ((long long)pc.slot * C::ROWS + (m - pc.m0)) * 2) =
              make_float2(ref, sum);
      }
      if constexpr (!MT2) {  // both states read: the next unit may begin
        fence_before();
        bar_sync(4, 256);
        fence_after();
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (mi.failed && warp == 8 && lane == 0) {  // copies in flight land before the CTA ends
    for (int i = max(0, kc - C::SK); i < kc; ++i) mbar_wait(&mi.k_full[i % C::SK], (i / C::SK) & 1, &g_error, 1);
    for (int i = max(0, vc - C::SV); i < vc; ++i) mbar_wait(&mi.v_full[i % C::SV], (i / C::SV) & 1, &g_error, 1);
  }
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Joins the pieces of each unit that more than one CTA worked on; one warp per row.
template <int HD, int ROWS, int PER>
__global__ void __launch_bounds__(256) tree_join_t5_kernel(const Params p, int ctas) {
  __shared__ int prefix[kMaxBatch + 1];
  const int G = p.n_heads / p.n_kv;
  const int b = blockIdx.z, mt = blockIdx.y / p.n_kv, kvh = blockIdx.y % p.n_kv;
  Span s;
  const int n = unit_steps<ROWS, PER>(p, b, mt, G, s);
  if (n == 0) return;
  steps_prefix<ROWS, PER>(p, G, prefix, 256);
  const int W = prefix[p.batch];
  int u0 = prefix[b];
  for (int i = 0; i < mt; ++i) {
    Span q;
    u0 += p.n_kv * unit_steps<ROWS, PER>(p, b, i, G, q);
  }
  u0 += kvh * n;
  // the CTAs whose parts hold the unit's first and last step
  int c0 = (int)((long long)u0 * ctas / W);
  while (part_begin(W, c0 + 1, ctas) <= u0) ++c0;
  while (part_begin(W, c0, ctas) > u0) --c0;
  int c1 = c0;
  while (part_begin(W, c1 + 1, ctas) < u0 + n) ++c1;
  if (c1 == c0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int rr = blockIdx.x * 8 + warp; rr < ROWS; rr += gridDim.x * 8) {
    const int m = mt * ROWS + rr, t = m / G;
    if (t >= s.T) break;
    // a CTA's place for this unit: its first piece begins with the CTA's part
    auto state = [&](int c) { return (long long)(2 * c + (part_begin(W, c, ctas) < u0 ? 1 : 0)) * ROWS + rr; };
    auto empty = [&](int c) { return part_begin(W, c, ctas) == part_begin(W, c + 1, ctas); };
    float top = -INFINITY;
    for (int c = c0; c <= c1; ++c)
      if (!empty(c)) top = fmaxf(top, p.part_ml[state(c) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f, acc[HD / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) acc[e] = 0.f;
    for (int c = c0; c <= c1; ++c) {
      if (empty(c)) continue;  // fewer steps than CTAs
      const long long st = state(c);
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + st * 2);
      const float w = ex2(ml.x - base);
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // nothing seen in this piece
      total = fmaf(w, ml.y, total);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) acc[e] = fmaf(w, p.part_o[st * HD + e * 32 + lane], acc[e]);
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const long long at = (long long)(s.row0 + t) * p.ldout + (long long)(kvh * G + m % G) * HD;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) store_out(p, at + e * 32 + lane, acc[e] * inv);
  }
}

// Whether this kernel serves the call (the other one has no limits of this kind).
static bool serves(int head_dim, int batch, long long max_steps) {
  return (head_dim == 64 || head_dim == 128) && batch <= kMaxBatch && max_steps < (1ll << 31);
}

// Rows of a unit, key tiles per step.  256 rows where a sequence may fill more than 128 (each K/V
// tile then serves two row tiles), unless hi + lo planes need the room.
struct Shape {
  bool mt2;
  int rows, m_tiles, grid;
  long long max_steps;
  size_t off_ml, bytes;
};
static Shape shape_of(int batch, int n_heads, int n_kv, int head_dim, int max_q, int max_ctx, bool x2) {
  Shape h;
  const long long m = (long long)max_q * (n_heads / n_kv);
  h.mt2 = !x2 && m > 128;
  h.rows = h.mt2 ? 256 : 128;
  h.m_tiles = (int)((m + h.rows - 1) / h.rows);
  const int keys = h.mt2 ? kKeys : 2 * kKeys;
  // + 1: with a window, a unit's first tile may begin anywhere
  h.max_steps = (long long)batch * n_kv * h.m_tiles * ((max_ctx + keys - 1) / keys + 1);
  h.grid = (int)std::min<long long>(num_sms(), h.max_steps);
  h.off_ml = (size_t)2 * h.grid * h.rows * head_dim * sizeof(float);
  h.bytes = h.off_ml + (size_t)2 * h.grid * h.rows * 2 * sizeof(float);
  return h;
}

template <int HD, bool MT2, bool X2>
static int launch(Params& p, const Shape& h, cudaStream_t stream) {
  using C = Cfg<HD, MT2, X2>;
  auto kern = tree_attn_t5_kernel<HD, MT2, X2>;
  const int smem = C::OFF_MISC + (int)sizeof(Misc) + 1024;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return B2D_ERR_CUDA;
  }
  kern<<<h.grid, kThreads, smem, stream>>>(p);
  B2D_TRY(launch_status());
  tree_join_t5_kernel<HD, C::ROWS, MT2 ? 1 : 2>
      <<<dim3(C::ROWS / 32, h.m_tiles * p.n_kv, p.batch), 256, 0, stream>>>(p, h.grid);
  return launch_status();
}

}  // namespace t5
}  // namespace tree
}  // namespace b2d
