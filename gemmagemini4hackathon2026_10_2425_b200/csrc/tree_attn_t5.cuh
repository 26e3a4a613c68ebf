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
// Roles: warps 0-7 softmax (warp w reads TMEM lanes 32 (w % 4) ..), warps 8 and 10 load K and V
// (TMA), warp 9 issues the MMAs, warp 11 loads the next unit's Q while this one ends.
//
// Weights are 2^((s - ref) c + 7), c = scale log2(e), ref a score: a product ref c of its own would be off
// by up to half a step, which is 2^9 for |ref c| near 2^33.  The difference is one more operation per
// pair of scores than a fused s c - ref c.
//
// O is rescaled only when a row's largest weight has grown by more than 2^8 since the last time: it
// starts at 2^7 and stays below 2^15, inside fp16's range, where what fp16 drops (2^-25) is 2^-32 of
// it.  After the first tiles of a unit that is almost never; the sum and the weights always use the
// same reference, so nothing else is lost.
//
// Included by tree_attn.cu, whose Params, Span and row helpers it uses.
#pragma once

namespace b2d {
namespace tree {

namespace t5 {

constexpr int kKeys = 128;
constexpr int kSoftmax = 256;               // threads of the two warpgroups
constexpr int kThreads = kSoftmax + 128;    // + K, MMA, V and Q warps
// Registers: a softmax thread holds a row of 128 scores.  384 threads launch with 168 each
// (64512); the split 256 * 224 + 128 * 56 uses the same number.
constexpr int kRegsSoftmax = 224, kRegsOther = 56;
constexpr int kGroups = 320;                // prefix sums kept, one per `stride` sequences
constexpr float kSlack = 8.f;               // log2 of the growth that O is rescaled for
constexpr float kLift = 7.f;                // log2 of the weight of a row's reference

template <int HD, bool MT2, bool X2>
struct Cfg {
  static constexpr int BOXES = HD / 64;
  static constexpr int TILE = kKeys * HD * 2;
  static constexpr int ROWS = MT2 ? 256 : 128;     // rows of a unit
  static constexpr int PLANES = MT2 || X2 ? 2 : 1;  // 128-row fp16 planes of Q
  // K and V stages.  A V tile waits for the weights, a K tile only for its turn: the room left over
  // goes to V (HD 128: 2 + 2 stages made the MMAs wait for V 1400 cycles a tile).
  static constexpr int SK = HD == 64 ? 4 : 2;
  static constexpr int SV = HD == 64 ? 4 : (X2 ? 2 : 3);
  static constexpr int OFF_K = PLANES * TILE;  // a Q plane is as large as a tile
  static constexpr int OFF_V = OFF_K + SK * TILE;
  static constexpr int OFF_MISC = OFF_V + SV * TILE;
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
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  return r;
}
// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* tm, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* tm) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// 128-byte swizzled operands.  K-major (Q, K): 8-row groups 1024 bytes apart.  MN-major (V, whose
// rows are the reduction): 8-row groups 1024 bytes apart, 64-column blocks `block` bytes apart.
// A descriptor's high word is a constant and its low word holds the address (in 16-byte units,
// below 2^14, so that adding to it stays in the field) and the block stride: the MMAs of one
// product differ by an addition of a constant.
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);  // group stride 1024, version, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr, uint32_t block) { return (addr >> 4) | ((block >> 4) << 16); }
// Byte offset of 16-byte chunk ch of row r in a V tile: pages of HD/64 blocks of 16 swizzled rows.
template <int HD>
__device__ __forceinline__ uint32_t v_at(int r, int ch) {
  return (uint32_t)((r >> 4) * (HD * 32) + (ch >> 3) * 2048 + (r & 15) * 128 + (((ch & 7) ^ (r & 7)) << 4));
}
// kind::f16, D fp32, A and B fp16, M = 128; bit 16: B is MN-major.
constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\t"
      "mov.b64 y, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"((uint32_t)acc), "r"(kDescHigh));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id) {  // accumulates
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, 1, 0;\n\tmov.b64 y, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(kDescHigh));
}
// One lane of the warp (the same each time), in code that all of it runs: the operands stay in
// uniform registers, which a branch on the lane number would load anew for every MMA.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// The part of one unit that a CTA works on.
struct Piece {
  Span s;
  int b, kvh, m0;
  int t0, nt;      // first key tile of the piece (of the unit's), number of them
  bool whole;      // the whole unit
  bool starts;     // its first steps
  int u_end;       // the unit's last step + 1
  int slot;        // place in the workspace, if not
};

// What beginning and ending a unit costs, in steps: the line counts it in, or the CTAs with many
// short units end last (4 x 512 causal rows over 0-8k places 348 us without, 203 us with; 32 trees of
// 5-24 nodes over 512-4k places 70 and 60 us).
template <int PER>
constexpr __host__ __device__ int unit_cost() {
  return PER == 1 ? 3 : 2;
}

// Steps of one unit of sequence b, row tile mt.
template <int ROWS, int PER>
__device__ __forceinline__ int unit_steps(const Params& p, int b, int mt, int G, Span& s) {
  if (!span_of(p, b, mt * ROWS, mt * ROWS + ROWS, G, kKeys, s)) return 0;
  return max(1, (s.hi - s.lo + kKeys * PER - 1) / (kKeys * PER));
}

// Steps of sequence b, with its units' cost.
template <int ROWS, int PER>
__device__ int sequence_steps(const Params& p, int b, int G) {
  int n = 0;
  Span s;
  for (int mt = 0; mt < p.m_tiles; ++mt) {
    const int u = unit_steps<ROWS, PER>(p, b, mt, G, s);
    if (u == 0) break;
    n += u + unit_cost<PER>();
  }
  return n * p.n_kv;
}

// prefix[j] = steps (with the units' cost) of the sequences before j * stride; all threads of the CTA.
struct Scan {
  int carry, wsum[32];
};
__device__ __forceinline__ int groups_of(int batch, int stride) { return (batch + stride - 1) / stride; }
template <int ROWS, int PER>
__device__ void steps_prefix(const Params& p, int G, int stride, int* prefix, Scan& sc) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int groups = groups_of(p.batch, stride);
  if (tid == 0) {
    sc.carry = 0;
    prefix[0] = 0;
  }
  __syncthreads();
  for (int j0 = 0; j0 < groups; j0 += threads) {
    const int j = j0 + tid;
    int n = 0;
    if (j < groups)
      for (int b = j * stride; b < min((j + 1) * stride, p.batch); ++b) n += sequence_steps<ROWS, PER>(p, b, G);
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sc.wsum[warp] = x;
    __syncthreads();
    int base = sc.carry;
    for (int w = 0; w < warp; ++w) base += sc.wsum[w];
    if (j < groups) prefix[j + 1] = base + x;
    __syncthreads();
    if (j0 + threads < groups) {
      if (tid == threads - 1) sc.carry = base + x;
      __syncthreads();
    }
  }
}

// CTA cta's part of the line of W steps.
__device__ __forceinline__ int part_begin(int W, int cta, int ctas) { return (int)((long long)W * cta / ctas); }

// Walks the pieces of steps [x, end) of the line.
template <int ROWS, int PER>
struct Walk {
  int x, end;
  int b, mt, n, at0;  // the units of row tile mt of sequence b, n steps each, begin at step at0
  int begun;          // where the CTA's part begins
  __device__ void begin(const Params& p, const int* prefix, int stride, int W) {
    x = begun = part_begin(W, blockIdx.x, gridDim.x);
    end = part_begin(W, blockIdx.x + 1, gridDim.x);
    int lo = 0, hi = groups_of(p.batch, stride);  // the group of sequences that holds step x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid;
    }
    b = lo * stride - 1;  // the first call of next() goes on to the next sequence
    mt = p.m_tiles;
    n = 0;
    at0 = prefix[lo];
  }
  // A unit's place in the line is its cost, then its steps; a part that holds the cost alone holds
  // none of the unit.
  __device__ bool next(const Params& p, int G, Piece& pc) {
    constexpr int cost = unit_cost<PER>();
    while (x < end) {
      Span s = pc.s;
      while (n == 0 || x >= at0 + (n + cost) * p.n_kv) {  // on to the next row tile, or sequence
        if (n) at0 += (n + cost) * p.n_kv;
        n = ++mt < p.m_tiles ? unit_steps<ROWS, PER>(p, b, mt, G, s) : 0;
        if (n == 0) {
          mt = 0;
          n = unit_steps<ROWS, PER>(p, ++b, 0, G, s);
        }
        pc.s = s;
      }
      const int kvh = (x - at0) / (n + cost), u = at0 + kvh * (n + cost);
      const int v1 = min(u + n + cost, end), s0 = max(0, x - u - cost), s1 = max(0, v1 - u - cost);
      pc.slot = 2 * (int)blockIdx.x + (x == begun ? 0 : 1);
      x = v1;
      if (s1 == s0) continue;
      const int tiles = (pc.s.hi - pc.s.lo + kKeys - 1) / kKeys;
      pc.b = b;
      pc.m0 = mt * ROWS;
      pc.kvh = kvh;
      pc.t0 = s0 * PER;
      pc.nt = max(0, min(s1 * PER, tiles) - pc.t0);
      pc.whole = s0 == 0 && s1 == n;
      pc.starts = s0 == 0;
      pc.u_end = u + n + cost;
      return true;
    }
    return false;
  }
};

template <int ROWS, int PER>
struct Misc {
  static constexpr bool MT2 = PER == 1;
  float2 ml[2][MT2 ? 1 : 128];  // key split: the warpgroups' (reference, sum) per row
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2], pv_done[2], q_full, q_empty, v_seen[2];
  uint64_t drained;             // after a wait that gave up: every MMA issued has ended
  unsigned bad[2][3][4];        // non-finite V rows of a tile that was looked over
  uint32_t tmem;
  int failed;
  int prefix[kGroups + 1];      // first step of each group of sequences
  Scan scan;
  // What each warp works on.  In shared memory on purpose: a softmax thread's registers hold a row
  // of scores, and values spilled to local memory may come from L2 (next to 200 KB of shared memory
  // the L1 holds little for long), some 300 cycles each.  What still is spilled (132-208 bytes a
  // thread) is on the loop's path: 6 loads and 2.6 stores per warp and tile, of 730 instructions.
  Piece pc[kThreads / 32];
  Walk<ROWS, PER> walk[kThreads / 32];
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
    __syncwarp();
    tmem_st32(o_col + c, o);
  }
  tmem_wait_st();
}

// The block-table entries of a piece's tiles, lane 0-7 a page each (-1: none).  Callers load an
// entry a tile ahead and compare it only when they come to the tile: a comparison would wait for
// the load on the spot.
struct Pages {
  const int* at;  // the lane's entry of tile 0
  int left;       // entries of the lane's column, from tile 0 on, that hold a page (in pages)
  __device__ Pages(const Params& p, const Piece& pc, int lane) {
    const int pg = pc.s.lo / 16 + pc.t0 * (kKeys / 16) + lane;
    at = p.block_table + (long long)pc.b * p.max_blocks + pg;
    left = lane < kKeys / 16 ? min(min(p.max_blocks, (pc.s.hi + 15) / 16), pg - lane + pc.nt * (kKeys / 16)) - pg : 0;
  }
  __device__ int operator()(int tile) const { return tile * (kKeys / 16) < left ? at[tile * (kKeys / 16)] : -1; }
};
// Bit per page of the tile that does not exist (the loaders skip it).
__device__ __forceinline__ unsigned missing(const Params& p, int entry) {
  return ~__ballot_sync(0xffffffffu, entry >= 0 && entry < p.n_blocks) & 0xffu;
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
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_t5_kernel(const __grid_constant__ Params p, const int stride) {
  using C = Cfg<HD, MT2, X2>;
  constexpr int PER = MT2 ? 1 : 2;  // key tiles per step
  extern __shared__ __align__(1024) uint8_t sm[];  // the kernel has no static shared memory
  Misc<C::ROWS, PER>& mi = *reinterpret_cast<Misc<C::ROWS, PER>*>(sm + C::OFF_MISC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.n_heads / p.n_kv;

  // fp16 rows whose heads fill a 128-row tile exactly come by TMA; others the softmax warps load
  const bool q_tma = p.q_f16 && 128 % G == 0;

  pdl_launch_dependents();  // the join waits for this grid's end before it reads anything
  if (tid == 0) {
    for (int i = 0; i < C::SK; ++i) {
      mbar_init(&mi.k_full[i], 1);
      mbar_init(&mi.k_empty[i], 1);
    }
    for (int i = 0; i < C::SV; ++i) {
      mbar_init(&mi.v_full[i], 1);
      mbar_init(&mi.v_empty[i], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&mi.s_full[g], 1);
      mbar_init(&mi.p_full[g], 4);
      mbar_init(&mi.pv_done[g], 1);
      mbar_init(&mi.v_seen[g], MT2 ? 8 : 4);
      for (int w = 0; w < 12; ++w) mi.bad[g][0][w] = 0u;
    }
    mbar_init(&mi.q_full, q_tma ? 1 : 8);
    mbar_init(&mi.q_empty, 1);
    mbar_init(&mi.drained, 1);
    mi.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32) {
    prefetch_map(&p.tmK);
    prefetch_map(&p.tmV);
    if (q_tma) prefetch_map(&p.tmQ);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&mi.tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (X2 && q_tma) {  // an fp16 q has nothing beyond its high part
    for (int x = tid; x < C::TILE / 16; x += kThreads)
      *reinterpret_cast<uint4*>(sm + C::TILE + x * 16) = make_uint4(0u, 0u, 0u, 0u);
    fence_async();
  }
  fence_before();
  steps_prefix<C::ROWS, PER>(p, G, stride, mi.prefix, mi.scan);
  fence_after();
  const uint32_t tmem = mi.tmem;
  const int W = mi.prefix[groups_of(p.batch, stride)];
  Piece& pc = mi.pc[warp];
  if (lane == 0) mi.walk[warp].begin(p, mi.prefix, stride, W);
  auto next_warp = [&]() {
    __syncwarp();  // the lanes are done with the piece before
    bool more = false;
    if (lane == 0) more = mi.walk[warp].next(p, G, pc);
    __syncwarp();  // and see the next one: a shuffle orders no memory
    return __shfl_sync(0xffffffffu, (int)more, 0) != 0;
  };
  bool dead = false;
  int kc = 0, vc = 0;  // tiles (warp 11: units) through the rings so far; every role counts them alike
  auto wait = [&](uint64_t* bar, uint32_t phase) {
    // after a wait that gave up nobody waits any more, but every role runs to its end
    if (!dead && !mbar_wait(bar, phase, &g_error, 1)) {
      dead = true;
      mi.failed = 1;
    }
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 8 || warp == 10) {
      // ---------------- TMA: page loads of K (warp 8) or V (warp 10), lane = page of the tile ----
      // A K page comes as HD/64 boxes of 16 rows x 128 bytes, each to its 64-column block of the
      // tile; a V page as one box of all of them (the MMA takes a page per 16 keys of reduction).
      const bool is_k = warp == 8;
      const int stages = is_k ? C::SK : C::SV;
      uint64_t* full = is_k ? mi.k_full : mi.v_full;
      uint64_t* empty = is_k ? mi.k_empty : mi.v_empty;
      while (!dead && next_warp()) {
        const Pages pages(p, pc, lane);
        const int nt = pc.nt, kvh = pc.kvh;
        int entry = pages(0);
        for (int i = 0; i < nt; ++i, ++kc) {
          const int id = entry >= 0 && entry < p.n_blocks ? entry : -1;
          entry = pages(i + 1);
          const unsigned have = __ballot_sync(0xffffffffu, id >= 0);
          const int row = (id * p.n_kv + kvh) * 16, st = kc % stages;
          if (kc >= stages) wait(&empty[st], (kc / stages - 1) & 1);
          dead = __any_sync(0xffffffffu, dead);
          if (dead) break;
          if (lane == 0) {
            if (have) mbar_expect_tx(&full[st], __popc(have) * 16 * HD * 2);
            else mbar_arrive(&full[st]);
          }
          __syncwarp();
          if (id >= 0) {
            if (is_k) {
#pragma unroll
              for (int bx = 0; bx < C::BOXES; ++bx)
                tma_load_2d(sm + C::OFF_K + st * C::TILE + bx * kKeys * 128 + lane * 2048, &p.tmK, bx * 64, row,
                            &full[st]);
            } else {
              tma_load_3d(sm + C::OFF_V + st * C::TILE + lane * (HD * 32), &p.tmV, 0, row, 0, &full[st]);
            }
          }
        }
      }
    } else if (warp == 9) {
      // ---------------- MMA: one elected lane, the warpgroups in turn ----------------
      // A turn is P V of one warpgroup's tile and the scores of its next one, back to back: while the
      // tensor cores do that, the other warpgroup has the exponential units to itself, and the two
      // keep alternating.  (Two issuing threads let both warpgroups do the same thing at the same
      // time.)
      // After a wait that gave up it hands nothing back to the loaders: a barrier with a copy in
      // flight must not be armed again.
      const uint32_t sm0 = smem_u32(sm);
      int np[2] = {0, 0}, nq = 0;  // products issued per warpgroup, pieces begun
      while (next_warp()) {
        auto qk = [&](int g, int i, bool first, bool last) {  // S_g = Q_g K^T of tile i of the piece
          const int c = kc + i, ks = c % C::SK;
          if (first) {
            wait(&mi.k_full[ks], (c / C::SK) & 1);
            fence_after();
          }
          const uint32_t q = desc_k(sm0 + (MT2 ? g * C::TILE : 0)), k = desc_k(sm0 + C::OFF_K + ks * C::TILE);
          if (elect_one()) {
#pragma unroll
            for (int pl = 0; pl < (X2 ? 2 : 1); ++pl)
#pragma unroll
              for (int e = 0; e < HD / 16; ++e) {
                const uint32_t o = ((e >> 2) * kKeys * 128 + (e & 3) * 32) >> 4;
                mma_ss(tmem + g * 128, q + pl * (C::TILE >> 4) + o, k + o, idesc(kKeys, false), pl > 0 || e > 0);
              }
            commit(&mi.s_full[g]);
            if (last && !dead) commit(&mi.k_empty[ks]);
          }
          __syncwarp();
        };
        auto pv = [&](int g, int i, bool first, bool last) {  // O_g += P_g V of tile i
          const int c = vc + i, vs = c % C::SV;
          // (a tile that some row must not see all of has been looked over before its weights are
          // announced: no wait of its own for that)
          if (first) wait(&mi.v_full[vs], (c / C::SV) & 1);
          wait(&mi.p_full[g], np[g] & 1);
          fence_after();
          const uint32_t v = desc_mn(sm0 + C::OFF_V + vs * C::TILE, 2048);
          if (elect_one()) {
#pragma unroll
            for (int pl = 0; pl < (X2 ? 2 : 1); ++pl)
#pragma unroll
              for (int e = 0; e < kKeys / 16; ++e)
                mma_ts(tmem + 256 + g * HD, tmem + g * 128 + pl * 64 + e * 8, v + e * (HD * 2), idesc(HD, true));
            commit(&mi.pv_done[g]);
            if (last && !dead) commit(&mi.v_empty[vs]);
          }
          __syncwarp();
        };
        auto pv_wait = [&](int g) {  // the next scores overwrite the P that the product reads
          wait(&mi.pv_done[g], np[g] & 1);
          fence_after();
        };
        wait(&mi.q_full, nq & 1);
        ++nq;
        // the first scores overwrite the last unit's weights
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (np[g] > 0) wait(&mi.pv_done[g], (np[g] - 1) & 1);
        fence_after();
        auto q_done = [&]() {  // every score of the unit is on its way: Q may go once they are formed
          if (elect_one() && !dead) commit(&mi.q_empty);
          __syncwarp();
        };
        if constexpr (MT2) {
          qk(0, 0, true, false);
          qk(1, 0, false, true);
          if (pc.nt == 1) q_done();
          for (int i = 0; i < pc.nt; ++i) {
            const bool more = i + 1 < pc.nt;
            pv(0, i, true, false);
            if (more) {
              pv_wait(0);
              qk(0, i + 1, true, false);
            }
            ++np[0];
            pv(1, i, false, true);
            if (more) {
              pv_wait(1);
              qk(1, i + 1, false, true);
              if (i + 2 == pc.nt) q_done();
            }
            ++np[1];
          }
        } else {
          qk(0, 0, true, true);
          if (pc.nt > 1) qk(1, 1, true, true);
          if (pc.nt <= 2) q_done();
          for (int i0 = 0; i0 < pc.nt; i0 += 2)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int i = i0 + g;
              if (i >= pc.nt) break;
              pv(g, i, true, true);
              if (i + 2 < pc.nt) {
                pv_wait(g);
                qk(g, i + 2, true, true);
                if (i + 3 == pc.nt) q_done();
              }
              ++np[g];
            }
        }
        kc += pc.nt;
        vc += pc.nt;
      }
    } else if (q_tma) {
      // ---------------- TMA: Q, as soon as the scores of the unit before are formed ----------------
      while (next_warp()) {
        if (kc > 0) wait(&mi.q_empty, (kc - 1) & 1);
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        ++kc;
        if (lane == 0) {
          constexpr int TILES = MT2 ? 2 : 1;
          mbar_expect_tx(&mi.q_full, TILES * C::TILE);
          for (int g = 0; g < TILES; ++g)
            for (int bx = 0; bx < C::BOXES; ++bx)
              tma_load_4d(sm + g * C::TILE + bx * 128 * 128, &p.tmQ, 0, pc.kvh * G,
                          pc.s.row0 + (pc.m0 + g * 128) / G, bx, &mi.q_full);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------- softmax: one thread per row ----------------
    const int g = warp >> 2, r = tid & 127;          // warpgroup, row of its 128-row tile
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane of the warp's first row
    const uint32_t s_col = tmem + lanes + g * 128, o_col = tmem + lanes + 256 + g * HD;
    Split shared_unit = {0, -1, 0, 0, 0, 0, 0};  // thread 0: the unit that other CTAs go on with
    int ns = 0, nl = 0;  // score tiles of this warpgroup so far, tiles looked over
    while (next_warp()) {
      const Span& s = pc.s;
      const int m = pc.m0 + (MT2 ? g * 128 : 0) + r, t = m / G, head = pc.kvh * G + m % G;
      const bool live = t < s.T;
      const int pos = live ? row_position(p, s, t) : s.ctx;
      const bool warp_live = __any_sync(0xffffffffu, live);
      if (!q_tma) {
        // Q rows into shared memory: MT2, own tile; key split, half of the one tile each.  This
        // warpgroup's (key split: both) scores of the unit before are formed.
        constexpr int QN = MT2 ? 128 : 256;
#pragma unroll 2
        for (int x = MT2 ? r : tid; x < 128 * (HD / 8); x += QN) {
          const int rr = x / (HD / 8), ch = x % (HD / 8), mm = pc.m0 + (MT2 ? g * 128 : 0) + rr, tt = mm / G;
          uint4 h = make_uint4(0u, 0u, 0u, 0u), l = h;
          if (tt < s.T) q_chunk(p, (long long)(s.row0 + tt) * p.ldq + (long long)(pc.kvh * G + mm % G) * HD + ch * 8, h, l);
          uint8_t* dst = sm + (MT2 ? g * C::TILE : 0) + sw(rr, ch, 128);
          *reinterpret_cast<uint4*>(dst) = h;
          if (X2) *reinterpret_cast<uint4*>(dst + C::TILE) = l;
        }
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&mi.q_full);
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
      const Pages pages(p, pc, lane);
      const int nt = pc.nt, first_j = s.lo + pc.t0 * kKeys;
      // tiles before this place are seen whole by every row, unless a page is missing or the window cuts
      const int whole_end = s.all - kKeys, whole_begin = p.window == 0 ? INT_MIN : s.pmax - p.window + 1;
      int entry = pages(MT2 ? 0 : g);

      for (int i = MT2 ? 0 : g; i < nt; i += PER) {
        const int c = vc + i, vs = c % C::SV, j0 = first_j + i * kKeys;
        const unsigned miss = missing(p, entry);
        entry = pages(i + PER);
        const bool whole = miss == 0 && j0 <= whole_end && j0 >= whole_begin;
        // the scores being there, this warpgroup's last product is done: its V stage has turned over,
        // and a wait for the next tile in it cannot mistake the phase
        wait(&mi.s_full[g], ns & 1);
        ++ns;
        fence_after();
        if (warp_live) {
          unsigned see[4];  // formed before the scores fill the registers
          if (!whole) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              see[w] = live ? see_bits(p, s, t, pos, j0 + 32 * w) : 0u;
              if ((miss >> (2 * w)) & 1) see[w] &= 0xffff0000u;
              if ((miss >> (2 * w + 1)) & 1) see[w] &= 0x0000ffffu;
            }
            __syncwarp();  // the lanes' branches end here: TMEM is read by the whole warp at once
          }
          float x[kKeys];
#pragma unroll
          for (int e = 0; e < kKeys; e += 32) tmem_ld32(s_col + e, reinterpret_cast<uint32_t*>(x) + e);
          tmem_wait_ld();
          if (!whole) {  // places the row does not see, whatever they hold
#pragma unroll
            for (int e = 0; e < kKeys; ++e)
              if (!((see[e >> 5] >> (e & 31)) & 1u)) x[e] = -INFINITY;
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
          float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int e = 4; e < kKeys; e += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              m4[k] = e + 4 + k < kKeys ? fmaxf(fmaxf(m4[k], x[e + k]), x[e + 4 + k]) : fmaxf(m4[k], x[e + k]);
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          // (the first place seen: inf > kSlack; none yet: NaN > kSlack)
          const bool grow = (mx - ref) * p.scale_log2 > kSlack;
          if (__any_sync(0xffffffffu, grow)) {
            const float corr = grow ? ex2((ref - mx) * p.scale_log2) : 1.f;
            if (grow) ref = mx;
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
          // weights as fp16 over the scores: relative 2^-11, the output's own rounding; with X2
          // their remainders behind them
          const uint64_t c2 = two(p.scale_log2, p.scale_log2), b2 = two(-base, -base), lift = two(kLift, kLift);
          uint64_t acc[2] = {0ull, 0ull};
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float& x0 = x[32 * h + 2 * e];
              float& x1 = x[32 * h + 2 * e + 1];
              const float2 z = split(fma2(add2(two(x0, x1), b2), c2, lift));
              x0 = ex2(z.x);
              x1 = ex2(z.y);
              acc[e & 1] = add2(acc[e & 1], two(x0, x1));
              w[e] = pack2(x0, x1);
            }
            tmem_st16(s_col + 16 * h, w);
            if constexpr (X2) {
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = pack2_rest(x[32 * h + 2 * e], x[32 * h + 2 * e + 1], w[e]);
              tmem_st16(s_col + 64 + 16 * h, w);
            }
          }
          const float2 s01 = split(add2(acc[0], acc[1]));
          sum += s01.x + s01.y;
          tmem_wait_st();
        }
        if (!whole) {
          // V rows past the end or without a page become zero and non-finite ones are found, by the
          // warps that share the tile (MT2: all eight); each of them hears of it through v_seen
          const int id = MT2 ? 0 : g, n = MT2 ? 256 : 128;
          unsigned* bad = mi.bad[id][nl % 3];
          wait(&mi.v_full[vs], (c / C::SV) & 1);
          uint8_t* V = sm + C::OFF_V + vs * C::TILE;
#pragma unroll 4
          for (int x = MT2 ? tid : r; x < kKeys * (HD / 8); x += n) {
            const int rr = x / (HD / 8), ch = x % (HD / 8);
            uint4* v = reinterpret_cast<uint4*>(V + v_at<HD>(rr, ch));
            const uint4 u = *v;
            if (j0 + rr >= s.hi || ((miss >> (rr >> 4)) & 1)) *v = make_uint4(0u, 0u, 0u, 0u);
            else if (nonfinite(u)) atomicOr(&bad[rr >> 5], 1u << (rr & 31));
          }
          // the flags of the next such tile: everyone is past the tile that used them last
          if ((MT2 ? tid : r) < 4) mi.bad[id][(nl + 1) % 3][tid & 3] = 0u;
          fence_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&mi.v_seen[id]);
          wait(&mi.v_seen[id], nl & 1);
          ++nl;
          if (bad[0] | bad[1] | bad[2] | bad[3]) {
            // the whole rows go (each warpgroup does it before its own product), and their products
            // are formed for the rows that see them alone
            for (int x = r; x < kKeys * (HD / 8); x += 128) {
              const int rr = x / (HD / 8), ch = x % (HD / 8);
              if ((bad[rr >> 5] >> (rr & 31)) & 1)
                *reinterpret_cast<uint4*>(V + v_at<HD>(rr, ch)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async();
            if (warp_live)
#pragma unroll 1
              for (int k = 0; k < kKeys; ++k) {
                if (!((bad[k >> 5] >> (k & 31)) & 1u)) continue;
                const float2 w2 = h2f2(tmem_ld1(s_col + k / 2));
                float w = (k & 1) ? w2.y : w2.x;
                if constexpr (X2) {
                  const float2 l2 = h2f2(tmem_ld1(s_col + 64 + k / 2));
                  w += (k & 1) ? l2.y : l2.x;
                }
                add_place<HD>(p, pc.b, pc.kvh, j0 + k, w, o_col);
              }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&mi.p_full[g]);
      }
      kc += pc.nt;
      vc += pc.nt;
      if (tid == 0 && pc.starts && !pc.whole) {
        int last = blockIdx.x;  // the CTA with the unit's last piece
        while (part_begin(W, last + 1, gridDim.x) < pc.u_end) ++last;
        shared_unit = Split{W, last, pc.slot, s.row0, s.T, pc.m0, pc.kvh};
      }

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
        w0 = ex2((a.x - base) * p.scale_log2);
        w1 = ex2((b.x - base) * p.scale_log2);
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
          if (live && pc.whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            store_row32(p, (long long)(s.row0 + t) * p.ldout + (long long)head * HD + c0 + cc, o);
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + cc + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          __syncwarp();  // rows that are not live come along: TMEM is read by the whole warp at once
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
    if (tid == 0) p.splits[blockIdx.x] = shared_unit;
  }
  fence_before();
  __syncthreads();
  fence_after();
  // a wait gave up somewhere: copies and MMAs in flight end before the CTA does
  if (mi.failed) {
    const bool k = warp == 8;
    const int stages = k ? C::SK : C::SV;
    if (k || warp == 10)
      for (int i = max(0, kc - stages); i < kc; ++i)
        mbar_wait(&(k ? mi.k_full : mi.v_full)[i % stages], (i / stages) & 1, &g_error, 1);
    if (warp == 11 && q_tma && kc > 0) mbar_wait(&mi.q_full, (kc - 1) & 1, &g_error, 1);
    if (warp == 9) {
      if (elect_one()) commit(&mi.drained);
      __syncwarp();
      mbar_wait(&mi.drained, 0, &g_error, 1);
    }
    __syncthreads();
  }
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Joins the pieces of each unit that more than one CTA worked on: blockIdx.x is the CTA with the
// unit's first piece (a CTA has one such unit at most, its last), one warp per row.
template <int HD, int ROWS>
__global__ void __launch_bounds__(256) tree_join_t5_kernel(const Params p, int ctas) {
  pdl_wait();
  const Split sp = p.splits[blockIdx.x];
  const int rr = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int G = p.n_heads / p.n_kv, t = (sp.m0 + rr) / G;
  if (sp.last <= (int)blockIdx.x || t >= sp.T) return;
  constexpr int E = HD / 32;
  // the places of the unit's pieces: the CTA's last one here, the first one of the CTAs after it
  // (those without any step hold nothing)
  auto state = [&](int c) { return (long long)(c == (int)blockIdx.x ? sp.slot : 2 * c) * ROWS + rr; };
  auto none = [&](int c) { return part_begin(sp.W, c, ctas) == part_begin(sp.W, c + 1, ctas); };
  float top = -INFINITY, total = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int c0 = blockIdx.x; c0 <= sp.last; c0 += 4) {  // four pieces' loads at a time
    float2 ml[4];
    float v[4][E];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + k;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (c > sp.last || none(c)) continue;
      const long long st = state(c);
      ml[k] = *reinterpret_cast<const float2*>(p.part_ml + st * 2);
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = p.part_o[st * HD + e * 32 + lane];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // nothing seen in this piece, or no piece
      const float m = fmaxf(top, ml[k].x), base = m == -INFINITY ? 0.f : m;
      const float w0 = ex2((top - base) * p.scale_log2), w1 = ex2((ml[k].x - base) * p.scale_log2);
      top = m;
      total = total * w0 + ml[k].y * w1;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + v[k][e] * w1;
    }
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  const long long at = (long long)(sp.row0 + t) * p.ldout + (long long)(sp.kvh * G + (sp.m0 + rr) % G) * HD;
#pragma unroll
  for (int e = 0; e < E; ++e) store_out(p, at + e * 32 + lane, acc[e] * inv);
}

// Rows of a unit, key tiles per step.  256 rows where a sequence may fill more than 128 (each K/V
// tile then serves two row tiles), unless hi + lo planes need the room.
struct Shape {
  bool mt2;
  int rows, live_rows, m_tiles, grid, stride;  // live_rows: of a unit, at most
  long long max_steps;
  size_t off_ml, off_splits, bytes;
};
static Shape shape_of(int batch, int n_heads, int n_kv, int head_dim, int max_q, int max_ctx, bool x2) {
  Shape h;
  const long long m = (long long)max_q * (n_heads / n_kv);
  h.mt2 = !x2 && m > 128;
  h.rows = h.mt2 ? 256 : 128;
  h.live_rows = (int)std::min<long long>(m, h.rows);
  h.m_tiles = (int)((m + h.rows - 1) / h.rows);
  const int keys = h.mt2 ? kKeys : 2 * kKeys;
  // + 1: with a window, a unit's first tile may begin anywhere
  h.max_steps = (long long)batch * n_kv * h.m_tiles * ((max_ctx + keys - 1) / keys + 1 + (h.mt2 ? unit_cost<1>() : unit_cost<2>()));
  h.stride = (batch + kGroups - 1) / kGroups;
  h.grid = (int)std::min<long long>(num_sms(), h.max_steps);
  h.off_ml = (size_t)2 * h.grid * h.rows * head_dim * sizeof(float);
  h.off_splits = h.off_ml + (size_t)2 * h.grid * h.rows * 2 * sizeof(float);
  h.bytes = h.off_splits + h.grid * sizeof(Split);
  return h;
}

template <int HD, bool MT2, bool X2>
static int launch(Params& p, const Shape& h, cudaStream_t stream) {
  using C = Cfg<HD, MT2, X2>;
  auto kern = tree_attn_t5_kernel<HD, MT2, X2>;
  const int smem = C::OFF_MISC + (int)sizeof(Misc<C::ROWS, MT2 ? 1 : 2>);
  static_assert(C::OFF_MISC + sizeof(Misc<C::ROWS, MT2 ? 1 : 2>) <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<unsigned long long> done;
  B2D_TRY(allow_smem(kern, smem, done));
  kern<<<h.grid, kThreads, smem, stream>>>(p, h.stride);
  B2D_TRY(launch_status());
  return launch_pdl(tree_join_t5_kernel<HD, C::ROWS>, dim3(h.grid, (h.live_rows + 7) / 8), dim3(256), 0, stream, p, h.grid);
}

}  // namespace t5
}  // namespace tree
}  // namespace b2d
