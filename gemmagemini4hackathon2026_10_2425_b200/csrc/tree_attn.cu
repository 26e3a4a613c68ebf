// Attention of several query rows per sequence over the paged cache: drafted trees, drafted
// chains, chunks of a prompt.
//
// The decode step's attention (attention.cu) has one query row per sequence; the reference's
// (LK/kernels.metal:235-305, window GK/kernels.metal:343) runs one row per threadgroup.  Here row
// t of sequence b (T_b rows, already rotated, K/V of the rows already in the cache at places
// ctx_b .. ctx_b + T_b - 1) sees every cached place j < ctx_b and, of the step's own rows, those
// its mask names (a tree) or those up to itself (no mask):
//   O_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = exp(scale q_t . k_j - m_t)   over the places seen.
//
// The T_b * G query rows of one KV head (G = heads per KV head) are the M side of two tensor-core
// products per key tile.  head_dim 64 and 128 run on tcgen05 (tree_attn_t5.cuh: 128 or 256 rows
// share each read of the cache); at head_dim 256 that kernel's two output tiles and two score tiles
// of 128 rows are 768 columns of TMEM, which has 512 (one output tile of 256 columns with 64-key tiles
// would fit; it is not built), so it runs on the kernel of this file:
//  * one CTA per (chunk of keys, 64-row tile of a KV head, sequence): four consumer warps of 16
//    rows each and one producer warp that streams key tiles (64 keys = 4 pages, TMA, 128-byte
//    swizzle) through a shared-memory ring;
//  * S = Q K^T and O += P V on mma.sync m16n8k16, running maximum and sum in registers;
//  * a sequence cut into several chunks leaves (max, sum, unnormalized output) per row and chunk
//    in the workspace and a second kernel joins them.
// Measured for 8 trees of 64 nodes over 8k-32k places at head_dim 128: 874 us on mma.sync, 205 us
// on tcgen05; for one draft of 8 rows over 1021 places 43.7 and 16 us.  So every size goes to
// tcgen05 where it can.  At head_dim 256 (8 heads on one KV head, 8 trees of 61-64 nodes over 4k-8k
// places, 25 GFLOP) this kernel takes 155 us in fp16, 210 us in fp32, 64 us in fp16 with a window of
// 512: bound by its four MMA warps per SM.
//
// fp32 q (or an output wider than fp16) carries q and the weights as hi + lo fp16 pairs, as the decode
// attention does: two MMAs for one.  A pair has 22 bits down to 2^-14 and no step below 2^-24, so the
// weights are lifted: the largest is 2^7 .. 2^15 (head_dim 256: 2^15), and what a place loses is 2^-32
// (2^-40) of it at most.  No state survives a call, so the workspace
// needs no initial contents and calls on different streams share nothing.
//
// Places a row must not see contribute nothing whatever they hold: scores are replaced, not
// added to, and a tile that any row sees only in part has its V checked -- rows past the end are
// zeroed, and a non-finite V row is zeroed and its product formed for the rows that see it alone
// (0 * NaN would otherwise reach every row of the MMA).
#include <algorithm>

#include "async.cuh"
#include "common.cuh"

namespace b2d {

int make_tmap_f16(CUtensorMap* m, const void* base, uint64_t rows, int cols, int ld, int box_rows);
int make_tmap_f16_blocks(CUtensorMap* m, const void* base, uint64_t rows, int cols, int box_rows);
int make_tmap_f16_heads(CUtensorMap* m, const void* base, uint64_t rows, int heads, int hd, int ld, int box_heads,
                        int box_rows);

namespace tree {

constexpr int kWarps = 4;                       // consumer warps
constexpr int kThreads = 32 * kWarps + 32;      // + the producer warp
constexpr int kRows = 16 * kWarps;              // query rows (t, g) per CTA
constexpr int kKeys = 64;                       // keys per tile
constexpr int kMaxChunk = 32768;                // keys per CTA (their page ids are in shared memory)
constexpr int kMaxWords = 8;
constexpr float kLift = 15.f;                   // log2 of a row's largest weight

__device__ int g_error;  // a bounded wait gave up (b2d_paged_tree_attn_error)

// A unit of work that several CTAs share (tcgen05 kernel): CTAs blockIdx.x .. last.
struct Split {
  int W, last, slot, row0, T, m0, kvh;
};

struct Params {
  // page pools as [n_blocks * Hkv * 16, HD] fp16: boxes of 64 columns x 16 rows (tcgen05 kernel's V:
  // 16 rows x all 64-column blocks)
  CUtensorMap tmK, tmV;
  CUtensorMap tmQ;  // q rows as [64-column block][row][head]: G heads x 128 / G rows per box
  const void* q;
  int q_f16;
  long long ldq;
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  const int* block_table;
  int max_blocks, n_blocks;
  const int* ctx_lens;
  const int* cu_q;
  const uint32_t* mask;
  int words;
  const int* positions;
  int n_heads, n_kv, batch, rows, max_q, max_ctx;
  int m_tiles;  // row tiles of the longest sequence
  float scale_log2;  // scale * log2(e)
  int window;
  void* out;
  int out_f16;
  uint16_t* out_lo;
  long long ldout;
  int chunk;       // keys per CTA (a multiple of kKeys)
  int max_chunks;  // chunks per sequence
  float* part_o;   // [rows][n_heads][max_chunks][HD]
  float* part_ml;  // [rows][n_heads][max_chunks][2]
  Split* splits;   // tcgen05 kernel: one per CTA; its part_o and part_ml are [2 * CTAs][unit rows]
};


// What the row tile m0 .. m1 - 1 of sequence b works on; the same in every kernel.
struct Span {
  int row0, T, ctx;  // first row, rows, cached places
  int lo, hi;        // places [lo, hi) that any of the tile's rows may see; lo a multiple of `keys`
  int all;           // every row sees the places before this one (but for the window)
  int pmax;          // no row's position is larger
  __device__ int chunks(int chunk) const { return hi > lo ? (hi - lo + chunk - 1) / chunk : 0; }
};

__device__ __forceinline__ bool span_of(const Params& p, int b, int m0, int m1, int G, int keys, Span& s) {
  s.ctx = p.ctx_lens[b];
  s.row0 = p.cu_q[b];
  s.T = min(min(p.cu_q[b + 1] - s.row0, p.max_q), p.rows - s.row0);
  if (s.row0 < 0 || s.T <= 0 || s.ctx < 0 || s.ctx > p.max_ctx - s.T) return false;
  const int t0 = m0 / G, t1 = min((m1 - 1) / G, s.T - 1);  // the tile's rows
  if (t0 >= s.T) return false;
  s.all = p.mask ? s.ctx : s.ctx + t0 + 1;
  s.pmax = s.ctx + t1;
  s.hi = p.mask ? s.ctx + s.T : s.ctx + t1 + 1;
  // row t's position is at least ctx (a tree) or ctx + t
  s.lo = p.window > 0 ? max(0, min(s.ctx + (p.mask ? 0 : t0) - p.window + 1, s.ctx)) / keys * keys : 0;
  return true;
}

// Position of row i of a sequence: given ones are held to ctx .. ctx + i, where a tree's are.
__device__ __forceinline__ int row_position(const Params& p, const Span& s, int i) {
  if (!p.mask || p.window <= 0) return s.ctx + i;
  return min(max(p.positions[s.row0 + i], s.ctx), s.ctx + i);
}

template <int HD>
struct Cfg {
  static constexpr int BOXES = HD / 64;
  static constexpr int TILE = kKeys * HD * 2;  // one K (or V) tile
  static constexpr int STAGES = 2;
  static constexpr int Q_PLANE = kRows * HD * 2;
  static constexpr int SMEM(bool x2) {
    return 1024 + STAGES * 2 * TILE + (x2 ? 2 : 1) * Q_PLANE + kMaxChunk / 16 * 4;
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What fp16 left of (a, b) after rounding them to `hi`.
__device__ __forceinline__ uint32_t pack2_rest(float a, float b, uint32_t hi) {
  const float2 h = h2f2(hi);
  return pack2(a - h.x, b - h.y);
}
// Byte offset of 16-byte chunk c of row r in a [rows][HD] fp16 tile of 128-byte swizzled rows
// (64 columns per box, `rows` rows per box).
__device__ __forceinline__ uint32_t sw(int r, int c, int rows) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// v = x if a == b, opaque to the compiler (which would put the array x comes from into memory).
__device__ __forceinline__ void take_if(float& v, float x, int a, int b) {
  asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %2, %3;\n\tselp.f32 %0, %1, %0, p;\n\t}"
      : "+f"(v)
      : "f"(x), "r"(a), "r"(b));
}
__device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, 128;" ::: "memory");
}

// 8 elements of q from element `at` on as fp16, and what fp32 elements have beyond that.
__device__ __forceinline__ void q_chunk(const Params& p, long long at, uint4& h, uint4& l) {
  if (p.q_f16) {
    h = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at);
  } else {
    const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at);
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + 4);
    h = make_uint4(pack2(u.x, u.y), pack2(u.z, u.w), pack2(v.x, v.y), pack2(v.z, v.w));
    l = make_uint4(pack2_rest(u.x, u.y, h.x), pack2_rest(u.z, u.w, h.y), pack2_rest(v.x, v.y, h.z),
                   pack2_rest(v.z, v.w, h.w));
  }
}
// Any of 8 fp16 values infinite or NaN.
__device__ __forceinline__ bool nonfinite(uint4 u) {
  // an exponent of all ones, and only that, carries into the sign's place
  auto carry = [](uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; };
  return ((carry(u.x) | carry(u.y) | carry(u.z) | carry(u.w)) & 0x80008000u) != 0;
}

// 32 consecutive output elements from i on (16-byte aligned).
__device__ __forceinline__ void store_row32(const Params& p, long long i, const float* v) {
  if (!p.out_f16) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    return;
  }
  uint32_t h[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) h[e] = pack2(v[2 * e], v[2 * e + 1]);
  uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
  if (p.out_lo) {
#pragma unroll
    for (int e = 0; e < 16; ++e) h[e] = pack2_rest(v[2 * e], v[2 * e + 1], h[e]);
    o = reinterpret_cast<uint4*>(p.out_lo + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
  }
}

__device__ __forceinline__ void store_out(const Params& p, long long i, float v) {
  if (p.out_f16)
    store_f16_split(static_cast<uint16_t*>(p.out), p.out_lo, (size_t)i, v);
  else
    static_cast<float*>(p.out)[i] = v;
}

// q . k of one row's head and a key, in fp32.
template <int HD, class Key>
__device__ __forceinline__ float dot_row(const Params& p, int row, int head, Key key) {
  const long long at = (long long)row * p.ldq + (long long)head * HD;
  float a = 0.f;
  for (int d = 0; d < HD; ++d)
    a = fmaf(p.q_f16 ? h2f(static_cast<const uint16_t*>(p.q)[at + d]) : static_cast<const float*>(p.q)[at + d],
             key(d), a);
  return a;
}
template <int HD>
__device__ __noinline__ float dot_tile(const Params& p, int row, int head, const uint8_t* Kt, int r) {
  return dot_row<HD>(p, row, head, [&](int d) {
    return h2f(*reinterpret_cast<const uint16_t*>(Kt + sw(r, d / 8, kKeys) + (d & 7) * 2));
  });
}

template <int HD, bool X2>
__global__ void __launch_bounds__(kThreads) paged_tree_attn_kernel(const __grid_constant__ Params p) {
  using C = Cfg<HD>;
  constexpr int KS = HD / 16, ND = HD / 8, NT = kKeys / 8;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* qs = ring + C::STAGES * 2 * C::TILE;  // [planes][BOXES][64 rows][128 bytes]
  int* blk = reinterpret_cast<int*>(qs + (X2 ? 2 : 1) * C::Q_PLANE);
  __shared__ __align__(8) uint64_t full[C::STAGES], empty[C::STAGES];
  __shared__ unsigned long long bad_keys[3];  // non-finite V rows of a looked-over tile, in turn
  __shared__ int failed;

  const int G = p.n_heads / p.n_kv;
  const int m_tiles = p.m_tiles;
  const int c = blockIdx.x, b = blockIdx.z;
  const int kvh = blockIdx.y / m_tiles, m0 = (blockIdx.y % m_tiles) * kRows;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Span s;
  if (!span_of(p, b, m0, m0 + kRows, G, kKeys, s)) return;
  const int nact = s.chunks(p.chunk);
  if (c >= max(nact, 1)) return;
  const int lo = s.lo + c * p.chunk, hi = min(lo + p.chunk, s.hi);
  const int tiles = hi > lo ? (hi - lo + kKeys - 1) / kKeys : 0;

  // page ids of the chunk (-1: outside the pool, never read), barriers
  const int* bt = p.block_table + (long long)b * p.max_blocks;
  for (int i = tid; i < tiles * (kKeys / 16); i += kThreads) {
    const int pg = lo / 16 + i;
    const int id = (pg < p.max_blocks && pg * 16 < s.hi) ? bt[pg] : -1;
    blk[i] = (id >= 0 && id < p.n_blocks) ? id : -1;
  }
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
    bad_keys[0] = bad_keys[1] = bad_keys[2] = 0ull;
  }
  // q rows of the tile into shared memory, as fp16 (hi and lo parts of fp32)
  for (int i = tid; i < kRows * (HD / 8); i += kThreads) {
    const int r = i / (HD / 8), ch = i % (HD / 8);
    const int m = m0 + r, t = m / G, g = m % G;
    uint4 h = make_uint4(0u, 0u, 0u, 0u), l = h;
    if (t < s.T) q_chunk(p, (long long)(s.row0 + t) * p.ldq + (long long)(kvh * G + g) * HD + ch * 8, h, l);
    *reinterpret_cast<uint4*>(qs + sw(r, ch, kRows)) = h;
    if (X2) *reinterpret_cast<uint4*>(qs + C::Q_PLANE + sw(r, ch, kRows)) = l;
  }
  __syncthreads();

  int issued = 0;  // the producer's
  if (warp == kWarps) {
    // ---------------- producer ----------------
    if (lane == 0) {
      for (int i = 0; i < tiles; ++i) {
        const int st = i % C::STAGES;
        if (i >= C::STAGES && !mbar_wait(&empty[st], (i / C::STAGES - 1) & 1, &g_error, 1)) {
          failed = 1;
          break;
        }
        issued = i + 1;
        uint8_t* dst = ring + st * 2 * C::TILE;
        int n = 0;
        for (int pg = 0; pg < kKeys / 16; ++pg) n += blk[i * (kKeys / 16) + pg] >= 0;
        if (n == 0) {
          mbar_arrive(&full[st]);
          continue;
        }
        mbar_expect_tx(&full[st], n * 2 * 16 * HD * 2);
        for (int pg = 0; pg < kKeys / 16; ++pg) {
          const int id = blk[i * (kKeys / 16) + pg];
          if (id < 0) continue;
          const int row = (id * p.n_kv + kvh) * 16;
#pragma unroll
          for (int bx = 0; bx < C::BOXES; ++bx) {
            tma_load_2d(dst + bx * kKeys * 128 + pg * 2048, &p.tmK, bx * 64, row, &full[st]);
            tma_load_2d(dst + C::TILE + bx * kKeys * 128 + pg * 2048, &p.tmV, bx * 64, row, &full[st]);
          }
        }
      }
    }
  } else {
    // ---------------- consumers ----------------
    const int g8 = lane >> 2, t4 = lane & 3, r8 = lane & 7, mat = lane >> 3;
    const int mr0 = m0 + warp * 16 + g8;           // this lane's rows: mr0 and mr0 + 8
    const int ts[2] = {mr0 / G, (mr0 + 8) / G};
    const bool live[2] = {ts[0] < s.T, ts[1] < s.T};
    int pos[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      pos[e] = live[e] ? row_position(p, s, ts[e]) : s.ctx;
    const uint32_t* words[2] = {p.mask + (long long)(s.row0 + (live[0] ? ts[0] : 0)) * p.words,
                                p.mask + (long long)(s.row0 + (live[1] ? ts[1] : 0)) * p.words};
    float o[ND][4];
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) o[nd][0] = o[nd][1] = o[nd][2] = o[nd][3] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    const uint32_t qb = smem_u32(qs);
    bool dead = false;
    int nl = 0;  // tiles looked over

    for (int i = 0; i < tiles; ++i) {
      const int st = i % C::STAGES, j0 = lo + i * kKeys;
      // a wait that gave up: no more waits, but the warp keeps its place in the CTA's barriers
      if (!dead && !__all_sync(0xffffffffu, mbar_wait(&full[st], (i / C::STAGES) & 1, &g_error, 1))) {
        dead = true;
        failed = 1;
      }
      uint8_t* Kt = ring + st * 2 * C::TILE;
      uint8_t* Vt = Kt + C::TILE;
      // does every row of the tile see every key of it?
      bool whole = j0 + kKeys <= s.all && (p.window == 0 || j0 > s.pmax - p.window);
#pragma unroll
      for (int pg = 0; pg < kKeys / 16; ++pg) whole &= blk[i * (kKeys / 16) + pg] >= 0;
      unsigned long long bad = 0ull;
      if (!whole) {
        // zero the V rows past the end or without a page; find and zero non-finite ones.  A warp may
        // be a tile ahead of another between two barriers, so three words take turns: the next
        // tile's is cleared before this tile's barrier, when everyone is past the tile that used it
        unsigned long long* const found = &bad_keys[nl % 3];
        for (int x = tid; x < kKeys * (HD / 8); x += 32 * kWarps) {
          const int r = x / (HD / 8), ch = x % (HD / 8);
          uint4* v = reinterpret_cast<uint4*>(Vt + sw(r, ch, kKeys));
          const bool out = j0 + r >= s.hi || blk[i * (kKeys / 16) + r / 16] < 0;
          if (!out) {
            if (nonfinite(*v)) atomicOr(found, 1ull << r);
          } else {
            *v = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        if (tid == 0) bad_keys[(nl + 1) % 3] = 0ull;
        ++nl;
        consumers_sync();
        bad = *reinterpret_cast<volatile unsigned long long*>(found);
        if (bad) {  // whole rows of V go, finite elements too: bad rows are added by hand
          for (int x = tid; x < kKeys * (HD / 8); x += 32 * kWarps) {
            const int r = x / (HD / 8), ch = x % (HD / 8);
            if ((bad >> r) & 1) *reinterpret_cast<uint4*>(Vt + sw(r, ch, kKeys)) = make_uint4(0u, 0u, 0u, 0u);
          }
          consumers_sync();
        }
      }

      // S = Q K^T
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      const uint32_t kb = smem_u32(Kt), vb = smem_u32(Vt);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t qa[4], ql[4];
        const uint32_t qo = sw(warp * 16 + (mat & 1) * 8 + r8, 2 * ks + (mat >> 1), kRows);
        ldsm4(qb + qo, qa);
        if (X2) ldsm4(qb + C::Q_PLANE + qo, ql);
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t kf[4];
          ldsm4(kb + sw(n * 8 + (mat >> 1) * 8 + r8, 2 * ks + (mat & 1), kKeys), kf);
          mma(sc[n], qa, kf[0], kf[1]);
          mma(sc[n + 1], qa, kf[2], kf[3]);
          if (X2) {
            mma(sc[n], ql, kf[0], kf[1]);
            mma(sc[n + 1], ql, kf[2], kf[3]);
          }
        }
      }
      if constexpr (X2) {
        // q as hi + lo parts makes NaN of an infinite k (or of a q past fp16's range) where the
        // product itself is fine: such scores are formed again, one by one
        float any = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) any += (sc[n][0] + sc[n][1]) + (sc[n][2] + sc[n][3]);
        if (__any_sync(0xffffffffu, any != any)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sc[n][e] != sc[n][e] && live[e >> 1])
                sc[n][e] = dot_tile<HD>(p, s.row0 + ts[e >> 1], kvh * G + (mr0 + 8 * (e >> 1)) % G, Kt,
                                       n * 8 + 2 * t4 + (e & 1));
        }
      }
      // scores outside a row's places are replaced, whatever they are
      if (!whole) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + n * 8 + 2 * t4 + (e & 1), h = e >> 1;
            bool see = live[h] && j < s.hi && blk[i * (kKeys / 16) + (n >> 1)] >= 0;
            if (see && j >= s.ctx) {
              const int own = j - s.ctx;
              see = p.mask ? own < 32 * p.words && ((words[h][own >> 5] >> (own & 31)) & 1u)
                           : own <= ts[h];
            }
            if (see && p.window > 0) {
              const int kp = j >= s.ctx ? row_position(p, s, j - s.ctx) : j;
              see = kp > pos[h] - p.window;
            }
            if (!see) sc[n][e] = -INFINITY;
          }
      }
      // running maximum and sum.  Weights are 2^((s - m) c): a product m c of its own would be off by up
      // to half a step, which is 2^9 for |m c| near 2^33.  kLift makes the largest one 2^15: fp16 has
      // no steps below 2^-24, so the smallest that are kept then are 2^-40 of it
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        m = fmaxf(mx[h], m);
        const float base = m == -INFINITY ? 0.f : m;  // nothing seen yet: every weight is 2^-inf
        const float corr = ex2((mx[h] - base) * p.scale_log2);
        mx[h] = m;
        float part = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sc[n][2 * h] = ex2(fmaf(sc[n][2 * h] - base, p.scale_log2, kLift));
          sc[n][2 * h + 1] = ex2(fmaf(sc[n][2 * h + 1] - base, p.scale_log2, kLift));
          part += sc[n][2 * h] + sc[n][2 * h + 1];
        }
        sum[h] = fmaf(sum[h], corr, part);
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) {
          o[nd][2 * h] *= corr;
          o[nd][2 * h + 1] *= corr;
        }
      }
      // O += P V.  P is rounded to fp16 for the product (relative 2^-11, the output's own
      // rounding) unless the result is kept in fp32: then its remainder follows in a second MMA.
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk) {
        const float* s0 = sc[2 * kk];
        const float* s1 = sc[2 * kk + 1];
        const uint32_t pa[4] = {pack2(s0[0], s0[1]), pack2(s0[2], s0[3]), pack2(s1[0], s1[1]),
                                pack2(s1[2], s1[3])};
        uint32_t pl[4];
        if (X2) {
          pl[0] = pack2_rest(s0[0], s0[1], pa[0]);
          pl[1] = pack2_rest(s0[2], s0[3], pa[1]);
          pl[2] = pack2_rest(s1[0], s1[1], pa[2]);
          pl[3] = pack2_rest(s1[2], s1[3], pa[3]);
        }
#pragma unroll
        for (int nd = 0; nd < ND; nd += 2) {
          uint32_t vf[4];
          ldsm4t(vb + sw(kk * 16 + (mat & 1) * 8 + r8, nd + (mat >> 1), kKeys), vf);
          mma(o[nd], pa, vf[0], vf[1]);
          mma(o[nd + 1], pa, vf[2], vf[3]);
          if (X2) {
            mma(o[nd], pl, vf[0], vf[1]);
            mma(o[nd + 1], pl, vf[2], vf[3]);
          }
        }
      }
      // non-finite V rows: only the rows that see them
      while (bad) {
        const int k = __ffsll((long long)bad) - 1;
        bad &= bad - 1;
        const int id = blk[i * (kKeys / 16) + k / 16];
        const uint16_t* v = p.v_pages + (((long long)id * p.n_kv + kvh) * 16 + k % 16) * HD;
        float w0 = 0.f, w1 = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          take_if(w0, (k & 1) ? sc[n][1] : sc[n][0], k / 8, n);
          take_if(w1, (k & 1) ? sc[n][3] : sc[n][2], k / 8, n);
        }
        const int src = (lane & ~3) | ((k & 7) >> 1);
        w0 = __shfl_sync(0xffffffffu, w0, src);
        w1 = __shfl_sync(0xffffffffu, w1, src);
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) {
          const float2 f = h2f2(*reinterpret_cast<const uint32_t*>(v + nd * 8 + 2 * t4));
          if (w0 != 0.f) {
            o[nd][0] = fmaf(w0, f.x, o[nd][0]);
            o[nd][1] = fmaf(w0, f.y, o[nd][1]);
          }
          if (w1 != 0.f) {
            o[nd][2] = fmaf(w1, f.x, o[nd][2]);
            o[nd][3] = fmaf(w1, f.y, o[nd][3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our writes before the refill
        mbar_arrive(&empty[st]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      if (!live[h]) continue;
      const int head = kvh * G + (mr0 + 8 * h) % G, row = s.row0 + ts[h];
      if (nact <= 1) {
        const float inv = sum[h] == 0.f ? 0.f : 1.0f / sum[h];  // no place seen: zeros
        const long long at = (long long)row * p.ldout + (long long)head * HD + 2 * t4;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) {
          store_out(p, at + nd * 8, o[nd][2 * h] * inv);
          store_out(p, at + nd * 8 + 1, o[nd][2 * h + 1] * inv);
        }
      } else {
        const long long pi = ((long long)row * p.n_heads + head) * p.max_chunks + c;
        float* po = p.part_o + pi * HD + 2 * t4;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
          *reinterpret_cast<float2*>(po + nd * 8) = make_float2(o[nd][2 * h], o[nd][2 * h + 1]);
        if (t4 == 0)
          *reinterpret_cast<float2*>(p.part_ml + pi * 2) = make_float2(mx[h], sum[h]);
      }
    }
  }
  // after a wait that gave up: copies in flight land before the CTA ends
  __syncthreads();
  if (failed)
    for (int i = max(0, issued - C::STAGES); i < issued; ++i)
      mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1, &g_error, 1);
}

// Joins the chunks of one row of one head: weights 2^((m_c - m) c), one warp per (row, head).
template <int HD>
__global__ void __launch_bounds__(256) tree_join_kernel(const Params p) {
  const int G = p.n_heads / p.n_kv;
  const int m_tiles = p.m_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y / m_tiles, m0 = (blockIdx.y % m_tiles) * kRows;
  Span s;
  if (!span_of(p, b, m0, m0 + kRows, G, kKeys, s)) return;
  const int nact = s.chunks(p.chunk);
  const int m = m0 + blockIdx.x * 8 + warp, t = m / G, head = kvh * G + m % G;
  if (nact <= 1 || t >= s.T) return;
  const long long row = s.row0 + t, pi = (row * p.n_heads + head) * p.max_chunks;
  float top = -INFINITY;
  for (int c = lane; c < nact; c += 32) top = fmaxf(top, p.part_ml[(pi + c) * 2]);
  top = warp_max(top);
  if (top == -INFINITY) top = 0.f;
  float total = 0.f, acc[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) acc[e] = 0.f;
  for (int c = 0; c < nact; ++c) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (pi + c) * 2);
    const float w = ex2((ml.x - top) * p.scale_log2);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // nothing seen in this chunk
    total = fmaf(w, ml.y, total);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e)
      acc[e] = fmaf(w, p.part_o[(pi + c) * HD + e * 32 + lane], acc[e]);
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e)
    store_out(p, row * p.ldout + (long long)head * HD + e * 32 + lane, acc[e] * inv);
}

// Keys per CTA: the largest chunk that still gives two CTAs per SM when every sequence is half of
// max_ctx long (no device data is read: captured graphs keep their shape).
static int chunk_keys(long long tiles_bh, int max_ctx) {
  const long long target = 2LL * num_sms();
  const int half = std::max(1, max_ctx / 2);
  for (int ch = kMaxChunk; ch > 128; ch >>= 1)
    if (tiles_bh * ((half + ch - 1) / ch) >= target) return ch;
  return 128;
}

struct Plan {
  int m_tiles, chunk, max_chunks;
  size_t off_ml, bytes;
};
static Plan plan_of(int batch, int rows, int n_heads, int n_kv, int head_dim, int max_q, int max_ctx) {
  Plan pl;
  const int G = n_heads / n_kv;
  pl.m_tiles = (int)(((long long)max_q * G + kRows - 1) / kRows);
  pl.chunk = chunk_keys((long long)batch * n_kv * pl.m_tiles, max_ctx);
  pl.max_chunks = (max_ctx + pl.chunk - 1) / pl.chunk;
  const size_t states = (size_t)rows * n_heads * pl.max_chunks;
  pl.off_ml = states * head_dim * sizeof(float);
  pl.bytes = pl.max_chunks > 1 ? pl.off_ml + states * 2 * sizeof(float) : 0;
  return pl;
}

}  // namespace tree
}  // namespace b2d

#include "tree_attn_t5.cuh"

namespace b2d {
namespace tree {

template <int HD, bool X2>
static int launch(const Params& p, int m_tiles, int batch, cudaStream_t stream) {
  auto kern = paged_tree_attn_kernel<HD, X2>;
  const int smem = Cfg<HD>::SMEM(X2);
  static std::atomic<unsigned long long> done;
  B2D_TRY(allow_smem(kern, smem, done));
  kern<<<dim3(p.max_chunks, m_tiles * p.n_kv, batch), kThreads, smem, stream>>>(p);
  B2D_TRY(launch_status());
  if (p.max_chunks > 1) {
    tree_join_kernel<HD><<<dim3(kRows / 8, m_tiles * p.n_kv, batch), 256, 0, stream>>>(p);
    B2D_TRY(launch_status());
  }
  return B2D_OK;
}

static bool shape_ok(int batch, int rows, int n_heads, int n_kv, int max_q, int max_ctx) {
  return batch > 0 && batch <= 65535 && rows > 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 &&
         n_heads / n_kv <= 64 && max_q > 0 && max_ctx > 0 && max_q <= max_ctx &&
         (((long long)max_q * (n_heads / n_kv) + kRows - 1) / kRows) * n_kv <= 65535;
}

}  // namespace tree

// The larger of the two operand forms' needs: the query does not know the types.
size_t paged_tree_attn_workspace_bytes(int batch, int rows, int n_heads, int n_kv_heads, int head_dim,
                                       int max_q, int max_ctx) {
  if (!tree::shape_ok(batch, rows, n_heads, n_kv_heads, max_q, max_ctx) || head_dim <= 0) return 0;
  if (head_dim == 256)
    return tree::plan_of(batch, rows, n_heads, n_kv_heads, head_dim, max_q, max_ctx).bytes;
  size_t need = 0;
  for (const bool x2 : {false, true}) {
    const tree::t5::Shape h = tree::t5::shape_of(batch, n_heads, n_kv_heads, head_dim, max_q, max_ctx, x2);
    if (h.max_steps < (1ll << 31)) need = std::max(need, h.bytes);
  }
  return need;
}

int paged_tree_attn(const void* q, int q_dtype, int ldq, const uint16_t* k_pages,
                    const uint16_t* v_pages, const int* block_table, int max_blocks, int n_blocks,
                    const int* ctx_lens, const int* cu_q, const uint32_t* mask, int mask_words,
                    const int* positions, int n_heads, int n_kv_heads, int head_dim, int batch,
                    int rows, int max_q, int max_ctx, float scale, int window, void* out,
                    int out_dtype, int ldout, void* workspace, size_t workspace_bytes,
                    cudaStream_t stream) {
  if (!q || !k_pages || !v_pages || !block_table || !ctx_lens || !cu_q || !out) return B2D_ERR_NULL;
  if (mask && window > 0 && !positions) return B2D_ERR_NULL;
  if (!tree::shape_ok(batch, rows, n_heads, n_kv_heads, max_q, max_ctx) || n_blocks <= 0 ||
      max_blocks <= 0 || (long long)max_blocks * 16 < max_ctx || window < 0)
    return B2D_ERR_SHAPE;
  if (mask ? (mask_words <= 0 || mask_words > tree::kMaxWords) : mask_words != 0) return B2D_ERR_SHAPE;
  const uint64_t prows = (uint64_t)n_blocks * n_kv_heads * 16;  // TMA coordinates are 32 bits
  if (prows > 0x7fffffffull) return B2D_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return B2D_ERR_UNSUPPORTED;
  if (q_dtype != B2D_F32 && q_dtype != B2D_F16) return B2D_ERR_UNSUPPORTED;
  if (out_dtype != B2D_F32 && out_dtype != B2D_F16 && out_dtype != B2D_F16X2) return B2D_ERR_UNSUPPORTED;
  if (ldq < n_heads * head_dim || ldout < n_heads * head_dim) return B2D_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      ldq % (q_dtype == B2D_F16 ? 8 : 4) || ldout % (out_dtype == B2D_F32 ? 4 : 8))
    return B2D_ERR_ALIGN;
  const bool x2 = q_dtype == B2D_F32 || out_dtype != B2D_F16;
  const tree::t5::Shape h = tree::t5::shape_of(batch, n_heads, n_kv_heads, head_dim, max_q, max_ctx, x2);
  if (head_dim != 256 && h.max_steps >= (1ll << 31)) return B2D_ERR_SHAPE;  // steps are counted in 32 bits
  const size_t need =
      paged_tree_attn_workspace_bytes(batch, rows, n_heads, n_kv_heads, head_dim, max_q, max_ctx);
  if (need && (!workspace || workspace_bytes < need)) return B2D_ERR_WORKSPACE;
  if (!aligned16(workspace)) return B2D_ERR_ALIGN;
  // rows of q are read while rows of out are written
  const int qe = q_dtype == B2D_F16 ? 2 : 4, oe = out_dtype == B2D_F32 ? 4 : 2;
  const long long width = (long long)n_heads * head_dim;
  if (rows_overlap(q, rows, (long long)ldq * qe, width * qe, out, out_dtype == B2D_F16X2 ? 2ll * rows : rows,
                   (long long)ldout * oe, width * oe))
    return B2D_ERR_UNSUPPORTED;
  tree::Params p = {};
  B2D_TRY(make_tmap_f16(&p.tmK, k_pages, prows, head_dim, head_dim, 16));
  p.q = q;
  p.q_f16 = q_dtype == B2D_F16;
  p.ldq = ldq;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.block_table = block_table;
  p.max_blocks = max_blocks;
  p.n_blocks = n_blocks;
  p.ctx_lens = ctx_lens;
  p.cu_q = cu_q;
  p.mask = mask;
  p.words = mask_words;
  p.positions = positions;
  p.n_heads = n_heads;
  p.n_kv = n_kv_heads;
  p.batch = batch;
  p.rows = rows;
  p.max_q = max_q;
  p.max_ctx = max_ctx;
  p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf((float)head_dim)) * 1.44269504088896340736f;
  p.window = window;
  p.out = out;
  p.out_f16 = out_dtype != B2D_F32;
  p.out_lo = out_dtype == B2D_F16X2 ? static_cast<uint16_t*>(out) + (size_t)rows * ldout : nullptr;
  p.ldout = ldout;
  p.part_o = static_cast<float*>(workspace);
  if (head_dim != 256) {
    B2D_TRY(make_tmap_f16_blocks(&p.tmV, v_pages, prows, head_dim, 16));
    const int G = n_heads / n_kv_heads;
    if (p.q_f16 && 128 % G == 0)
      B2D_TRY(make_tmap_f16_heads(&p.tmQ, q, rows, n_heads, head_dim, ldq, G, 128 / G));
    p.m_tiles = h.m_tiles;
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + h.off_ml);
    p.splits = reinterpret_cast<tree::Split*>(static_cast<char*>(workspace) + h.off_splits);
    if (head_dim == 64)
      return h.mt2 ? tree::t5::launch<64, true, false>(p, h, stream)
                   : (x2 ? tree::t5::launch<64, false, true>(p, h, stream)
                         : tree::t5::launch<64, false, false>(p, h, stream));
    return h.mt2 ? tree::t5::launch<128, true, false>(p, h, stream)
                 : (x2 ? tree::t5::launch<128, false, true>(p, h, stream)
                       : tree::t5::launch<128, false, false>(p, h, stream));
  }
  const tree::Plan pl = tree::plan_of(batch, rows, n_heads, n_kv_heads, head_dim, max_q, max_ctx);
  B2D_TRY(make_tmap_f16(&p.tmV, v_pages, prows, head_dim, head_dim, 16));
  p.m_tiles = pl.m_tiles;
  p.chunk = pl.chunk;
  p.max_chunks = pl.max_chunks;
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.off_ml);
  return x2 ? tree::launch<256, true>(p, pl.m_tiles, batch, stream)
            : tree::launch<256, false>(p, pl.m_tiles, batch, stream);
}

int paged_tree_attn_error() {
  int v = 0;
  const int zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, tree::g_error, sizeof(v));
  if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(tree::g_error, &zero, sizeof(zero));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return B2D_ERR_CUDA;
  }
  return v ? B2D_ERR_TIMEOUT : B2D_OK;
}

}  // namespace b2d
