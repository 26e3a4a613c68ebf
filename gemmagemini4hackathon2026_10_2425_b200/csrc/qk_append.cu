// Per-head norms of queries and keys, the position rotation and the paged append, in one pass
// over the QKV projection's rows (any number of rows per sequence).
//
// Reference: qkv_norm_rope (GK/kernels.metal:246-304: RMS of q and k per head with a weight, of v
// without one, rotation, cache write) and rope_kv (LK/kernels.metal:182-224); the decode step's
// own rope_kv_append covers one row per sequence without norms.
//
//   r = rsqrt(mean_i x_i^2 + eps),  y_i = x_i r gamma_i,
//   (y_i, y_{i + HD/2}) <- (y_i cos a_i - y_{i+HD/2} sin a_i, y_{i+HD/2} cos a_i + y_i sin a_i),
//   a_i = pos * inv_freq_i.
//
// The angle is formed in double: pos * inv_freq in fp32 is off by half a step of a number as
// large as pos (2^-7 rad at 131072), which is far more than fp16 keeps of a sine.  In double the
// product is exact for every position below 2^24, and what is left after taking whole turns out
// fits the fp32 sine's short-range path.  HD/2 angles per row serve all its heads.
//
// What bounds it: memory (each value read once and written once, ~20 flops per value).  One CTA
// per row; a head is spread over HD/8 lanes, each holding 4 values of the lower half and the 4
// they rotate with, so a row's loads are 16 bytes (fp32) or 8 bytes (fp16) wide, all issued
// before the angles are computed, and the norm is a shuffle within the head's lanes.
#include "common.cuh"

namespace b2d {

namespace qka {

constexpr int kThreads = 128;
constexpr int kRounds = 3;  // heads per lane in flight

struct Params {
  const void* qkv;
  long long ldqkv;
  const float* q_gamma;
  const float* k_gamma;
  float eps;
  int v_norm;
  const int* positions;
  const long long* slots;
  const int* n_rows;
  const float* inv_freq;
  void* q_out;
  long long ldq;
  uint16_t* k_pages;
  uint16_t* v_pages;
  long long n_slots;
  int n_heads, n_kv;
  int rows;
};

template <bool F16>
__device__ __forceinline__ float4 load4(const void* p, long long i) {
  if constexpr (F16) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    const float2 a = h2f2(u.x), b = h2f2(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  }
}

__device__ __forceinline__ uint2 pack4(float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <bool F16>
__device__ __forceinline__ void store4(void* p, long long i, float4 v) {
  if constexpr (F16)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = pack4(v);
  else
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
}

// cos and sin of pos * f (see the head of the file).
__device__ __forceinline__ float2 turn(int pos, float f) {
  constexpr double kTwoPi = 6.283185307179586476925;
  const double a = (double)pos * (double)f;
  const double r = fma(-rint(a * (1.0 / kTwoPi)), kTwoPi, a);
  float s, c;
  sincosf((float)r, &s, &c);
  return make_float2(c, s);
}

// XF16: qkv is fp16; QF16: q_out is fp16
template <int HD, bool XF16, bool QF16>
__global__ void __launch_bounds__(kThreads, 8) qk_norm_rope_append_kernel(const Params p) {
  constexpr int L = HD / 8;             // lanes per head
  constexpr int SLOTS = kThreads / L;   // heads in flight per CTA
  __shared__ __align__(16) float2 cs[HD / 2];
  const int row = blockIdx.x;
  if (p.n_rows && row >= *p.n_rows) return;  // padding behind the last request: left as it is
  const int pos = p.positions[row];
  if (pos < 0) return;
  const long long slot = p.slots ? p.slots[row] : -1;
  const int tid = threadIdx.x, li = tid % L, h0 = tid / L;
  const int heads = p.n_heads + 2 * p.n_kv;
  const long long x0 = (long long)row * p.ldqkv + 4 * li;
  const bool put = slot >= 0 && slot < p.n_slots;
  // heads are walked in whole rounds so that every lane of a warp takes part in the shuffles, the
  // loads of kRounds rounds first of all (before the angles the first time)
  for (int hb = 0; hb < heads; hb += kRounds * SLOTS) {
    float4 va[kRounds], vb[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int h = hb + j * SLOTS + h0;
      va[j] = vb[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (h < heads) {
        va[j] = load4<XF16>(p.qkv, x0 + (long long)h * HD);
        vb[j] = load4<XF16>(p.qkv, x0 + (long long)h * HD + HD / 2);
      }
    }
    if (hb == 0) {
      if (tid < HD / 2) cs[tid] = turn(pos, p.inv_freq[tid]);
      __syncthreads();
    }
    const float4 ca = *reinterpret_cast<const float4*>(&cs[4 * li]);      // c0 s0 c1 s1
    const float4 cb = *reinterpret_cast<const float4*>(&cs[4 * li + 2]);  // c2 s2 c3 s3
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int h = hb + j * SLOTS + h0;
      if (hb + j * SLOTS >= heads) break;
      float4 a = va[j], b = vb[j];
      const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv;
      const float* gamma = is_q ? p.q_gamma : (is_k ? p.k_gamma : nullptr);
      float ss = a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w + b.x * b.x + b.y * b.y + b.z * b.z +
                 b.w * b.w;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (h >= heads) continue;
      if (gamma || (!is_q && !is_k && p.v_norm)) {
        const float r = rsqrtf(ss * (1.0f / HD) + p.eps);
        float4 ga = make_float4(1.f, 1.f, 1.f, 1.f), gb = ga;
        if (gamma) {
          ga = *reinterpret_cast<const float4*>(gamma + 4 * li);
          gb = *reinterpret_cast<const float4*>(gamma + HD / 2 + 4 * li);
        }
        a = make_float4(a.x * r * ga.x, a.y * r * ga.y, a.z * r * ga.z, a.w * r * ga.w);
        b = make_float4(b.x * r * gb.x, b.y * r * gb.y, b.z * r * gb.z, b.w * r * gb.w);
      }
      if (is_q || is_k) {
        const float4 u = a;
        a = make_float4(u.x * ca.x - b.x * ca.y, u.y * ca.z - b.y * ca.w, u.z * cb.x - b.z * cb.y,
                        u.w * cb.z - b.w * cb.w);
        b = make_float4(b.x * ca.x + u.x * ca.y, b.y * ca.z + u.y * ca.w, b.z * cb.x + u.z * cb.y,
                        b.w * cb.z + u.w * cb.w);
      }
      if (is_q) {
        const long long o = (long long)row * p.ldq + (long long)h * HD + 4 * li;
        store4<QF16>(p.q_out, o, a);
        store4<QF16>(p.q_out, o + HD / 2, b);
      } else if (put) {
        const int kvh = is_k ? h - p.n_heads : h - p.n_heads - p.n_kv;
        uint16_t* pages = is_k ? p.k_pages : p.v_pages;
        const long long o = ((slot / 16 * p.n_kv + kvh) * 16 + slot % 16) * HD + 4 * li;
        *reinterpret_cast<uint2*>(pages + o) = pack4(a);
        *reinterpret_cast<uint2*>(pages + o + HD / 2) = pack4(b);
      }
    }
  }
}

template <int HD>
static int launch(const Params& p, bool x16, bool q16, cudaStream_t stream) {
  auto kern = x16 ? (q16 ? qk_norm_rope_append_kernel<HD, true, true>
                         : qk_norm_rope_append_kernel<HD, true, false>)
                  : (q16 ? qk_norm_rope_append_kernel<HD, false, true>
                         : qk_norm_rope_append_kernel<HD, false, false>);
  kern<<<p.rows, kThreads, 0, stream>>>(p);
  return launch_status();
}

}  // namespace qka

int qk_norm_rope_append(const void* qkv, int qkv_dtype, int ldqkv, const float* q_gamma,
                        const float* k_gamma, float eps, int v_norm, const int* positions,
                        const long long* slots, const int* n_rows, const float* inv_freq,
                        void* q_out, int q_dtype, int ldq, uint16_t* k_pages, uint16_t* v_pages,
                        int n_blocks, int n_heads, int n_kv_heads, int head_dim, int rows,
                        cudaStream_t stream) {
  if (!qkv || !positions || !inv_freq || !q_out) return B2D_ERR_NULL;
  if (slots && (!k_pages || !v_pages)) return B2D_ERR_NULL;
  if (rows <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads > 4096 || n_kv_heads > 4096 ||
      (slots && n_blocks <= 0))
    return B2D_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return B2D_ERR_UNSUPPORTED;
  if ((qkv_dtype != B2D_F32 && qkv_dtype != B2D_F16) || (q_dtype != B2D_F32 && q_dtype != B2D_F16))
    return B2D_ERR_UNSUPPORTED;
  if (ldqkv < (n_heads + 2 * n_kv_heads) * head_dim || ldq < n_heads * head_dim) return B2D_ERR_SHAPE;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(q_gamma) || !aligned16(k_gamma) || ldqkv % (qkv_dtype == B2D_F16 ? 8 : 4) ||
      ldq % (q_dtype == B2D_F16 ? 8 : 4))
    return B2D_ERR_ALIGN;
  // a value may be written where it was read (in place), but nowhere else in qkv: other lanes and
  // rows read there at the same time
  const int xe = qkv_dtype == B2D_F16 ? 2 : 4, oe = q_dtype == B2D_F16 ? 2 : 4;
  const bool in_place = q_out == qkv && q_dtype == qkv_dtype && (ldq == ldqkv || rows == 1);
  if (!in_place && rows_overlap(qkv, rows, (long long)ldqkv * xe, (long long)(n_heads + 2 * n_kv_heads) * head_dim * xe,
                                q_out, rows, (long long)ldq * oe, (long long)n_heads * head_dim * oe))
    return B2D_ERR_UNSUPPORTED;
  const qka::Params p = {qkv,      ldqkv,   q_gamma,  k_gamma, eps,
                         v_norm,   positions, slots,  n_rows,  inv_freq,
                         q_out,    ldq,     k_pages,  v_pages, (long long)n_blocks * 16,
                         n_heads,  n_kv_heads, rows};
  const bool x16 = qkv_dtype == B2D_F16, q16 = q_dtype == B2D_F16;
  switch (head_dim) {
    case 64: return qka::launch<64>(p, x16, q16, stream);
    case 128: return qka::launch<128>(p, x16, q16, stream);
    default: return qka::launch<256>(p, x16, q16, stream);
  }
}

}  // namespace b2d
