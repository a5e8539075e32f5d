// Root-mean-square norm of query and key heads with the position rotation in
// the same pass:
//   u = x * rsqrt(mean(x^2) + eps) * w          (over the head's d columns)
//   (u_a, u_b) <- (u_a cos - u_b sin, u_a sin + u_b cos)
// for the pairs of the first `rot` columns: (2i, 2i+1) interleaved (as the
// encoder's own RoPE, ops_simd.go:127-137) or (i, i + rot/2) half-split.
// Everything is float32 between one load and one store of each value, so a
// result is rounded once.  Bound by memory: each head vector is read and
// written once, the cos / sin rows and weights stay in L1 and L2 (32767 tokens,
// 32 + 8 heads of 128, bf16: 114 us, 5.9 TB/s, 0.90 of a measured copy; 18431
// tokens, 12 + 12 heads of 64 in packed fp16 rows: 21 us, 5.3 TB/s).
#include "elem.cuh"
#include "kernels.h"

namespace le {
namespace qkn {

constexpr int THREADS = 64;

// Quotient of item (< 2^30) by n; inv = floor(2^32 / n) + 1 (the high product
// is exact or one too large).
__device__ __forceinline__ uint32_t div_by(uint32_t item, uint32_t n, uint32_t inv) {
  uint32_t q = n == 1 ? item : __umulhi(item, inv);
  if (q * n > item) q--;
  return q;
}

// G lanes per head vector, eight columns per lane; U heads of one token and
// one kind (query or key) per lane, so that the token's rotation and the
// kind's weights are loaded and multiplied once for them:
//   y_i = r (x_i A_i + x_p(i) B_i),  A = w_i cos, B = -+ w_p(i) sin
// with p(i) the other column of i's pair, in the same lane (interleaved) or
// rot/16 lanes away (half-split), whose loaded words are exchanged as they
// are.  d is a multiple of 8, rot of 16, rows 16-byte aligned.
// PART: some columns are not rotated.  Interleaved pairs then leave the other
// column out of theirs, whose infinity times 0 would be NaN where the formula has
// 0 (half-split, B is 0 and the other column the same one).
// ONCE: more bytes than the L2 holds, so nothing is kept there.
template <class T, int G, int U, bool HALF, bool PART, bool ONCE>
__global__ void __launch_bounds__(THREADS) qk_norm_vec_kernel(QkNormParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % G, c = lane * 8;
  const uint32_t item = blockIdx.x * (uint32_t)(THREADS / G) + threadIdx.x / G;
  const bool live = c < p.d && item < p.items;
  const uint32_t tok = div_by(item, p.chunks, p.inv_chunks), chunk = item - tok * p.chunks;
  const bool is_q = chunk < (uint32_t)p.q_chunks;
  const int h0 = (int)(is_q ? chunk : chunk - p.q_chunks) * U, heads = is_q ? p.q_heads : p.k_heads;
  const long row = p.token0 + (long)tok;
  const T* in = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.q_stride : p.k_stride) + (long)h0 * p.d + c;
  Raw8<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    raw[u] = zero8<T>();
    if (live && h0 + u < heads) raw[u] = ONCE ? load8_once(in + u * p.d) : load8(in + u * p.d);
  }
  const int pos = item >= p.items ? -1 : p.positions ? p.positions[row] : 0;
  const bool in_table = (unsigned)pos < (unsigned)p.max_pos;
  const int lanes = p.rot / 16;  // lanes of one half of the rotated columns
  const int partner = HALF ? (lane < lanes ? lane + lanes : lane < 2 * lanes ? lane - lanes : lane) : lane;

  float A[8], B[8];
  {
    const float* w = is_q ? p.q_weight : p.k_weight;
    float wo[8], wp[8];  // weights of the own columns and of their partners
#pragma unroll
    for (int i = 0; i < 8; i++) wo[i] = wp[i] = 1.f;
    if (w && live) {
      load_f32x8(w + c, wo);
      if (HALF)
        load_f32x8(w + partner * 8, wp);
      else
#pragma unroll
        for (int i = 0; i < 8; i++) wp[i] = wo[i ^ 1];
    }
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      cs[i] = 1.f;
      sn[i] = 0.f;
    }
    if (c < p.rot && in_table) {
      const long at = (long)pos * (p.rot / 2);
      if (HALF) {
        const int j = lane < lanes ? c : c - p.rot / 2;
        load_f32x8(p.cos + at + j, cs);
        load_f32x8(p.sin + at + j, sn);
#pragma unroll
        for (int i = 0; i < 8; i++) sn[i] = lane < lanes ? -sn[i] : sn[i];
      } else {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos + at + c / 2));
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin + at + c / 2));
        cs[0] = cs[1] = c4.x, cs[2] = cs[3] = c4.y, cs[4] = cs[5] = c4.z, cs[6] = cs[7] = c4.w;
        sn[1] = s4.x, sn[3] = s4.y, sn[5] = s4.z, sn[7] = s4.w;
#pragma unroll
        for (int i = 0; i < 8; i += 2) sn[i] = -sn[i + 1];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      A[i] = wo[i] * cs[i];
      B[i] = wp[i] * sn[i];
    }
  }
  T* out = static_cast<T*>(is_q ? p.q_out : p.k_out) + row * (is_q ? p.qo_stride : p.ko_stride) + (long)h0 * p.d + c;
#pragma unroll
  for (int u = 0; u < U; u++) {
    float v[8], o[8];
    values8(raw[u], v);
    if (HALF) {
      Raw8<T> other;
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) * 2); i++)
        reinterpret_cast<uint32_t*>(&other)[i] =
            __shfl_sync(0xffffffffu, reinterpret_cast<const uint32_t*>(&raw[u])[i], partner, G);
      values8(other, o);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = !PART || c < p.rot ? v[i ^ 1] : 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
#pragma unroll
    for (int s = G / 2; s > 0; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    const float r = rsqrtf(fmaf(ss, p.inv_d, p.eps));
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = r * fmaf(v[i], A[i], o[i] * B[i]);
    if (live && in_table && h0 + u < heads) {
      if constexpr (ONCE)
        store8_once(out + u * p.d, v);
      else
        store8(out + u * p.d, v);
    }
  }
  if (item < p.items && !in_table && lane == 0) report(p.status, DE_BOUNDS, 70, pos);
}

// Any head size up to MAX_D, rotation and alignment: one warp per head
// vector, staged through shared memory for the rotation's pairs.  Bound by
// instructions and latency, about the same for every head size (18431 tokens,
// 12 + 12 heads of 50, 64 or 80: 229 us; 22 for 64 aligned columns).
constexpr int MAX_D = 256;
template <class T>
__global__ void __launch_bounds__(THREADS) qk_norm_any_kernel(QkNormParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float buf[THREADS / 32][MAX_D];
  const int lane = threadIdx.x & 31;
  float* b = buf[threadIdx.x >> 5];
  const uint32_t item = blockIdx.x * (uint32_t)(THREADS / 32) + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const uint32_t token = div_by(item, p.chunks, p.inv_chunks), head = item - token * p.chunks;
  const bool is_q = head < (uint32_t)p.q_heads;
  const long row = p.token0 + (long)token, h = is_q ? head : head - p.q_heads;
  const T* in = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.q_stride : p.k_stride) + h * p.d;
  T* out = static_cast<T*>(is_q ? p.q_out : p.k_out) + row * (is_q ? p.qo_stride : p.ko_stride) + h * p.d;
  const float* w = is_q ? p.q_weight : p.k_weight;
  const int pos = p.positions ? p.positions[row] : 0;
  if ((unsigned)pos >= (unsigned)p.max_pos) {
    if (lane == 0) report(p.status, DE_BOUNDS, 71, pos);
    return;
  }
  float ss = 0.f;
  for (int i = lane; i < p.d; i += 32) {
    const float x = to_f32(in[i]);
    b[i] = x;
    ss = fmaf(x, x, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(fmaf(ss, p.inv_d, p.eps));
  for (int i = lane; i < p.d; i += 32) b[i] = b[i] * r * (w ? w[i] : 1.f);
  __syncwarp();
  const int half = p.rot / 2;
  for (int i = lane; i < half; i += 32) {
    const int ia = p.half_split ? i : 2 * i, ib = p.half_split ? i + half : 2 * i + 1;
    const float c = p.cos[(long)pos * half + i], s = p.sin[(long)pos * half + i], x = b[ia], y = b[ib];
    b[ia] = fmaf(x, c, -y * s);
    b[ib] = fmaf(x, s, y * c);
  }
  __syncwarp();
  for (int i = lane; i < p.d; i += 32) out[i] = from_f32<T>(b[i]);
}

// cos and sin of pos * base^(-2i/rot), computed in 64 bits and rounded once:
// float32 angles lose 1e-3 of a turn by position 65536.
__global__ void rope_table_kernel(int max_pos, int half, int rot, double base, float* c, float* s) {
  const long n = (long)max_pos * half;
  for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
    const double a = (double)(i / half) * pow(base, -2.0 * (double)(i % half) / (double)rot);
    double sn, cs;
    sincos(a, &sn, &cs);
    c[i] = (float)cs;
    s[i] = (float)sn;
  }
}

// Sets the launch's items: chunks of U heads of each token.
static unsigned set_items(QkNormParams& p, int n_tokens, int U, int per_block) {
  p.q_chunks = (p.q_heads + U - 1) / U;
  p.chunks = p.q_chunks + (p.k_heads + U - 1) / U;
  p.inv_chunks = p.chunks == 1 ? 0 : (uint32_t)((1ull << 32) / p.chunks) + 1;
  p.items = (uint32_t)n_tokens * p.chunks;
  return (p.items + per_block - 1) / per_block;
}

template <class T, int G, int U, bool ONCE = false>
static cudaError_t launch_vec(QkNormParams p, int n, cudaStream_t s) {
  const unsigned blocks = set_items(p, n, U, THREADS / G);
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3(blocks), dim3(THREADS), 0, s, attr);
  // The choice between the interleaved ones costs 3% (18431 tokens, 12 + 12 heads
  // of 64, fp16: 20.0 and 20.6 us).
  return p.half_split  ? cudaLaunchKernelEx(&cfg, qk_norm_vec_kernel<T, G, U, true, false, ONCE>, p)
         : p.rot < p.d ? cudaLaunchKernelEx(&cfg, qk_norm_vec_kernel<T, G, U, false, true, ONCE>, p)
                       : cudaLaunchKernelEx(&cfg, qk_norm_vec_kernel<T, G, U, false, false, ONCE>, p);
}

template <class T, int G>
static cudaError_t launch_g(const QkNormParams& p, int n, cudaStream_t s) {
  // Four heads per lane once that still gives every one of the 148 SMs sixteen
  // blocks of them; eight of the 2-byte types where both kinds come in eights
  // (32 + 8 heads of 128, bf16: 132 -> 121 us; 12 + 12 heads of 64 padded to 16:
  // 22.7 -> 26.4 us), past the L2's 126 MB with loads and stores that are not
  // kept there (121 -> 114 us).  Four a lane keeps them: 24 + 6 heads of 128 in
  // 94 us, 5.4 TB/s; float32, 32 + 8 heads, 210 us, 6.4 TB/s.
  const long vectors = (long)n * (p.q_heads + p.k_heads);
  if (vectors < 148L * 16 * 4 * (THREADS / G)) return launch_vec<T, G, 1>(p, n, s);
  if constexpr (sizeof(T) == 2)
    if (p.q_heads % 8 == 0 && p.k_heads % 8 == 0)
      return 4 * vectors * p.d > 126L << 20 ? launch_vec<T, G, 8, true>(p, n, s) : launch_vec<T, G, 8>(p, n, s);
  return launch_vec<T, G, 4>(p, n, s);
}

template <class T>
static cudaError_t launch(QkNormParams p, int n, cudaStream_t s) {
  auto al = [](const void* q, long stride) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (stride * (long)sizeof(T)) % 16 == 0;
  };
  const bool vec = p.d % 8 == 0 && p.rot % 16 == 0 &&
                   (p.q_heads == 0 || (al(p.q, p.q_stride) && al(p.q_out, p.qo_stride))) &&
                   (p.k_heads == 0 || (al(p.k, p.k_stride) && al(p.k_out, p.ko_stride))) &&
                   reinterpret_cast<uintptr_t>(p.q_weight) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.k_weight) % 16 == 0;
  if (!vec) {
    const unsigned blocks = set_items(p, n, 1, THREADS / 32);
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3(blocks), dim3(THREADS), 0, s, attr);
    return cudaLaunchKernelEx(&cfg, qk_norm_any_kernel<T>, p);
  }
  if (p.d <= 32) return launch_g<T, 4>(p, n, s);
  if (p.d <= 64) return launch_g<T, 8>(p, n, s);
  if (p.d <= 128) return launch_g<T, 16>(p, n, s);
  return launch_g<T, 32>(p, n, s);
}

}  // namespace qkn

cudaError_t launch_rope_table(int max_pos, int rot, double base, float* cos, float* sin, cudaStream_t s) {
  if (rot == 0) return cudaSuccess;
  qkn::rope_table_kernel<<<296, 256, 0, s>>>(max_pos, rot / 2, rot, base, cos, sin);
  return cudaGetLastError();
}

cudaError_t launch_qk_norm(int dt, QkNormParams p, int n_tokens, cudaStream_t s) {
  const int H = p.q_heads + p.k_heads;
  if (n_tokens == 0 || H == 0) return cudaSuccess;
  p.inv_d = 1.f / (float)p.d;
  // Vectors are numbered in 32 bits within a launch.
  const int step = (1 << 30) / H;
  for (int t0 = 0; t0 < n_tokens; t0 += step) {
    const int n = n_tokens - t0 < step ? n_tokens - t0 : step;
    p.token0 = t0;
    const cudaError_t e = dt == DT_F32   ? qkn::launch<float>(p, n, s)
                          : dt == DT_F16 ? qkn::launch<__half>(p, n, s)
                                         : qkn::launch<__nv_bfloat16>(p, n, s);
    if (e != cudaSuccess) return e;
    if (n_tokens - t0 <= step) break;
  }
  return cudaSuccess;
}

}  // namespace le
