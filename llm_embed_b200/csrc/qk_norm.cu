// Root-mean-square norm of query and key heads with the position rotation in
// the same pass:
//   u = x * rsqrt(mean(x^2) + eps) * w          (over the head's d columns)
//   (u_a, u_b) <- (u_a cos - u_b sin, u_a sin + u_b cos)
// for the pairs of the first `rot` columns: (2i, 2i+1) interleaved (as the
// encoder's own RoPE, ops_simd.go:127-137) or (i, i + rot/2) half-split.
// Everything is float32 between one load and one store of each value, so a
// result is rounded once.  Bound by memory: each head vector is read and
// written once; the cos / sin rows and weights stay in L1 and L2.
#include "elem.cuh"
#include "kernels.h"

namespace le {
namespace qkn {

constexpr int THREADS = 256;

// Token of `item` among vectors of H heads per token; inv = floor(2^32 / H) + 1
// (the quotient from the high product is exact or one too large).
__device__ __forceinline__ uint32_t div_heads(uint32_t item, uint32_t H, uint32_t inv) {
  uint32_t q = H == 1 ? item : __umulhi(item, inv);
  if (q * H > item) q--;
  return q;
}

// A head vector's place: pointers to the input and output rows, its weight.
template <class T>
struct Vec {
  const T* in;
  T* out;
  const float* w;
};
template <class T>
__device__ __forceinline__ Vec<T> locate(const QkNormParams& p, uint32_t token, uint32_t head) {
  const bool is_q = head < (uint32_t)p.q_heads;
  const uint32_t h = is_q ? head : head - p.q_heads;
  const long row = (long)(p.token0 + token);
  Vec<T> v;
  v.in = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.q_stride : p.k_stride) + (long)h * p.d;
  v.out = static_cast<T*>(is_q ? p.q_out : p.k_out) + row * (is_q ? p.qo_stride : p.ko_stride) + (long)h * p.d;
  v.w = is_q ? p.q_weight : p.k_weight;
  return v;
}

// G lanes per head vector, eight columns per lane; U vectors per lane in
// flight.  d is a multiple of 8, rot of 16, rows 16-byte aligned.
template <class T, int G, int U, bool HALF>
__global__ void __launch_bounds__(THREADS) qk_norm_vec_kernel(QkNormParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int PER = THREADS / G;  // vectors per block and step
  const int lane = threadIdx.x % G, c = lane * 8;
  const bool live = c < p.d;
  const uint32_t H = p.q_heads + p.k_heads;
  const uint32_t item0 = blockIdx.x * (uint32_t)(PER * U) + threadIdx.x / G;
  Raw8<T> raw[U];
  uint32_t tok[U], head[U];
  int pos[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t item = item0 + u * PER;
    tok[u] = div_heads(item, H, p.inv_heads);
    head[u] = item - tok[u] * H;
    raw[u] = zero8<T>();
    pos[u] = -1;
    if (item < p.items) {
      if (live) raw[u] = load8(locate<T>(p, tok[u], head[u]).in + c);
      pos[u] = p.positions ? p.positions[p.token0 + tok[u]] : 0;
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    float v[8];
    values8(raw[u], v);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss / (float)p.d + p.eps);
    const Vec<T> at = locate<T>(p, tok[u], head[u]);
    const bool here = item0 + u * PER < p.items;
    const bool in_table = (unsigned)pos[u] < (unsigned)p.max_pos;
    if (at.w && live) {
      const float4 w0 = __ldg(reinterpret_cast<const float4*>(at.w + c));
      const float4 w1 = __ldg(reinterpret_cast<const float4*>(at.w + c) + 1);
      const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = v[i] * r * w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= r;
    }
    if constexpr (HALF) {
      const int lanes = p.rot / 16;  // lanes of one half
      const int partner = lane < lanes ? lane + lanes : lane - lanes;
      float other[8];
#pragma unroll
      for (int i = 0; i < 8; i++) other[i] = __shfl_sync(0xffffffffu, v[i], partner, G);
      if (c < p.rot && in_table) {
        const long row = (long)pos[u] * (p.rot / 2) + (lane < lanes ? c : c - p.rot / 2);
        const float4* cp = reinterpret_cast<const float4*>(p.cos + row);
        const float4* sp = reinterpret_cast<const float4*>(p.sin + row);
        const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
        const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
        const float sg = lane < lanes ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fmaf(v[i], cs[i], sg * other[i] * sn[i]);
      }
    } else if (c < p.rot && in_table) {
      const long row = (long)pos[u] * (p.rot / 2) + c / 2;
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos + row));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin + row));
      const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = v[2 * i], b = v[2 * i + 1];
        v[2 * i] = fmaf(a, cs[i], -b * sn[i]);
        v[2 * i + 1] = fmaf(a, sn[i], b * cs[i]);
      }
    }
    if (here) {
      if (!in_table) {
        if (lane == 0) report(p.status, DE_BOUNDS, 70, pos[u]);
      } else if (live) {
        store8(at.out + c, v);
      }
    }
  }
}

// Any head size up to MAX_D, rotation and alignment: one warp per head
// vector, staged through shared memory for the rotation's pairs.
constexpr int MAX_D = 256;
template <class T>
__global__ void __launch_bounds__(THREADS) qk_norm_any_kernel(QkNormParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float buf[THREADS / 32][MAX_D];
  const int lane = threadIdx.x & 31;
  float* b = buf[threadIdx.x >> 5];
  const uint32_t H = p.q_heads + p.k_heads;
  const uint32_t item = blockIdx.x * (uint32_t)(THREADS / 32) + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const uint32_t token = div_heads(item, H, p.inv_heads), head = item - token * H;
  const Vec<T> at = locate<T>(p, token, head);
  const int pos = p.positions ? p.positions[p.token0 + token] : 0;
  if ((unsigned)pos >= (unsigned)p.max_pos) {
    if (lane == 0) report(p.status, DE_BOUNDS, 71, pos);
    return;
  }
  float ss = 0.f;
  for (int i = lane; i < p.d; i += 32) {
    const float x = to_f32(at.in[i]);
    b[i] = x;
    ss = fmaf(x, x, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / (float)p.d + p.eps);
  for (int i = lane; i < p.d; i += 32) b[i] = b[i] * r * (at.w ? at.w[i] : 1.f);
  __syncwarp();
  const int half = p.rot / 2;
  for (int i = lane; i < half; i += 32) {
    const int ia = p.half_split ? i : 2 * i, ib = p.half_split ? i + half : 2 * i + 1;
    const float c = p.cos[(long)pos * half + i], s = p.sin[(long)pos * half + i], x = b[ia], y = b[ib];
    b[ia] = fmaf(x, c, -y * s);
    b[ib] = fmaf(x, s, y * c);
  }
  __syncwarp();
  for (int i = lane; i < p.d; i += 32) at.out[i] = from_f32<T>(b[i]);
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

template <class T, int G, int U>
static cudaError_t launch_vec(const QkNormParams& p, cudaStream_t s) {
  constexpr uint32_t per = THREADS / G * U;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3((p.items + per - 1) / per), dim3(THREADS), 0, s, attr);
  return p.half_split ? cudaLaunchKernelEx(&cfg, qk_norm_vec_kernel<T, G, U, true>, p)
                      : cudaLaunchKernelEx(&cfg, qk_norm_vec_kernel<T, G, U, false>, p);
}

template <class T, int G>
static cudaError_t launch_g(const QkNormParams& p, cudaStream_t s) {
  // Four vectors in flight per lane once that still fills the GPU's 148 SMs
  // with blocks.
  return p.items >= 148u * 4 * 4 * (THREADS / G) ? launch_vec<T, G, 4>(p, s) : launch_vec<T, G, 1>(p, s);
}

template <class T>
static cudaError_t launch(const QkNormParams& p, cudaStream_t s) {
  auto al = [](const void* q, long stride) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (stride * (long)sizeof(T)) % 16 == 0;
  };
  const bool vec = p.d % 8 == 0 && p.rot % 16 == 0 && (p.d * sizeof(T)) % 16 == 0 &&
                   (p.q_heads == 0 || (al(p.q, p.q_stride) && al(p.q_out, p.qo_stride))) &&
                   (p.k_heads == 0 || (al(p.k, p.k_stride) && al(p.k_out, p.ko_stride))) &&
                   reinterpret_cast<uintptr_t>(p.q_weight) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.k_weight) % 16 == 0;
  if (!vec) {
    constexpr uint32_t per = THREADS / 32;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3((p.items + per - 1) / per), dim3(THREADS), 0, s, attr);
    return cudaLaunchKernelEx(&cfg, qk_norm_any_kernel<T>, p);
  }
  if (p.d <= 32) return launch_g<T, 4>(p, s);
  if (p.d <= 64) return launch_g<T, 8>(p, s);
  if (p.d <= 128) return launch_g<T, 16>(p, s);
  return launch_g<T, 32>(p, s);
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
  p.inv_heads = H == 1 ? 0 : (uint32_t)((1ull << 32) / (uint32_t)H) + 1;
  // Vectors are numbered in 32 bits within a launch.
  const int step = (1 << 30) / H;
  for (int t0 = 0; t0 < n_tokens; t0 += step) {
    const int n = n_tokens - t0 < step ? n_tokens - t0 : step;
    p.token0 = t0;
    p.items = (uint32_t)n * (uint32_t)H;
    const cudaError_t e = dt == DT_F32   ? qkn::launch<float>(p, s)
                          : dt == DT_F16 ? qkn::launch<__half>(p, s)
                                         : qkn::launch<__nv_bfloat16>(p, s);
    if (e != cudaSuccess) return e;
    if (n_tokens - t0 <= step) break;
  }
  return cudaSuccess;
}

}  // namespace le
