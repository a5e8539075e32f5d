// Eight-bit product for few tokens (mma.sync m16n8k32 e4m3, sm_100a):
//   y[m][n] = sum_b xs[b][m] ws[n/128][b] sum_{k in block b} xq[m][k] wq[n][k]
// with the activations quantised on the fly (f8.cuh), so a call is one launch
// and reads each weight byte once.  Bound by the weight's bytes, or by latency
// when those are few.
//
// A CTA computes 16 weight rows x 8*NT tokens; its eight warps take the K
// blocks in turn, each keeping its own float32 sums, which are added in warp
// order at the end.  The weight rows are the MMA's 16 rows and the tokens its
// eight columns.  A sum over k does not depend on the order of k, so a lane
// takes 16 consecutive bytes of a row, the same for weights and activations,
// as two instructions' fragments: wide loads and no shuffles.  The four lanes
// that hold a token's 128 columns of a block find its scale with two
// shuffles.
#include "f8.cuh"
#include "kernels.h"

namespace le {
namespace f8s {

using namespace f8;

constexpr int WARPS = 8;
constexpr int ROWS = 16;  // weight rows per CTA

struct E4m3 {};  // activations that are quantised already

__device__ __forceinline__ void mma_e4m3(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ldw(const uint8_t* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

// This lane's 32 activations of block kb of token m, as fragments, and the
// block's scale.  Columns from K on are zero.
template <class X>
__device__ __forceinline__ float act_frag(const F8GemmParams& p, int m, int kb, int t, uint32_t (&b)[8]) {
  const int k0 = kb * BLOCK + 16 * t;
  const bool row = m < p.M;
  if constexpr (sizeof(X) == 1) {
    const uint8_t* x = static_cast<const uint8_t*>(p.x) + (long)m * p.ldx;
#pragma unroll
    for (int c = 0; c < 2; c++) *reinterpret_cast<uint4*>(b + 4 * c) = ldw(x + k0 + 64 * c, row && k0 + 64 * c < p.K);
    return row ? __ldg(p.xs + (long)kb * p.M + m) : 0.f;
  } else {
    const X* x = static_cast<const X*>(p.x) + (long)m * p.ldx;
    Raw8<X> raw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int k = k0 + 64 * (i >> 1) + 8 * (i & 1);
      raw[i] = row && k < p.K ? load8(x + k) : zero8<X>();
    }
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float v[8];
      values8(raw[i], v);
#pragma unroll
      for (int j = 0; j < 8; j++) a = max(a, abs_bits(v[j]));
    }
    a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
    float inv;
    const float s = block_scale(a, &inv);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float v[8];
      values8(raw[i], v);
      b[2 * i] = pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      b[2 * i + 1] = pack_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    }
    return s;
  }
}

template <class X, class Y, int NT>
__global__ void __launch_bounds__(WARPS * 32) f8_small_kernel(F8GemmParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[WARPS][NT * 8][ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * ROWS, m0 = blockIdx.y * (8 * NT);
  const int KB = (p.K + BLOCK - 1) / BLOCK;
  const float* ws = p.ws + (long)(n0 / BLOCK) * KB;
  const uint8_t* wa = p.w + (long)(n0 + g) * p.K;
  const uint8_t* wb = wa + 8L * p.K;
  const bool ra = n0 + g < p.N, rb = n0 + g + 8 < p.N;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 2
  for (int kb = warp; kb < KB; kb += WARPS) {
    uint4 a[2], b[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = kb * BLOCK + 64 * c + 16 * t;
      a[c] = ldw(wa + k, ra && k < p.K);
      b[c] = ldw(wb + k, rb && k < p.K);
    }
    const float wsc = __ldg(ws + kb);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      uint32_t f[8];
      const float xs = act_frag<X>(p, m0 + 8 * j + g, kb, t, f);
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; c++) {
        mma_e4m3(d, a[c].x, b[c].x, a[c].y, b[c].y, f[4 * c], f[4 * c + 1]);
        mma_e4m3(d, a[c].z, b[c].z, a[c].w, b[c].w, f[4 * c + 2], f[4 * c + 3]);
      }
      // Columns 2t and 2t + 1 of the result: the scales of those tokens.
      const float s0 = __shfl_sync(0xffffffffu, xs, 8 * t) * wsc, s1 = __shfl_sync(0xffffffffu, xs, 8 * t + 4) * wsc;
      acc[j][0] = fmaf(d[0], s0, acc[j][0]);
      acc[j][1] = fmaf(d[1], s1, acc[j][1]);
      acc[j][2] = fmaf(d[2], s0, acc[j][2]);
      acc[j][3] = fmaf(d[3], s1, acc[j][3]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; j++) {
    red[warp][8 * j + 2 * t][g] = acc[j][0];
    red[warp][8 * j + 2 * t + 1][g] = acc[j][1];
    red[warp][8 * j + 2 * t][g + 8] = acc[j][2];
    red[warp][8 * j + 2 * t + 1][g + 8] = acc[j][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * ROWS; i += WARPS * 32) {
    const int m = i / ROWS, n = i % ROWS;
    float v = red[0][m][n];
#pragma unroll
    for (int w = 1; w < WARPS; w++) v += red[w][m][n];
    if (m0 + m < p.M && n0 + n < p.N) static_cast<Y*>(p.y)[(long)(m0 + m) * p.ldy + n0 + n] = from_f32<Y>(v);
  }
}

template <class X, class Y, int NT>
static cudaError_t launch_nt(const F8GemmParams& p, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3((p.N + ROWS - 1) / ROWS, (p.M + 8 * NT - 1) / (8 * NT)),
                                            dim3(WARPS * 32), 0, s, attr);
  return cudaLaunchKernelEx(&cfg, f8_small_kernel<X, Y, NT>, p);
}
template <class X, class Y>
static cudaError_t launch_xy(const F8GemmParams& p, cudaStream_t s) {
  if (p.M <= 8) return launch_nt<X, Y, 1>(p, s);
  if (p.M <= 16) return launch_nt<X, Y, 2>(p, s);
  return launch_nt<X, Y, 4>(p, s);
}
template <class X>
static cudaError_t launch_x(int ydt, const F8GemmParams& p, cudaStream_t s) {
  return ydt == DT_F32   ? launch_xy<X, float>(p, s)
         : ydt == DT_F16 ? launch_xy<X, __half>(p, s)
                         : launch_xy<X, __nv_bfloat16>(p, s);
}

}  // namespace f8s

cudaError_t launch_f8_gemm_small(int xdt, int ydt, const F8GemmParams& p, cudaStream_t s) {
  if (p.M == 0) return cudaSuccess;
  switch (xdt) {
    case DT_F32: return f8s::launch_x<float>(ydt, p, s);
    case DT_F16: return f8s::launch_x<__half>(ydt, p, s);
    case DT_BF16: return f8s::launch_x<__nv_bfloat16>(ydt, p, s);
    default: return f8s::launch_x<f8s::E4m3>(ydt, p, s);
  }
}

}  // namespace le
