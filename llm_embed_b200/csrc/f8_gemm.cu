// Eight-bit product for few tokens (mma.sync m16n8k32 e4m3, sm_100a):
//   y[m][n] = sum_b xs[b][m] ws[n/128][b] sum_{k in block b} xq[m][k] wq[n][k]
// with the activations of up to 8 rows quantised on the fly (f8.cuh), so that
// such a call is one launch; each weight byte is read once.  Bound by the weight's bytes, or by latency
// when those are few (1 x 768 . 2304: 1.8 us; 24 x 4096 . 4096: 6.5 us, 2.6 TB/s
// of weight, behind a quantiser of 1.5 us).
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

constexpr int ROWS = 16;  // weight rows per CTA
constexpr int WARPS = 8;

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

// This lane's 32 activations of block kb of token m as they lie in memory
// (zero from column K and row M on), and as fragments with the block's scale.
template <class X>
struct Act {
  Raw8<X> raw[4];
  __device__ __forceinline__ void load(const F8GemmParams& p, int m, int kb, int t) {
    const X* x = static_cast<const X*>(p.x) + (long)m * p.ldx;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int k = kb * BLOCK + 16 * t + 64 * (i >> 1) + 8 * (i & 1);
      raw[i] = m < p.M && k < p.K ? load8(x + k) : zero8<X>();
    }
  }
  __device__ __forceinline__ float frag(uint32_t (&b)[8]) const {
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
};
template <>
struct Act<E4m3> {
  uint4 raw[2];
  float scale;
  __device__ __forceinline__ void load(const F8GemmParams& p, int m, int kb, int t) {
    const uint8_t* x = static_cast<const uint8_t*>(p.x) + (long)m * p.ldx;
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = kb * BLOCK + 16 * t + 64 * c;
      raw[c] = m < p.M && k < p.K ? *reinterpret_cast<const uint4*>(x + k) : make_uint4(0, 0, 0, 0);
    }
    scale = m < p.M && kb * BLOCK < p.K ? p.xs[(long)kb * p.M + m] : 0.f;
  }
  __device__ __forceinline__ float frag(uint32_t (&b)[8]) const {
#pragma unroll
    for (int c = 0; c < 2; c++) *reinterpret_cast<uint4*>(b + 4 * c) = raw[c];
    return scale;
  }
};

// NT groups of eight tokens.
template <class X, class Y, int NT>
__global__ void __launch_bounds__(WARPS * 32, 2) f8_small_kernel(F8GemmParams p) {
  __shared__ float red[WARPS][NT * 8][ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * ROWS, m0 = blockIdx.y * (8 * NT);
  const int KB = (p.K + BLOCK - 1) / BLOCK;
  const float* ws = p.ws + (long)(n0 / BLOCK) * KB;
  const uint8_t* wrow = p.w + (long)(n0 + g) * p.K;
  uint4 w[2][2];
  float wsc;
  // Rows g and g + 8 of block kb: two pieces of 16 bytes each.
  auto load_w = [&](int kb) {
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int k = kb * BLOCK + 64 * c + 16 * t;
        w[r][c] = ldw(wrow + (long)(8 * r) * p.K + k, n0 + g + 8 * r < p.N && k < p.K);
      }
    wsc = kb < KB ? __ldg(ws + kb) : 0.f;
  };
  // The weight is no other kernel's result, so its first blocks are under way
  // before the previous kernel (the quantiser, if there is one) has ended.
  load_w(warp);
  pdl_wait();
  pdl_trigger();
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  for (int kb = warp; kb < KB; kb += WARPS) {
    Act<X> x[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) x[j].load(p, m0 + 8 * j + g, kb, t);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      uint32_t f[8];
      const float xs = x[j].frag(f);
      // Columns 2t and 2t + 1 of the result: the scales of those tokens.
      const float s0 = __shfl_sync(0xffffffffu, xs, 8 * t) * wsc;
      const float s1 = __shfl_sync(0xffffffffu, xs, 8 * t + 4) * wsc;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const uint4 a = w[0][c], b = w[1][c];
        mma_e4m3(v, a.x, b.x, a.y, b.y, f[4 * c], f[4 * c + 1]);
        mma_e4m3(v, a.z, b.z, a.w, b.w, f[4 * c + 2], f[4 * c + 3]);
      }
      acc[j][0] = fmaf(v[0], s0, acc[j][0]);
      acc[j][1] = fmaf(v[1], s1, acc[j][1]);
      acc[j][2] = fmaf(v[2], s0, acc[j][2]);
      acc[j][3] = fmaf(v[3], s1, acc[j][3]);
    }
    load_w(kb + WARPS);
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
    for (int k = 1; k < WARPS; k++) v += red[k][m][n];
    if (m0 + m < p.M && n0 + n < p.N) static_cast<Y*>(p.y)[(long)(m0 + m) * p.ldy + n0 + n] = from_f32<Y>(v);
  }
}

template <class X, class Y, int NT>
static cudaError_t launch_nt(const F8GemmParams& p, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg =
      pdl_config(dim3((p.N + ROWS - 1) / ROWS, (p.M + 8 * NT - 1) / (8 * NT)), dim3(WARPS * 32), 0, s, attr);
  return cudaLaunchKernelEx(&cfg, f8_small_kernel<X, Y, NT>, p);
}
template <class X, class Y>
static cudaError_t launch_xy(const F8GemmParams& p, cudaStream_t s) {
  if constexpr (sizeof(X) == 1) {
    if (p.M > 24) return launch_nt<X, Y, 4>(p, s);
    if (p.M > 16) return launch_nt<X, Y, 3>(p, s);
    if (p.M > 8) return launch_nt<X, Y, 2>(p, s);
  }
  return launch_nt<X, Y, 1>(p, s);
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
