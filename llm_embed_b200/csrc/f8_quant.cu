// Quantisation to e4m3 with a power-of-two scale per block of 128 (f8.cuh):
// activations by row and 128 columns, weights by 128 x 128.  Bound by memory:
// one read and one write of each value (18431 x 4096, bf16: 39 us, 5.9 TB/s,
// 0.90 of a measured copy; 44 us with loads that are not kept in the L2; 8 x
// 768: 1.3 us).
#include "f8.cuh"
#include "kernels.h"

namespace le {
namespace f8q {

using namespace f8;

constexpr int THREADS = 256;
constexpr int G = 16;  // lanes per block of 128 columns, eight columns each

__device__ __forceinline__ uint32_t group_max(uint32_t a, int width) {
  for (int o = width / 2; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// x [M][K] (row stride ldx) -> q [M][K] bytes, scales [ceil(K/128)][M].
// Rows 16-byte aligned, K a multiple of 8.  A block has 16 rows, each lane
// group U consecutive K blocks of one: U loads in flight, and the rows'
// scales of a K block lie side by side.
template <class T, int U>
__global__ void __launch_bounds__(THREADS) quant_vec_kernel(const T* __restrict__ x, long ldx, int M, int K, int KB,
                                                            int steps, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % G;
  const long row = (long)(blockIdx.x / steps) * (THREADS / G) + threadIdx.x / G;
  const int kb0 = blockIdx.x % steps * U;
  const bool live = row < M;
  Raw8<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = (kb0 + u) * BLOCK + lane * 8;
    raw[u] = live && c < K ? load8(x + row * ldx + c) : zero8<T>();
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    float v[8];
    values8(raw[u], v);
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, abs_bits(v[i]));
    a = group_max(a, G);
    float inv;
    const float s = block_scale(a, &inv);
    const int c = (kb0 + u) * BLOCK + lane * 8;
    if (live && c < K)
      *reinterpret_cast<uint2*>(q + row * K + c) =
          make_uint2(pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                     pack_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
    if (live && lane == 0 && kb0 + u < KB) scales[(long)(kb0 + u) * M + row] = s;
  }
}

// Any K, row stride and alignment: one warp per block of 128 columns.  Bound by
// its instructions, with single elements loaded and stored: 18431 x 4095 of bf16
// in 94 us, 2.4 TB/s, where rows on 16 bytes take 38.
template <class T>
__global__ void __launch_bounds__(THREADS) quant_any_kernel(const T* __restrict__ x, long ldx, long items, int M,
                                                            int K, int KB, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (item >= items) return;
  const long row = item / KB;
  const int kb = (int)(item - row * KB);
  float v[BLOCK / 32];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < BLOCK / 32; i++) {
    const int c = kb * BLOCK + i * 32 + lane;
    v[i] = c < K ? to_f32(x[row * ldx + c]) : 0.f;
    a = max(a, abs_bits(v[i]));
  }
  a = group_max(a, 32);
  float inv;
  const float s = block_scale(a, &inv);
#pragma unroll
  for (int i = 0; i < BLOCK / 32; i++) {
    const int c = kb * BLOCK + i * 32 + lane;
    if (c < K) q[row * K + c] = (uint8_t)pack_e4m3(v[i] * inv, 0.f, 0.f, 0.f);
  }
  if (lane == 0) scales[(long)kb * M + row] = s;
}

// w [N][K] float32 -> q [N][K] bytes, scales [ceil(N/128)][ceil(K/128)] (KB
// columns): one CTA per 128 x 128 block (its second read comes from L1 or L2).
__global__ void __launch_bounds__(THREADS) quant_weight_kernel(const float* __restrict__ w, int N, int K, int KB,
                                                               uint8_t* __restrict__ q, float* __restrict__ scales) {
  __shared__ uint32_t top;
  const int k0 = blockIdx.x % KB * BLOCK, n0 = blockIdx.x / KB * BLOCK;
  const int nk = min(BLOCK, K - k0), nn = min(BLOCK, N - n0);
  if (threadIdx.x == 0) top = 0;
  __syncthreads();
  uint32_t a = 0;
  for (int i = threadIdx.x; i < BLOCK * BLOCK; i += THREADS) {
    const int r = i / BLOCK, c = i % BLOCK;
    if (r < nn && c < nk) a = max(a, abs_bits(w[(long)(n0 + r) * K + k0 + c]));
  }
  atomicMax(&top, group_max(a, 32));
  __syncthreads();
  float inv;
  const float s = block_scale(top, &inv);
  for (int i = threadIdx.x; i < BLOCK * BLOCK; i += THREADS) {
    const int r = i / BLOCK, c = i % BLOCK;
    if (r < nn && c < nk) {
      const long at = (long)(n0 + r) * K + k0 + c;
      q[at] = (uint8_t)pack_e4m3(w[at] * inv, 0.f, 0.f, 0.f);
    }
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = s;
}

template <class T>
static cudaError_t launch(const void* x, long ldx, int M, int K, uint8_t* q, float* scales, cudaStream_t s) {
  const int KB = (K + BLOCK - 1) / BLOCK;
  const long items = (long)M * KB;
  const bool vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * (long)sizeof(T)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 8 == 0;
  // Four K blocks in flight per lane once that still gives every one of the
  // 148 SMs four blocks.
  const int u = vec && items >= 148L * 4 * 4 * (THREADS / G) ? 4 : 1, steps = (KB + u - 1) / u;
  const long blocks = vec ? ((long)M + THREADS / G - 1) / (THREADS / G) * steps
                          : (items + THREADS / 32 - 1) / (THREADS / 32);
  if (blocks > 0x7fffffffL) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)blocks), dim3(THREADS), 0, s, attr);
  const T* xt = static_cast<const T*>(x);
  if (!vec) return cudaLaunchKernelEx(&cfg, quant_any_kernel<T>, xt, ldx, items, M, K, KB, q, scales);
  if (u == 4) return cudaLaunchKernelEx(&cfg, quant_vec_kernel<T, 4>, xt, ldx, M, K, KB, steps, q, scales);
  return cudaLaunchKernelEx(&cfg, quant_vec_kernel<T, 1>, xt, ldx, M, K, KB, steps, q, scales);
}

}  // namespace f8q

cudaError_t launch_f8_quantize(int dt, const void* x, long ldx, int M, int K, uint8_t* q, float* scales,
                               cudaStream_t s) {
  if (M == 0) return cudaSuccess;
  return dt == DT_F32   ? f8q::launch<float>(x, ldx, M, K, q, scales, s)
         : dt == DT_F16 ? f8q::launch<__half>(x, ldx, M, K, q, scales, s)
                        : f8q::launch<__nv_bfloat16>(x, ldx, M, K, q, scales, s);
}

cudaError_t launch_f8_quantize_weight(const float* w, int N, int K, uint8_t* q, float* scales, cudaStream_t s) {
  const int kb = (K + f8::BLOCK - 1) / f8::BLOCK, nb = (N + f8::BLOCK - 1) / f8::BLOCK;
  const long blocks = (long)kb * nb;
  if (blocks > 0x7fffffffL) return cudaErrorInvalidValue;
  f8q::quant_weight_kernel<<<(unsigned)blocks, f8q::THREADS, 0, s>>>(w, N, K, kb, q, scales);
  return cudaGetLastError();
}

}  // namespace le
