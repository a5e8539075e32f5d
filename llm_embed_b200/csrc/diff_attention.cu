// Differential attention over packed sequences (mma.sync tiles):
//   A_i = softmax(q_i k_i^T / sqrt(d)), i = 1, 2
//   o   = (A_1 - lambda A_2) v
//   out = (1 - lambda_init) o rsqrt(mean(o^2) + eps) w     (o itself without w)
// for every head, whose two query and key parts have d columns each and whose
// values have 2d.
//
// A CTA has 64 queries of one head and sequence, 16 per warp, and goes once
// over the keys in blocks of 64, two in flight (cp.async).  Each map keeps a
// running maximum and sum per query and its own float32 result O_i, rescaled
// when the maximum grows; at the end o = O_1 / l_1 - lambda O_2 / l_2.  A block's values are read
// from shared memory once for both maps.  Weights P are rounded to the
// operands' type (16 bits) for the second product, their sums are not.
// Keys past the sequence get weight 0 and their values are zeros in shared
// memory, whatever the rows behind hold.
#include <mutex>

#include "diff_attention.cuh"

namespace le {
namespace dif {

constexpr int BQ = 64, BKEY = 64, WARPS = 4;

template <class T>
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// A tile's rows hold W = 2d elements as 16-byte chunks, chunk c of row r at
// c ^ (r & 7): eight rows of one chunk lie on distinct banks for ldmatrix.
template <int W>
__device__ __forceinline__ uint32_t at(uint32_t base, int row, int chunk) {
  return base + row * (W * 2) + ((chunk ^ (row & 7)) << 4);
}

// Rows [0, 64) of a tile from src (row stride ld); rows from `n` on are zero.
template <int W, class T>
__device__ __forceinline__ void load_tile(uint32_t base, const T* src, long ld, int n) {
  constexpr int CH = W / 8;
#pragma unroll
  for (int i = threadIdx.x; i < 64 * CH; i += WARPS * 32) {
    const int r = i / CH, c = i % CH;
    const int bytes = r < n ? 16 : 0;
    const T* g = src + (long)(r < n ? r : 0) * ld + c * 8;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at<W>(base, r, c)), "l"(g), "r"(bytes));
  }
}

template <class T, int D>
__global__ void __launch_bounds__(WARPS * 32) diff_mma_kernel(DiffParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int W = 2 * D, TILE = 64 * W * 2;
  if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(p, WARPS * 32);
  Where wh;
  if (!find_block(p, p.offsets, blockIdx.x, BQ, wh) || wh.len < p.min_len || wh.len > p.max_len) return;
  extern __shared__ __align__(128) uint8_t smem_diff[];
  const uint32_t sq = (uint32_t)__cvta_generic_to_shared(smem_diff), skv = sq + TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y, kvh = head / p.group;
  const T* q = static_cast<const T*>(p.q) + (long)(wh.t0 + wh.q0) * p.q_stride + (long)head * W;
  const T* k = static_cast<const T*>(p.k) + (long)wh.t0 * p.k_stride + (long)kvh * W;
  const T* v = static_cast<const T*>(p.v) + (long)wh.t0 * p.v_stride + (long)kvh * W;
  const int nkb = (wh.len + BKEY - 1) / BKEY;
  auto load_kv = [&](int j) {
    const uint32_t b = skv + (j & 1) * 2 * TILE;
    load_tile<W>(b, k + (long)j * BKEY * p.k_stride, p.k_stride, wh.len - j * BKEY);
    load_tile<W>(b + TILE, v + (long)j * BKEY * p.v_stride, p.v_stride, wh.len - j * BKEY);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load_tile<W>(sq, q, p.q_stride, wh.len - wh.q0);
  load_kv(0);

  uint32_t qa[2][D / 16][4];
  float o[2][W / 8][4], m[2][2], l[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    m[i][0] = m[i][1] = -INFINITY;
    l[i][0] = l[i][1] = 0.f;
#pragma unroll
    for (int n = 0; n < W / 8; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
  }
  const float scale2 = 1.4426950408889634f * rsqrtf((float)D);
  for (int j = 0; j < nkb; j++) {
    if (j + 1 < nkb) {
      load_kv(j + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    if (j == 0) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < D / 16; c++)
          ldsm4(qa[i][c], at<W>(sq, warp * 16 + (lane & 15), i * (D / 8) + 2 * c + (lane >> 4)));
    }
    const uint32_t sk = skv + (j & 1) * 2 * TILE, sv = sk + TILE;
    const int left = wh.len - j * BKEY;  // keys of this block and behind
    uint32_t pa[2][BKEY / 16][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float s[BKEY / 8][4];
#pragma unroll
      for (int n = 0; n < BKEY / 8; n++) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
          uint32_t b[4];
          ldsm4(b, at<W>(sk, n * 8 + (lane & 7), i * (D / 8) + 2 * c + (lane >> 3)));
          mma16<T>(s[n], qa[i][c], b[0], b[1]);
          mma16<T>(s[n], qa[i][c + 1], b[2], b[3]);
        }
      }
      float mx0 = m[i][0], mx1 = m[i][1];
#pragma unroll
      for (int n = 0; n < BKEY / 8; n++) {
        if (left < BKEY) {
          const int key = n * 8 + 2 * t;
          if (key >= left) s[n][0] = s[n][2] = -INFINITY;
          if (key + 1 >= left) s[n][1] = s[n][3] = -INFINITY;
        }
        mx0 = fmaxf(mx0, fmaxf(s[n][0], s[n][1]));
        mx1 = fmaxf(mx1, fmaxf(s[n][2], s[n][3]));
      }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      const float c0 = ex2f((m[i][0] - mx0) * scale2), c1 = ex2f((m[i][1] - mx1) * scale2);
      m[i][0] = mx0;
      m[i][1] = mx1;
      const float off0 = -mx0 * scale2, off1 = -mx1 * scale2;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int n = 0; n < BKEY / 8; n++) {
        s[n][0] = ex2f(fmaf(s[n][0], scale2, off0));
        s[n][1] = ex2f(fmaf(s[n][1], scale2, off0));
        s[n][2] = ex2f(fmaf(s[n][2], scale2, off1));
        s[n][3] = ex2f(fmaf(s[n][3], scale2, off1));
        l0 += s[n][0] + s[n][1];
        l1 += s[n][2] + s[n][3];
      }
      l[i][0] = fmaf(l[i][0], c0, l0);
      l[i][1] = fmaf(l[i][1], c1, l1);
#pragma unroll
      for (int n = 0; n < W / 8; n++) {
        o[i][n][0] *= c0;
        o[i][n][1] *= c0;
        o[i][n][2] *= c1;
        o[i][n][3] *= c1;
      }
#pragma unroll
      for (int n = 0; n < BKEY / 16; n++) {
        pa[i][n][0] = pack2<T>(s[2 * n][0], s[2 * n][1]);
        pa[i][n][1] = pack2<T>(s[2 * n][2], s[2 * n][3]);
        pa[i][n][2] = pack2<T>(s[2 * n + 1][0], s[2 * n + 1][1]);
        pa[i][n][3] = pack2<T>(s[2 * n + 1][2], s[2 * n + 1][3]);
      }
    }
#pragma unroll
    for (int c = 0; c < BKEY / 16; c++)
#pragma unroll
      for (int n = 0; n < W / 8; n += 2) {
        uint32_t b[4];
        ldsm4_t(b, at<W>(sv, c * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n + (lane >> 4)));
#pragma unroll
        for (int i = 0; i < 2; i++) {
          mma16<T>(o[i][n], pa[i][c], b[0], b[1]);
          mma16<T>(o[i][n + 1], pa[i][c], b[2], b[3]);
        }
      }
    __syncthreads();
  }

  const float lam = p.lambda[head];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int r = 0; r < 2; r++) {
      l[i][r] += __shfl_xor_sync(0xffffffffu, l[i][r], 1);
      l[i][r] += __shfl_xor_sync(0xffffffffu, l[i][r], 2);
    }
  const float a0 = 1.f / l[0][0], a1 = 1.f / l[0][1], b0 = lam / l[1][0], b1 = lam / l[1][1];
  float ss0 = 0.f, ss1 = 0.f;
#pragma unroll
  for (int n = 0; n < W / 8; n++) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      o[0][n][c] = o[0][n][c] * a0 - o[1][n][c] * b0;
      o[0][n][2 + c] = o[0][n][2 + c] * a1 - o[1][n][2 + c] * b1;
      ss0 = fmaf(o[0][n][c], o[0][n][c], ss0);
      ss1 = fmaf(o[0][n][2 + c], o[0][n][2 + c], ss1);
    }
  }
  float r0 = 1.f, r1 = 1.f;
  if (p.norm_w) {
    ss0 += __shfl_xor_sync(0xffffffffu, ss0, 1);
    ss0 += __shfl_xor_sync(0xffffffffu, ss0, 2);
    ss1 += __shfl_xor_sync(0xffffffffu, ss1, 1);
    ss1 += __shfl_xor_sync(0xffffffffu, ss1, 2);
    r0 = p.out_scale * rsqrtf(ss0 / (float)W + p.eps);
    r1 = p.out_scale * rsqrtf(ss1 / (float)W + p.eps);
  }
  const int q0 = wh.q0 + warp * 16 + g;
  T* out = static_cast<T*>(p.out) + (long)(wh.t0 + q0) * p.o_stride + (long)head * W + 2 * t;
#pragma unroll
  for (int n = 0; n < W / 8; n++) {
    const float w0 = p.norm_w ? __ldg(p.norm_w + 8 * n + 2 * t) : 1.f;
    const float w1 = p.norm_w ? __ldg(p.norm_w + 8 * n + 2 * t + 1) : 1.f;
    if (q0 < wh.len)
      *reinterpret_cast<uint32_t*>(out + 8 * n) = pack2<T>(o[0][n][0] * r0 * w0, o[0][n][1] * r0 * w1);
    if (q0 + 8 < wh.len)
      *reinterpret_cast<uint32_t*>(out + 8 * p.o_stride + 8 * n) =
          pack2<T>(o[0][n][2] * r1 * w0, o[0][n][3] * r1 * w1);
  }
}

template <class T, int D>
static cudaError_t launch(const DiffParams& p, cudaStream_t s) {
  constexpr int SMEM = 5 * 64 * 2 * D * 2;
  static std::mutex mu;
  static uint64_t attr_set = 0;  // per-device bit: the attribute is a per-device setting
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(attr_set >> dev & 1)) {
      const cudaError_t e =
          cudaFuncSetAttribute(diff_mma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
      if (e != cudaSuccess) return e;
      if (dev < 64) attr_set |= 1ull << dev;
    }
  }
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg =
      pdl_config(dim3(block_count(p.T, p.nseq, BQ), p.heads), dim3(WARPS * 32), SMEM, s, attr);
  return cudaLaunchKernelEx(&cfg, diff_mma_kernel<T, D>, p);
}

}  // namespace dif

cudaError_t launch_diff_attention(int dt, int d, const DiffParams& p, cudaStream_t s) {
  if (p.nseq == 0 || p.T == 0) return cudaSuccess;
  if (dt == DT_F16) return d == 64 ? dif::launch<__half, 64>(p, s) : dif::launch<__half, 32>(p, s);
  return d == 64 ? dif::launch<__nv_bfloat16, 64>(p, s) : dif::launch<__nv_bfloat16, 32>(p, s);
}

}  // namespace le
