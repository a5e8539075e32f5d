// Eight-bit product on the tensor cores (tcgen05 kind::f8f6f4, sm_100a):
//   y[m][n] = sum_b xs[b][m] ws[n/128][b] sum_{k in block b} xq[m][k] wq[n][k]
//
// The weight's scales are any float32, so they cannot be left to the MMA's
// own power-of-two scaling: each K block of 128 is one accumulator of its own
// in TMEM (four MMAs of K = 32, the first overwriting), and the epilogue warps
// add it, times the row's and the weight block's scale, to float32 sums in
// registers while the tensor cores fill the other accumulators.  A thread
// holds one row's columns of one weight block, so a block costs it one
// multiplier and half a packed fma per column.
//
// Bound by that addition: of about 1000 clocks a K block of 128 x 256 columns
// costs, the tensor cores need 512 and the warps that add 256 for their fmas,
// the rest is the way from MMA to addition and back.  Without the loads of the
// sums it would be 121 us where it is 129 (8192 x 4096 . 4096), without the
// wait for the accumulator 90.  Measured with rows that are quantised already,
// 50 calls in a graph:
//   8192 x 4096 . 4096    129 us  2.13 PFLOP/s (to 142 once the chip is at its power limit)
//   32768 x 768 . 2304     70 us  1.66 PFLOP/s
//   512 x 4096 . 4096    14.4 us  (12.6 before the narrow tiles' present form)
//   333 x 768 . 2304      4.7 us
//
// Persistent kernel; tile = 128 * CG token rows x BN weight rows.  CG = 2: a
// cluster of two CTAs computes it with one MMA of M = 256 (cta_group::2), each
// CTA loading its 128 token rows and half of the weight rows.
//   warp 0     producer: TMA loads, one K block (128 bytes a row, 128B
//              swizzle) per stage
//   warp 1     TMEM allocation; one lane (of the even CTA) issues the MMAs
//   warp 2     copies of the scales, three K blocks ahead
//   warps 4-   epilogue: TMEM lanes by warp % 4, columns by group of four;
//              rows go out through shared memory and TMA stores, or by plain
//              stores where y's rows do not begin and end on 16 bytes
// Rows and columns past M, N and K are zeros from TMA and are not stored.
// Every mbarrier wait is bounded (WAIT_LIMIT_NS); after one that ran out the CTA
// lets its copies and MMAs end before it exits.
#include <cudaTypedefs.h>

#include <mutex>

#include "elem.cuh"
#include "gemm_epi_tc.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace le {
namespace f8t {

using namespace tcx;

constexpr int BM = 128;
constexpr int BK = 128;  // one scale block
constexpr int EPI_WARP0 = 4;
constexpr int SLOTS = 3, SLOT_BYTES = (BM + 4) * 4;  // K blocks whose scales are in shared memory

template <int CG, int BN, int STAGES, int NACC>
struct Cfg {
  static constexpr int cg = CG, bn = BN, stages = STAGES, nacc = NACC;
  // Two groups of four epilogue warps share the columns of the wider tiles; a
  // group has at least 64 (a 128-byte row of a 16-bit result).
  static constexpr int EPI_WARPS = BN >= 128 ? 8 : 4;
  static constexpr int COLS = BN / (EPI_WARPS / 4);  // columns of a warp
  // Columns of a TMEM load: two loads of 32 beside 128 sums spill.
  static constexpr int CHUNK = COLS >= 128 ? 16 : 32;
  static constexpr int NTHREADS = (EPI_WARP0 + EPI_WARPS) * 32;
  static constexpr int B_ROWS = BN / CG;  // weight rows per CTA
  static constexpr int A_BYTES = BM * BK, B_BYTES = B_ROWS * BK;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = OFF_A + STAGES * A_BYTES;
  static constexpr int OFF_STAGE = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_SCALE = OFF_STAGE + EPI_WARPS * 2 * 4096;  // [SLOTS][128 rows, up to 2 columns' groups]
  static constexpr int OFF_BAR = OFF_SCALE + SLOTS * SLOT_BYTES;
  static constexpr int NBAR = 2 * STAGES + 2 * NACC + 2 * SLOTS;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static constexpr int TMEM_COLS = NACC * BN;
  static_assert(ALLOC <= 232448, "shared memory of one CTA");
  static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM columns");
};

template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 2)
    mma_commit_pair(bar, 0x3);
  else
    mma_commit(bar);
}

// 32 or 16 TMEM columns of the warp's lanes; the registers hold them after
// wait_ld, which names them so that no use moves above it.
__device__ __forceinline__ void ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%"
      "20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])::"memory");
}

// acc += v * s in both halves, kept in its place between the loads and waits.
__device__ __forceinline__ void add_scaled(unsigned long long& acc, unsigned long long v, unsigned long long s) {
  asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s));
}

// Plain stores of 32 rows x 128 bytes (words[32] of a lane: its row), turned in
// the warp's shared memory so that consecutive lanes write consecutive words of
// a row (word j of row i lies at j ^ i: distinct banks both ways).  `even`:
// rows begin on 4-byte boundaries; else a word of two columns goes out in
// halves.
template <class Y>
__device__ __forceinline__ void store_plain(uint32_t* stg, const uint32_t* words, Y* y, long ldy, int row0, int col0,
                                            int M, int N, bool even) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; j++) stg[lane * 32 + (j ^ lane)] = words[j];
  __syncwarp();
  constexpr int PER = 4 / sizeof(Y);  // columns of a word
  const int col = col0 + lane * PER, n = min(32, M - row0);
  Y* out = y + (long)row0 * ldy + col;
  if (n == 32 && col0 + 32 * PER <= N) {  // a whole block: nothing to decide in the loops
    if (PER == 1 || even) {
#pragma unroll
      for (int i = 0; i < 32; i++, out += ldy) *reinterpret_cast<uint32_t*>(out) = stg[i * 32 + (lane ^ i)];
    } else {
#pragma unroll 8
      for (int i = 0; i < 32; i++, out += ldy) {
        const uint32_t w = stg[i * 32 + (lane ^ i)];
        reinterpret_cast<uint16_t*>(out)[0] = (uint16_t)w;
        reinterpret_cast<uint16_t*>(out)[1] = (uint16_t)(w >> 16);
      }
    }
    return;
  }
#pragma unroll 4
  for (int i = 0; i < n; i++, out += ldy) {
    const uint32_t w = stg[i * 32 + (lane ^ i)];
    if constexpr (PER == 1) {
      if (col < N) *reinterpret_cast<uint32_t*>(out) = w;
    } else {
      if (col < N) reinterpret_cast<uint16_t*>(out)[0] = (uint16_t)w;
      if (col + 1 < N) reinterpret_cast<uint16_t*>(out)[1] = (uint16_t)(w >> 16);
    }
  }
}

template <class C, class Y>
__global__ void __launch_bounds__(C::NTHREADS, 1)
    f8_tc_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_y, int use_tma, F8GemmParams p, int m_tiles, int n_tiles,
                 DevStatus* status) {
  constexpr int CG = C::cg, BN = C::bn, S = C::stages, NACC = C::nacc, COLS = C::COLS, EPI_WARPS = C::EPI_WARPS;
  constexpr uint32_t IDESC = idesc_f16(CG * BM, BN);  // e4m3 x e4m3 has the same type fields (0)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (S + s); };
  auto tfull = [&](int a) { return bar0 + 8 * (2 * S + a); };
  auto tempty = [&](int a) { return bar0 + 8 * (2 * S + NACC + a); };
  auto sfull = [&](int s) { return bar0 + 8 * (2 * S + 2 * NACC + s); };
  auto sempty = [&](int s) { return bar0 + 8 * (2 * S + 2 * NACC + SLOTS + s); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int KB = (p.K + BK - 1) / BK;
  const int total = m_tiles * n_tiles;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < S; s++) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < NACC; a++) {
      mbar_init(tfull(a), 1);
      mbar_init(tempty(a), CG * EPI_WARPS);
    }
    for (int s = 0; s < SLOTS; s++) {
      mbar_init(sfull(s), 32);
      mbar_init(sempty(s), EPI_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // both CTAs' barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  // The widest tile's epilogue holds 128 sums a thread: of the 384 x 168
  // registers at launch the first warpgroup keeps 40 each, the two of the
  // epilogue take 232.
  if (warp < EPI_WARP0) {
  if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_a)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_b)) : "memory");
      auto load = [&](const CUtensorMap* map, uint32_t dst, int kb, int row, int s) {
        if constexpr (CG == 2)
          tma_load_2d_pair(dst, map, kb * BK, row, map_to_rank(full(s), 0));
        else
          tma_load_2d(dst, map, kb * BK, row, full(s));
      };
      auto load_weight = [&](int tile, int kb, int s) {
        if (leader) mbar_expect_tx(full(s), CG * (C::A_BYTES + C::B_BYTES));
        load(&tmap_b, sbase + C::OFF_B + s * C::B_BYTES, kb, tile % n_tiles * BN + (int)rank * C::B_ROWS, s);
      };
      // The weight is no other kernel's result: the first stages' part of it is
      // on its way before the previous kernel (the quantiser) has ended.
      const int early = min(S, KB);
      for (int kb = 0; kb < early; kb++) load_weight(first, kb, kb);
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += step) {
        const int row = (tile / n_tiles * CG + (int)rank) * BM;
        for (int kb = 0; kb < KB; kb++, it++) {
          const int s = it % S;
          if (!mbar_wait(empty(s), ((it / S) & 1) ^ 1, abort_flag, status, 50)) {
            ok = false;
            break;
          }
          if (it >= (uint32_t)early) load_weight(tile, kb, s);
          load(&tmap_a, sbase + C::OFF_A + s * C::A_BYTES, kb, row, s);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    // The whole warp walks the loop, so that its addresses are uniform; one
    // lane issues.
    if (leader) {
      const bool issuer = elect_one();
      const uint64_t a0 = sw128_desc(sbase + C::OFF_A), b0 = sw128_desc(sbase + C::OFF_B);
      uint32_t it = 0;
      bool ok = true;
      // The rows come once the previous kernel has ended, however long that
      // takes: the bounded waits for them begin there too.
      pdl_wait();
      for (int tile = first; tile < total && ok; tile += step) {
        for (int kb = 0; kb < KB && ok; kb++, it++) {
          const uint32_t s = it % S, acc = it % NACC;
          ok = mbar_wait(full(s), (it / S) & 1, abort_flag, status, 52) &&
               mbar_wait(tempty(acc), ((it / NACC) & 1) ^ 1, abort_flag, status, 51);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (issuer) {
            // Descriptor addresses count 16-byte units.
            const uint64_t a = a0 + s * (C::A_BYTES / 16), b = b0 + s * (C::B_BYTES / 16);
#pragma unroll
            for (int kk = 0; kk < BK / 32; kk++) mma_f8<CG>(tmem + acc * BN, a + kk * 2, b + kk * 2, IDESC, kk != 0);
            commit<CG>(tfull(acc));
            commit<CG>(empty(s));
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales
    // Copied ahead by a warp that has nothing else to do: a load from L2 takes
    // as long as a K block or two, and the epilogue has no registers to wait in.
    auto copy = [](uint32_t dst, const float* src) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
    };
    pdl_wait();
    uint32_t it = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += step) {
      // Clamped rows and columns read a scale that exists and are not stored.
      const int row = (tile / n_tiles * CG + (int)rank) * BM + lane;
      const float* ws = p.ws + (long)(min(tile % n_tiles * BN + lane * COLS, p.N - 1) / 128) * KB;
      for (int kb = 0; kb < KB; kb++, it++) {
        const int s = it % SLOTS;
        ok = __all_sync(0xffffffffu, mbar_wait(sempty(s), ((it / SLOTS) & 1) ^ 1, abort_flag, status, 54));
        if (!ok) break;
        const uint32_t dst = sbase + C::OFF_SCALE + s * SLOT_BYTES + lane * 4;
        const float* xs = p.xs + (long)kb * p.M;
#pragma unroll
        for (int i = 0; i < BM / 32; i++) copy(dst + i * 128, xs + min(row + 32 * i, p.M - 1));
        if (lane < EPI_WARPS / 4) copy(dst + BM * 4, ws + kb);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sfull(s)) : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, ew = warp - EPI_WARP0;
    const int c0 = (ew >> 2) * COLS;  // this warp's columns of the tile
    const uint32_t stage = sbase + C::OFF_STAGE + ew * 2 * 4096;
    uint32_t* stg = reinterpret_cast<uint32_t*>(smem + C::OFF_STAGE + ew * 2 * 4096);
    const bool even = p.ldy % 2 == 0 && reinterpret_cast<uintptr_t>(p.y) % 4 == 0;
    int buf = 0;
    uint32_t it = 0;
    bool ok = true;
    const float* scales = reinterpret_cast<const float*>(smem + C::OFF_SCALE);
    pdl_wait();  // y's memory is the previous kernels'
    for (int tile = first; tile < total && ok; tile += step) {
      const int mt = tile / n_tiles, nt = tile % n_tiles;
      const int row0 = (mt * CG + (int)rank) * BM + quarter * 32, n0 = nt * BN + c0;
      unsigned long long acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; i++) acc[i] = 0;
      for (int kb = 0; kb < KB; kb++, it++) {
        const int a = it % NACC;
        const int s = it % SLOTS;
        if (!__all_sync(0xffffffffu, mbar_wait(sfull(s), (it / SLOTS) & 1, abort_flag, status, 55) &&
                                         mbar_wait(tfull(a), (it / NACC) & 1, abort_flag, status, 53))) {
          ok = false;
          break;
        }
        const float* slot = scales + s * (SLOT_BYTES / 4);
        const float sc = slot[quarter * 32 + lane] * slot[BM + (ew >> 2)];
        tc_fence_after();
        const unsigned long long sc2 = f2_pack(sc, sc);
        const uint32_t t = tmem + a * BN + c0 + ((uint32_t)(quarter * 32) << 16);
        // The next columns are on their way while these are added.
        constexpr int CH = C::CHUNK;
        uint32_t v[2][CH];
        ld(t, v[0]);
#pragma unroll
        for (int c = 0; c < COLS; c += CH) {
          uint32_t(&u)[CH] = v[(c / CH) & 1];
          wait_ld(u);
          if (c + CH < COLS) {
            ld(t + c + CH, v[(c / CH + 1) & 1]);
          } else {  // all read: the accumulator is free while the last columns are added
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(sempty(s));
              if constexpr (CG == 2)
                mbar_arrive_cluster(map_to_rank(tempty(a), 0));
              else
                mbar_arrive(tempty(a));
            }
          }
#pragma unroll
          for (int i = 0; i < CH / 2; i++)
            add_scaled(acc[c / 2 + i], f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), sc2);
        }
      }
      if (!ok) break;
      if (row0 >= p.M) continue;  // warp-uniform
      constexpr int PER = 128 / sizeof(Y);  // columns of a 128-byte block
#pragma unroll
      for (int c = 0; c < COLS; c += PER) {
        if (n0 + c >= p.N) break;
        uint32_t words[32];
#pragma unroll
        for (int i = 0; i < PER / 2; i++) {
          float lo, hi;
          f2_unpack(acc[c / 2 + i], lo, hi);
          if constexpr (sizeof(Y) == 4) {
            words[2 * i] = __float_as_uint(lo);
            words[2 * i + 1] = __float_as_uint(hi);
          } else {
            words[i] = pack2<Y>(lo, hi);
          }
        }
        if (use_tma)
          emit_block(&tmap_y, stage, buf, words, n0 + c, row0);
        else
          store_plain<Y>(stg, words, static_cast<Y*>(p.y), p.ldy, row0, n0 + c, p.M, p.N, even);
      }
    }
    if (use_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) settle(abort_flag);
  if constexpr (CG == 2) cluster_sync();  // the peer is done with this CTA's shared memory and TMEM
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
  }
}

// ---------------------------------------------------------------- host ----

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// 2-D row-major map of bytes_per-element elements with 128B-swizzled boxes.
static bool encode(PFN_cuTensorMapEncodeTiled_v12000 enc, CUtensorMap* map, CUtensorMapDataType type, int esz,
                   const void* p, long rows, long cols, long ld, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * esz};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class C, class Y>
static cudaError_t launch(int ydt, const F8GemmParams& p, DevStatus* status, cudaStream_t s) {
  auto enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  CUtensorMap amap, bmap, ymap = {};
  if (!encode(enc, &amap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.x, p.M, p.K, p.ldx, BK, BM) ||
      !encode(enc, &bmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.N, p.K, p.K, BK, C::B_ROWS))
    return cudaErrorInvalidValue;
  // A TMA store clips the last columns at 16-byte steps only, so N must end on
  // one for the columns behind to stay as they were.
  const int use_tma = reinterpret_cast<uintptr_t>(p.y) % 16 == 0 && (p.ldy * (long)sizeof(Y)) % 16 == 0 &&
                      (p.N * (long)sizeof(Y)) % 16 == 0;
  const CUtensorMapDataType yt = ydt == DT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : ydt == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (use_tma && !encode(enc, &ymap, yt, sizeof(Y), p.y, p.M, p.N, p.ldy, 128 / sizeof(Y), 32))
    return cudaErrorInvalidValue;
  // Per device: the shared-memory attribute and how many clusters fit at once.
  static std::mutex mu;
  static int resident[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64) return cudaErrorInvalidDevice;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C::cg;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (resident[dev] == 0) {
      cudaError_t e = cudaFuncSetAttribute(f8_tc_kernel<C, Y>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::ALLOC);
      if (e != cudaSuccess) return e;
      int sms = 0, n = 0;
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(sms / C::cg * C::cg);
      cfg.blockDim = dim3(C::NTHREADS);
      cfg.dynamicSmemBytes = C::ALLOC;
      cfg.attrs = attr + 1;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&n, f8_tc_kernel<C, Y>, &cfg);
      if (e != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = sms / C::cg;
      }
      resident[dev] = n;
    }
  }
  const int m_tiles = (p.M + C::cg * BM - 1) / (C::cg * BM), n_tiles = (p.N + C::bn - 1) / C::bn;
  const long total = (long)m_tiles * n_tiles;
  if (total > 0x7fffffff) return cudaErrorInvalidValue;
  const int clusters = total < resident[dev] ? (int)total : resident[dev];
  cudaLaunchConfig_t cfg = pdl_config(dim3(clusters * C::cg), dim3(C::NTHREADS), C::ALLOC, s, attr);
  cfg.numAttrs = C::cg == 2 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, f8_tc_kernel<C, Y>, amap, bmap, ymap, use_tma, p, m_tiles, n_tiles, status);
}

using Pair = Cfg<2, 256, 5, 2>;
using Tile128 = Cfg<1, 128, 5, 4>;
using Tile64 = Cfg<1, 64, 8, 4>;

template <class Y>
static cudaError_t pick(int ydt, const F8GemmParams& p, DevStatus* status, cudaStream_t s) {
  switch (f8_tile(p.M, p.N)) {
    case 256: return launch<Pair, Y>(ydt, p, status, s);
    case 128: return launch<Tile128, Y>(ydt, p, status, s);
    default: return launch<Tile64, Y>(ydt, p, status, s);
  }
}

}  // namespace f8t

int f8_tile(int M, int N) {
  // Measured cost of one wave of tiles, 64 : 128 : 256 wide, about 4 : 5 : 8
  // (K = 768: 4.1, 5.0 and 6.6 us, K = 4096: 10.4, 13.6 and 20 us).
  const long sms = 148, m1 = ((long)M + 127) / 128, m2 = (m1 + 1) / 2, n = N;
  auto waves = [](long tiles, long slots) { return (tiles + slots - 1) / slots; };
  const long c64 = 4 * waves(m1 * ((n + 63) / 64), sms), c128 = 5 * waves(m1 * ((n + 127) / 128), sms),
             c256 = 8 * waves(m2 * ((n + 255) / 256), sms / 2);
  return c256 <= c128 && c256 <= c64 ? 256 : c128 <= c64 ? 128 : 64;
}

cudaError_t launch_f8_gemm_tc(int ydt, const F8GemmParams& p, DevStatus* status, cudaStream_t s) {
  if (p.M == 0) return cudaSuccess;
  return ydt == DT_F32   ? f8t::pick<float>(ydt, p, status, s)
         : ydt == DT_F16 ? f8t::pick<__half>(ydt, p, status, s)
                         : f8t::pick<__nv_bfloat16>(ydt, p, status, s);
}

}  // namespace le
