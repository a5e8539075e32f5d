// Differential attention on the tensor cores (tcgen05, sm_100a), for the
// sequences that are long enough to fill its tiles:
//   A_i = softmax(q_i k_i^T / sqrt(d)), o = (A_1 - lambda A_2) v, then the
//   head's norm (diff_attention.cu has the formulas in full).
//
// One CTA per SM, which goes from tile to tile (cluster launch control hands
// out the grid's CTAs that have not started).  A tile is 128 queries of one
// head and sequence; its two maps are two chains that share the keys' and values'
// loads and take turns on the tensor cores: while one map's scores are
// exponentiated, the other's products run.  A thread of a map's warpgroup has
// one query row (TMEM lane): it reads the 64 scores of a key block, writes
// the weights back over them as 16-bit pairs (the A operand of P.V), and keeps
// the row's maximum and sum.  The maximum that the weights refer to is only
// moved when it has grown by more than 2^8 (the weights then stay within 2^8 of
// its own, inside the operand's range, and the sums are float32), so rescaling
// the result in TMEM is rare.  The weights are the only values rounded to 16 bits
// before the result: the tensor cores take no wider operand at their rate.
//
// Bound by the exponentials, two per query, key and head, 16 a clock and SM,
// and by what they delay: instructions on barriers, TMEM and shared memory share
// the special-function unit's queue.  16 texts of 1024 to 2047 tokens, 6 heads of
// 64, bf16: 203 us (902 TFLOP/s; the exponentials alone 105 us at 1.9 GHz).  Of
// 1860 clocks that a block of 64 keys takes a map's warps, 630 are exponentials
// (512 at least), 390 the maximum and scaling, 270 packing and writing the
// weights, 320 the wait for scores, 170 the turn.  256 texts of 16 to 128: 51 us;
// the longest part of a tile of one or two key blocks is its epilogue.
//
//   warp 0      producer: TMA loads of Q (two stages), K and V (four each)
//   warps 1, 2  MMAs of a map each: S_i = Q_i K_i^T, O_i += P_i V (one warp
//               for both spent more time on its waits than the tensor cores
//               on their work: 2070 clocks a block, 775 of them busy)
//   warp 3      takes the tiles, finds their sequences and publishes them
//   warps 4-7   softmax of map 1, warps 8-11 of map 2
//   warps 12-15 combine O_1 and O_2, norm and store, beside the next tile's
//               first two blocks
// TMEM (512 columns): two buffers of S_i / P_i for each map (64 each), O_1,
// O_2 (2d each).  A map's MMAs run in the order they are issued - S of block
// j + 2 after P.V of block j, whose buffer it takes, also where those are blocks
// of the next tiles - so a map has a block of scores waiting while another's
// weights are multiplied.
//
// Keys past the sequence: their scores count as -inf; P.V stops at the next
// multiple of 16 keys, and the values between (another sequence's, or
// garbage) are overwritten with zeros in shared memory before it, so nothing
// but the sequence's own rows reaches a result.  Query rows past it are not
// stored.  Every mbarrier wait is bounded (WAIT_LIMIT_NS); after one that ran out
// the CTA lets its copies and MMAs end before it exits.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "diff_attention.cuh"
#include "gemm_epi_tc.cuh"
#include "softmax_tc.cuh"
#include "tcgen05.cuh"

namespace le {
namespace dtc {

using namespace tcx;
using namespace dif;

constexpr int BQ = 128, BKEY = 64;
constexpr int QTILE = 128 * 128, KTILE = 64 * 128;  // bytes of 128 and 64 rows x 64 columns
constexpr int KV = 4;                               // stages of K and of V
constexpr int NTHREADS = 512;
constexpr int RING = 4;
constexpr int EPI = 32;  // columns of a result that the epilogue loads at a time
constexpr int AHEAD = 8;    // tiles of more key blocks are taken one at a time
constexpr int OFFS = 1024;  // sequences whose offsets are copied to shared memory
constexpr float GROW = 8.f;  // log2 of the growth that moves the maximum
// log2 of the weight of a score at that maximum.  fp16 has all its bits from
// 2^-14 to 2^16 only, so its weights go up to 2^15 and those down to 2^-21 of the
// maximum's keep their 11 bits; bf16 has the range of float32.  The sums are of
// the same scale, so the result does not know of it.
template <class T>
constexpr float LIFT = std::is_same<T, __half>::value ? 15.f - GROW : 0.f;

template <int D>
struct Lay {
  static constexpr int NT = 2 * D / 64;   // 64-column tiles of an operand
  static constexpr int QB = NT * QTILE;   // bytes of a query tile
  static constexpr int KB = NT * KTILE;   // bytes of a block of K or V
  static constexpr int OFF_Q = 0;         // [2]
  static constexpr int OFF_K = 2 * QB;    // [KV]
  static constexpr int OFF_V = OFF_K + KV * KB;  // [KV]
  static constexpr int OFF_OUT = OFF_V + KV * KB;  // results on their way out [4 warps][32 rows][64]
  static constexpr int OFF_L = OFF_OUT + 4 * 4096;  // sums [2 tiles][2 maps][128]
  static constexpr int OFF_RING = OFF_L + 2 * 2 * 128 * 4;
  static constexpr int OFF_ITEM = OFF_RING + RING * 16;  // the answer that holds the next item
  static constexpr int OFF_OFFS = OFF_ITEM + 16;
  static constexpr int OFF_BAR = OFF_OFFS + (OFFS + 2) * 4;
  // q_full q_empty [2 each], k_full k_empty v_full v_empty [KV each], s_full
  // p_full [2 maps][2], o_done [2], o_full o_empty, sum_full sum_empty [2 each],
  // ring_full ring_empty [RING], turn [2 maps][4 quarters], next item
  static constexpr int B_Q = 0, B_K = 4, B_V = B_K + 2 * KV, B_S = B_V + 2 * KV, B_P = B_S + 4, B_D = B_P + 4,
                       B_O = B_D + 2, B_R = B_O + 6, B_T = B_R + 2 * RING, NBAR = B_T + 9;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory of one CTA");
};

__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%"
      "20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// D (TMEM) (+)= A (TMEM: lane = row, two 16-bit values of K per column) . B.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
// The norm's weights as a kernel parameter: reads from shared memory wait in the
// queue behind the exponentials.
template <int W>
struct NormWeight {
  float w[W];
};

// The maximum that weights refer to: scores that are all -inf so far have
// weight 0 (0 - 0 would be NaN), and a row of nothing else ends with 0 / 0.
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }

template <class T, int D>
__global__ void __launch_bounds__(NTHREADS, 1)
    diff_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_o,
                   const __grid_constant__ NormWeight<2 * D> norm, DiffParams p) {
  using L = Lay<D>;
  constexpr int NT = L::NT, W = 2 * D;
  constexpr uint32_t FMT = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0;
  constexpr uint32_t IDESC_S = idesc_f16(BQ, BKEY) | FMT;
  constexpr uint32_t IDESC_O = idesc_f16(BQ, W) | FMT | (1u << 16);  // B (V) MN-major
  constexpr uint32_t TM_O = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem), bar0 = sbase + L::OFF_BAR;
  auto q_full = [&](int s) { return bar0 + 8 * (L::B_Q + s); };
  auto q_empty = [&](int s) { return bar0 + 8 * (L::B_Q + 2 + s); };
  auto k_full = [&](int s) { return bar0 + 8 * (L::B_K + s); };
  auto k_empty = [&](int s) { return bar0 + 8 * (L::B_K + KV + s); };
  auto v_full = [&](int s) { return bar0 + 8 * (L::B_V + s); };
  auto v_empty = [&](int s) { return bar0 + 8 * (L::B_V + KV + s); };
  auto s_full = [&](int i, uint32_t b) { return bar0 + 8 * (L::B_S + 2 * i + (b & 1)); };
  auto p_full = [&](int i, uint32_t b) { return bar0 + 8 * (L::B_P + 2 * i + (b & 1)); };
  auto o_done = [&](int i) { return bar0 + 8 * (L::B_D + i); };
  const uint32_t o_full = bar0 + 8 * L::B_O, o_empty = o_full + 8;
  auto sum_full = [&](uint32_t n) { return bar0 + 8 * (L::B_O + 2 + (n & 1)); };
  auto sum_empty = [&](uint32_t n) { return bar0 + 8 * (L::B_O + 4 + (n & 1)); };
  auto ring_full = [&](int e) { return bar0 + 8 * (L::B_R + e); };
  auto ring_empty = [&](int e) { return bar0 + 8 * (L::B_R + RING + e); };
  auto turn = [&](int i, int q) { return bar0 + 8 * (L::B_T + 4 * i + q); };
  const uint32_t item_bar = turn(0, 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC + 4);
  int4* ring = reinterpret_cast<int4*>(smem + L::OFF_RING);  // {t0, len, q0, head}, len 0: no more
  DevStatus* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; i++) {
      mbar_init(q_full(i), 1);
      mbar_init(q_empty(i), 2);  // the two maps' MMAs
      mbar_init(o_done(i), 1);
      for (int b = 0; b < 2; b++) {
        mbar_init(s_full(i, b), 1);
        mbar_init(p_full(i, b), 4);
      }
    }
    for (int s = 0; s < KV; s++) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 2);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 2);
    }
    mbar_init(o_full, 2);
    for (int i = 0; i < 9; i++) mbar_init(turn(0, i), 1);  // and item_bar
    mbar_init(o_empty, 4);
    for (int i = 0; i < 2; i++) {
      mbar_init(sum_full(i), 8);
      mbar_init(sum_empty(i), 4);
    }
    for (int e = 0; e < RING; e++) {
      mbar_init(ring_full(e), 1);
      mbar_init(ring_empty(e), 15);  // producer, two MMA, eight softmax, four epilogue warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  // No pdl_trigger: the next kernel waits for this one's CTAs, started or
  // cancelled, to be done.

  // The next tile of the ring, for a whole warp; false at the end.
  auto next_tile = [&](uint32_t n, int4& tile) -> bool {
    const int e = n % RING;
    if (!__all_sync(0xffffffffu, mbar_wait(ring_full(e), (n / RING) & 1, abort_flag, status, 60))) return false;
    tile = ring[e];
    __syncwarp();
    if (lane == 0) mbar_arrive(ring_empty(e));
    return tile.y > 0;
  };

  // 512 threads of 128 registers at launch: 56 + 2 * 128 + 200 = 4 * 128.  Short
  // tiles wait for the epilogue, whose 128 results a thread and two loads of 32
  // columns need the most (256 texts of 16 to 128: 54 us with 144 and 168
  // registers, loads of 16 and weights in shared memory, 49 to 51 us so).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 3) {
      // -------------------------------------------------------------- tiles
      uint32_t n = 0;
      auto publish = [&](int4 t) -> bool {
        const int e = n % RING;
        if (!__all_sync(0xffffffffu, mbar_wait(ring_empty(e), ((n / RING) & 1) ^ 1, abort_flag, status, 61)))
          return false;
        if (lane == 0) {
          ring[e] = t;
          mbar_arrive(ring_full(e));
        }
        n++;
        return true;
      };
      auto ring_free = [&]() -> bool {  // every reader has taken the last tile
        return __all_sync(0xffffffffu, mbar_wait(ring_empty((n - 1) % RING), ((n - 1) / RING) & 1, abort_flag, status,
                                                 82)) != 0;
      };
      const int32_t* offsets = p.offsets;
      if (p.nseq <= OFFS) {
        int32_t* copy = reinterpret_cast<int32_t*>(smem + L::OFF_OFFS);
        for (int s = lane; s <= p.nseq; s += 32) copy[s] = p.offsets[s];
        __syncwarp();
        offsets = copy;
      }
      // The first item is the CTA's own; further ones are CTAs of the grid that
      // have not started, cancelled one at a time, so that the items go to
      // whichever SM is free.  The next is asked for while this one is looked
      // up, but behind a long tile only when every reader has taken it: what
      // a CTA holds, no other can do.
      const uint32_t answer = sbase + L::OFF_ITEM;
      auto ask = [&]() {
        if (lane == 0) {
          mbar_expect_tx(item_bar, 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::
                           "r"(answer),
                       "r"(item_bar)
                       : "memory");
        }
        __syncwarp();
      };
      Where w{};
      int last = -1;
      bool found = false, ok = true, asked = false;
      uint32_t item = blockIdx.x;
      for (uint32_t k = 0;; k++) {
        const int tile = (int)(item / (uint32_t)p.heads), head = (int)(item - (uint32_t)tile * p.heads);
        if (item == 0) check_offsets(p);  // whichever CTA has it: the first may itself be cancelled
        if (tile != last) found = find_block(p, offsets, tile, BQ, w);
        last = tile;
        asked = !found || w.len <= AHEAD * BKEY;
        if (asked) ask();
        if (found) ok = publish(make_int4(w.t0, w.len, w.q0, head));
        if (!asked) {
          ok = ok && ring_free();
          if (ok) ask();
        }
        if (!ok) break;
        ok = __all_sync(0xffffffffu, mbar_wait(item_bar, k & 1, abort_flag, status, 81));
        if (!ok) break;
        uint64_t lo, hi;
        uint32_t more;
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(answer) : "memory");
        asm volatile(
            "{\n.reg .b128 a;\n.reg .pred p;\nmov.b128 a, {%2, %3};\n"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\nselp.u32 %0, 1, 0, p;\n"
            "mov.u32 %1, 0;\n"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n}\n"
            : "=r"(more), "=&r"(item)
            : "l"(lo), "l"(hi));
        // Every lane has read the answer before lane 0 asks for the next one,
        // which overwrites it.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (!more) break;
      }
      if (ok) publish(make_int4(0, 0, 0, 0));
    } else if (warp == 0) {
      // ----------------------------------------------------------- producer
      const bool issuer = elect_one();
      uint32_t n = 0, ib = 0;  // tiles, key blocks
      int4 t;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, uint32_t dst, int bytes, int col, int row, uint32_t bar) {
        mbar_expect_tx(bar, NT * bytes);
#pragma unroll
        for (int c = 0; c < NT; c++) tma_load_2d(dst + c * bytes, map, col + c * 64, row, bar);
      };
      while (ok && next_tile(n, t)) {
        const int qs = n & 1, kcol = t.w / p.group * W, nkb = (t.y + BKEY - 1) / BKEY;
        ok = __all_sync(0xffffffffu, mbar_wait(q_empty(qs), ((n >> 1) & 1) ^ 1, abort_flag, status, 62));
        if (!ok) break;
        if (issuer) load(&tmap_q, sbase + L::OFF_Q + qs * L::QB, QTILE, t.w * W, t.x + t.z, q_full(qs));
        for (int j = 0; j < nkb && ok; j++, ib++) {
          const int s = ib % KV, row = t.x + j * BKEY;
          const uint32_t ph = ((ib / KV) & 1) ^ 1;
          ok = __all_sync(0xffffffffu, mbar_wait(k_empty(s), ph, abort_flag, status, 63));
          if (!ok) break;
          if (issuer) load(&tmap_k, sbase + L::OFF_K + s * L::KB, KTILE, kcol, row, k_full(s));
          ok = __all_sync(0xffffffffu, mbar_wait(v_empty(s), ph, abort_flag, status, 64));
          if (!ok) break;
          if (issuer) load(&tmap_v, sbase + L::OFF_V + s * L::KB, KTILE, kcol, row, v_full(s));
        }
        n++;
      }
    } else {
      // ---------------------------------------------------------------- MMA
      const int i = warp - 1;  // map
      const bool issuer = elect_one();
      const uint32_t s_tm = tmem + i * 128, o_tm = tmem + TM_O + i * W;
      uint32_t n = 0, ib = 0;
      int4 t;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int site) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, site));
        return ok;
      };
      // Operand descriptors (their addresses count 16-byte units).  Map i of an
      // operand with d = 64 is a tile of its own, with d = 32 half of the
      // 128-byte rows.  V [keys][64] tiles side by side: KTILE bytes from one
      // 64-column group to the next (leading offset), 16 keys = 2048 bytes.
      const uint64_t q0 = sw128_desc(sbase + L::OFF_Q + i * (D == 64 ? QTILE : 64));
      const uint64_t k0 = sw128_desc(sbase + L::OFF_K + i * (D == 64 ? KTILE : 64));
      const uint64_t v0 = (sw128_desc(sbase + L::OFF_V) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(KTILE >> 4) << 16);
      // The scores run two blocks ahead of the values, into the next tiles too:
      // S of block b + 2 goes out behind P.V of block b, whose buffer it takes.
      uint32_t sn = 0, sb = 0;  // tiles and blocks whose scores are issued
      bool ended = false;
      int s_left = 0;           // blocks of the last of those tiles without scores
      int len1 = 0, len2 = 0;   // lengths of the tiles between (at most two)
      auto scores = [&]() {
        if (s_left == 0) {
          if (!next_tile(sn, t)) {
            ended = true;
            return;
          }
          s_left = (t.y + BKEY - 1) / BKEY;
          if (len1 == 0)
            len1 = t.y;
          else
            len2 = t.y;
          if (!wait(q_full(sn & 1), (sn >> 1) & 1, 65)) return;
          sn++;
        }
        s_left--;
        // Once its keys are there; then they are free, with the tile's last
        // block the queries too.
        if (!wait(k_full(sb % KV), (sb / KV) & 1, 66)) return;
        tc_fence_after();
        if (issuer) {
          const uint32_t qs = (sn - 1) & 1;
          const uint64_t qd = q0 + qs * (L::QB / 16), kd = k0 + (sb % KV) * (L::KB / 16);
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)
            mma_f16(s_tm + (sb & 1) * BKEY, qd + 2 * kk, kd + 2 * kk, IDESC_S, kk != 0);
          mma_commit(s_full(i, sb));
          mma_commit(k_empty(sb % KV));
          if (s_left == 0) mma_commit(q_empty(qs));
        }
        __syncwarp();
        sb++;
      };
      scores();
      if (ok && !ended) scores();
      while (ok && ib < sb) {
        const int len = len1, nkb = (len + BKEY - 1) / BKEY;
        len1 = len2;
        len2 = 0;
        if (!wait(o_empty, (n & 1) ^ 1, 68)) break;
        for (int j = 0; j < nkb && ok; j++, ib++) {
          const int left = len - j * BKEY, steps = min(BKEY, left + 15) / 16;
          if (!wait(v_full(ib % KV), (ib / KV) & 1, 67)) break;
          if (!wait(p_full(i, ib), (ib >> 1) & 1, 73)) break;
          tc_fence_after();
          if (issuer) {
            const uint64_t vd = v0 + (ib % KV) * (L::KB / 16);
            const uint32_t pt = s_tm + (ib & 1) * BKEY;
            if (steps == BKEY / 16) {
#pragma unroll
              for (int kk = 0; kk < BKEY / 16; kk++)
                mma_ts(o_tm, pt + kk * 8, vd + kk * (2048 / 16), IDESC_O, j != 0 || kk != 0);
            } else {
              for (int kk = 0; kk < steps; kk++)
                mma_ts(o_tm, pt + kk * 8, vd + kk * (2048 / 16), IDESC_O, j != 0 || kk != 0);
            }
            mma_commit(o_done(i));
            mma_commit(v_empty(ib % KV));
            if (j + 1 == nkb) mma_commit(o_full);
          }
          __syncwarp();
          if (!ended) scores();
        }
        n++;
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    // -------------------------------------------------------------- softmax
    const int map = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t to = tmem + TM_O + map * W + lanes;
    const float scale = 1.4426950408889634f * rsqrtf((float)D);
    const unsigned long long scale2 = f2_pack(scale, scale);
    float* sums = reinterpret_cast<float*>(smem + L::OFF_L);
    uint32_t n = 0, ib = 0;
    int4 t;
    bool ok = true;
    while (ok && next_tile(n, t)) {
      const int nkb = (t.y + BKEY - 1) / BKEY;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nkb; j++, ib++) {
        const uint32_t ts = tmem + map * 128 + (ib & 1) * BKEY + lanes;
        ok = __all_sync(0xffffffffu, mbar_wait(s_full(map, ib), (ib >> 1) & 1, abort_flag, status, 74));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[BKEY];
        ld32(ts, r);
        ld32(ts + 32, r + 32);
        wait_ld();
        const int left = t.y - j * BKEY;  // keys of this block and behind
        if (left < BKEY) {
#pragma unroll
          for (int e = 0; e < BKEY; e++) r[e] = e < left ? r[e] : 0xff800000u;
        }
        float m0 = m, m1 = __uint_as_float(r[0]), m2 = __uint_as_float(r[1]), m3 = __uint_as_float(r[2]);
#pragma unroll
        for (int e = 0; e < BKEY; e += 8) {
          m0 = max3(m0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
          m1 = max3(m1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
          m2 = max3(m2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
          m3 = max3(m3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
        }
        m0 = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        if (j == 0) {
          m = m0;
        } else if (__any_sync(0xffffffffu, (m0 - m) * scale > GROW)) {
          const float f = ex2((m - finite(m0)) * scale);
          const unsigned long long f2 = f2_pack(f, f);
          // The result of the blocks before, complete.
          ok = __all_sync(0xffffffffu, mbar_wait(o_done(map), (ib - 1) & 1, abort_flag, status, 79));
          if (!ok) break;
          tc_fence_after();
          m = m0;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < W; c += 16) {
            float v[16];
            uint32_t w[16];
            tmem_ld16(to + c, v);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float a, b;
              f2_unpack(f2_mul(f2_pack(v[e], v[e + 1]), f2), a, b);
              w[e] = __float_as_uint(a);
              w[e + 1] = __float_as_uint(b);
            }
            st16(to + c, w);
          }
        }
        const float from = fmaf(-finite(m), scale, LIFT<T>);
        const unsigned long long off = f2_pack(from, from);
#pragma unroll
        for (int e = 0; e < BKEY; e += 2) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), scale2, off), x0, x1);
          r[e] = __float_as_uint(x0);
          r[e + 1] = __float_as_uint(x1);
        }
        // The maps take turns at the exponentials, so that one's other work
        // runs beside them; the turn is passed on a little before the end.
        ok = __all_sync(0xffffffffu, mbar_wait(turn(map, quarter), (ib & 1) ^ (map ^ 1), abort_flag, status, 80));
        if (!ok) break;
#pragma unroll
        for (int e = 0; e < BKEY; e++) {
          if (e == BKEY - 12) {
            __syncwarp();
            if (lane == 0) mbar_arrive(turn(map ^ 1, quarter));
          }
          r[e] = __float_as_uint(ex2(__uint_as_float(r[e])));
        }
        unsigned long long s0 = 0, s1 = 0;
#pragma unroll
        for (int c = 0; c < BKEY; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float x0 = __uint_as_float(r[c + 2 * e]), x1 = __uint_as_float(r[c + 2 * e + 1]);
            w[e] = pack2<T>(x0, x1);
            if (e & 1)
              s1 = f2_add(s1, f2_pack(x0, x1));
            else
              s0 = f2_add(s0, f2_pack(x0, x1));
          }
          st16(ts + c / 2, w);
        }
        float a, b;
        f2_unpack(f2_add(s0, s1), a, b);
        l += a + b;
        if (left < BKEY && left % 16 != 0) {
          // The values between the last key and the end of its 16 (both maps'
          // threads write the same zeros, each before its own product).
          ok = __all_sync(0xffffffffu, mbar_wait(v_full(ib % KV), (ib / KV) & 1, abort_flag, status, 75));
          if (!ok) break;
          const int rows = 16 - left % 16;
          uint8_t* v = smem + L::OFF_V + (ib % KV) * L::KB + left * 128;
          for (int e = row; e < rows * 8 * NT; e += 128)
            *reinterpret_cast<uint4*>(v + e / (rows * 8) * KTILE + e % (rows * 8) * 16) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(map, ib));
      }
      if (!ok) break;
      // The row's sum, for the epilogue: two buffers, since the softmax of short
      // tiles runs ahead of the results.
      ok = __all_sync(0xffffffffu, mbar_wait(sum_empty(n), ((n >> 1) & 1) ^ 1, abort_flag, status, 78));
      if (!ok) break;
      sums[(n & 1) * 256 + map * 128 + row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_full(n));
      n++;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ------------------------------------------------------------- epilogue
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t o1 = tmem + TM_O + ((uint32_t)(quarter * 32) << 16);
    const float* sums = reinterpret_cast<const float*>(smem + L::OFF_L);
    const uint32_t stage = sbase + L::OFF_OUT + quarter * 4096;
    uint32_t n = 0;
    int4 t;
    while (next_tile(n, t)) {
      const float lambda = p.lambda[t.w];
      if (!__all_sync(0xffffffffu, mbar_wait(sum_full(n), (n >> 1) & 1, abort_flag, status, 77)) ||
          !__all_sync(0xffffffffu, mbar_wait(o_full, n & 1, abort_flag, status, 76)))
        break;
      tc_fence_after();
      const float* sum = sums + (n & 1) * 256;
      const float w1 = 1.f / sum[row], w2 = -lambda / sum[128 + row];
      const unsigned long long w1s = f2_pack(w1, w1), w2s = f2_pack(w2, w2);
      unsigned long long o[W / 2], ss2 = 0;
#pragma unroll
      for (int c = 0; c < W; c += EPI) {
        uint32_t a[EPI], b[EPI];
        ld32(o1 + c, a);
        ld32(o1 + W + c, b);
        wait_ld();
#pragma unroll
        for (int e = 0; e < EPI; e += 2) {
          unsigned long long& x = o[(c + e) / 2];
          x = f2_fma(f2_pack(__uint_as_float(a[e]), __uint_as_float(a[e + 1])), w1s,
                     f2_mul(f2_pack(__uint_as_float(b[e]), __uint_as_float(b[e + 1])), w2s));
          ss2 = f2_fma(x, x, ss2);
        }
      }
      tc_fence_before();  // all read: the next tile's values may come
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(o_empty);
        mbar_arrive(sum_empty(n));
      }
      if (p.norm_w) {
        float s0, s1;
        f2_unpack(ss2, s0, s1);
        const float f = p.out_scale * rsqrtf((s0 + s1) * (1.f / W) + p.eps);
#pragma unroll
        for (int c = 0; c < W; c += 2) o[c / 2] = f2_mul(o[c / 2], f2_pack(f * norm.w[c], f * norm.w[c + 1]));
      }
      // 64 columns at a time; a warp whose 32 rows are all the sequence's
      // stores them through shared memory with TMA, others row by row.
      const bool whole = t.z + quarter * 32 + 32 <= t.y;
#pragma unroll
      for (int c = 0; c < W; c += 64) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; e++) {
          float x, y;
          f2_unpack(o[c / 2 + e], x, y);
          w[e] = pack2<T>(x, y);
        }
        if (whole) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; q++)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((q ^ (lane & 7)) << 4)),
                         "r"(w[4 * q]), "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                         : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) tma_store_2d(&tmap_o, stage, t.w * W + c, t.x + t.z + quarter * 32);
        } else if (t.z + row < t.y) {
          uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (long)(t.x + t.z + row) * p.o_stride +
                                                (long)t.w * W + c);
#pragma unroll
          for (int q = 0; q < 8; q++) out[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        }
      }
      n++;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    settle(abort_flag);
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
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

template <class T, int D>
static cudaError_t launch(const DiffParams& p, cudaStream_t s) {
  auto enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  auto encode = [&](CUtensorMap* map, const void* ptr, int heads, long ld, int rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)heads * 2 * D, (cuuint64_t)p.T};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)rows};
    const cuuint32_t estr[2] = {1, 1};
    const auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  CUtensorMap mq, mk, mv, mo;
  const int kvh = p.heads / p.group;
  if (!encode(&mq, p.q, p.heads, p.q_stride, BQ) || !encode(&mk, p.k, kvh, p.k_stride, BKEY) || !encode(&mv, p.v, kvh, p.v_stride, BKEY) ||
      !encode(&mo, p.out, p.heads, p.o_stride, 32))
    return cudaErrorInvalidValue;
  static std::mutex mu;
  static uint64_t attr_set = 0;  // per-device bit: the attribute is a per-device setting
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(attr_set >> dev & 1)) {
      const cudaError_t e =
          cudaFuncSetAttribute(diff_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::ALLOC);
      if (e != cudaSuccess) return e;
      if (dev < 64) attr_set |= 1ull << dev;
    }
  }
  const int tiles = block_count(p.T, p.nseq, BQ);
  const long items = (long)tiles * p.heads;
  if (items > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)items), dim3(NTHREADS),
                                            Lay<D>::ALLOC, s, attr);
  NormWeight<2 * D> norm = {};
  if (p.norm_w) std::copy_n(p.norm_host, 2 * D, norm.w);
  return cudaLaunchKernelEx(&cfg, diff_tc_kernel<T, D>, mq, mk, mv, mo, norm, p);
}

}  // namespace dtc

cudaError_t launch_diff_attention_tc(int dt, int d, const DiffParams& p, cudaStream_t s) {
  if (p.nseq == 0 || p.T == 0) return cudaSuccess;
  if (dt == DT_F16) return d == 64 ? dtc::launch<__half, 64>(p, s) : dtc::launch<__half, 32>(p, s);
  return d == 64 ? dtc::launch<__nv_bfloat16, 64>(p, s) : dtc::launch<__nv_bfloat16, 32>(p, s);
}

}  // namespace le
