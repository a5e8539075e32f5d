// Differential attention over packed sequences (mma.sync tiles):
//   A_i = softmax(q_i k_i^T / sqrt(d)), i = 1, 2
//   o   = (A_1 - lambda A_2) v
//   out = (1 - lambda_init) o rsqrt(mean(o^2) + eps) w     (o itself without w)
// for every head, whose two query and key parts have d columns each and whose
// values have 2d.
//
// For short sequences, where a call is bound by latency, by instructions and by
// how many sequences are in flight: a CTA of four or eight warps holds 64 or 128
// rows of Q, K and V, which are one head of a text that long or several heads of
// a shorter one; a warp has 16 query rows.  The scores stay in registers, so the
// maxima and sums are known before the second product, and it runs once, on
// P = P_1 / l_1 - lambda P_2 / l_2, rounded to the operands' type (16 bits, in
// the upper part of fp16's range); the sums are not.  Longer sequences (a caller whose hint of the longest was too
// small) take the same steps block by block, in two passes: maxima and sums,
// then weights and values.
// Spilled registers: none in the 64-row kernels' own path, 44 to 80 bytes in the
// 128-row ones (both maps of 128 keys), the rest in that of longer sequences.
// Keys past the sequence get weight 0 and their values are zeros in shared
// memory, whatever the rows behind hold.
#include <mutex>
#include <type_traits>

#include "diff_attention.cuh"

namespace le {
namespace dif {

constexpr int BKEY = 64;  // keys per block; a CTA has ROWS (64 or 128) rows and a warp for each 16

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

// ROWS rows of a tile, 2^lg to a head: row r is token r % 2^lg of head r / 2^lg,
// from src + token * ld + head * W; tokens from `n` on and heads from `heads` on
// are zero.  `group` query heads share a head of src.  A thread keeps its chunk
// and goes down the rows in steps whose token and head are the same for the
// whole CTA.
template <int W, int ROWS, class T>
__device__ __forceinline__ void load_tile(uint32_t base, const T* src, long ld, int lg, int n, int head0, int heads,
                                          int group) {
  constexpr int CH = W / 8, STEP = ROWS * 2 / CH;  // rows that the CTA's threads cover: at most 2^lg
  const int r0 = threadIdx.x / CH, c = threadIdx.x % CH;
  const T* mine = src + (long)r0 * ld + c * 8;
  const uint32_t dst = at<W>(base, r0, c);
#pragma unroll
  for (int r = 0; r < ROWS; r += STEP) {
    const int token = r & ((1 << lg) - 1), head = head0 + (r >> lg);
    const int h = group == 1 ? head : head / group;
    const bool in = token + r0 < n && head < heads;
    const T* g = in ? mine + (long)token * ld + h * W : src;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + r * (W * 2)), "l"(g), "r"(in ? 16 : 0));
  }
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Scores of a warp's 16 rows against keys key0 .. key0 + 63 of a tile (those of
// the first `left`; -inf behind), for part `i` of the head.
template <class T, int D>
__device__ __forceinline__ void scores(float (*s)[4], uint32_t sq, uint32_t sk, int i, int row0, int key0, int left) {
  constexpr int W = 2 * D;
  const int lane = threadIdx.x & 31, t = lane & 3;
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int c = 0; c < D / 16; c++) ldsm4(qa[c], at<W>(sq, row0 + (lane & 15), i * (D / 8) + 2 * c + (lane >> 4)));
#pragma unroll
  for (int n = 0; n < 8; n++) {
    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    if (n * 8 < left) {
#pragma unroll
      for (int c = 0; c < D / 16; c += 2) {
        uint32_t b[4];
        ldsm4(b, at<W>(sk, key0 + n * 8 + (lane & 7), i * (D / 8) + 2 * c + (lane >> 3)));
        mma16<T>(s[n], qa[c], b[0], b[1]);
        mma16<T>(s[n], qa[c + 1], b[2], b[3]);
      }
    }
    if (n * 8 + 8 > left) {
      const int key = n * 8 + 2 * t;
      if (key >= left) s[n][0] = s[n][2] = -INFINITY;
      if (key + 1 >= left) s[n][1] = s[n][3] = -INFINITY;
    }
  }
}

// A row pair's running maximum and sum of one map.
struct Stat {
  float m[2], l[2];
};

// The part of N tiles of eight keys in the statistics; s becomes exp2(scale (s - m)).
// Scores that are all -inf so far have weight 0 (0 - 0 would be NaN), and a row
// of nothing else ends with 0 / 0.
template <int N>
__device__ __forceinline__ void add_block(Stat& st, float (&s)[N][4], float scale) {
  float m0 = st.m[0], m1 = st.m[1];
#pragma unroll
  for (int n = 0; n < N; n++) {
    m0 = fmaxf(m0, fmaxf(s[n][0], s[n][1]));
    m1 = fmaxf(m1, fmaxf(s[n][2], s[n][3]));
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
  }
  const float f0 = m0 == -INFINITY ? 0.f : m0, f1 = m1 == -INFINITY ? 0.f : m1;
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int n = 0; n < N; n++) {
    s[n][0] = ex2f(fmaf(s[n][0], scale, -f0 * scale));
    s[n][1] = ex2f(fmaf(s[n][1], scale, -f0 * scale));
    s[n][2] = ex2f(fmaf(s[n][2], scale, -f1 * scale));
    s[n][3] = ex2f(fmaf(s[n][3], scale, -f1 * scale));
    l0 += s[n][0] + s[n][1];
    l1 += s[n][2] + s[n][3];
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
  }
  st.l[0] = fmaf(st.l[0], ex2f((st.m[0] - f0) * scale), l0);
  st.l[1] = fmaf(st.l[1], ex2f((st.m[1] - f1) * scale), l1);
  st.m[0] = m0;
  st.m[1] = m1;
}

// The power of two that P is multiplied by before its rounding, and the result
// divided by: P is at most 1 + |lambda| and as small as 1 / keys, and fp16 has all
// its bits from 2^-14 to 2^16 only, so P goes up to 2^15 and a bit; bf16 needs
// nothing.  Powers of two change no other rounding.
template <class T>
struct Lift {
  float up = 1.f, down = 1.f;
  __device__ __forceinline__ explicit Lift(float lambda) {
    if constexpr (std::is_same<T, __half>::value) {
      // 2^(14 - e) with 2^e <= max(1, |lambda|) < 2^(e + 1): P below 3 * 2^14
      const uint32_t e = (__float_as_uint(fmaxf(fabsf(lambda), 1.f)) >> 23) - 127;
      up = __uint_as_float((127 + 14 - e) << 23);
      down = __uint_as_float((127 - 14 + e) << 23);
    }
  }
};

// P = w1 a - w2 b of 64 keys as the second product's operand.
template <class T>
__device__ __forceinline__ void weights(uint32_t (*pa)[4], const float (*a)[4], const float (*b)[4], const float (&w1)[2],
                                        const float (&w2)[2]) {
#pragma unroll
  for (int n = 0; n < 8; n++) {
    pa[n / 2][2 * (n & 1)] = pack2<T>(fmaf(a[n][0], w1[0], -b[n][0] * w2[0]), fmaf(a[n][1], w1[0], -b[n][1] * w2[0]));
    pa[n / 2][2 * (n & 1) + 1] = pack2<T>(fmaf(a[n][2], w1[1], -b[n][2] * w2[1]), fmaf(a[n][3], w1[1], -b[n][3] * w2[1]));
  }
}

// o += P V for the first `left` of KEYS keys from key0.
template <class T, int W, int KEYS>
__device__ __forceinline__ void values(float (&o)[W / 8][4], const uint32_t (*pa)[4], uint32_t sv, int key0, int left) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < KEYS / 16; c++)
    if (c * 16 < left) {
#pragma unroll
      for (int n = 0; n < W / 8; n += 2) {
        uint32_t f[4];
        ldsm4_t(f, at<W>(sv, key0 + c * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n + (lane >> 4)));
        mma16<T>(o[n], pa[c], f[0], f[1]);
        mma16<T>(o[n + 1], pa[c], f[2], f[3]);
      }
    }
}

// Where a warp's 16 rows lie: in the tiles, and which head and tokens they are.
struct Rows {
  int row0, key0, head, first;
  bool work;  // any of them is the sequence's
};
__device__ __forceinline__ Rows rows_of(const DiffParams& p, const Where& wh, int lg, int head0) {
  Rows r;
  r.row0 = (threadIdx.x >> 5) * 16;
  r.key0 = r.row0 >> lg << lg;
  r.head = head0 + (r.row0 >> lg);
  r.first = wh.q0 + r.row0 - r.key0;
  r.work = r.head < p.heads && r.first < wh.len;
  return r;
}

// Scaled back (down) and normed, then out through the warp's own rows of the query tile: whole 16-byte
// chunks of a row instead of pairs of elements.
template <class T, int W>
__device__ __forceinline__ void finish(const DiffParams& p, const Where& wh, const Rows& rw, float (&o)[W / 8][4],
                                       uint32_t sq) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const float down = Lift<T>(__ldg(p.lambda + rw.head)).down;  // not held since the weights
  float r0 = down, r1 = down;
  if (p.norm_w) {
    float ss0 = 0.f, ss1 = 0.f;
#pragma unroll
    for (int n = 0; n < W / 8; n++) {
      ss0 = fmaf(o[n][0], o[n][0], fmaf(o[n][1], o[n][1], ss0));
      ss1 = fmaf(o[n][2], o[n][2], fmaf(o[n][3], o[n][3], ss1));
    }
#pragma unroll
    for (int e = 1; e < 4; e <<= 1) {
      ss0 += __shfl_xor_sync(0xffffffffu, ss0, e);
      ss1 += __shfl_xor_sync(0xffffffffu, ss1, e);
    }
    r0 *= p.out_scale * rsqrtf(ss0 * (down * down) / (float)W + p.eps);
    r1 *= p.out_scale * rsqrtf(ss1 * (down * down) / (float)W + p.eps);
  }
  __syncwarp();
#pragma unroll
  for (int n = 0; n < W / 8; n++) {
    float2 w = make_float2(1.f, 1.f);
    if (p.norm_w) w = __ldg(reinterpret_cast<const float2*>(p.norm_w + 8 * n + 2 * t));
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at<W>(sq, rw.row0 + g, n) + 4 * t),
                 "r"(pack2<T>(o[n][0] * r0 * w.x, o[n][1] * r0 * w.y))
                 : "memory");
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at<W>(sq, rw.row0 + g + 8, n) + 4 * t),
                 "r"(pack2<T>(o[n][2] * r1 * w.x, o[n][3] * r1 * w.y))
                 : "memory");
  }
  __syncwarp();
  T* out = static_cast<T*>(p.out) + (long)(wh.t0 + rw.first) * p.o_stride + (long)rw.head * W;
#pragma unroll
  for (int e = lane; e < 16 * (W / 8); e += 32) {
    const int r = e / (W / 8), c = e % (W / 8);
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(at<W>(sq, rw.row0 + r, c))
                 : "memory");
    if (rw.first + r < wh.len) *reinterpret_cast<uint4*>(out + (long)r * p.o_stride + c * 8) = x;
  }
}

__device__ __forceinline__ void clear(Stat& st) {
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
}

// A sequence of at most ROWS tokens: every key is in shared memory.  Of more
// than 64 keys, the first map's weights of all keys are kept and the second
// map's scores made twice, for its statistics and for its weights: both maps'
// would not fit the registers.
template <class T, int D, int ROWS>
__device__ __forceinline__ void short_rows(const DiffParams& p, const Where& wh, int lg, int head0, uint32_t sq) {
  constexpr int W = 2 * D, TILE = ROWS * W * 2;
  const uint32_t sk = sq + TILE, sv = sk + TILE;
  const T* q = static_cast<const T*>(p.q) + (long)wh.t0 * p.q_stride;
  const T* k = static_cast<const T*>(p.k) + (long)wh.t0 * p.k_stride;
  const T* v = static_cast<const T*>(p.v) + (long)wh.t0 * p.v_stride;
  load_tile<W, ROWS>(sq, q, p.q_stride, lg, wh.len, head0, p.heads, 1);
  load_tile<W, ROWS>(sk, k, p.k_stride, lg, wh.len, head0, p.heads, p.group);
  commit_copies();
  load_tile<W, ROWS>(sv, v, p.v_stride, lg, wh.len, head0, p.heads, p.group);
  commit_copies();
  const Rows rw = rows_of(p, wh, lg, head0);
  const float scale = 1.4426950408889634f * rsqrtf((float)D);
  const float lambda = rw.work ? p.lambda[rw.head] : 0.f;
  const Lift<T> lift(lambda);
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  __syncthreads();
  uint32_t pa[ROWS / 16][4];
  if (rw.work) {
    Stat st[2];
    clear(st[0]);
    clear(st[1]);
    if (ROWS == BKEY || wh.len <= BKEY) {
      float s[2][8][4];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        scores<T, D>(s[i], sq, sk, i, rw.row0, rw.key0, wh.len);
        add_block<8>(st[i], s[i], scale);
      }
      const float w1[2] = {lift.up / st[0].l[0], lift.up / st[0].l[1]};
      const float w2[2] = {lift.up * lambda / st[1].l[0], lift.up * lambda / st[1].l[1]};
      weights<T>(pa, s[0], s[1], w1, w2);
    } else if constexpr (ROWS > BKEY) {
      float a[16][4], s[8][4];
      scores<T, D>(a, sq, sk, 0, rw.row0, 0, wh.len);
      scores<T, D>(a + 8, sq, sk, 0, rw.row0, BKEY, wh.len - BKEY);
      add_block<16>(st[0], a, scale);
#pragma unroll 1
      for (int j = 0; j < 2; j++) {
        scores<T, D>(s, sq, sk, 1, rw.row0, j * BKEY, wh.len - j * BKEY);
        add_block<8>(st[1], s, scale);
      }
      const float w1[2] = {lift.up / st[0].l[0], lift.up / st[0].l[1]};
      const float w2[2] = {lift.up * lambda / st[1].l[0], lift.up * lambda / st[1].l[1]};
#pragma unroll
      for (int j = 0; j < 2; j++) {
        scores<T, D>(s, sq, sk, 1, rw.row0, j * BKEY, wh.len - j * BKEY);
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[n][e] = ex2f(fmaf(s[n][e], scale, -st[1].m[e >> 1] * scale));
        weights<T>(pa + 4 * j, a + 8 * j, s, w1, w2);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if (!rw.work) return;
  float o[W / 8][4];
#pragma unroll
  for (int n = 0; n < W / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  values<T, W, ROWS>(o, pa, sv, rw.key0, wh.len);
  finish<T, W>(p, wh, rw, o, sq);
}

// Queries wh.q0 .. wh.q0 + ROWS - 1 of a longer sequence and one head, in two
// passes over blocks of ROWS keys, 64 at a time.
template <class T, int D, int ROWS>
__device__ __noinline__ void long_rows(const DiffParams& p, const Where& wh, int head0, uint32_t sq) {
  constexpr int W = 2 * D, TILE = ROWS * W * 2, lg = ROWS == 64 ? 6 : 7;
  const uint32_t sk = sq + TILE, sv = sk + TILE;
  const T* q = static_cast<const T*>(p.q) + (long)(wh.t0 + wh.q0) * p.q_stride;
  const T* k = static_cast<const T*>(p.k) + (long)wh.t0 * p.k_stride;
  const T* v = static_cast<const T*>(p.v) + (long)wh.t0 * p.v_stride;
  const Rows rw = rows_of(p, wh, lg, head0);
  const float scale = 1.4426950408889634f * rsqrtf((float)D), lambda = p.lambda[head0];
  const Lift<T> lift(lambda);
  float o[W / 8][4];
#pragma unroll
  for (int n = 0; n < W / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  Stat st[2];
  clear(st[0]);
  clear(st[1]);
  load_tile<W, ROWS>(sq, q, p.q_stride, lg, wh.len - wh.q0, head0, p.heads, 1);
  for (int pass = 0; pass < 2; pass++) {
    float w1[2], w2[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      w1[r] = lift.up / st[0].l[r];
      w2[r] = lift.up * lambda / st[1].l[r];
    }
    for (int j = 0; j < wh.len; j += ROWS) {
      load_tile<W, ROWS>(sk, k + (long)j * p.k_stride, p.k_stride, lg, wh.len - j, head0, p.heads, p.group);
      if (pass == 1)
        load_tile<W, ROWS>(sv, v + (long)j * p.v_stride, p.v_stride, lg, wh.len - j, head0, p.heads, p.group);
      commit_copies();
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      for (int key0 = 0; key0 < ROWS && j + key0 < wh.len && rw.work; key0 += BKEY) {
        const int left = wh.len - j - key0;
        float s[2][8][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          scores<T, D>(s[i], sq, sk, i, rw.row0, key0, left);
          if (pass == 0) {
            add_block<8>(st[i], s[i], scale);
          } else {
#pragma unroll
            for (int n = 0; n < 8; n++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                s[i][n][e] = ex2f(fmaf(s[i][n][e], scale, -st[i].m[e >> 1] * scale));
          }
        }
        if (pass == 1) {
          uint32_t pa[BKEY / 16][4];
          weights<T>(pa, s[0], s[1], w1, w2);
          values<T, W, BKEY>(o, pa, sv, key0, left);
        }
      }
      __syncthreads();
    }
  }
  if (rw.work) finish<T, W>(p, wh, rw, o, sq);
}

// One CTA per sequence and ROWS rows of heads (of a longer sequence than the
// kernel is for: its query blocks in turn).
template <class T, int D, int ROWS>
__global__ void __launch_bounds__(ROWS * 2, ROWS == 128 ? 2 : D == 64 ? 4 : 5)
    diff_short_kernel(const __grid_constant__ DiffParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(128) uint8_t smem_diff[];
  const uint32_t sq = (uint32_t)__cvta_generic_to_shared(smem_diff);
  constexpr int TOP = ROWS == 64 ? 6 : 7;
  Where wh;
  if (!sequence(p, blockIdx.x, wh)) return;
  // 16 to ROWS rows of a head in the tiles, and no fewer than one step of
  // load_tile covers.
  int lg = ROWS == 128 && D == 32 ? 5 : 4;
  while (lg < TOP && wh.len > 1 << lg) lg++;
  const int head0 = blockIdx.y << (TOP - lg);
  if (head0 >= p.heads) return;
  if (wh.len <= ROWS) {
    short_rows<T, D, ROWS>(p, wh, lg, head0, sq);
    return;
  }
  for (; wh.q0 < wh.len; wh.q0 += ROWS) {
    long_rows<T, D, ROWS>(p, wh, head0, sq);
    __syncthreads();
  }
}

template <class T, int D, int ROWS>
static cudaError_t launch(const DiffParams& p, cudaStream_t s) {
  constexpr int SMEM = 3 * ROWS * 2 * D * 2;
  static std::mutex mu;
  static uint64_t attr_set = 0;  // per-device bit: the attribute is a per-device setting
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(attr_set >> dev & 1)) {
      const cudaError_t e =
          cudaFuncSetAttribute(diff_short_kernel<T, D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
      if (e != cudaSuccess) return e;
      if (dev < 64) attr_set |= 1ull << dev;
    }
  }
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = pdl_config(dim3(p.nseq, p.heads), dim3(ROWS * 2), SMEM, s, attr);
  return cudaLaunchKernelEx(&cfg, diff_short_kernel<T, D, ROWS>, p);
}
template <class T, int D>
static cudaError_t launch_rows(const DiffParams& p, int rows, cudaStream_t s) {
  return rows == 64 ? launch<T, D, 64>(p, s) : launch<T, D, 128>(p, s);
}

}  // namespace dif

static cudaError_t launch_short(int dt, int d, const DiffParams& p, int rows, cudaStream_t s) {
  if (dt == DT_F16) return d == 64 ? dif::launch_rows<__half, 64>(p, rows, s) : dif::launch_rows<__half, 32>(p, rows, s);
  return d == 64 ? dif::launch_rows<__nv_bfloat16, 64>(p, rows, s) : dif::launch_rows<__nv_bfloat16, 32>(p, rows, s);
}

// max_len, where it is known, tells the texts that this file's kernels are for;
// they are right for others too, and slow.  Measured (us, 6 heads of 64 and 12 of
// 32; 64 rows / 128 rows / tcgen05 tiles):
//   256 texts of 16:        8.8 / -  / 39       9.0 / -   / 54
//   256 of 64:              30  / 32 / 41       31  / 37  / 48
//   256 of 30 to 70:        -   / 39 / 45       -   / 45  / 64
//   256 of 40 to 90:        -   / 56 / 48       -   / 67  / 74
//   256 of 50 to 100:       -   / 65 / 49       -   / 78  / 78
//   256 of 128:             -   / 90 / 48       -   / 103 / 68
cudaError_t launch_diff_attention(int dt, int d, const DiffParams& p, int max_len, cudaStream_t s) {
  if (p.nseq == 0 || p.T == 0) return cudaSuccess;
  if (max_len > 0 && max_len <= 64) return launch_short(dt, d, p, 64, s);
  if (max_len > 0 && max_len <= 128 && (long)p.T < (d == 64 ? 56L : 75L) * p.nseq)
    return launch_short(dt, d, p, 128, s);
  return launch_diff_attention_tc(dt, d, p, s);
}

}  // namespace le
