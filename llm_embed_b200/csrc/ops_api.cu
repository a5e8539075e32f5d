// C ABI of the stand-alone operators (include/llmembed.h): handles, argument
// checks and dispatch.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <new>

#include "../../include/llmembed.h"
#include "common.cuh"
#include "elem.cuh"
#include "kernels.h"

using namespace le;

int le_fail(int code, const char* fmt, ...);

#define CK(call)                                                                                     \
  do {                                                                                               \
    cudaError_t e_ = (call);                                                                         \
    if (e_ != cudaSuccess) {                                                                         \
      cudaGetLastError();                                                                            \
      return le_fail(e_ == cudaErrorMemoryAllocation ? LE_ENOMEM : LE_ECUDA, "%s: %s (%s:%d)", #call, \
                     cudaGetErrorString(e_), __FILE__, __LINE__);                                    \
    }                                                                                                \
  } while (0)

#define TRY(call)               \
  do {                          \
    int r_ = (call);            \
    if (r_ != LE_OK) return r_; \
  } while (0)

// The Python binding packs these by field (llm_embed_b200/ops.py).
static_assert(sizeof(le_f8gemm_args) == 72 && sizeof(le_qk_norm_args) == 112 && sizeof(le_diffattn_args) == 88,
              "argument structures");

namespace {

// Makes `dev` current and the caller's device current again at the end.
struct DeviceGuard {
  int prev = -1;
  cudaError_t err;
  explicit DeviceGuard(int dev) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != dev)
      err = cudaSetDevice(dev);
    else
      prev = -1;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

struct Buf {
  void* p = nullptr;
  ~Buf() {
    if (p) cudaFree(p);
  }
  int alloc(size_t n) {
    CK(cudaMalloc(&p, n ? n : 16));
    return LE_OK;
  }
  template <class T>
  T* as() const {
    return static_cast<T*>(p);
  }
};

// What every operator's handle has: its device, its own stream, and one
// allocation with the status word that its kernels report to and its arrays
// behind (256-byte steps).
struct OpBase {
  int dev = 0;
  cudaStream_t stream = nullptr;
  Buf mem;
  static size_t step(size_t n) { return (n + 255) / 256 * 256; }
  int open(int d, size_t bytes) {
    dev = d;
    CK(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));
    TRY(mem.alloc(256 + bytes));
    CK(cudaMemsetAsync(mem.p, 0, sizeof(DevStatus), cudaStreamLegacy));
    return LE_OK;
  }
  template <class T>
  T* at(size_t offset) const {
    return reinterpret_cast<T*>(mem.as<uint8_t>() + 256 + offset);
  }
  ~OpBase() {
    if (stream) cudaStreamDestroy(stream);
  }
  cudaStream_t pick(void* s) const { return s ? static_cast<cudaStream_t>(s) : stream; }
  DevStatus* st() const { return mem.as<DevStatus>(); }
  int sync() {
    DeviceGuard g(dev);
    CK(g.err);
    CK(cudaDeviceSynchronize());
    DevStatus h{};
    CK(cudaMemcpy(&h, mem.p, sizeof h, cudaMemcpyDeviceToHost));
    if (h.code == DE_OK) return LE_OK;
    CK(cudaMemset(mem.p, 0, sizeof h));
    return le_fail(LE_EDEVICE, "kernel failure code %d at site %d (info %d)", h.code, h.where, h.info);
  }
};

// Whether `dev` is an sm_100 device (asked of the runtime once per device).
int usable_device(int dev) {
  static std::atomic<uint64_t> known{0};
  if (dev >= 0 && dev < 64 && (known.load(std::memory_order_relaxed) >> dev & 1)) return LE_OK;
  int n = 0, total = 0;
  TRY(le_init(&n));
  CK(cudaGetDeviceCount(&total));
  if (dev < 0 || dev >= total) return le_fail(LE_EINVAL, "device %d out of range (%d devices)", dev, total);
  cudaDeviceProp prop{};
  CK(cudaGetDeviceProperties(&prop, dev));
  if (prop.major != 10) return le_fail(LE_ECUDA, "device %d is not an sm_100 device", dev);
  if (dev < 64) known.fetch_or(1ull << dev, std::memory_order_relaxed);
  return LE_OK;
}

bool is_float_type(int t) { return t == LE_DT_F32 || t == LE_DT_F16 || t == LE_DT_BF16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t blocks128(int64_t n) { return (n + 127) / 128; }
// Rows and columns of the e4m3 operators and sequences of a call: the kernels
// count them in 32 bits, rounded up to whole tiles.
constexpr int MAX_DIM = 1 << 30;

// Frees a handle on its device, after its own stream's work.
template <class H>
int free_handle(H* h) {
  if (!h) return LE_OK;
  DeviceGuard g(h->dev);
  if (h->stream) cudaStreamSynchronize(h->stream);
  delete h;
  return LE_OK;
}

template <class H>
struct Owner {
  H* h = new (std::nothrow) H;
  ~Owner() { delete h; }
  H* release() {
    H* r = h;
    h = nullptr;
    return r;
  }
};

}  // namespace

struct le_f8weight : OpBase {
  int N = 0, K = 0;
  size_t w_bytes() const { return (size_t)N * K; }
  size_t ws_bytes() const { return (size_t)(blocks128(N) * blocks128(K)) * 4; }
  uint8_t* w() const { return at<uint8_t>(0); }
  float* ws() const { return at<float>(step(w_bytes())); }
};
struct le_rope : OpBase {
  int max_pos = 0, rot = 0, half_split = 0;
  size_t table_bytes() const { return (size_t)max_pos * (rot / 2) * 4; }
  float* cos() const { return at<float>(0); }
  float* sin() const { return at<float>(step(table_bytes())); }
};
struct le_diffattn : OpBase {
  int heads = 0, kv_heads = 0, d = 0;
  float out_scale = 1.f, eps = 0.f;
  bool norm = false;
  float norm_host[128] = {};
  float* lambda() const { return at<float>(0); }
  float* norm_w() const { return at<float>(step((size_t)heads * 4)); }
};

extern "C" {

// ---------------------------------------------------------------- e4m3 ----

int le_f8_quantize_device(int dev, int x_type, const void* d_x, int64_t ldx, int M, int K, uint8_t* d_q,
                          float* d_scales, void* stream) {
  if (M < 0 || K < 1 || M > MAX_DIM || K > MAX_DIM) return le_fail(LE_EINVAL, "bad shape (M %d, K %d)", M, K);
  if (!is_float_type(x_type)) return le_fail(LE_EINVAL, "x_type %d is not LE_DT_F32, LE_DT_F16 or LE_DT_BF16", x_type);
  if (ldx == 0) ldx = K;
  if (ldx < K) return le_fail(LE_EINVAL, "ldx %lld < K %d", (long long)ldx, K);
  if (M > 0 && (!d_x || !d_q || !d_scales)) return le_fail(LE_EINVAL, "null argument");
  if (!aligned(d_x, elem_size(x_type)) || !aligned(d_scales, 4))
    return le_fail(LE_EINVAL, "x or scales not aligned to their elements");
  TRY(usable_device(dev));
  DeviceGuard g(dev);
  CK(g.err);
  CK(launch_f8_quantize(x_type, d_x, ldx, M, K, d_q, d_scales,
                        stream ? static_cast<cudaStream_t>(stream) : cudaStreamLegacy));
  return LE_OK;
}

static int f8weight_open(int dev, const void* src, int N, int K, Owner<le_f8weight>& o) {
  if (!src) return le_fail(LE_EINVAL, "null argument");
  if (N < 1 || K < 16 || K % 16 || N > MAX_DIM || K > MAX_DIM)
    return le_fail(LE_EINVAL, "bad shape (N %d in [1, 2^30], K %d a multiple of 16 to 2^30)", N, K);
  TRY(usable_device(dev));
  if (!o.h) return le_fail(LE_ENOMEM, "out of host memory");
  return LE_OK;
}

static int f8weight_alloc(le_f8weight* w, int dev, int N, int K) {
  w->N = N;
  w->K = K;
  return w->open(dev, OpBase::step(w->w_bytes()) + w->ws_bytes());
}

int le_f8weight_create(int dev, const uint8_t* wq, const float* scales, int N, int K, le_f8weight** out) {
  if (!out) return le_fail(LE_EINVAL, "null argument");
  *out = nullptr;
  if (!scales) return le_fail(LE_EINVAL, "null argument");
  Owner<le_f8weight> o;
  TRY(f8weight_open(dev, wq, N, K, o));
  DeviceGuard g(dev);
  CK(g.err);
  TRY(f8weight_alloc(o.h, dev, N, K));
  CK(cudaMemcpy(o.h->w(), wq, o.h->w_bytes(), cudaMemcpyDefault));
  CK(cudaMemcpy(o.h->ws(), scales, o.h->ws_bytes(), cudaMemcpyDefault));
  CK(cudaStreamSynchronize(cudaStreamLegacy));
  *out = o.release();
  return LE_OK;
}

int le_f8weight_quantize(int dev, const float* w, int N, int K, le_f8weight** out) {
  if (!out) return le_fail(LE_EINVAL, "null argument");
  *out = nullptr;
  Owner<le_f8weight> o;
  TRY(f8weight_open(dev, w, N, K, o));
  DeviceGuard g(dev);
  CK(g.err);
  TRY(f8weight_alloc(o.h, dev, N, K));
  Buf src;
  TRY(src.alloc((size_t)N * K * 4));
  CK(cudaMemcpy(src.p, w, (size_t)N * K * 4, cudaMemcpyDefault));
  CK(launch_f8_quantize_weight(src.as<float>(), N, K, o.h->w(), o.h->ws(), cudaStreamLegacy));
  CK(cudaStreamSynchronize(cudaStreamLegacy));
  *out = o.release();
  return LE_OK;
}

int le_f8weight_read(le_f8weight* w, uint8_t* wq, float* scales) {
  if (!w) return le_fail(LE_EINVAL, "null argument");
  DeviceGuard g(w->dev);
  CK(g.err);
  if (wq) CK(cudaMemcpy(wq, w->w(), w->w_bytes(), cudaMemcpyDeviceToHost));
  if (scales) CK(cudaMemcpy(scales, w->ws(), w->ws_bytes(), cudaMemcpyDeviceToHost));
  return LE_OK;
}

// Quantised activations [M][K], then their scales on a 16-byte boundary.
static int64_t f8_work_scales_at(int64_t M, int64_t K) { return (M * K + 15) / 16 * 16; }

int le_f8gemm_workspace(const le_f8weight* w, int M, int x_type, int64_t* bytes) {
  if (!w || !bytes) return le_fail(LE_EINVAL, "null argument");
  if (M < 0 || M > MAX_DIM) return le_fail(LE_EINVAL, "M %d outside [0, 2^30]", M);
  if (x_type != LE_DT_E4M3 && !is_float_type(x_type)) return le_fail(LE_EINVAL, "unknown x_type %d", x_type);
  *bytes = x_type == LE_DT_E4M3 ? 0 : f8_work_scales_at(M, w->K) + blocks128(w->K) * M * 4;
  return LE_OK;
}

int le_f8gemm_tile(int M, int N) { return M <= 0 || N <= 0 ? 0 : M <= F8_SMALL_MAX_M ? 16 : f8_tile(M, N); }

int le_f8gemm_device(le_f8weight* w, const le_f8gemm_args* a, void* stream) {
  if (!w || !a) return le_fail(LE_EINVAL, "null argument");
  F8GemmParams p{};
  p.M = a->M;
  p.N = w->N;
  p.K = w->K;
  p.ldx = a->ldx ? a->ldx : w->K;
  p.ldy = a->ldy ? a->ldy : w->N;
  int64_t need = 0;
  TRY(le_f8gemm_workspace(w, a->M, a->x_type, &need));
  if (!is_float_type(a->y_type)) return le_fail(LE_EINVAL, "y_type %d is not LE_DT_F32, LE_DT_F16 or LE_DT_BF16", a->y_type);
  if (p.ldx < p.K || p.ldy < p.N) return le_fail(LE_EINVAL, "row stride shorter than a row");
  if (a->M == 0) return LE_OK;
  if (!a->x || !a->y || (a->x_type == LE_DT_E4M3 && !a->x_scales)) return le_fail(LE_EINVAL, "null argument");
  if (a->work_bytes < need || (need && !a->work))
    return le_fail(LE_EINVAL, "workspace of %lld bytes, %lld needed", (long long)a->work_bytes, (long long)need);
  if (need && !aligned(a->work, 16)) return le_fail(LE_EINVAL, "workspace not 16-byte aligned");
  if (!aligned(a->x, elem_size(a->x_type)) || !aligned(a->y, elem_size(a->y_type)) || !aligned(a->x_scales, 4))
    return le_fail(LE_EINVAL, "x, y or x_scales not aligned to its elements");
  if (a->x_type == LE_DT_E4M3 && (!aligned(a->x, 16) || p.ldx % 16))
    return le_fail(LE_EINVAL, "e4m3 rows of x must be 16-byte aligned");
  DeviceGuard g(w->dev);
  CK(g.err);
  const cudaStream_t s = w->pick(stream);
  p.x = a->x;
  p.xs = a->x_scales;
  p.w = w->w();
  p.ws = w->ws();
  p.y = a->y;
  int xt = a->x_type;
  // Up to F8_FUSED_MAX_M rows are quantised by the product's own kernel; more
  // are quantised once, before it.
  const bool small = p.M <= F8_SMALL_MAX_M;
  if (xt != LE_DT_E4M3 && (p.M > F8_FUSED_MAX_M || !aligned(p.x, 16) || (p.ldx * elem_size(xt)) % 16)) {
    uint8_t* q = static_cast<uint8_t*>(a->work);
    float* sc = reinterpret_cast<float*>(q + f8_work_scales_at(p.M, p.K));
    CK(launch_f8_quantize(xt, p.x, p.ldx, p.M, p.K, q, sc, s));
    p.x = q;
    p.xs = sc;
    p.ldx = p.K;
    xt = LE_DT_E4M3;
  }
  CK(small ? launch_f8_gemm_small(xt, a->y_type, p, s) : launch_f8_gemm_tc(a->y_type, p, w->st(), s));
  return LE_OK;
}

int le_f8weight_sync(le_f8weight* w) { return w ? w->sync() : le_fail(LE_EINVAL, "null argument"); }
int le_f8weight_free(le_f8weight* w) { return free_handle(w); }

// ------------------------------------------------- norm and rotation ------

int le_rope_create(int dev, int max_pos, int rot_dim, double base, int pairing, le_rope** out) {
  if (!out) return le_fail(LE_EINVAL, "null argument");
  *out = nullptr;
  if (max_pos < 1) return le_fail(LE_EINVAL, "max_pos %d < 1", max_pos);
  if (rot_dim < 0 || rot_dim > 256 || rot_dim % 2)
    return le_fail(LE_EINVAL, "rot_dim %d is not an even number in [0, 256]", rot_dim);
  if (!(base > 0) || !std::isfinite(base)) return le_fail(LE_EINVAL, "base must be positive and finite");
  if (pairing != LE_ROPE_INTERLEAVED && pairing != LE_ROPE_HALF) return le_fail(LE_EINVAL, "unknown pairing %d", pairing);
  TRY(usable_device(dev));
  Owner<le_rope> o;
  if (!o.h) return le_fail(LE_ENOMEM, "out of host memory");
  DeviceGuard g(dev);
  CK(g.err);
  o.h->max_pos = max_pos;
  o.h->rot = rot_dim;
  o.h->half_split = pairing == LE_ROPE_HALF;
  TRY(o.h->open(dev, OpBase::step(o.h->table_bytes()) + o.h->table_bytes()));
  CK(launch_rope_table(max_pos, rot_dim, base, o.h->cos(), o.h->sin(), cudaStreamLegacy));
  CK(cudaStreamSynchronize(cudaStreamLegacy));
  *out = o.release();
  return LE_OK;
}

int le_qk_norm_device(le_rope* r, const le_qk_norm_args* a, void* stream) {
  if (!r || !a) return le_fail(LE_EINVAL, "null argument");
  if (!is_float_type(a->type)) return le_fail(LE_EINVAL, "type %d is not LE_DT_F32, LE_DT_F16 or LE_DT_BF16", a->type);
  if (a->n_tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads > 65536 || a->k_heads > 65536)
    return le_fail(LE_EINVAL, "bad sizes (tokens %d, heads %d and %d)", a->n_tokens, a->q_heads, a->k_heads);
  if (a->head_dim < 1 || a->head_dim > 256 || a->head_dim < r->rot)
    return le_fail(LE_EINVAL, "head_dim %d outside [max(1, rot_dim %d), 256]", a->head_dim, r->rot);
  if (!(a->eps >= 0)) return le_fail(LE_EINVAL, "eps must not be negative");
  if (a->n_tokens == 0 || a->q_heads + a->k_heads == 0) return LE_OK;
  QkNormParams p{};
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  const int64_t qw = (int64_t)a->q_heads * a->head_dim, kw = (int64_t)a->k_heads * a->head_dim;
  p.q_stride = a->q_stride ? a->q_stride : qw;
  p.k_stride = a->k_stride ? a->k_stride : kw;
  p.qo_stride = a->q_out_stride ? a->q_out_stride : qw;
  p.ko_stride = a->k_out_stride ? a->k_out_stride : kw;
  if (p.q_stride < qw || p.k_stride < kw || p.qo_stride < qw || p.ko_stride < kw)
    return le_fail(LE_EINVAL, "token stride shorter than its heads");
  if ((a->q_heads && (!a->q || !a->q_out)) || (a->k_heads && (!a->k || !a->k_out)) || (r->rot && !a->positions))
    return le_fail(LE_EINVAL, "null argument");
  if ((a->q_heads && a->q == a->q_out && p.q_stride != p.qo_stride) ||
      (a->k_heads && a->k == a->k_out && p.k_stride != p.ko_stride))
    return le_fail(LE_EINVAL, "in place needs equal strides");
  const int es = elem_size(a->type);
  if (!aligned(a->q, es) || !aligned(a->k, es) || !aligned(a->q_out, es) || !aligned(a->k_out, es) ||
      !aligned(a->positions, 4) || !aligned(a->q_weight, 4) || !aligned(a->k_weight, 4))
    return le_fail(LE_EINVAL, "a pointer is not aligned to its elements");
  p.q_heads = a->q_heads;
  p.k_heads = a->k_heads;
  p.d = a->head_dim;
  p.rot = r->rot;
  p.half_split = r->half_split;
  p.max_pos = r->max_pos;
  p.q_weight = a->q_weight;
  p.k_weight = a->k_weight;
  p.cos = r->cos();
  p.sin = r->sin();
  p.positions = r->rot ? a->positions : nullptr;
  p.eps = a->eps;
  p.status = r->st();
  DeviceGuard g(r->dev);
  CK(g.err);
  CK(launch_qk_norm(a->type, p, a->n_tokens, r->pick(stream)));
  return LE_OK;
}

int le_rope_sync(le_rope* r) { return r ? r->sync() : le_fail(LE_EINVAL, "null argument"); }
int le_rope_free(le_rope* r) { return free_handle(r); }

// ------------------------------------------------ differential attention --

int le_diffattn_create(int dev, int heads, int kv_heads, int head_dim, const float* lambdas, int n_lambda,
                       float lambda_init, const float* norm_weight, float eps, le_diffattn** out) {
  if (!out) return le_fail(LE_EINVAL, "null argument");
  *out = nullptr;
  if (!lambdas) return le_fail(LE_EINVAL, "null argument");
  if (heads < 1 || heads > 65535 || kv_heads < 1 || heads % kv_heads)
    return le_fail(LE_EINVAL, "heads %d must be a positive multiple of kv_heads %d (<= 65535)", heads, kv_heads);
  if (head_dim != 32 && head_dim != 64) return le_fail(LE_EINVAL, "head_dim %d is not 32 or 64", head_dim);
  if (n_lambda != 1 && n_lambda != heads) return le_fail(LE_EINVAL, "n_lambda %d is neither 1 nor heads %d", n_lambda, heads);
  if (!(eps >= 0)) return le_fail(LE_EINVAL, "eps must not be negative");
  TRY(usable_device(dev));
  Owner<le_diffattn> o;
  if (!o.h) return le_fail(LE_ENOMEM, "out of host memory");
  DeviceGuard g(dev);
  CK(g.err);
  o.h->heads = heads;
  o.h->kv_heads = kv_heads;
  o.h->d = head_dim;
  o.h->out_scale = 1.f - lambda_init;
  o.h->eps = eps;
  o.h->norm = norm_weight != nullptr;
  TRY(o.h->open(dev, OpBase::step((size_t)heads * 4) + (size_t)2 * head_dim * 4));
  std::unique_ptr<float[]> lam(new (std::nothrow) float[heads]);
  if (!lam) return le_fail(LE_ENOMEM, "out of host memory");
  for (int i = 0; i < heads; i++) {
    const float* l = lambdas + (n_lambda == 1 ? 0 : (size_t)i * 4 * head_dim);
    double a = 0, b = 0;
    for (int j = 0; j < head_dim; j++) {
      a += (double)l[j] * l[head_dim + j];
      b += (double)l[2 * head_dim + j] * l[3 * head_dim + j];
    }
    lam[i] = (float)(std::exp(a) - std::exp(b) + (double)lambda_init);
  }
  CK(cudaMemcpy(o.h->lambda(), lam.get(), (size_t)heads * 4, cudaMemcpyHostToDevice));
  if (norm_weight) std::copy_n(norm_weight, 2 * head_dim, o.h->norm_host);
  if (norm_weight) CK(cudaMemcpy(o.h->norm_w(), norm_weight, (size_t)2 * head_dim * 4, cudaMemcpyHostToDevice));
  CK(cudaStreamSynchronize(cudaStreamLegacy));
  *out = o.release();
  return LE_OK;
}

int le_diffattn_device(le_diffattn* h, const le_diffattn_args* a, void* stream) {
  if (!h || !a) return le_fail(LE_EINVAL, "null argument");
  if (a->type != LE_DT_F16 && a->type != LE_DT_BF16) return le_fail(LE_EINVAL, "type %d is not LE_DT_F16 or LE_DT_BF16", a->type);
  if (a->nseq < 0 || a->nseq > MAX_DIM || a->n_tokens < 0 || a->max_len < 0)
    return le_fail(LE_EINVAL, "bad sizes (nseq %d, tokens %d, max_len %d)", a->nseq, a->n_tokens, a->max_len);
  if (a->nseq == 0 || a->n_tokens == 0) return LE_OK;
  DiffParams p{};
  const int64_t qw = (int64_t)h->heads * 2 * h->d, kw = (int64_t)h->kv_heads * 2 * h->d;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.q_stride = a->q_stride ? a->q_stride : qw;
  p.k_stride = a->k_stride ? a->k_stride : kw;
  p.v_stride = a->v_stride ? a->v_stride : kw;
  p.o_stride = a->out_stride ? a->out_stride : qw;
  if (p.q_stride < qw || p.k_stride < kw || p.v_stride < kw || p.o_stride < qw)
    return le_fail(LE_EINVAL, "token stride shorter than its heads");
  if (!a->q || !a->k || !a->v || !a->out || !a->offsets) return le_fail(LE_EINVAL, "null argument");
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) || p.q_stride % 8 ||
      p.k_stride % 8 || p.v_stride % 8 || p.o_stride % 8)
    return le_fail(LE_EINVAL, "q, k, v and out need 16-byte aligned pointers and strides that are multiples of 8");
  if (!aligned(a->offsets, 4)) return le_fail(LE_EINVAL, "offsets not aligned");
  p.offsets = a->offsets;
  p.nseq = a->nseq;
  p.T = a->n_tokens;
  p.heads = h->heads;
  p.group = h->heads / h->kv_heads;
  p.lambda = h->lambda();
  p.norm_w = h->norm ? h->norm_w() : nullptr;
  p.norm_host = h->norm_host;
  p.out_scale = h->out_scale;
  p.eps = h->eps;
  p.status = h->st();
  DeviceGuard g(h->dev);
  CK(g.err);
  CK(launch_diff_attention(a->type, h->d, p, a->max_len, h->pick(stream)));
  return LE_OK;
}

int le_diffattn_sync(le_diffattn* h) { return h ? h->sync() : le_fail(LE_EINVAL, "null argument"); }
int le_diffattn_free(le_diffattn* h) { return free_handle(h); }

}  // extern "C"
