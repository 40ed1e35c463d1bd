// Scores of given tokens from rows of logits, and their gradient.
//
// Of a row x[0..V), a temperature T and a set A of columns (allowed by the caller's mask, x != -inf), with z = x / T:
//   m = max_A x,  s = sum_A exp((x - m) / T),  logp_j = (x_j - m) / T - log s,  p = exp(logp)
//   H = -sum_A p logp = log s - (1 / (T s)) sum_A exp((x - m) / T) (x - m)
//   top alternatives: the k largest x of A, equal values by the lower index
//   d logp_t / d x_j = ([j = t] - p_j) / T,   d H / d x_j = -p_j (logp_j + H) / T
// Differences x - m are taken before they are scaled: they are exact (or rounded once) where a product x / T first would
// lose the low bits of large logits.  m and log s are kept apart for the gradient for the same reason.
// Sums are fp32 over partial sums of a thread's own elements, joined in a fixed order: results are reproducible.
// Where exp((x - m) / T) is 0, x - m may be -inf (the difference of a type's lowest value overflows); as a factor it is
// held at -1e20, so that the product is 0 and not NaN.  A NaN or +inf among A makes s, logp and H NaN.
#include "drk_common.h"
#include "../../include/drakes_hip.h"

#define TSCHECK(cond, name) \
  if (!(cond)) return drk_set_error_msg(DRK_EINVAL, name ": bad arguments")

#define TS_THREADS 256

struct ts_f32 {
  typedef float T;
  static __device__ __forceinline__ float get(const T* p) { return *p; }
  static __device__ __forceinline__ T put(float v) { return v; }
};
struct ts_bf16 {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
  static __device__ __forceinline__ T put(float v) { return (__bf16)v; }
};
struct ts_f16 {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
  static __device__ __forceinline__ T put(float v) { return (_Float16)v; }
};

#define TS_LOG2E 1.4426950408889634f
__device__ __forceinline__ float ts_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float ts_factor(float d) { return fmaxf(d, -1e20f); }
__device__ __forceinline__ float ts_ref(float m) { return m == -INFINITY ? 0.f : m; }   // what an empty row's differences are taken from

// (m, s, t) of a set of elements: s = sum exp2(c (x - m)), t = sum exp2(c (x - m)) (x - m)
struct ts_acc {
  float m, s, t;
};
__device__ __forceinline__ ts_acc ts_join(ts_acc a, ts_acc b, float c) {
  const float m = fmaxf(a.m, b.m), r = ts_ref(m);
  const float da = a.m - r, db = b.m - r;
  const float fa = ts_exp2(c * da), fb = ts_exp2(c * db);
  ts_acc o;
  o.m = m;
  o.s = a.s * fa + b.s * fb;
  o.t = (a.t + a.s * ts_factor(da)) * fa + (b.t + b.s * ts_factor(db)) * fb;
  return o;
}

struct TsArgs {
  const void* x;
  const int64_t* tok;
  const unsigned char* allowed;
  long allowed_stride, row_stride;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
  int V, k;
  float inv_temp;
};

// A row's written results, by one thread: x_t is read again.
template <class D>
__device__ __forceinline__ void ts_finish(const TsArgs& a, long row, ts_acc v) {
  const typename D::T* x = (const typename D::T*)a.x + row * a.row_stride;
  const unsigned char* al = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  const float ls = v.s == 0.f ? 0.f : logf(v.s);
  a.stats[2 * row] = v.m;
  a.stats[2 * row + 1] = ls;
  if (a.entropy) a.entropy[row] = v.s == 0.f ? 0.f : ls - a.inv_temp * (v.t / v.s);
  const int64_t t = a.tok[row];
  float lp = 0.f;
  if (t >= a.V) {
    lp = NAN;
  } else if (t >= 0) {
    const float xt = D::get(x + t);
    const bool in = (!al || al[t]) && xt != -INFINITY;
    lp = v.s != v.s ? NAN : in ? (xt - v.m) * a.inv_temp - ls : -INFINITY;
  }
  a.logp[row] = lp;
}

template <class D>
__global__ void __launch_bounds__(TS_THREADS) k_token_scores(TsArgs a) {
  __shared__ ts_acc red[TS_THREADS];
  __shared__ float bv[TS_THREADS];
  __shared__ int bi[TS_THREADS];
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const typename D::T* x = (const typename D::T*)a.x + row * a.row_stride;
  const unsigned char* al = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  const float c = a.inv_temp * TS_LOG2E;
  ts_acc v = {-INFINITY, 0.f, 0.f};
  for (int j = tid; j < a.V; j += TS_THREADS)
    if (!al || al[j]) {
      const float e = D::get(x + j);
      v = ts_join(v, ts_acc{e, e == -INFINITY ? 0.f : e != e ? NAN : 1.f, 0.f}, c);
    }
  red[tid] = v;
  for (int w = TS_THREADS / 2; w > 0; w >>= 1) {
    __syncthreads();
    if (tid < w) red[tid] = ts_join(red[tid], red[tid + w], c);
  }
  __syncthreads();
  v = red[0];
  if (tid == 0) ts_finish<D>(a, row, v);
  // the k largest, one after the other: the best element that comes after the last one taken
  float pv = INFINITY;
  int pi = -1;
  for (int r = 0; r < a.k; ++r) {
    float best = -INFINITY;
    int at = a.V;
    for (int j = tid; j < a.V; j += TS_THREADS)
      if (!al || al[j]) {
        const float e = D::get(x + j);
        if ((e < pv || (e == pv && j > pi)) && e > best) { best = e; at = j; }
      }
    __syncthreads();
    bv[tid] = best;
    bi[tid] = at;
    for (int w = TS_THREADS / 2; w > 0; w >>= 1) {
      __syncthreads();
      if (tid < w && (bv[tid + w] > bv[tid] || (bv[tid + w] == bv[tid] && bi[tid + w] < bi[tid]))) {
        bv[tid] = bv[tid + w];
        bi[tid] = bi[tid + w];
      }
    }
    __syncthreads();
    pv = bv[0];
    pi = bi[0];
    if (tid == 0) {
      const long o = row * a.k + r;
      a.top_ids[o] = pi < a.V ? pi : -1;
      a.top_logp[o] = pi < a.V ? (v.s != v.s ? NAN : (pv - v.m) * a.inv_temp - logf(v.s)) : -INFINITY;
    }
    if (pi >= a.V) pv = -INFINITY;      // nothing is left: the remaining places come out the same
  }
}

struct TsBwdArgs {
  const void* x;
  const int64_t* tok;
  const unsigned char* allowed;
  long allowed_stride, row_stride;
  const float *stats, *entropy, *g_logp, *g_entropy, *g_top;
  const int64_t* top_ids;
  void* dx;
  int V, k;
  float inv_temp;
};

template <class D>
__global__ void __launch_bounds__(TS_THREADS) k_token_scores_bwd(TsBwdArgs a) {
  const long row = blockIdx.x;
  const typename D::T* x = (const typename D::T*)a.x + row * a.row_stride;
  typename D::T* dx = (typename D::T*)a.dx + row * a.V;
  const unsigned char* al = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  const float m = a.stats[2 * row], ls = a.stats[2 * row + 1];
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f, H = a.g_entropy ? a.entropy[row] : 0.f;
  const int64_t t = a.tok[row];
  float g1 = 0.f;
  if (a.g_logp && t >= 0 && t < a.V && (!al || al[t]) && D::get(x + t) != -INFINITY) g1 = a.g_logp[row];
  float whole = g1;
  for (int r = 0; r < a.k; ++r)
    if (a.top_ids[row * a.k + r] >= 0) whole += a.g_top[row * a.k + r];
  __syncthreads();                      // dlogits may be the logits: x_t has been read by every thread
  for (int j = threadIdx.x; j < a.V; j += TS_THREADS) {
    const float e = D::get(x + j);
    float d = 0.f;
    if ((!al || al[j]) && e != -INFINITY) {
      const float lp = (e - m) * a.inv_temp - ls, p = ts_exp2(lp * TS_LOG2E);
      d = -p * (whole + gh * (ts_factor(lp) + H));
      if (j == t) d += g1;
      for (int r = 0; r < a.k; ++r)
        if (a.top_ids[row * a.k + r] == j) d += a.g_top[row * a.k + r];
      d *= a.inv_temp;
    }
    dx[j] = D::put(d);
  }
}

// ------------------------------------------------------------------------------------------------ C ABI
static bool ts_shape_ok(long rows, int V, long row_stride, long allowed_stride, int k, float temp) {
  return rows >= 0 && rows < (1L << 31) && V >= 1 && row_stride >= 0 && (allowed_stride == 0 || allowed_stride >= V) && k >= 0 &&
         k <= DRK_TOPK_MAX && k <= V && temp > 0.f && temp < INFINITY && 1.f / temp < INFINITY;
}

extern "C" int drk_token_scores(const void* logits, int dtype, long row_stride, const int64_t* tokens, const unsigned char* allowed,
                                long allowed_stride, float temp, int k, float* logp, float* entropy, int64_t* top_ids,
                                float* top_logp, float* stats, long rows, int V, void* stream) {
  TSCHECK(ts_shape_ok(rows, V, row_stride, allowed_stride, k, temp), "drk_token_scores (rows, V, strides, k or temp)");
  if (rows == 0) return DRK_OK;
  TSCHECK(logits && tokens && logp && stats && (k == 0 || (top_ids && top_logp)), "drk_token_scores");
  const TsArgs a = {logits, tokens, allowed, allowed_stride, row_stride, logp, entropy, stats, top_logp, top_ids, V, k, 1.f / temp};
  const dim3 grid((unsigned)rows), block(TS_THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DRK_F32) hipLaunchKernelGGL(k_token_scores<ts_f32>, grid, block, 0, st, a);
  else if (dtype == DRK_BF16) hipLaunchKernelGGL(k_token_scores<ts_bf16>, grid, block, 0, st, a);
  else if (dtype == DRK_F16) hipLaunchKernelGGL(k_token_scores<ts_f16>, grid, block, 0, st, a);
  else return drk_set_error_msg(DRK_EINVAL, "drk_token_scores: dtype is DRK_F32, DRK_BF16 or DRK_F16");
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}

extern "C" int drk_token_scores_bwd(const void* logits, int dtype, long row_stride, const int64_t* tokens,
                                    const unsigned char* allowed, long allowed_stride, float temp, int k, const float* stats,
                                    const float* entropy, const int64_t* top_ids, const float* g_logp, const float* g_entropy,
                                    const float* g_top, void* dlogits, long rows, int V, void* stream) {
  TSCHECK(ts_shape_ok(rows, V, row_stride, allowed_stride, k, temp), "drk_token_scores_bwd (rows, V, strides, k or temp)");
  if (rows == 0) return DRK_OK;
  TSCHECK(logits && tokens && stats && dlogits && (!g_entropy || entropy) && (k == 0 || (top_ids && g_top)), "drk_token_scores_bwd");
  const TsBwdArgs a = {logits, tokens, allowed, allowed_stride, row_stride, stats, entropy, g_logp, g_entropy, g_top, top_ids, dlogits, V, k, 1.f / temp};
  const dim3 grid((unsigned)rows), block(TS_THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DRK_F32) hipLaunchKernelGGL(k_token_scores_bwd<ts_f32>, grid, block, 0, st, a);
  else if (dtype == DRK_BF16) hipLaunchKernelGGL(k_token_scores_bwd<ts_bf16>, grid, block, 0, st, a);
  else if (dtype == DRK_F16) hipLaunchKernelGGL(k_token_scores_bwd<ts_f16>, grid, block, 0, st, a);
  else return drk_set_error_msg(DRK_EINVAL, "drk_token_scores_bwd: dtype is DRK_F32, DRK_BF16 or DRK_F16");
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}
