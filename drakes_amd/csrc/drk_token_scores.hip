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
// held at -1e29, so that the product is 0 and not NaN: 2^30 of them do not overflow, and up to T = 1e26 the exponential of
// anything below it is 0.  From T = 1e-38 on log2(e) / T is a number.  A NaN or +inf among A makes s, logp and H NaN.
//
// A forward pass reads every logit once, a backward pass reads them again and writes as much.  Kernel times, forward +
// backward: 204 800 x 5 fp32 5.2 + 5.5 us; 4 080 x 1 001 fp16, masked, 4 alternatives 10.7 + 9.4 us; 2 049 x 50 021 bf16 58 +
// 75 us (205 and 410 MB: 3.5 and 5.5 TB/s; the forward takes 41 us where the Infinity Cache holds the logits: its vector work,
// which hides the reads from HBM only in part); forward 3 x 131 072 bf16 with 8 alternatives 9.1 + 6.7 us (split and join).  Up to some thousand rows of this a call is bound by its launches.  Three
// shapes of work, chosen by V and the number of rows alone:
//   V <= 64        one thread per row; 64 rows at a time come through LDS, so that short rows are still read and written as
//                  whole cache lines (k_scores_small, k_scores_small_bwd);
//   longer rows    one wave (up to 256 16-byte pieces) or four waves per row, one pass with a running maximum, sum and
//                  entropy sum per thread (k_scores_row, k_scores_row_bwd);
//   few long rows  a row is split over workgroups, whose partial results a second launch joins in order (k_scores_join).
// Top alternatives without a second pass over the row: every thread has the maximum of its own elements; the k-th largest
// of a wave's 64 maxima is a lower bound of the row's k-th largest element, so only threads whose maximum reaches the
// largest such bound can hold an alternative.  Their elements are read again (a few hundred per row), those above the bound
// are listed, and the k that fewest others precede are the answer.  A row with more equal elements at the bound than the
// list holds (a constant row) is searched k times instead.
#include <type_traits>

#include "drk_common.h"
#include "../../include/drakes_hip.h"

#define TSCHECK(cond, name) \
  if (!(cond)) return drk_set_error_msg(DRK_EINVAL, name ": bad arguments")

struct ts_f32 {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};
struct ts_bf16 {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(T v) { return (float)v; }
  static __device__ __forceinline__ T put(float v) { return (__bf16)v; }
};
struct ts_f16 {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(T v) { return (float)v; }
  static __device__ __forceinline__ T put(float v) { return (_Float16)v; }
};

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
#define TS_LOG2E 1.4426950408889634f
__device__ __forceinline__ float ts_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float ts_factor(float d) { return fmaxf(d, -1e29f); }
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
// Over the 64 lanes, every lane gets the result: lanes 1, 2, 7, 15 apart by DPP, then rows of 16 and halves by exchange.
template <class Op>
__device__ __forceinline__ float ts_wave(float v, Op op) {
  auto dpp = [](float x, auto ctrl) __attribute__((always_inline)) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = op(v, dpp(v, std::integral_constant<int, 0xB1>()));
  v = op(v, dpp(v, std::integral_constant<int, 0x4E>()));
  v = op(v, dpp(v, std::integral_constant<int, 0x141>()));
  v = op(v, dpp(v, std::integral_constant<int, 0x140>()));
  const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const u32x2 h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ ts_acc ts_join_wave(ts_acc v, float c) {
  ts_acc o;
  o.m = ts_wave(v.m, [](float a, float b) { return fmaxf(a, b); });
  const float d = v.m - ts_ref(o.m), f = ts_exp2(c * d);
  auto add = [](float a, float b) { return a + b; };
  o.s = ts_wave(v.s * f, add);
  o.t = ts_wave((v.t + v.s * ts_factor(d)) * f, add);
  return o;
}

struct TsArgs {
  const void* x;
  const int64_t* tok;
  const unsigned char* allowed;
  long allowed_stride, row_stride, rows, row0;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
  void* parts;                 // split rows: [rows][splits] TsPart
  int V, k, splits, per_part;  // per_part: 16-byte pieces of a part
  float inv_temp;
};
struct TsPart {                // partial result of a part of a row: 16 + 8 * DRK_TOPK_MAX bytes
  ts_acc v;
  int n;
  float x[DRK_TOPK_MAX];
  int at[DRK_TOPK_MAX];
};

__device__ __forceinline__ float ts_logp(float x, ts_acc v, float ls, float inv_temp) {
  return v.s != v.s ? NAN : (x - v.m) * inv_temp - ls;
}
__device__ __forceinline__ float ts_log_sum(ts_acc v) { return v.s == 0.f ? 0.f : logf(v.s); }

// A row's scalars, by one thread; xt: the given token's logit, -inf where its column does not count.
__device__ __forceinline__ void ts_finish(const TsArgs& a, long row, ts_acc v, float ls, int64_t t, float xt) {
  *(float2*)(a.stats + 2 * row) = make_float2(v.m, ls);
  if (a.entropy) a.entropy[row] = v.s == 0.f ? 0.f : ls - a.inv_temp * (v.t / v.s);
  a.logp[row] = t < 0 ? 0.f : t >= a.V ? NAN : xt == -INFINITY ? (v.s != v.s ? NAN : -INFINITY) : ts_logp(xt, v, ls, a.inv_temp);
}
template <class D>
__device__ __forceinline__ float ts_token(const TsArgs& a, long row, int64_t t) {
  if (t < 0 || t >= a.V || (a.allowed && !a.allowed[row * a.allowed_stride + t])) return -INFINITY;
  return D::get(((const typename D::T*)a.x)[row * a.row_stride + t]);
}

// ---------------------------------------------------------------------------------------------- V <= 64: a thread per row
#define TS_SMALL_V 64
// a row's word j in LDS: one pad word after every 64, so that 64 threads at a stride of V words meet few banks twice
__device__ __forceinline__ int ts_pad(int i) { return i + (i >> 6); }
#define TS_SMALL_LDS(V) (65 * (V) * (int)sizeof(float))      // 64 rows and a pad word per 64

// n consecutive rows -> LDS as floats, -inf in columns that a per-row list leaves out.  VEC: the rows are dense and 16-byte
// aligned (and so is the list, by its own width): whole 16-byte pieces.
template <class D, bool VEC>
__device__ __forceinline__ void ts_stage(const typename D::T* x, const unsigned char* al, long row_stride, long al_stride, int V, int n, float* lds) {
  constexpr int E = 16 / sizeof(typename D::T);
  const int lane = threadIdx.x, total = n * V;
  if (VEC) {
    struct alignas(16) piece { typename D::T v[E]; };
    struct alignas(E) bytes { unsigned char v[E]; };
    const int whole = total / E;
    for (int i0 = lane; i0 < whole; i0 += 256) {           // four requests in flight
      piece p[4];
      bytes b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u < whole ? i0 + 64 * u : i0;
        p[u] = ((const piece*)x)[i];
        if (al) b[u] = ((const bytes*)al)[i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u;
        if (i < whole) {
#pragma unroll
          for (int j = 0; j < E; ++j) lds[ts_pad(E * i) + j] = al && !b[u].v[j] ? -INFINITY : D::get(p[u].v[j]);
        }
      }
    }
    for (int i = whole * E + lane; i < total; i += 64) lds[ts_pad(i)] = al && !al[i] ? -INFINITY : D::get(x[i]);
  } else {
    const float inv = 1.f / (float)V;
    for (int i = lane; i < total; i += 64) {
      const int r = (int)(((float)i + 0.5f) * inv), c = i - r * V;      // i < 4096: the quotient is exact
      lds[ts_pad(i)] = al && !al[r * al_stride + c] ? -INFINITY : D::get(x[r * row_stride + c]);
    }
  }
}
// columns j0 .. j0 + 7 of a row in LDS, -inf where `on` has no bit (none beyond V)
__device__ __forceinline__ void ts_eight(const float* lds, int base, int j0, int V, uint64_t on, float x[8]) {
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float e = lds[ts_pad(base + min(j0 + u, V - 1))];
    x[u] = (on >> (j0 + u)) & 1 ? e : -INFINITY;
  }
}
// the columns of a list that all rows share, as bits
__device__ __forceinline__ uint64_t ts_shared_list(const unsigned char* al, int V) {
  const bool on = (int)threadIdx.x < V && (!al || al[threadIdx.x]);
  return __ballot(on);
}

template <class D, bool VEC>
__global__ void __launch_bounds__(64) k_scores_small(TsArgs a) {
  extern __shared__ float lds[];
  const long row0 = (long)blockIdx.x * 64, row = row0 + threadIdx.x;
  const int n = (int)(a.rows - row0 < 64 ? a.rows - row0 : 64), V = a.V, base = threadIdx.x * V;
  const bool own_list = a.allowed && a.allowed_stride;
  const uint64_t on = ts_shared_list(own_list ? nullptr : a.allowed, V);
  const int64_t t = row < a.rows ? a.tok[row] : -1;
  ts_stage<D, VEC>((const typename D::T*)a.x + row0 * a.row_stride, own_list ? a.allowed + row0 * a.allowed_stride : nullptr, a.row_stride, a.allowed_stride, V, n, lds);
  __syncthreads();
  if (row >= a.rows) return;
  const float c = a.inv_temp * TS_LOG2E;
  ts_acc v = {-INFINITY, 0.f, 0.f};
  float x[8];
  for (int j = 0; j < V; j += 8) {
    ts_eight(lds, base, j, V, on, x);
#pragma unroll
    for (int u = 0; u < 8; ++u) v.m = fmaxf(v.m, x[u]);
  }
  const float r = ts_ref(v.m);
  for (int j = 0; j < V; j += 8) {
    ts_eight(lds, base, j, V, on, x);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float d = x[u] - r, e = ts_exp2(c * d);
      v.s += e;
      v.t = fmaf(e, ts_factor(d), v.t);
    }
  }
  const float ls = ts_log_sum(v);
  ts_finish(a, row, v, ls, t, t >= 0 && t < V && ((on >> t) & 1) ? lds[ts_pad(base + (int)t)] : -INFINITY);
  for (int i = 0; i < a.k; ++i) {            // the best that is left, and out with it
    float best = -INFINITY;
    int at = -1;
    for (int j = 0; j < V; j += 8) {
      ts_eight(lds, base, j, V, on, x);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (x[u] > best) { best = x[u]; at = j + u; }
    }
    a.top_ids[row * a.k + i] = at;
    a.top_logp[row * a.k + i] = at < 0 ? -INFINITY : ts_logp(best, v, ls, a.inv_temp);
    if (at >= 0) lds[ts_pad(base + at)] = -INFINITY;
  }
}

struct TsBwdArgs {
  const void* x;
  const int64_t* tok;
  const unsigned char* allowed;
  long allowed_stride, row_stride, rows, row0;
  const float *stats, *logp, *entropy, *g_logp, *g_entropy, *g_top;
  const int64_t* top_ids;
  void* dx;
  int V, k, splits, per_part;
  float inv_temp;
};

// What a row's gradient is made of: d_j = inv_temp * (hot_j - p_j * (whole + gh * (logp_j + H))).  A row into which nothing
// comes gets zeros whatever its p, which may be NaN: a batch's padding may hold anything.
struct TsRowGrad {
  float m, ls, gh, H, g1, whole;
  int64_t t;
};
__device__ __forceinline__ TsRowGrad ts_row_grad(const TsBwdArgs& a, long row) {      // (`whole` without the alternatives)
  TsRowGrad g;
  const float2 st = *(const float2*)(a.stats + 2 * row);
  g.m = st.x;
  g.ls = st.y;
  g.gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  g.H = a.g_entropy ? a.entropy[row] : 0.f;
  g.t = a.tok[row];
  const float lp = a.g_logp ? a.logp[row] : -INFINITY, g1 = a.g_logp ? a.g_logp[row] : 0.f;
  g.g1 = g.t >= 0 && g.t < a.V && lp != -INFINITY ? g1 : 0.f;
  g.whole = g.g1;
  return g;
}
__device__ __forceinline__ float ts_dense_grad(float x, const TsRowGrad& g, float inv_temp) {
  const float lp = (x - g.m) * inv_temp - g.ls, p = ts_exp2(lp * TS_LOG2E);      // (p is 0 from lp = -128 on)
  return x == -INFINITY ? 0.f : -p * (g.whole + g.gh * (fmaxf(lp, -128.f) + g.H));
}

template <class D, bool VEC>
__global__ void __launch_bounds__(64) k_scores_small_bwd(TsBwdArgs a) {
  constexpr int E = 16 / sizeof(typename D::T);
  extern __shared__ float lds[];
  const long row0 = (long)blockIdx.x * 64, row = row0 + threadIdx.x;
  const int n = (int)(a.rows - row0 < 64 ? a.rows - row0 : 64), V = a.V, base = threadIdx.x * V;
  const bool own_list = a.allowed && a.allowed_stride;
  const uint64_t on = ts_shared_list(own_list ? nullptr : a.allowed, V);
  ts_stage<D, VEC>((const typename D::T*)a.x + row0 * a.row_stride, own_list ? a.allowed + row0 * a.allowed_stride : nullptr, a.row_stride, a.allowed_stride, V, n, lds);
  __syncthreads();
  if (row < a.rows) {
    TsRowGrad g = ts_row_grad(a, row);
    bool any = g.g1 != 0.f || g.gh != 0.f;
#pragma unroll 4
    for (int r = 0; r < a.k; ++r) {
      const int64_t j = a.top_ids[row * a.k + r];
      const float gr = j >= 0 ? a.g_top[row * a.k + r] : 0.f;
      g.whole += gr;
      any |= gr != 0.f;
    }
    // (a row with NaN has a NaN for a token that does not count: its column gets nothing all the same)
    const int tc = g.g1 != 0.f ? (int)g.t : 0;
    const float xt = (on >> tc) & 1 ? lds[ts_pad(base + tc)] : -INFINITY;
    for (int j = 0; j < V; j += 8) {
      float x[8];
      ts_eight(lds, base, j, V, on, x);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j + u < V) lds[ts_pad(base + j + u)] = ts_dense_grad(x[u], g, a.inv_temp) * a.inv_temp;
    }
    if (!any)
      for (int j = 0; j < V; ++j) lds[ts_pad(base + j)] = 0.f;
    if (g.g1 != 0.f && xt != -INFINITY) lds[ts_pad(base + (int)g.t)] += g.g1 * a.inv_temp;
    for (int r = 0; r < a.k; ++r) {
      const int64_t j = a.top_ids[row * a.k + r];
      if (j >= 0 && j < V) lds[ts_pad(base + (int)j)] += a.g_top[row * a.k + r] * a.inv_temp;
    }
  }
  __syncthreads();
  typename D::T* dx = (typename D::T*)a.dx + row0 * V;
  const int total = n * V, whole = VEC ? total / E : 0;
  for (int i = threadIdx.x; i < whole; i += 64) {
    struct alignas(16) piece { typename D::T v[E]; } p;
#pragma unroll
    for (int j = 0; j < E; ++j) p.v[j] = D::put(lds[ts_pad(E * i) + j]);
    ((piece*)dx)[i] = p;
  }
  for (int i = whole * E + threadIdx.x; i < total; i += 64) dx[i] = D::put(lds[ts_pad(i)]);
}

// ---------------------------------------------------------------------------------------------- longer rows
// A row as whole 16-byte pieces from its first 16-byte boundary on, and up to E - 1 elements before the first and behind the
// last of them, which one thread each of the row's first part takes (`edge`).
template <class D>
struct TsRow {
  static constexpr int E = 16 / sizeof(typename D::T);
  struct alignas(16) piece { typename D::T v[E]; };
  const typename D::T* x;
  const unsigned char* al;
  int V, head, full, tail;      // elements before the pieces, pieces, first element behind them
  __device__ __forceinline__ TsRow(const void* base, const unsigned char* allowed, long row, long row_stride, long allowed_stride, int V_) {
    x = (const typename D::T*)base + row * row_stride;
    al = allowed ? allowed + row * allowed_stride : nullptr;
    V = V_;
    const int skew = (int)(((uintptr_t)x & 15) / sizeof(typename D::T));
    head = skew ? E - skew : 0;                          // (< V: these kernels take V > 64)
    full = (V - head) / E;
    tail = head + full * E;
  }
  __device__ __forceinline__ int edge(int tid) const {
    return tid < head ? tid : tid >= E && tid - E < V - tail ? tail + tid - E : -1;
  }
  __device__ __forceinline__ float one(int j) const { return j >= 0 && (!al || al[j]) ? D::get(x[j]) : -INFINITY; }
  // pieces c, c + step, ... as floats, -inf where no column counts and in pieces from c1 on (whose place an earlier one is
  // read from): all requests before the first use.  c < c1.
  template <int N>
  __device__ __forceinline__ void load(int c, int step, int c1, float v[N][E]) const {
    piece p[N];
    uint64_t b[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int at = head + (c + (long)u * step < c1 ? c + u * step : c) * E;
      p[u] = *(const piece*)(x + at);
      if (al) __builtin_memcpy(&b[u], al + at, E);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const bool on = c + (long)u * step < c1;
#pragma unroll
      for (int j = 0; j < E; ++j) v[u][j] = on && (!al || ((b[u] >> (8 * j)) & 255)) ? D::get(p[u].v[j]) : -INFINITY;
    }
  }
};
// The pieces of a part of a row, and whether the row's edges are among it.
__device__ __forceinline__ void ts_part(int full, int splits, int per_part, int part, int* c0, int* c1) {
  const long lo = (long)part * per_part, hi = lo + per_part;
  *c0 = (int)(lo < full ? lo : full);
  *c1 = (int)(part == splits - 1 || hi > full ? full : hi);
}

// floats as unsigned integers of the same order (no NaN among them)
__device__ __forceinline__ unsigned ts_key(float v) {
  const unsigned u = __float_as_uint(v + 0.f);            // -0 -> 0: the two are equal
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float ts_unkey(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

#define TS_BATCH 4              // pieces that a thread requests before it uses the first
#define TS_LIST 512
struct TsList {
  int n;
  float x[TS_LIST];
  int at[TS_LIST];
};
__device__ __forceinline__ bool ts_before(float x, int at, float y, int bt) { return x > y || (x == y && at < bt); }

// A lower bound of the k-th largest of all elements, from the maxima of T threads: the largest of the waves' k-th largest
// maxima, rounded down to 16 bits.  Ends with a barrier.
template <int T>
__device__ __forceinline__ float ts_bound(float mine, int k, unsigned* wave_bound) {
  const unsigned key = ts_key(mine);
  unsigned bound = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const unsigned c = bound | (1u << b);
    if (__popcll(__ballot(key >= c)) >= k) bound = c;
  }
  if ((threadIdx.x & 63) == 0) wave_bound[threadIdx.x >> 6] = bound;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 64; ++w) bound = wave_bound[w] > bound ? wave_bound[w] : bound;
  return bound < 0x00800000u ? -INFINITY : ts_unkey(bound);       // (smaller keys are -inf's own, rounded down)
}

// The k best of the elements of pieces [c0, c1), which this workgroup's threads walked in steps of T, and of the threads' own
// `xe` at column je (-inf: none); mine: a thread's maximum of all; ONE: x holds all of a thread's pieces (one batch).
// put(i, x, at) receives the i-th best; the number found is returned to every thread.
template <class D, int T, bool ONE, class Put>
__device__ __forceinline__ int ts_top(const TsRow<D>& R, int c0, int c1, const float (&x)[TS_BATCH][TsRow<D>::E], float xe, int je,
                                      float mine, int k, TsList* list, unsigned* wave_bound, Put put) {
  constexpr int E = TsRow<D>::E;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) list->n = 0;
  const float least = ts_bound<T>(mine, k, wave_bound);
  auto add = [&](float x, int at) __attribute__((always_inline)) {
    if (x > -INFINITY && x >= least) {
      const int p = atomicAdd(&list->n, 1);
      if (p < TS_LIST) {
        list->x[p] = x;
        list->at[p] = at;
      }
    }
  };
  add(xe, je);
  if (ONE) {
    if (mine >= least) {
#pragma unroll
      for (int u = 0; u < TS_BATCH; ++u)
#pragma unroll
        for (int j = 0; j < E; ++j) add(x[u][j], R.head + (c0 + tid + T * u) * E + j);
    }
  } else {
    uint64_t todo = __ballot(mine >= least && mine > -INFINITY);
    while (todo) {                           // the wave reads these threads' pieces together, four threads' at a time
      int first[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        first[u] = todo ? c0 + wave * 64 + (int)__builtin_ctzll(todo) : c1;
        todo &= todo - 1;
      }
      for (long off = (long)T * lane; first[0] + off < c1; off += (long)T * 64) {
        float v[4][1][E];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const long c = first[u] + off;
          R.template load<1>(c < c1 ? (int)c : c0, 0, c1, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (first[u] + off < c1) {
#pragma unroll
            for (int j = 0; j < E; ++j) add(v[u][0][j], R.head + (int)(first[u] + off) * E + j);
          }
      }
    }
  }
  __syncthreads();
  const int n = list->n;
  if (n <= TS_LIST) {                        // the order of the list does not matter: every entry finds its own place
    for (int i = tid; i < n; i += T) {
      const float x = list->x[i];
      const int at = list->at[i];
      int place = 0;
      for (int o = 0; o < n; ++o) place += ts_before(list->x[o], list->at[o], x, at);
      if (place < k) put(place, x, at);
    }
    return n < k ? n : k;
  }
  float px = INFINITY;
  int pat = -1, found = 0;
  for (; found < k; ++found) {               // too many equals: one search per place
    float best = -INFINITY;
    int at = 0x7fffffff;
    auto look = [&](float x, int i) __attribute__((always_inline)) {
      if (x > -INFINITY && ts_before(px, pat, x, i) && ts_before(x, i, best, at)) { best = x; at = i; }
    };
    look(xe, je);
    for (long c = c0 + tid; c < c1; c += T) {
      float v[1][E];
      R.template load<1>((int)c, 0, c1, v);
#pragma unroll
      for (int j = 0; j < E; ++j) look(v[0][j], R.head + (int)c * E + j);
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) {
      const float ox = __shfl_xor(best, w);
      const int oi = __shfl_xor(at, w);
      if (ts_before(ox, oi, best, at)) { best = ox; at = oi; }
    }
    __syncthreads();
    if (lane == 0) { list->x[wave] = best; list->at[wave] = at; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w)
      if (ts_before(list->x[w], list->at[w], best, at)) { best = list->x[w]; at = list->at[w]; }
    if (best == -INFINITY) break;            // (uniform)
    if (tid == 0) put(found, best, at);
    px = best;
    pat = at;
  }
  return found;
}

// ONE: a part is at most one batch per thread.
template <class D, int T, bool ONE>
__global__ void __launch_bounds__(T) k_scores_row(TsArgs a) {
  constexpr int E = TsRow<D>::E;
  __shared__ TsList list;
  __shared__ ts_acc wave_acc[T / 64];
  __shared__ unsigned wave_bound[T / 64];
  const int tid = threadIdx.x;
  const long row = a.row0 + (a.splits == 1 ? blockIdx.x : blockIdx.x / a.splits);
  const int part = a.splits == 1 ? 0 : (int)(blockIdx.x % a.splits);
  const TsRow<D> R(a.x, a.allowed, row, a.row_stride, a.allowed_stride, a.V);
  int c0, c1;
  ts_part(R.full, a.splits, a.per_part, part, &c0, &c1);
  const float c = a.inv_temp * TS_LOG2E;
  int64_t t = -1;
  float xt = -INFINITY;
  if (tid == 0 && a.splits == 1) {           // requested ahead of the row
    t = a.tok[row];
    xt = ts_token<D>(a, row, t);
  }
  const int je = part == 0 ? R.edge(tid) : -1;
  const float xe = R.one(je);
  ts_acc v = {xe != xe ? -INFINITY : xe, xe == -INFINITY ? 0.f : xe != xe || xe == INFINITY ? NAN : 1.f, 0.f};
  float x[TS_BATCH][E];
  auto batch = [&](int i) __attribute__((always_inline)) {
    R.template load<TS_BATCH>(i, T, c1, x);
    float m = v.m;
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u)
#pragma unroll
      for (int j = 0; j < E; ++j) m = fmaxf(m, x[u][j]);
    const float r = ts_ref(m);
    if (m > v.m) {                           // the running sums move to the new maximum
      const float d = v.m - r, f = ts_exp2(c * d);
      v.t = (v.t + v.s * ts_factor(d)) * f;
      v.s *= f;
      v.m = m;
    }
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = x[u][j] - r, e = ts_exp2(c * d);
        v.s += e;
        v.t = fmaf(e, ts_factor(d), v.t);
      }
  };
  if (ONE) {
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u)
#pragma unroll
      for (int j = 0; j < E; ++j) x[u][j] = -INFINITY;
    if (c0 + tid < c1) batch(c0 + tid);
  } else {
    for (long i = c0 + tid; i < c1; i += (long)T * TS_BATCH) batch((int)i);
  }
  const float mine = v.m;
  v = ts_join_wave(v, c);
  if (T > 64) {
    if ((tid & 63) == 0) wave_acc[tid >> 6] = v;
    __syncthreads();
    v = wave_acc[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = ts_join(v, wave_acc[w], c);
  }
  const float ls = ts_log_sum(v);
  if (a.splits > 1) {
    TsPart* P = (TsPart*)a.parts + row * a.splits + part;
    int n = 0;
    if (a.k) n = ts_top<D, T, ONE>(R, c0, c1, x, xe, je, mine, a.k, &list, wave_bound, [&](int i, float x, int at) {
      P->x[i] = x;
      P->at[i] = at;
    });
    if (tid == 0) {
      P->v = v;
      P->n = n;
    }
    return;
  }
  if (tid == 0) ts_finish(a, row, v, ls, t, xt);
  if (a.k == 0) return;
  const int n = ts_top<D, T, ONE>(R, c0, c1, x, xe, je, mine, a.k, &list, wave_bound, [&](int i, float x, int at) {
    a.top_ids[row * a.k + i] = at;
    a.top_logp[row * a.k + i] = ts_logp(x, v, ls, a.inv_temp);
  });
  for (int i = n + tid; i < a.k; i += T) {
    a.top_ids[row * a.k + i] = -1;
    a.top_logp[row * a.k + i] = -INFINITY;
  }
}

#define TS_MAX_SPLITS 64
// The parts of a row, joined: the sums by a wave (every wave the same), the alternatives from the parts'
// own k best as in ts_top.
template <class D>
__global__ void __launch_bounds__(256) k_scores_join(TsArgs a) {
  constexpr int MOST = TS_MAX_SPLITS * DRK_TOPK_MAX / 256;
  __shared__ float lx[TS_MAX_SPLITS * DRK_TOPK_MAX];
  __shared__ int lat[TS_MAX_SPLITS * DRK_TOPK_MAX];
  __shared__ unsigned wave_bound[4];
  __shared__ int kept;
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const TsPart* P = (const TsPart*)a.parts + row * a.splits;
  const float c = a.inv_temp * TS_LOG2E;
  const int total = a.splits * a.k;
  int64_t t = -1;
  float xt = -INFINITY;
  if (tid == 0) {
    kept = 0;
    t = a.tok[row];
    xt = ts_token<D>(a, row, t);
  }
  ts_acc v = {-INFINITY, 0.f, 0.f};
  if ((tid & 63) < a.splits) v = P[tid & 63].v;
  v = ts_join_wave(v, c);
  float x[MOST], mine = -INFINITY;
  int at[MOST];
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    const int i = tid + 256 * u;
    x[u] = -INFINITY;
    at[u] = 0;
    if (i < total) {
      const int p = i / a.k, j = i - p * a.k;
      if (j < P[p].n) {
        x[u] = P[p].x[j];
        at[u] = P[p].at[j];
      }
    }
    mine = fmaxf(mine, x[u]);
  }
  const float ls = ts_log_sum(v);
  if (tid == 0) ts_finish(a, row, v, ls, t, xt);
  if (a.k == 0) return;
  const float least = ts_bound<256>(mine, a.k, wave_bound);
#pragma unroll
  for (int u = 0; u < MOST; ++u)
    if (x[u] > -INFINITY && x[u] >= least) {
      const int p = atomicAdd(&kept, 1);     // (in any order: every entry finds its own place)
      lx[p] = x[u];
      lat[p] = at[u];
    }
  __syncthreads();
  const int n = kept;
  for (int i = tid; i < n; i += 256) {
    int place = 0;
    for (int o = 0; o < n; ++o) place += ts_before(lx[o], lat[o], lx[i], lat[i]);
    if (place < a.k) {
      a.top_ids[row * a.k + place] = lat[i];
      a.top_logp[row * a.k + place] = ts_logp(lx[i], v, ls, a.inv_temp);
    }
  }
  for (int i = n + tid; i < a.k; i += 256) {
    a.top_ids[row * a.k + i] = -1;
    a.top_logp[row * a.k + i] = -INFINITY;
  }
}

// One pass: piece in, piece out.  The columns of the one-hot terms are stored once more at the end, by a thread each, from
// logits that were read before the first store (dlogits may be the logits: a workgroup reads only what it writes itself, and
// what a batch reads in the place of a piece behind the end is its own thread's, not yet stored).
// ALIKE: a row of dlogits lies on the 16-byte grid as the row of logits does, so that whole pieces are stored.
template <class D, int T, bool ALIKE>
__global__ void __launch_bounds__(T) k_scores_row_bwd(TsBwdArgs a) {
  constexpr int E = TsRow<D>::E;
  const int tid = threadIdx.x;
  const long row = a.row0 + (a.splits == 1 ? blockIdx.x : blockIdx.x / a.splits);
  const int part = a.splits == 1 ? 0 : (int)(blockIdx.x % a.splits);
  const TsRow<D> R(a.x, a.allowed, row, a.row_stride, a.allowed_stride, a.V);
  int c0, c1;
  ts_part(R.full, a.splits, a.per_part, part, &c0, &c1);
  typename D::T* dx = (typename D::T*)a.dx + row * a.V;
  TsRowGrad g = ts_row_grad(a, row);
  // lane r of every wave holds alternative r; the sum runs over the lanes
  const int lane = tid & 63;
  int id = -1;
  float gr = 0.f;
  if (lane < a.k) {
    id = (int)a.top_ids[row * a.k + lane];
    gr = id >= 0 ? a.g_top[row * a.k + lane] : 0.f;
  }
  if (a.k) g.whole += ts_wave(gr, [](float u, float v) { return u + v; });
  const bool none = g.g1 == 0.f && g.gh == 0.f && !__ballot(gr != 0.f);
  // thread r < k stores alternative r's column once more, thread k the given token's: what the one-hot terms add to it
  int mine = tid < a.k ? id : tid == a.k && g.g1 != 0.f ? (int)g.t : -1;
  float xm = -INFINITY, hot = mine >= 0 && mine == g.t ? g.g1 : 0.f;
  for (int r = 0; r < a.k; ++r) {
    const int other = __builtin_amdgcn_readlane(id, r);
    const float go = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gr), r));
    hot += other == mine ? go : 0.f;
  }
  if (mine >= 0) {
    if (mine >= a.V) mine = -1;
    else if (mine < R.head || mine >= R.tail) mine = part == 0 ? mine : -1;
    else if ((mine - R.head) / E < c0 || (mine - R.head) / E >= c1) mine = -1;
    if (mine >= 0) {
      xm = D::get(R.x[mine]);
      if (R.al && !R.al[mine]) xm = -INFINITY;
      if (xm == -INFINITY) hot = 0.f;        // (the token of a row with NaN may be one that does not count)
    }
  }
  const int je = part == 0 ? R.edge(tid) : -1;
  const float xe = R.one(je);
  if (T > 64) __syncthreads();
  if (je >= 0) dx[je] = D::put(ts_dense_grad(xe, g, a.inv_temp) * a.inv_temp);
  for (long i = c0 + tid; i < c1; i += (long)T * TS_BATCH) {
    float x[TS_BATCH][E];
    R.template load<TS_BATCH>((int)i, T, c1, x);
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u) {
      const long at = i + (long)T * u;
      typename TsRow<D>::piece p;
#pragma unroll
      for (int j = 0; j < E; ++j) p.v[j] = D::put(ts_dense_grad(x[u][j], g, a.inv_temp) * a.inv_temp);
      if (at >= c1) continue;
      if (ALIKE) {
        *(typename TsRow<D>::piece*)(dx + R.head + at * E) = p;
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) dx[R.head + at * E + j] = p.v[j];
      }
    }
  }
  __syncthreads();
  if (none) {
    if (je >= 0) dx[je] = D::put(0.f);
    for (long i = R.head + (long)c0 * E + tid; i < R.head + (long)c1 * E; i += T) dx[i] = D::put(0.f);
    return;
  }
  if (mine >= 0) dx[mine] = D::put((ts_dense_grad(xm, g, a.inv_temp) + hot) * a.inv_temp);
}

// ------------------------------------------------------------------------------------------------ C ABI
static bool ts_shape_ok(long rows, int V, long row_stride, long allowed_stride, int k, float temp) {
  return rows >= 0 && rows < (1L << 31) && V >= 1 && V <= (1 << 30) && row_stride >= 0 && (allowed_stride == 0 || allowed_stride >= V) &&
         k >= 0 && k <= DRK_TOPK_MAX && k <= V && temp >= DRK_TEMP_MIN && temp <= DRK_TEMP_MAX;
}
static int ts_size(int dtype) { return dtype == DRK_F32 ? 4 : 2; }

// Pieces of 16 bytes per row, threads per row, parts per row.  A row of up to
// 256 pieces is one wave's: its four loads per lane are in flight together.  With fewer rows than `want` workgroups, a row
// is split as long as a part keeps one piece per thread.
static void ts_plan(long rows, int V, int size, long want, bool* wave, int* splits, int* per_part) {
  const int e = 16 / size;
  const long pieces = V / e;
  *wave = pieces <= 256;
  long s = 1;
  if (!*wave && rows < want) {
    s = (want + rows - 1) / rows;
    if (s > pieces / 256) s = pieces / 256;
    if (s > TS_MAX_SPLITS) s = TS_MAX_SPLITS;
    if (s < 1) s = 1;
  }
  const long per = (pieces + s - 1) / s;
  *per_part = (int)per;
  *splits = (int)((pieces + per - 1) / per);
}
#define TS_WANT_FWD 512
// A launch holds fewer than 2^32 threads: 256 per row make that 2^24 rows (which are never split).
#define TS_LAUNCH_ROWS ((1L << 24) - 1)
static unsigned ts_grid(long rows, long row0, int splits) {
  return (unsigned)((rows - row0 < TS_LAUNCH_ROWS ? rows - row0 : TS_LAUNCH_ROWS) * splits);
}

extern "C" long drk_token_scores_workspace_bytes(long rows, int V, int dtype) {
  if (rows <= 0 || V <= TS_SMALL_V) return 0;
  bool wave;
  int splits, per;
  ts_plan(rows, V, ts_size(dtype), TS_WANT_FWD, &wave, &splits, &per);
  return splits == 1 ? 0 : rows * splits * (long)sizeof(TsPart);
}

template <class D>
static int ts_forward(TsArgs a, bool dense, hipStream_t st) {
  if (a.V <= TS_SMALL_V) {
    const bool vec = dense && ((uintptr_t)a.x & 15) == 0 && (!a.allowed_stride || ((uintptr_t)a.allowed & 7) == 0);
    const dim3 grid((unsigned)((a.rows + 63) / 64));
    if (vec) hipLaunchKernelGGL((k_scores_small<D, true>), grid, dim3(64), TS_SMALL_LDS(a.V), st, a);
    else hipLaunchKernelGGL((k_scores_small<D, false>), grid, dim3(64), TS_SMALL_LDS(a.V), st, a);
    DRK_CHECK_LAUNCH();
    return DRK_OK;
  }
  bool wave;
  ts_plan(a.rows, a.V, (int)sizeof(typename D::T), TS_WANT_FWD, &wave, &a.splits, &a.per_part);
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += TS_LAUNCH_ROWS) {
    const dim3 grid(ts_grid(a.rows, a.row0, a.splits));
    if (wave) hipLaunchKernelGGL((k_scores_row<D, 64, true>), grid, dim3(64), 0, st, a);
    else if (a.per_part <= 256 * TS_BATCH) hipLaunchKernelGGL((k_scores_row<D, 256, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_scores_row<D, 256, false>), grid, dim3(256), 0, st, a);
    DRK_CHECK_LAUNCH();
  }
  if (a.splits > 1) {
    hipLaunchKernelGGL(k_scores_join<D>, dim3((unsigned)a.rows), dim3(256), 0, st, a);
    DRK_CHECK_LAUNCH();
  }
  return DRK_OK;
}

extern "C" int drk_token_scores(const void* logits, int dtype, long row_stride, const int64_t* tokens, const unsigned char* allowed,
                                long allowed_stride, float temp, int k, float* logp, float* entropy, int64_t* top_ids,
                                float* top_logp, float* stats, long rows, int V, void* workspace, long workspace_bytes, void* stream) {
  TSCHECK(ts_shape_ok(rows, V, row_stride, allowed_stride, k, temp), "drk_token_scores (rows, V, strides, k or temp)");
  if (rows == 0) return DRK_OK;
  TSCHECK(logits && tokens && logp && stats && (k == 0 || (top_ids && top_logp)), "drk_token_scores");
  TSCHECK(((uintptr_t)stats & 7) == 0, "drk_token_scores (stats: 8-byte aligned)");
  const long need = drk_token_scores_workspace_bytes(rows, V, dtype);
  TSCHECK(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
          "drk_token_scores (workspace: 16-byte aligned, drk_token_scores_workspace_bytes(rows, V, dtype) bytes)");
  const TsArgs a = {logits, tokens, allowed, allowed_stride, row_stride, rows, 0, logp, entropy, stats, top_logp, top_ids, workspace, V, k, 1, 0, 1.f / temp};
  const bool dense = row_stride == V && (allowed_stride == 0 || allowed_stride == V);
  if (dtype == DRK_F32) return ts_forward<ts_f32>(a, dense, (hipStream_t)stream);
  if (dtype == DRK_BF16) return ts_forward<ts_bf16>(a, dense, (hipStream_t)stream);
  if (dtype == DRK_F16) return ts_forward<ts_f16>(a, dense, (hipStream_t)stream);
  return drk_set_error_msg(DRK_EINVAL, "drk_token_scores: dtype is DRK_F32, DRK_BF16 or DRK_F16");
}

#define TS_WANT_BWD 1024
template <class D>
static int ts_backward(TsBwdArgs a, bool dense, hipStream_t st) {
  const int size = (int)sizeof(typename D::T);
  if (a.V <= TS_SMALL_V) {
    const bool vec = dense && ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.dx & 15) == 0 && (!a.allowed_stride || ((uintptr_t)a.allowed & 7) == 0);
    const dim3 grid((unsigned)((a.rows + 63) / 64));
    if (vec) hipLaunchKernelGGL((k_scores_small_bwd<D, true>), grid, dim3(64), TS_SMALL_LDS(a.V), st, a);
    else hipLaunchKernelGGL((k_scores_small_bwd<D, false>), grid, dim3(64), TS_SMALL_LDS(a.V), st, a);
    DRK_CHECK_LAUNCH();
    return DRK_OK;
  }
  bool wave;
  ts_plan(a.rows, a.V, size, TS_WANT_BWD, &wave, &a.splits, &a.per_part);
  const bool alike = (a.row_stride - a.V) * size % 16 == 0 && (((uintptr_t)a.x ^ (uintptr_t)a.dx) & 15) == 0;
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += TS_LAUNCH_ROWS) {
    const dim3 grid(ts_grid(a.rows, a.row0, a.splits));
    if (wave && alike) hipLaunchKernelGGL((k_scores_row_bwd<D, 64, true>), grid, dim3(64), 0, st, a);
    else if (wave) hipLaunchKernelGGL((k_scores_row_bwd<D, 64, false>), grid, dim3(64), 0, st, a);
    else if (alike) hipLaunchKernelGGL((k_scores_row_bwd<D, 256, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_scores_row_bwd<D, 256, false>), grid, dim3(256), 0, st, a);
    DRK_CHECK_LAUNCH();
  }
  return DRK_OK;
}

extern "C" int drk_token_scores_bwd(const void* logits, int dtype, long row_stride, const int64_t* tokens,
                                    const unsigned char* allowed, long allowed_stride, float temp, int k, const float* stats,
                                    const float* logp, const float* entropy, const int64_t* top_ids, const float* g_logp,
                                    const float* g_entropy, const float* g_top, void* dlogits, long rows, int V, void* stream) {
  TSCHECK(ts_shape_ok(rows, V, row_stride, allowed_stride, k, temp), "drk_token_scores_bwd (rows, V, strides, k or temp)");
  if (rows == 0) return DRK_OK;
  TSCHECK(logits && tokens && stats && dlogits && (!g_logp || logp) && (!g_entropy || entropy) && (k == 0 || (top_ids && g_top)),
          "drk_token_scores_bwd");
  TSCHECK(((uintptr_t)stats & 7) == 0, "drk_token_scores_bwd (stats: 8-byte aligned)");
  TSCHECK(dlogits != logits || row_stride == V, "drk_token_scores_bwd (in place: dense rows)");
  const TsBwdArgs a = {logits, tokens, allowed, allowed_stride, row_stride, rows, 0, stats, logp, entropy, g_logp, g_entropy, g_top, top_ids, dlogits, V, k, 1, 0, 1.f / temp};
  const bool dense = row_stride == V && (allowed_stride == 0 || allowed_stride == V);
  if (dtype == DRK_F32) return ts_backward<ts_f32>(a, dense, (hipStream_t)stream);
  if (dtype == DRK_BF16) return ts_backward<ts_bf16>(a, dense, (hipStream_t)stream);
  if (dtype == DRK_F16) return ts_backward<ts_f16>(a, dense, (hipStream_t)stream);
  return drk_set_error_msg(DRK_EINVAL, "drk_token_scores_bwd: dtype is DRK_F32, DRK_BF16 or DRK_F16");
}
