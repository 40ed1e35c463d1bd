// Activation checkpoints in 8 bits, and the backward kernels that read them.
//
// A residual layer's forward keeps, per row of 128 channels, x^ = (feat + tbias - mean) * rstd as 128 signed bytes and one
// power-of-two scale for each block of 32 channels (132 bytes, against 512 for an fp32 residual snapshot and 256 for a bf16
// LayerNorm output), rstd, and the ReLU gates of the layer below as bits.  With a = max |x^| of a block,
//     e = the smallest integer with a <= 127 * 2^e (e >= -126),  q = rint(x^ / 2^e) (ties to even),  x^ ~ xq = q * 2^e,
// so |x^ - xq| <= 2^(e-1), a / 127 at most.  The scale is a power of two so that xq is exact in bf16 (7 bits and a sign):
// the weight gradient's matrix instructions multiply it without another rounding.  The scale byte is e + 127; 0 = a block of
// zeros; 255 = a block that holds an infinity, a NaN or more than 127 * 2^120 (it reads back as NaN: an overflow is not lost
// on the way, and 128 * 2^e stays finite).
//   LayerNorm backward:  a = dh * gamma;  dx = rstd * (a - mean_c(a) - xq * mean_c(a * xq))
//   weight gradient:     h = gamma * xq + beta, so  dw[t] = gamma (x) P[t] + beta (x) S[t],
//                        P[t][ci][co] = sum_rows xq[row + off_t][ci] dc[row][co],  S[t][co] = sum of dc over the rows that
//                        tap t can reach: gamma and beta stay out of the matrix product, where h would have to be rounded.
#include <atomic>

#include "drk_common.h"
#include "../../include/drakes_hip.h"

typedef __bf16 bf16v8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16v4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define CKCHECK(cond, name) \
  if (!(cond)) return drk_set_error_msg(DRK_EINVAL, name ": bad arguments")

#define CK_BLK 32                       // channels per scale
#define CK_EXPS (DRK_C / CK_BLK)        // scale bytes per row
#define CK_LN_EPS 1e-5

// ---- sums over the 16 lanes that hold a row, every lane gets the total ------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0u, (unsigned)v, CTRL, 0xF, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0u, (unsigned)(v >> 32), CTRL, 0xF, 0xF, false);
  return ((uint64_t)hi << 32) | lo;
}
#define DPP_XOR1 0xB1       // quad_perm [1,0,3,2]
#define DPP_XOR2 0x4E       // quad_perm [2,3,0,1]
#define DPP_HALF 0x141      // row_half_mirror
#define DPP_ROW 0x140       // row_mirror
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_f32<DPP_XOR1>(v);
  v += dpp_f32<DPP_XOR2>(v);
  v += dpp_f32<DPP_HALF>(v);
  v += dpp_f32<DPP_ROW>(v);
  return v;
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  return __longlong_as_double((long long)dpp_u64<CTRL>((uint64_t)__double_as_longlong(v)));
}
__device__ __forceinline__ double row_sum(double v) {
  v += dpp_f64<DPP_XOR1>(v);
  v += dpp_f64<DPP_XOR2>(v);
  v += dpp_f64<DPP_HALF>(v);
  v += dpp_f64<DPP_ROW>(v);
  return v;
}

__device__ __forceinline__ void load8(const float* p, float v[8]) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void store8(float* p, const float v[8]) {
  *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
  *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8_bf16(void* p, const float v[8]) {
  bf16v8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (__bf16)v[i];
  *(bf16v8*)p = o;
}
// the eight values of eight codes: (q + 128) * 2^e - 128 * 2^e in one rounding, which is exact; scale byte 255 -> NaN
__device__ __forceinline__ void decode8(uint64_t q, unsigned e, float v[8]) {
  const float s = __uint_as_float(e << 23), b = e == 255u ? NAN : -128.f * s;
  const unsigned lo = (unsigned)q ^ 0x80808080u, hi = (unsigned)(q >> 32) ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = fmaf((float)((lo >> (8 * i)) & 255u), s, b);
    v[4 + i] = fmaf((float)((hi >> (8 * i)) & 255u), s, b);
  }
}

// ---- forward -------------------------------------------------------------------------------------------------------
// 16 lanes per row, 8 channels per lane (32 bytes of feat, 16 of h, 8 codes, 1 byte of gates).  Statistics and codes are
// computed in fp64: a code is then the rounding of the true value except within ~1e-15 of a border, whatever order a sum
// is taken in, and fp64 multiplies and adds run at the rate of unpacked fp32 ones on this chip, behind a memory-bound pass.
// 1 044 bytes per row with feat, mask and gates: 524 288 rows in 110 to 121 us, 4.5 to 5 TB/s (a copy reaches 5.1).
struct CkFwdArgs {
  const float *feat, *tbias, *gamma, *beta;
  const unsigned char* relu_mask;
  long tb_stride;
  void* h;
  uint64_t* codes;
  unsigned char *exps, *gates;
  float* rstd;
  long M;
  int L, gate_self;
};

template <bool LN>
__global__ void __launch_bounds__(256) k_ln_fwd_ck8(CkFwdArgs a) {
  const int lane = threadIdx.x & 15;
  float gm[8], bt[8];
  if (LN) {
    load8(a.gamma + 8 * lane, gm);
    load8(a.beta + 8 * lane, bt);
  }
  for (long row = (long)blockIdx.x * 16 + (threadIdx.x >> 4); row < a.M; row += (long)gridDim.x * 16) {
    float f[8], hv[8];
    load8(a.feat + row * DRK_C + 8 * lane, f);
    double x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (double)f[i];
    if (LN) {
      if (a.tbias) {
        float tb[8];
        load8(a.tbias + (a.tb_stride ? row / a.L * a.tb_stride : 0) + 8 * lane, tb);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += (double)tb[i];
      }
      double s = 0.0, v = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[i];
      const double mean = row_sum(s) * (1.0 / DRK_C);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] -= mean;
        v = fma(x[i], x[i], v);
      }
      const double r = 1.0 / sqrt(row_sum(v) * (1.0 / DRK_C) + CK_LN_EPS);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= r;
        hv[i] = (float)fma(x[i], (double)gm[i], (double)bt[i]);
      }
      if (lane == 0) a.rstd[row] = (float)r;
      store8_bf16((char*)a.h + row * (2 * DRK_C) + 16 * lane, hv);
    } else {
      store8_bf16((char*)a.h + row * (2 * DRK_C) + 16 * lane, f);
    }
    // the block's largest magnitude, compared as bit patterns: a NaN or an infinity comes out on top
    uint64_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t b = (uint64_t)__double_as_longlong(x[i]) & 0x7fffffffffffffffull;
      am = b > am ? b : am;
    }
    uint64_t o = dpp_u64<DPP_XOR1>(am);
    am = o > am ? o : am;
    o = dpp_u64<DPP_XOR2>(am);
    am = o > am ? o : am;
    const int be = (int)(am >> 52);                                     // a = 1.f * 2^(be - 1023)
    int e = be - 1023 - 6 + ((am & 0xfffffffffffffull) > 0xfc00000000000ull ? 1 : 0);   // 1.f <= 127 / 64 ?
    e = e < -126 ? -126 : e;
    const bool bad = e > 120, none = am == 0;      // (an infinity's or a NaN's exponent field gives e = 1018)
    const double inv = __longlong_as_double((long long)(1023 - e) << 52);
    uint64_t q = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) q |= (uint64_t)((unsigned)(int)rint(x[i] * inv) & 255u) << (8 * i);
    if (bad) q = 0;
    a.codes[row * (DRK_C / 8) + lane] = q;
    if ((lane & 3) == 0) a.exps[row * CK_EXPS + (lane >> 2)] = bad ? 255 : none ? 0 : (unsigned char)(e + 127);
    if (a.gates) {
      unsigned g = 0;
      if (a.relu_mask) {
        const uint64_t m = *(const uint64_t*)(a.relu_mask + row * DRK_C + 8 * lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) g |= ((m >> (8 * i)) & 255u) ? 1u << i : 0u;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g |= f[i] > 0.f ? 1u << i : 0u;
      }
      a.gates[row * (DRK_C / 8) + lane] = (unsigned char)g;
    }
  }
}

// 132 bytes in, 512 (bf16: 256) out, and nothing to compute: 524 288 rows to fp32 in 63 us, 5.3 TB/s.
// Four channels per thread, four groups in flight: a wave's store is 1 KB (bf16: 512 bytes) in one piece.
template <bool BF16>
__global__ void __launch_bounds__(256) k_ck8_unpack(const unsigned* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                    char* __restrict__ out, long n) {
  const long step = (long)gridDim.x * 256;
  for (long i0 = (long)blockIdx.x * 256 + threadIdx.x; i0 < n; i0 += 4 * step) {
    unsigned q[4], e[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long i = i0 + u * step < n ? i0 + u * step : i0;
      q[u] = codes[i];
      e[u] = exps[i >> 3];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long i = i0 + u * step;
      float v[8];
      decode8(q[u], e[u], v);
      if (i < n) {
        if (BF16) {
          bf16v4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = (__bf16)v[j];
          *(bf16v4*)(out + 8 * i) = o;
        } else {
          *(f32x4*)(out + 16 * i) = f32x4{v[0], v[1], v[2], v[3]};
        }
      }
    }
  }
}

// ---- LayerNorm backward --------------------------------------------------------------------------------------------
// Row layout as above.  Column sums stay in a lane's registers over the rows its workgroup walks; the 16 rows in flight
// are joined in order through LDS and leave as one [4][128] slab per workgroup, the slabs are added in order.
// Memory-bound: 524 288 rows (1.02 GB) in 193 us, 5.3 TB/s; 6 400 rows 5.6 us and 4.8 us for the sums.
struct CkBwdArgs {
  const float *dh, *gamma, *rstd, *g_resid;
  const uint64_t* codes;
  const unsigned char *exps, *gates;
  float *dfeat, *dxin, *slabs;
  void* dc;
  long M;
};

template <bool LN, bool SUMS>
__global__ void __launch_bounds__(256) k_ln_bwd_ck8(CkBwdArgs a) {
  __shared__ float red[16][DRK_C + 4];
  const int lane = threadIdx.x & 15, sub = threadIdx.x >> 4;
  float gm[8], sg[8], sb[8], sx[8], sc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = sb[i] = sx[i] = sc[i] = 0.f;
  if (LN) load8(a.gamma + 8 * lane, gm);
  for (long row = (long)blockIdx.x * 16 + sub; row < a.M; row += (long)gridDim.x * 16) {
    const long at = row * DRK_C + 8 * lane;
    float d[8], x[8], o[8];
    load8(a.dh + at, d);
    if (a.g_resid) load8(a.g_resid + at, o);
    if (LN) {
      decode8(a.codes[row * (DRK_C / 8) + lane], a.exps[row * CK_EXPS + (lane >> 2)], x);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = d[i] * gm[i];
        s1 += y;
        s2 = fmaf(y, x[i], s2);
      }
      const float r = a.rstd[row], m1 = row_sum(s1) * (1.f / DRK_C), m2 = row_sum(s2) * (1.f / DRK_C);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (SUMS) {
          sg[i] = fmaf(d[i], x[i], sg[i]);
          sb[i] += d[i];
        }
        d[i] = r * (fmaf(d[i], gm[i], -m1) - x[i] * m2);
      }
    }
    if (a.dxin) store8(a.dxin + at, d);
    unsigned g = 255u;
    if (a.gates) g = a.gates[row * (DRK_C / 8) + lane];
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (SUMS) sx[i] += d[i];
      o[i] = a.g_resid ? o[i] + d[i] : d[i];
      c[i] = (g >> i) & 1u ? o[i] : 0.f;
      if (SUMS) sc[i] += c[i];
    }
    if (a.dfeat) store8(a.dfeat + at, a.dc ? o : c);
    if (a.dc) store8_bf16((char*)a.dc + 2 * at, c);
  }
  if (!SUMS) return;
  for (int q = 0; q < 4; ++q) {
    __syncthreads();
    store8(&red[sub][8 * lane], q == 0 ? sg : q == 1 ? sb : q == 2 ? sx : sc);
    __syncthreads();
    if (threadIdx.x < DRK_C) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) s += red[k][threadIdx.x];
      a.slabs[((long)blockIdx.x * 4 + q) * DRK_C + threadIdx.x] = s;
    }
  }
}

// out[i] += slab 0 [i] + slab 1 [i] + ...: 32 threads per output take every 32nd slab, then join in a fixed tree
__global__ void __launch_bounds__(256) k_ck8_sums(const float* __restrict__ slabs, int n, float* __restrict__ out) {
  __shared__ float red[32][8];
  const int c = threadIdx.x & 7, s0 = threadIdx.x >> 3, i = blockIdx.x * 8 + c;
  float s = 0.f;
#pragma unroll 8
  for (int k = s0; k < n; k += 32) s += slabs[(long)k * (4 * DRK_C) + i];
  red[s0][c] = s;
  for (int w = 16; w > 0; w >>= 1) {
    __syncthreads();
    if (s0 < w) red[s0][c] += red[s0 + w][c];
  }
  if (s0 == 0) out[i] += red[0][c];
}

// ---- weight gradient -----------------------------------------------------------------------------------------------
// A matrix product whose K runs along the rows: 128 ci x 128 co per tap, 294 912 operations per row at 9 taps against 388
// bytes read, so it is bound by the matrix cores and by what feeds them.  Sequences follow each other without padding; a
// 32-row step of a tap has the rows that stay in their sequence as 32 bits, computed from the step's first position; the
// others are cleared in the xq fragment (an infinity or NaN of dc meets a zero there and makes NaN, as with padded rows; a step
// that k_wgrad_ck8_tap leaves out, since its tap reaches none of its rows, looks for one).
// Both operands are read transposed (ds_read_b64_tr_b16) from tiles in LDS.  S comes from the same product: a fragment whose
// row m is 1 where tap m is inside its sequence.
//   k_wgrad_ck8_ring: all taps in one workgroup, 32 of the 128 input channels.  The decoded xq rows form a ring: every row is
//     read and decoded once per chunk whatever the number of taps (decoded per tap, the vector instructions alone took
//     longer than the product).  8 waves, each four taps x 16 ci x 64 co, half of tap 8 and a quarter of S: 76 accumulator
//     registers, 9 fragments for 19 matrix instructions, the next step's fragments requested among this step's product.
//     262 144 rows, 9 taps, with the join: sequences of 1 024 83 to 99 us by dilation, of 200 94 to 124 us, where more
//     steps have rows that leave their sequence (all at dilation 64) and taps are multiplied whether they reach a row or not.
//     The matrix instructions of a step take 608 cycles of a SIMD (2 waves x 19 x 16), its fragments 74 KB of LDS reads, 576
//     cycles at 128 bytes a cycle: both are full at once, and only fewer fragments per product would change that.  Masks, the
//     staging of tiles and the join (9 us) are the rest.
//   k_wgrad_ck8_tap: one tap and 64 input channels per workgroup, for one tap, for few rows (nine times the workgroups per
//     row chunk, and every chunk costs a slab of P written and read) and for shifts that no ring in LDS can hold
//     ((taps - 1) * dilation > 832).  262 144 rows, with the join: one tap 38 us, 9 taps of dilation 128 208 us.
#define CW_TILE 64
#define CW_DC (CW_TILE * 256)            // bytes of a dc tile
#define CW_SLAB ((DRK_C + 1) * DRK_C)    // P [128][128], then S [128]
#define CW_MAX_TAPS 9

__device__ __forceinline__ int cw_dc_at(int row, int ch) { return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3))); }
__device__ __forceinline__ s16x4 cw_read(const char* p) {
  typedef s16x4 __attribute__((address_space(3))) * lds4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
}
__device__ __forceinline__ bf16v8 cw_frag(const char* p0, const char* p1) {
  const s16x4 lo = cw_read(p0), hi = cw_read(p1);
  return __builtin_bit_cast(bf16v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// Bit k: row k of 32 rows that follow each other from position lb of a sequence of L (then the next sequences') is inside
// its sequence after a shift of o, |o| <= L.
__device__ __forceinline__ unsigned cw_inside(int lb, int L, int o) {
  unsigned rows = 0;
  for (int s = -lb; s < 32; s += L) {                      // a sequence's rows are k = s .. s + L - 1
    const int lo = max(s + max(-o, 0), 0), n = min(s + min(L - o, L), 32) - lo;
    rows |= n > 0 ? (~0u >> (32 - n)) << lo : 0u;
  }
  return rows;
}
// eight bits -> eight halves of all ones or zeros
__device__ __forceinline__ u32x4 cw_mask(unsigned bits) {
  u32x4 m;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const unsigned a = (unsigned)((int)(bits << (31 - 2 * d)) >> 31), b = (unsigned)((int)(bits << (30 - 2 * d)) >> 31);
    m[d] = (a & 0xffffu) | (b & 0xffff0000u);
  }
  return m;
}

struct CwArgs {
  const uint64_t* codes;
  const unsigned char* exps;
  const char* dc;
  float* slabs;
  long M;
  int L, taps, dil, tiles_per_wg, total_tiles, chunks;
};

// What a chunk of rows is to a kernel: its first row, its tiles, and where its first row stands in its sequence.
struct CwChunk {
  long r0;
  int nt, lb;
};
__device__ __forceinline__ CwChunk cw_chunk(const CwArgs& a, int chunk) {
  const int T0 = chunk * a.tiles_per_wg;
  CwChunk c;
  c.r0 = (long)T0 * CW_TILE;
  c.nt = (T0 + a.tiles_per_wg < a.total_tiles ? T0 + a.tiles_per_wg : a.total_tiles) - T0;
  c.lb = (int)(c.r0 % a.L);
  return c;
}
__device__ __forceinline__ int cw_shift(const CwArgs& a, int tap) {      // at most L either way: nothing is inside there
  const long o = (long)(tap - a.taps / 2) * a.dil;
  return (int)(o > a.L ? a.L : o < -a.L ? -a.L : o);
}
__device__ __forceinline__ bf16v8 cw_clear(bf16v8 f, u32x4 mask) { return __builtin_bit_cast(bf16v8, __builtin_bit_cast(u32x4, f) & mask); }

__global__ void __launch_bounds__(256) k_wgrad_ck8_tap(CwArgs a) {
  __shared__ __attribute__((aligned(16))) char xs[2][CW_TILE * 128];      // xq, 64 channels
  __shared__ __attribute__((aligned(16))) char ds[2][CW_DC];
  __shared__ unsigned nan_at[DRK_C / 2];                                  // two channels of dc each, as `lost`
  // the two halves of a chunk read the same dc: 8 workgroups apart they run on the same XCD
  const int half = (blockIdx.x >> 3) & 1, chunk = (blockIdx.x >> 4) * 8 + (blockIdx.x & 7);
  if (chunk >= a.chunks) return;
  const int tid = threadIdx.x, lane = tid & 63, tap = blockIdx.y, L = a.L;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), ciq = w >> 1, coh = w & 1;
  const CwChunk c = cw_chunk(a, chunk);
  const long g0 = c.r0 + (long)(tap - a.taps / 2) * a.dil;
  const int shift = cw_shift(a, tap), lstep = 32 % L;
  int lb = c.lb;
  uint64_t rq[2];
  unsigned re[2];
  f32x4 rd[4];
  auto fetch = [&](int T) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int it = tid + 256 * i;
      const long g = g0 + 64L * T + (it >> 3);
      rq[i] = 0;
      re[i] = 0;
      if (g >= 0 && g < a.M) {
        rq[i] = a.codes[g * (DRK_C / 8) + 8 * half + (it & 7)];
        re[i] = a.exps[g * CK_EXPS + 2 * half + ((it >> 2) & 1)];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int it = tid + 256 * i;
      const long g = c.r0 + 64L * T + (it >> 4);
      rd[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (g < a.M) rd[i] = *(const f32x4*)(a.dc + g * 256 + 16 * (it & 15));
    }
  };
  unsigned live[2];              // of the stored tile's two steps: the rows that stay in their sequence
  u32x4 lost = {0u, 0u, 0u, 0u};      // bits 15, 31: dc of this thread's 8 channels was not finite in a step without such a row
  auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      live[ks] = cw_inside(lb, L, shift);
      lb += lstep;
      lb -= lb >= L ? L : 0;
      if (!live[ks]) {           // (rd[2 ks], rd[2 ks + 1] hold rows of step ks; an exponent of ones carries into the next bit)
        const u32x4 d0 = __builtin_bit_cast(u32x4, rd[2 * ks]), d1 = __builtin_bit_cast(u32x4, rd[2 * ks + 1]);
        lost |= ((d0 & 0x7f807f80u) + 0x00800080u) | ((d1 & 0x7f807f80u) + 0x00800080u);
      }
    }
    if (!(live[0] | live[1])) return;                      // nobody reads this tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int it = tid + 256 * i, row = it >> 3;
      float v[8];
      decode8(rq[i], re[i], v);
      store8_bf16(xs[buf] + 128 * row + 16 * ((it & 7) ^ (((row >> 1) & 1) << 1) ^ (((row >> 3) & 1) << 2)), v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int it = tid + 256 * i;
      *(f32x4*)(ds[buf] + cw_dc_at(it >> 4, it & 15)) = rd[i];
    }
  };
  // lane 16 kg + 4 q + p asks for row 8 kg + q (+ 4 in the second read), columns 4 p .. 4 p + 3 of a 16-channel tile.  The
  // 32-byte pairs of an xq row are exchanged by bits 1 and 3 of the row: 8 rows of 32 lanes fall into different banks.
  const int kg = lane >> 4, q = (lane >> 2) & 3, p = lane & 3, row = 8 * kg + q;
  const int aoff = 128 * row + 32 * ((2 * ciq) ^ ((row >> 1) & 1) ^ ((row >> 2) & 2)) + 16 * (p >> 1) + 8 * (p & 1);
  const int boff = cw_dc_at(row, 8 * coh + (p >> 1)) + 8 * (p & 1);
  f32x4 acc[2][4], accs[2];
#pragma unroll
  for (int n = 0; n < 4; ++n) acc[0][n] = acc[1][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  accs[0] = accs[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tid < 64) nan_at[tid] = 0u;
  fetch(0);
  store(0);
  __syncthreads();
  for (int T = 0; T < c.nt; ++T) {
    if (T + 1 < c.nt) fetch(T + 1);
    const char *xt = xs[T & 1], *dt = ds[T & 1];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const unsigned rows = live[ks];
      if (rows) {
        bf16v8 af[2], bf[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) bf[n] = cw_frag(dt + 8192 * ks + (boff ^ (32 * n)), dt + 8192 * ks + 1024 + (boff ^ (32 * n) ^ 16));
#pragma unroll
        for (int m = 0; m < 2; ++m) af[m] = cw_frag(xt + 4096 * ks + (aoff ^ (32 * m)), xt + 4096 * ks + 512 + (aoff ^ (32 * m)));
        u32x4 mask = cw_mask(rows >> (8 * kg));
        af[0] = cw_clear(af[0], mask);
        af[1] = cw_clear(af[1], mask);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 4; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], bf[n], acc[m][n], 0, 0, 0);
        if (half == 0) {
          mask &= 0x3f803f80u;                             // ones in the rows that count
#pragma unroll
          for (int n = 0; n < 2; ++n)
            accs[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16v8, mask), ciq ? bf[2 + n] : bf[n], accs[n], 0, 0, 0);
        }
      }
    }
    if (T + 1 < c.nt) {
      store((T + 1) & 1);                                  // its last readers passed the previous barrier
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (lost[d] & 0x80008000u) atomicOr(&nan_at[4 * (tid & 15) + d], lost[d] & 0x80008000u);
    }
    __syncthreads();
  }
  // D[row 4 g + v][col] of tile (m, n): ci = 64 half + 32 ciq + 16 m + 4 g + v, co = 64 coh + 16 n + (lane & 15)
  float* dst = a.slabs + ((long)chunk * a.taps + tap) * CW_SLAB;
  const int g = lane >> 4, cn = lane & 15;
  bool nan[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) nan[n] = (nan_at[(64 * coh + 16 * n + cn) >> 1] >> (cn & 1 ? 31 : 15)) & 1u;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v) dst[(64 * half + 32 * ciq + 16 * m + 4 * g + v) * DRK_C + 64 * coh + 16 * n + cn] = nan[n] ? NAN : acc[m][n][v];
  if (half == 0 && g == 0) {
#pragma unroll
    for (int n = 0; n < 2; ++n) dst[DRK_C * DRK_C + 64 * coh + 16 * (2 * ciq + n) + cn] = (ciq ? nan[2 + n] : nan[n]) ? NAN : accs[n][0];
  }
}

#define CW_NT 5                           // A fragments of a wave: four taps, and tap 8 for two of the four co tiles
#define CW_RING_MAX 1024                  // rows
#define CW_RD 288                         // bytes of a dc row: 32 more than it holds, so that 8 rows of 32 bytes meet no bank twice
#define CW_RDC (CW_TILE * CW_RD)
// Ring blocks of 64 rows: those a tile reads, one more for the next tile's first step, one that is being filled.
__host__ __device__ static inline int cw_ring_rows(int taps, int dilation) {
  const int need = (((taps - 1) * dilation + 63) / 64 + 3) * 64;
  int r = 256;
  while (r < need) r *= 2;
  return r;
}
#define CW_RING_LDS(rows) (((rows) + 16) * 64 + 3 * CW_RDC + 128)      // (the ring's first 16 rows once more behind its last)

// K slot 8 kg + j of a 32-row step is row 4 kg + j (j < 4) or 12 + 4 kg + j: the rows that 32 lanes read together follow each
// other.
__global__ void __launch_bounds__(512) k_wgrad_ck8_ring(CwArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];              // the ring, then three dc tiles
  typedef s16x4 __attribute__((address_space(3))) * lds4;
  // the four quarters of a chunk read the same dc: 8 workgroups apart they run on the same XCD
  const int quarter = (blockIdx.x >> 3) & 3, chunk = (blockIdx.x >> 5) * 8 + (blockIdx.x & 7);
  if (chunk >= a.chunks) return;
  const int tid = threadIdx.x, lane = tid & 63, L = a.L, jn = a.taps;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), tg = w >> 2, cih = (w >> 1) & 1, coh = w & 1;
  const CwChunk c = cw_chunk(a, chunk);
  const int span = (jn - 1) * a.dil, sb = (span + 63) / 64;                // a tile reads ring blocks T .. T + sb
  const int R = cw_ring_rows(jn, a.dil), bwrap = R / 64 - 1;
  const unsigned wrap = 64u * R - 1u;
  const long g0 = c.r0 - (long)(jn / 2) * a.dil;                          // the ring's first row
  const int dcs = (R + 16) * 64;

  // staging: 256 threads an xq block (row tid / 4, 8 channels), all of them a dc tile (rows tid / 16 and + 32).  The halves
  // of a ring row are exchanged by bit 2 of the row: the 8 rows of 32 lanes fall into different banks wherever they start.
  const int xrow = (tid & 255) >> 2, xch = tid & 3;
  const uint64_t* const xc = a.codes + 4 * quarter + xch;
  const unsigned char* const xe = a.exps + quarter;
  const int xput = 64 * xrow + 16 * (xch ^ (((xrow >> 2) & 1) << 1)), dput = dcs + (tid >> 4) * CW_RD + 16 * (tid & 15);
  auto fetch_x = [&](int b, uint64_t& q, unsigned& e) __attribute__((always_inline)) {
    const long g = g0 + 64L * b + xrow;
    const bool on = g >= 0 && g < a.M;
    q = on ? xc[g * (DRK_C / 8)] : 0;
    e = on ? xe[g * CK_EXPS] : 0;
  };
  auto store_x = [&](int b, uint64_t q, unsigned e) __attribute__((always_inline)) {
    float v[8];
    decode8(q, e, v);
    bf16v8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (__bf16)v[i];
    *(bf16v8*)(smem + (b & bwrap) * 4096 + xput) = o;
    if ((b & bwrap) == 0 && xrow < 16) *(bf16v8*)(smem + 64 * R + xput) = o;
  };
  const char* dp = a.dc + (c.r0 + (tid >> 4)) * 256 + 16 * (tid & 15);    // of the next tile to be read
  long left = a.M - c.r0 - (tid >> 4);                                     // rows from there to the end
  auto fetch_d = [&](f32x4 d[2]) __attribute__((always_inline)) {
    d[0] = d[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (left > 0) d[0] = *(const f32x4*)dp;
    if (left > 32) d[1] = *(const f32x4*)(dp + 32 * 256);
    dp += CW_DC;
    left -= CW_TILE;
  };
  auto store_d = [&](int buf, const f32x4 d[2]) __attribute__((always_inline)) {
    *(f32x4*)(smem + buf * CW_RDC + dput) = d[0];
    *(f32x4*)(smem + buf * CW_RDC + dput + 32 * CW_RD) = d[1];
  };

  // fragments: lane 16 kg + 4 q + p asks for row 4 kg + q (+ 16 in the second read), columns 4 p .. 4 p + 3 of a 16-channel
  // tile.  Wave (tg, cih, coh) multiplies taps 2 i + tg (i < 4) with the four co tiles of its half, tap 8 with the first two
  // of b, and the ones of S with b[0]: b's order is such that the waves of a half share tap 8 and S among them.
  const int kg = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
  unsigned aoff[CW_NT];
#pragma unroll
  for (int i = 0; i < CW_NT; ++i) {
    const int t = i < 4 ? 2 * i + tg : 8;
    const int row = (t < jn ? t : jn - 1) * a.dil + 4 * kg + q;      // (without such a tap: another one's rows, and not stored)
    aoff[i] = 64 * row + 32 * (cih ^ ((row >> 2) & 1)) + 8 * p;
  }
  const int co0 = 2 * tg + cih, co1 = co0 ^ 1, co2 = 2 * (1 - tg);   // b[0], b[1], b[2] (b[3] is the tile after b[2])
  const unsigned boff = dcs + (4 * kg + q) * CW_RD + 128 * coh + 8 * p, boff0 = boff + 32 * co0, boff1 = boff + 32 * co1, boff2 = boff + 32 * co2;
  struct Frags { bf16v8 a[CW_NT], b[4]; };
  // (addresses are offsets into LDS: smem is all that this kernel has there, so it starts at 0, which the host checks before the
  // first launch; as offsets from a pointer they cost 1 % more time, an addition each)
  auto frag = [&](unsigned at, int second) __attribute__((always_inline)) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at + second));
    return __builtin_bit_cast(bf16v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto load = [&](Frags& f, int T, int buf, int ks) __attribute__((always_inline)) {
    const unsigned at = buf * CW_RDC, base = (unsigned)T * 4096u + 2048u * ks;      // (base: modulo 2^32, a multiple of the ring)
    f.b[0] = frag(at + boff0 + 32 * ks * CW_RD, 16 * CW_RD);
    f.b[1] = frag(at + boff1 + 32 * ks * CW_RD, 16 * CW_RD);
    f.b[2] = frag(at + boff2 + 32 * ks * CW_RD, 16 * CW_RD);
    f.b[3] = frag(at + boff2 + 32 * ks * CW_RD + 32, 16 * CW_RD);
#pragma unroll
    for (int i = 0; i < CW_NT; ++i) f.a[i] = frag((base + aoff[i]) & wrap, 16 * 64);
  };
  // the rows of a lane's slots as masks: four bits -> two words, from a table of 16 entries behind the dc tiles
  const int table = dcs + 3 * CW_RDC;
  if (tid < 16) *(uint2*)(smem + table + 8 * tid) = make_uint2((tid & 1 ? 0xffffu : 0u) | (tid & 2 ? 0xffff0000u : 0u), (tid & 4 ? 0xffffu : 0u) | (tid & 8 ? 0xffff0000u : 0u));
  auto mask = [&](unsigned rows) __attribute__((always_inline)) {
    const uint2 lo = *(const uint2*)(smem + table + 8 * ((rows >> (4 * kg)) & 15u)), hi = *(const uint2*)(smem + table + 8 * ((rows >> (16 + 4 * kg)) & 15u));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };

  f32x4 acc[4][4], acc8[2], accs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[i][n] = accs;
  acc8[0] = acc8[1] = accs;
  const int my_tap = lane & 15, my_shift = cw_shift(a, my_tap), o_first = cw_shift(a, 0), o_last = cw_shift(a, jn - 1);
  const unsigned ones = my_tap < jn ? 0x3f803f80u : 0u;
  const int lstep = 32 % L;
  int lb = c.lb;
  // One step: rows that leave their sequence are cleared, and the next step's fragments (tile T, ks) are requested among this
  // one's matrix instructions.  There is no branch around a tap that reaches no row: 19 matrix instructions in one piece with
  // the next step's reads between them took less time than 14 to 16 behind branches.
  auto step = [&](Frags& f, Frags& next, int T, int buf, int ks) __attribute__((always_inline)) {
    u32x4 v = {ones, ones, ones, ones};
    if (!(lb + 31 < L && lb + o_first >= 0 && lb + 31 + o_last < L)) {
      const unsigned mine = cw_inside(lb, L, my_shift);    // lane t finds tap t's rows
      unsigned rows[CW_NT];
#pragma unroll
      for (int i = 0; i < CW_NT; ++i) rows[i] = __builtin_amdgcn_readlane(mine, i < 4 ? 2 * i + tg : 8);
      if (__ballot(mine != 0u && mine != ~0u)) {
#pragma unroll
        for (int i = 0; i < CW_NT; ++i) f.a[i] = cw_clear(f.a[i], mask(rows[i]));
        v &= mask(mine);
      } else {                                             // every tap all or nothing, as where shifts and lengths are multiples of 32
#pragma unroll
        for (int i = 0; i < CW_NT; ++i) f.a[i] = cw_clear(f.a[i], u32x4{rows[i], rows[i], rows[i], rows[i]});
        v &= mine;
      }
    }
    load(next, T, buf, ks);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.a[i], f.b[n], acc[i][n], 0, 0, 0);
#pragma unroll
    for (int n = 0; n < 2; ++n) acc8[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.a[4], f.b[n], acc8[n], 0, 0, 0);
    accs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16v8, v), f.b[0], accs, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 18; ++u) {                         // (a matrix instruction takes 16 cycles, its issue 4)
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    lb += lstep;
    lb -= lb >= L ? L : 0;
  };

  {
    f32x4 d0[2], d1[2];
    fetch_d(d0);
    fetch_d(d1);                                           // (past the chunk's end: rows that no step multiplies)
#pragma unroll 1
    for (int b = tid >> 8; b < sb + 2; b += 8) {           // two blocks at a time, four times in flight
      uint64_t xq[4];
      unsigned xs[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) fetch_x(b + 2 * u, xq[u], xs[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (b + 2 * u < sb + 2) store_x(b + 2 * u, xq[u], xs[u]);
    }
    store_d(0, d0);
    store_d(1, d1);
  }
  __syncthreads();
  // What tile T + 2 needs is stored at the end of tile T; it was requested at the start of tile T - 1.
  struct Staged { f32x4 d[2]; uint64_t q; unsigned e; };
  auto request = [&](Staged& s, int T) __attribute__((always_inline)) {
    fetch_d(s.d);
    if (tid < 256) fetch_x(T + sb, s.q, s.e);
  };
  Frags f0, f1;
  load(f0, 0, 0, 0);
  int buf = 0;                                             // T mod 3
  auto tile = [&](int T, Staged& now, Staged& later) __attribute__((always_inline)) {
    const int nbuf = buf == 2 ? 0 : buf + 1, fbuf = buf == 0 ? 2 : buf - 1;
    request(later, T + 3);                                 // (past the chunk's end: stored, and not used)
    step(f0, f1, T, buf, 1);
    step(f1, f0, T + 1, nbuf, 0);
    store_d(fbuf, now.d);                                  // the buffer and the block whose last readers passed the previous barrier
    if (tid < 256) store_x(T + 2 + sb, now.q, now.e);
    buf = nbuf;
    __syncthreads();
  };
  Staged s0, s1;
  request(s0, 2);
  for (int T = 0; T < c.nt; T += 2) {
    tile(T, s0, s1);
    if (T + 1 < c.nt) tile(T + 1, s1, s0);
  }

  // D[row 4 g + v][col]: ci = 32 quarter + 16 cih + 4 g + v, co = 64 coh + 16 (the fragment's co tile) + (lane & 15)
  const int g = lane >> 4, cn = lane & 15;
  const int co[4] = {16 * co0, 16 * co1, 16 * co2, 16 * co2 + 16};
#pragma unroll
  for (int i = 0; i < CW_NT; ++i) {
    const int t = i < 4 ? 2 * i + tg : 8;
    if (t >= jn) continue;
    float* dst = a.slabs + ((long)chunk * jn + t) * CW_SLAB + (32 * quarter + 16 * cih + 4 * g) * DRK_C + 64 * coh + cn;
#pragma unroll
    for (int n = 0; n < (i < 4 ? 4 : 2); ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v) dst[v * DRK_C + co[n]] = i < 4 ? acc[i][n][v] : acc8[n & 1][v];
  }
  if (quarter == 0) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (4 * g + v < jn) a.slabs[((long)chunk * jn + 4 * g + v) * CW_SLAB + DRK_C * DRK_C + 64 * coh + co[0] + cn] = accs[v];
  }
}

// dwt[t][ci][co] += gamma[ci] * sum of P + beta[ci] * sum of S over the chunks (gamma null: 1 and 0).  A workgroup joins 4
// rows of P: eight groups of threads take an eighth of the chunks each, in order, and are then added in order, so that
// enough loads are in flight to read the slabs at the rate they come from the Infinity Cache.
__global__ void __launch_bounds__(1024) k_wgrad_ck8_join(const float* __restrict__ slabs, int chunks, int taps,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta,
                                                         float* __restrict__ dwt) {
  __shared__ f32x4 lp[8][4][32], ls[8][32];
  const int col = threadIdx.x & 31, sub = (threadIdx.x >> 5) & 3, grp = threadIdx.x >> 7;
  const int t = blockIdx.y, ci = blockIdx.x * 4 + sub, per = (chunks + 7) / 8;
  const int k0 = grp * per, k1 = k0 + per < chunks ? k0 + per : chunks;
  const long step = (long)taps * CW_SLAB;
  const float* s = slabs + (long)t * CW_SLAB + 4 * col;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 P = zero, S = zero;
#pragma unroll 8
  for (int k = k0; k < k1; ++k) P += *(const f32x4*)(s + k * step + ci * DRK_C);
  if (gamma && sub == 0) {
#pragma unroll 8
    for (int k = k0; k < k1; ++k) S += *(const f32x4*)(s + k * step + DRK_C * DRK_C);
    ls[grp][col] = S;
  }
  lp[grp][sub][col] = P;
  __syncthreads();
  if (grp) return;
  P = S = zero;
#pragma unroll
  for (int g = 0; g < 8; ++g) P += lp[g][sub][col];
  if (gamma) {
#pragma unroll
    for (int g = 0; g < 8; ++g) S += ls[g][col];
    P = P * gamma[ci] + S * beta[ci];
  }
  f32x4* o = (f32x4*)(dwt + ((long)t * DRK_C + ci) * DRK_C + 4 * col);
  *o += P;
}

// ------------------------------------------------------------------------------------------------ C ABI
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
#define CK_FWD_WGS 8192

extern "C" int drk_ln_fwd_ck8(const float* feat, const float* tbias, long tb_stride, const float* gamma, const float* beta,
                              const unsigned char* relu_mask, int gate_self, void* h, signed char* codes, unsigned char* exps,
                              float* rstd, unsigned char* gates, int B, int L, int ln, void* stream) {
  DRK_SHAPE_GUARD("drk_ln_fwd_ck8");
  CKCHECK(feat && h && codes && exps && (!ln || (gamma && beta && rstd)) && (ln || !tbias), "drk_ln_fwd_ck8");
  CKCHECK((gates != nullptr) == (relu_mask || gate_self) && !(relu_mask && gate_self), "drk_ln_fwd_ck8 (gates need relu_mask or gate_self)");
  CKCHECK(aligned16(feat) && aligned16(tbias) && tb_stride % 4 == 0 && tb_stride >= 0 && aligned16(gamma) && aligned16(beta) && aligned16(h) &&
              ((uintptr_t)codes & 7) == 0 && ((uintptr_t)relu_mask & 7) == 0, "drk_ln_fwd_ck8 (alignment)");
  const CkFwdArgs a = {feat, tbias, gamma, beta, relu_mask, tb_stride, h, (uint64_t*)codes, exps, gates, rstd, (long)B * L, L, gate_self};
  long grid = (a.M + 15) / 16;
  if (grid > CK_FWD_WGS) grid = CK_FWD_WGS;
  if (ln) hipLaunchKernelGGL(k_ln_fwd_ck8<true>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(k_ln_fwd_ck8<false>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}

extern "C" int drk_ck8_unpack(const signed char* codes, const unsigned char* exps, void* out, int dtype, int B, int L, void* stream) {
  DRK_SHAPE_GUARD("drk_ck8_unpack");
  CKCHECK(codes && exps && out && aligned16(out) && ((uintptr_t)codes & 7) == 0, "drk_ck8_unpack");
  const long n = (long)B * L * (DRK_C / 4);
  long grid = (n + 1023) / 1024;
  if (grid > CK_FWD_WGS) grid = CK_FWD_WGS;
  if (dtype == DRK_F32) hipLaunchKernelGGL(k_ck8_unpack<false>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const unsigned*)codes, exps, (char*)out, n);
  else if (dtype == DRK_BF16) hipLaunchKernelGGL(k_ck8_unpack<true>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const unsigned*)codes, exps, (char*)out, n);
  else return drk_set_error_msg(DRK_EINVAL, "drk_ck8_unpack: dtype is DRK_F32 or DRK_BF16");
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}

#define CK_BWD_WGS 1024
static long ck_bwd_grid(long M) { return (M + 15) / 16 < CK_BWD_WGS ? (M + 15) / 16 : CK_BWD_WGS; }

extern "C" long drk_ln_bwd_ck8_workspace_bytes(int B, int L) {
  return B <= 0 || L <= 0 ? 0 : ck_bwd_grid((long)B * L) * 4 * DRK_C * (long)sizeof(float);
}

extern "C" int drk_ln_bwd_ck8(const float* dh, const signed char* codes, const unsigned char* exps, const float* rstd,
                              const float* gamma, const float* g_resid, const unsigned char* gates, float* dfeat, void* dc,
                              float* dxin, float* sums, int B, int L, void* workspace, long workspace_bytes, void* stream) {
  DRK_SHAPE_GUARD("drk_ln_bwd_ck8");
  CKCHECK(dh && (dfeat || dc) && (!dc || gates) && (!codes || (exps && rstd && gamma)), "drk_ln_bwd_ck8");
  CKCHECK(aligned16(dh) && aligned16(gamma) && aligned16(g_resid) && aligned16(dfeat) && aligned16(dc) && aligned16(dxin) && ((uintptr_t)codes & 7) == 0,
          "drk_ln_bwd_ck8 (alignment)");
  CKCHECK(!sums || (workspace && aligned16(workspace) && workspace_bytes >= drk_ln_bwd_ck8_workspace_bytes(B, L)),
          "drk_ln_bwd_ck8 (sums need a workspace of drk_ln_bwd_ck8_workspace_bytes(B, L) bytes, 16-byte aligned)");
  const CkBwdArgs a = {dh, gamma, rstd, g_resid, (const uint64_t*)codes, exps, gates, dfeat, dxin, (float*)workspace, dc, (long)B * L};
  const dim3 grid((unsigned)ck_bwd_grid(a.M)), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (codes && sums) hipLaunchKernelGGL((k_ln_bwd_ck8<true, true>), grid, block, 0, st, a);
  else if (codes) hipLaunchKernelGGL((k_ln_bwd_ck8<true, false>), grid, block, 0, st, a);
  else if (sums) hipLaunchKernelGGL((k_ln_bwd_ck8<false, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_ln_bwd_ck8<false, false>), grid, block, 0, st, a);
  DRK_CHECK_LAUNCH();
  if (sums) {
    hipLaunchKernelGGL(k_ck8_sums, dim3(4 * DRK_C / 8), block, 0, st, (const float*)workspace, (int)grid.x, sums);
    DRK_CHECK_LAUNCH();
  }
  return DRK_OK;
}

// How the work is cut.  All taps in one workgroup (the ring) or one tap per workgroup; row chunks so that every CU has one
// workgroup of the ring kernel or two of the other, no more, because every chunk costs a slab of P and S per tap written and
// read (half as many workgroups: 155 us instead of 99 at 262 144 rows; one tap, one against two: 50 and 40 us).
// From this many rows on the ring is the faster one.  Ring against one tap per workgroup, us, sequences of 200:
//                     6 400        12 800        25 600       102 400       262 000 rows
//   9 taps, d = 4   25.9  22.4    28.0  29.3    29.3  40.8    50.0 112.2    97.0 267.9
//   9 taps, d = 64  26.8  20.1    29.8  24.9    32.3  33.3    61.1  84.0   123.9 196.0
//   7 taps, d = 1   22.6  21.5    24.6  26.6    26.5  36.1    44.9  89.4    90.3 210.8
//   5 taps, d = 1   20.6  20.5    22.6  23.2    24.6  29.3    42.2  67.2    87.2 153.6
//   3 taps, d = 1   17.3  16.1    20.1  17.8    22.3  21.3    39.8  43.9    84.5  97.8
//   3 taps, d = 64  17.7  15.8    21.6  17.5    25.0  21.2    48.0  42.2   104.3  92.8
// (sequences of 1 024: the same within a tenth at d = 1 to 16, and the ring gains at d = 64: 100 and 238 at 262 144 rows.)  The
// rule is the model's own, nine taps; at three, and near the border at wide dilations, it gives up to 5 us away (12 us, a
// tenth, at three taps of dilation 64).
#define CW_RING_ROWS 12800
struct CwPlan {
  bool ring;
  int tiles_per_wg, chunks, total;
};
static CwPlan cw_plan(long M, int taps, int dilation) {
  CwPlan p;
  const long tiles = (M + CW_TILE - 1) / CW_TILE;
  p.ring = taps > 1 && (long)(taps - 1) * dilation <= CW_RING_MAX - 3 * 64 && M >= CW_RING_ROWS;
  const long most = p.ring ? 64 : 512 / (2 * taps);
  const long per = (tiles + most - 1) / most;
  p.tiles_per_wg = (int)per;
  p.chunks = (int)((tiles + per - 1) / per);
  p.total = (int)tiles;
  return p;
}
static bool cw_shape_ok(int taps, int dilation) { return taps >= 1 && taps <= CW_MAX_TAPS && (taps & 1) && dilation >= 0; }

extern "C" long drk_conv_wgrad_ck8_workspace_bytes(int B, int L, int taps, int dilation) {
  if (B <= 0 || L <= 0 || !cw_shape_ok(taps, 0)) return 0;
  if (dilation < 0) return 0;
  return (long)cw_plan((long)B * L, taps, dilation).chunks * taps * CW_SLAB * (long)sizeof(float);
}

extern "C" int drk_conv_wgrad_ck8(const signed char* codes, const unsigned char* exps, const float* gamma, const float* beta,
                                  const void* dc, float* dwt, int B, int L, int taps, int dilation, void* workspace,
                                  long workspace_bytes, void* stream) {
  DRK_SHAPE_GUARD("drk_conv_wgrad_ck8");
  CKCHECK(codes && exps && dc && dwt && !gamma == !beta && cw_shape_ok(taps, dilation), "drk_conv_wgrad_ck8");
  CKCHECK(((uintptr_t)codes & 7) == 0 && aligned16(dc) && aligned16(dwt), "drk_conv_wgrad_ck8 (alignment)");
  CKCHECK(workspace && aligned16(workspace) && workspace_bytes >= drk_conv_wgrad_ck8_workspace_bytes(B, L, taps, dilation),
          "drk_conv_wgrad_ck8 (workspace: 16-byte aligned, drk_conv_wgrad_ck8_workspace_bytes(B, L, taps, dilation) bytes)");
  const long M = (long)B * L;
  CKCHECK(M < (1L << 36) && L < (1 << 30), "drk_conv_wgrad_ck8 (too many rows)");
  const CwPlan pl = cw_plan(M, taps, dilation);
  const int chunks = pl.chunks;
  const CwArgs a = {(const uint64_t*)codes, exps, (const char*)dc, (float*)workspace, M, L, taps, dilation, pl.tiles_per_wg, pl.total, chunks};
  hipStream_t st = (hipStream_t)stream;
  const unsigned g8 = (unsigned)((chunks + 7) / 8);
  if (pl.ring) {
    static std::atomic<unsigned> lds_set[DRK_MAX_DEVICES];      // the kernel may use more than 64 KB of LDS: said once per device
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return drk_set_error(e, "drk_conv_wgrad_ck8(hipGetDevice)");
    if (dev < 0 || dev >= DRK_MAX_DEVICES || !lds_set[dev].load(std::memory_order_acquire)) {
      hipFuncAttributes at;
      e = hipFuncGetAttributes(&at, (const void*)k_wgrad_ck8_ring);
      if (e != hipSuccess) return drk_set_error(e, "drk_conv_wgrad_ck8(hipFuncGetAttributes)");
      if (at.sharedSizeBytes != 0) return drk_set_error_msg(DRK_EINVAL, "drk_conv_wgrad_ck8: this build's kernel has static LDS, its addresses take the ring to start at 0");
      e = hipFuncSetAttribute((const void*)k_wgrad_ck8_ring, hipFuncAttributeMaxDynamicSharedMemorySize, CW_RING_LDS(CW_RING_MAX));
      if (e != hipSuccess) return drk_set_error(e, "drk_conv_wgrad_ck8(LDS size)");
      if (dev >= 0 && dev < DRK_MAX_DEVICES) lds_set[dev].store(1u, std::memory_order_release);
    }
    hipLaunchKernelGGL(k_wgrad_ck8_ring, dim3(g8 * 32), dim3(512), CW_RING_LDS(cw_ring_rows(taps, dilation)), st, a);
  } else {
    hipLaunchKernelGGL(k_wgrad_ck8_tap, dim3(g8 * 16, (unsigned)taps), dim3(256), 0, st, a);
  }
  DRK_CHECK_LAUNCH();
  hipLaunchKernelGGL(k_wgrad_ck8_join, dim3(DRK_C / 4, (unsigned)taps), dim3(1024), 0, st, (const float*)workspace, chunks, taps, gamma, beta, dwt);
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}
