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
#include "drk_common.h"
#include "../../include/drakes_hip.h"

typedef __bf16 bf16v8 __attribute__((ext_vector_type(8)));
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

template <bool BF16>
__global__ void __launch_bounds__(256) k_ck8_unpack(const uint64_t* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                    char* __restrict__ out, long n) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {     // eight channels each
    float v[8];
    decode8(codes[i], exps[i >> 2], v);
    if (BF16) store8_bf16(out + 16 * i, v);
    else store8((float*)(out + 32 * i), v);
  }
}

// ---- LayerNorm backward --------------------------------------------------------------------------------------------
// Row layout as above.  Column sums stay in a lane's registers over the rows its workgroup walks; the 16 rows in flight
// are joined in order through LDS and leave as one [4][128] slab per workgroup, the slabs are added in order.
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
  for (int k = s0; k < n; k += 32) s += slabs[(long)k * (4 * DRK_C) + i];
  red[s0][c] = s;
  for (int w = 16; w > 0; w >>= 1) {
    __syncthreads();
    if (s0 < w) red[s0][c] += red[s0 + w][c];
  }
  if (s0 == 0) out[i] += red[0][c];
}

// ---- weight gradient -----------------------------------------------------------------------------------------------
// Workgroup = (chunk of rows, tap).  Tiles of 64 rows of xq (decoded to bf16, shifted by the tap) and of dc lie in LDS as
// plain 256-byte rows; rows that the tap shifts out of their sequence are zero in both.  Both operands of the product
// have their K along the rows, so fragments are read transposed (ds_read_b64_tr_b16).  4 waves of 64 ci x 64 co each; the
// column sums S come from two more matrix instructions per k-step with a fragment of ones.
#define CW_TILE 64
#define CW_IMG (CW_TILE * 256)
#define CW_SLAB ((DRK_C + 1) * DRK_C)    // P [128][128], then S [128]
#define CW_MAX_TAPS 9

// byte offset of 16-byte chunk `ch` of a row: the eight 32-byte pairs of four neighbouring rows fall into different banks
__device__ __forceinline__ int cw_at(int row, int ch) { return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3))); }
__device__ __forceinline__ bf16v8 cw_frag(const char* p0, const char* p1) {
  typedef s16x4 __attribute__((address_space(3))) * lds4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p0);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p1);
  return __builtin_bit_cast(bf16v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__global__ void __launch_bounds__(256) k_wgrad_ck8(const uint64_t* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                   const char* __restrict__ dc, float* __restrict__ slabs, long M, int L, int taps,
                                                   int dil, int tiles_per_wg, int total_tiles) {
  __shared__ __attribute__((aligned(16))) char smem[2 * CW_IMG];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wr = w >> 1, wc = w & 1;
  const int t = blockIdx.y;
  const long off = (long)(t - taps / 2) * dil;
  const int T0 = blockIdx.x * tiles_per_wg, T1 = T0 + tiles_per_wg < total_tiles ? T0 + tiles_per_wg : total_tiles;
  const int srow = tid >> 4, scol = tid & 15;
  const int kg = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
  f32x4 acc[4][4], accs[2];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  accs[0] = accs[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16v8 one;
#pragma unroll
  for (int i = 0; i < 8; ++i) one[i] = (__bf16)1.f;
  for (int T = T0; T < T1; ++T) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long r = (long)T * CW_TILE + srow + 16 * i;
      const int at = cw_at(srow + 16 * i, scol);
      f32x4 dv = {0.f, 0.f, 0.f, 0.f};
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (r < M) {
        const long l = r % L + off;
        if (l >= 0 && l < L) {
          dv = *(const f32x4*)(dc + r * 256 + 16 * scol);
          decode8(codes[(r + off) * (DRK_C / 8) + scol], exps[(r + off) * CK_EXPS + (scol >> 2)], v);
        }
      }
      store8_bf16(smem + at, v);
      *(f32x4*)(smem + CW_IMG + at) = dv;
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16v8 af[4], bf[4];
      const int row = 32 * ks + 8 * kg + q;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        af[m] = cw_frag(smem + cw_at(row, 2 * (4 * wr + m) + (p >> 1)) + 8 * (p & 1), smem + cw_at(row + 4, 2 * (4 * wr + m) + (p >> 1)) + 8 * (p & 1));
        bf[m] = cw_frag(smem + CW_IMG + cw_at(row, 2 * (4 * wc + m) + (p >> 1)) + 8 * (p & 1),
                        smem + CW_IMG + cw_at(row + 4, 2 * (4 * wc + m) + (p >> 1)) + 8 * (p & 1));
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], bf[n], acc[m][n], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < 2; ++n) accs[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(one, wr ? bf[2 + n] : bf[n], accs[n], 0, 0, 0);
    }
  }
  // D[row 4 g + i][col n] of tile (m, n): ci = 64 wr + 16 m + 4 g + i, co = 64 wc + 16 n + (lane & 15)
  float* dst = slabs + ((long)blockIdx.x * taps + t) * CW_SLAB;
  const int g = lane >> 4, cn = lane & 15;
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[(64 * wr + 16 * m + 4 * g + i) * DRK_C + 64 * wc + 16 * n + cn] = acc[m][n][i];
  if (g == 0) {
#pragma unroll
    for (int n = 0; n < 2; ++n) dst[DRK_C * DRK_C + 64 * wc + 16 * (2 * wr + n) + cn] = accs[n][0];
  }
}

// dwt[t][ci][co] += gamma[ci] * sum of P + beta[ci] * sum of S over the chunks, in order (gamma null: 1 and 0)
__global__ void __launch_bounds__(256) k_wgrad_ck8_join(const float* __restrict__ slabs, int chunks, int taps,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta,
                                                        float* __restrict__ dwt) {
  const int t = blockIdx.y, ci = blockIdx.x * 8 + (threadIdx.x >> 5), c4 = 4 * (threadIdx.x & 31);
  f32x4 P = {0.f, 0.f, 0.f, 0.f}, S = P;
  for (int k = 0; k < chunks; ++k) {
    const float* s = slabs + ((long)k * taps + t) * CW_SLAB;
    P += *(const f32x4*)(s + ci * DRK_C + c4);
    if (gamma) S += *(const f32x4*)(s + DRK_C * DRK_C + c4);
  }
  f32x4* o = (f32x4*)(dwt + ((long)t * DRK_C + ci) * DRK_C + c4);
  *o += gamma ? P * gamma[ci] + S * beta[ci] : P;
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
  const long n = (long)B * L * (DRK_C / 8);
  long grid = (n + 255) / 256;
  if (grid > CK_FWD_WGS) grid = CK_FWD_WGS;
  if (dtype == DRK_F32) hipLaunchKernelGGL(k_ck8_unpack<false>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const uint64_t*)codes, exps, (char*)out, n);
  else if (dtype == DRK_BF16) hipLaunchKernelGGL(k_ck8_unpack<true>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const uint64_t*)codes, exps, (char*)out, n);
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

// Row chunks per tap: enough workgroups for the 256 CUs, no more, because every chunk costs a slab written and read.
static void cw_plan(long M, int taps, int* tiles_per_wg, int* chunks) {
  const long tiles = (M + CW_TILE - 1) / CW_TILE;
  long most = 256 / taps;
  const long tpw = (tiles + most - 1) / most;
  *tiles_per_wg = (int)tpw;
  *chunks = (int)((tiles + tpw - 1) / tpw);
}
static bool cw_shape_ok(int taps, int dilation) { return taps >= 1 && taps <= CW_MAX_TAPS && (taps & 1) && dilation >= 0; }

extern "C" long drk_conv_wgrad_ck8_workspace_bytes(int B, int L, int taps) {
  if (B <= 0 || L <= 0 || !cw_shape_ok(taps, 0)) return 0;
  int tpw, chunks;
  cw_plan((long)B * L, taps, &tpw, &chunks);
  return (long)chunks * taps * CW_SLAB * (long)sizeof(float);
}

extern "C" int drk_conv_wgrad_ck8(const signed char* codes, const unsigned char* exps, const float* gamma, const float* beta,
                                  const void* dc, float* dwt, int B, int L, int taps, int dilation, void* workspace,
                                  long workspace_bytes, void* stream) {
  DRK_SHAPE_GUARD("drk_conv_wgrad_ck8");
  CKCHECK(codes && exps && dc && dwt && !gamma == !beta && cw_shape_ok(taps, dilation), "drk_conv_wgrad_ck8");
  CKCHECK(((uintptr_t)codes & 7) == 0 && aligned16(dc) && aligned16(dwt), "drk_conv_wgrad_ck8 (alignment)");
  CKCHECK(workspace && aligned16(workspace) && workspace_bytes >= drk_conv_wgrad_ck8_workspace_bytes(B, L, taps),
          "drk_conv_wgrad_ck8 (workspace: 16-byte aligned, drk_conv_wgrad_ck8_workspace_bytes(B, L, taps) bytes)");
  const long M = (long)B * L;
  int tpw, chunks;
  cw_plan(M, taps, &tpw, &chunks);
  CKCHECK(M < (1L << 36), "drk_conv_wgrad_ck8 (too many rows)");
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(k_wgrad_ck8, dim3((unsigned)chunks, (unsigned)taps), dim3(256), 0, st, (const uint64_t*)codes, exps, (const char*)dc,
                     (float*)workspace, M, L, taps, dilation, tpw, (int)((M + CW_TILE - 1) / CW_TILE));
  DRK_CHECK_LAUNCH();
  hipLaunchKernelGGL(k_wgrad_ck8_join, dim3(DRK_C / 8, (unsigned)taps), dim3(256), 0, st, (const float*)workspace, chunks, taps, gamma, beta, dwt);
  DRK_CHECK_LAUNCH();
  return DRK_OK;
}
