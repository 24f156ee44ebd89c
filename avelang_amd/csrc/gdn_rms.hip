// Root-mean-square norm over the last axis for gfx950, with the residual's
// addition, an output in 8 bits, and its gradients (declared in gdn_attn.h):
//     h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd (w + offset)
//     e = dy (w + offset),  hh = h rstd,  dx = rstd (e - hh mean(e hh)) + dh
//     dw = sum over rows of dy hh
// Every pass is bound by HBM: a row is read once into registers (16 bytes per
// lane and load), reduced there and written once; the 8-bit output's maximum is
// a second reduction of the same registers.  h is rounded to its type before
// the norm, so that y belongs to the h that the next layer adds to and the
// backward needs h alone.
//
// bf16 with a residual: 8192 rows of 2048 into e4m3 24 us, 4.9 TB/s; of 4096 46 us,
// 5.9 TB/s read and written, its backward 43 us, 6.2 TB/s, and 4 us for the weight's
// sum; one row of 2048 4.7 us: a row's reduction between two round trips to HBM, x and the
// residual's and, behind the stores of h, the weight's.  Rows of more than 8192 elements (bf16)
// are read again for each step: 2048 rows of 12288 46 us, into e4m3 48, the backward 80; of
// 16384 62, 64 and 101.
#include "gdn_norm_rows.h"
#include "gdn_bits8.h"
#include "../../include/gdn_attn.h"

namespace gdn {

// Largest value over the lanes of a row (as row_sum).
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x, uint32_t* red) {
#pragma unroll
  for (int off = 1; off < (LPR < 64 ? LPR : 64); off *= 2)
    x = max(x, (uint32_t)__shfl_xor((int)x, off));
  if constexpr (LPR > 64) {
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < LPR / 64; ++w) x = max(x, red[w]);
  }
  return x;
}

// 1 / sqrt(mean + eps) of a row's sum of squares.
__device__ __forceinline__ float rstd_of(float s, int D, float eps) { return rsqrtf(s * (1.f / D) + eps); }

struct RmsArgs {
  const void* x;
  const void* res;
  const void* w;
  void* y;
  void* h;
  float* scale;
  long long rows;
  int D;
  float eps, offset;
  int wt, code;   // code: the output's type where it is one of 8 bits
};

// Codes of VEC values from element c of a row of D (at byte base): the nearest fp32
// quotients by the scale (one correction), rounded.
template <int VEC>
__device__ __forceinline__ void st_codes(void* p, long long base, int c, int D, const float (&f)[VEC],
                                         const Row8& r, int code) {
  uint32_t w[VEC / 4];
  float q[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    q[j] = f[j] * r.inv;
    q[j] = fmaf(fmaf(-q[j], r.scale, f[j]), r.inv, q[j]);
  }
#pragma unroll
  for (int u = 0; u < VEC / 4; ++u)
    w[u] = code == GDN_DTYPE_E4M3 ? e4m3_4(q[4 * u], q[4 * u + 1], q[4 * u + 2], q[4 * u + 3])
                                  : int8_4(q[4 * u], q[4 * u + 1], q[4 * u + 2], q[4 * u + 3]);
  uint8_t* dst = static_cast<uint8_t*>(p) + base + c;
  if (c + VEC <= D) {
    if constexpr (VEC == 8)
      *reinterpret_cast<u32x2b*>(dst) = u32x2b{w[0], w[1]};
    else
      *reinterpret_cast<u32b*>(dst) = w[0];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j < D) dst[j] = static_cast<uint8_t>(w[j / 4] >> (8 * (j % 4)));
  }
}

// x + residual (rounded to the residual's type RT, and stored as h) of VEC
// elements from element c of a row.
template <int DT, int RT, int VEC>
__device__ __forceinline__ void add_row(const RmsArgs& a, long long base, int c, float (&f)[VEC],
                                        const float (&r)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = round_to<RT>(f[j] + r[j]);
  if (c < a.D) st_row<RT, VEC>(a.h, base, c, a.D, f);
}

template <int VEC>
__device__ __forceinline__ void scale_row(const RmsArgs& a, int c, float rstd, float (&f)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] *= rstd;
  if (a.w) {
    float p[VEC];
    ld_par<VEC>(a.w, 0, c, a.D, a.wt, p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] *= p[j] + a.offset;
  }
}

// One row per group of LPR lanes, VPT vectors of 16 bytes of x per lane.
template <int DT, int RT, int LPR, int VPT>
__global__ __launch_bounds__(256) void rms_fwd_kernel(RmsArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[4];
  __shared__ uint32_t redm[4];
  const int l = threadIdx.x % LPR;
  const long long r = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (LPR < 256 && r >= a.rows) return;
  const long long base = r * a.D;
  float f[VPT][VEC];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) ld_row<DT, VEC>(a.x, base, (l + LPR * i) * VEC, a.D, f[i]);
  if (a.res) {
    float q[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) ld_row<RT, VEC>(a.res, base, (l + LPR * i) * VEC, a.D, q[i]);
#pragma unroll
    for (int i = 0; i < VPT; ++i) add_row<DT, RT, VEC>(a, base, (l + LPR * i) * VEC, f[i], q[i]);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += f[i][j] * f[i][j];   // (past the row's end 0)
  s = row_sum<LPR>(s, red);
  const float rstd = rstd_of(s, a.D, a.eps);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (l + LPR * i) * VEC;
    if (c >= a.D) break;
    scale_row<VEC>(a, c, rstd, f[i]);
    if (!a.scale) {
      st_row<DT, VEC>(a.y, base, c, a.D, f[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j < a.D) m = max(m, abs_bits(f[i][j]));
    }
  }
  if (!a.scale) return;
  const Row8 q = row8(row_max<LPR>(m, redm), a.code, s);
  if (l == 0) a.scale[r] = q.scale;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (l + LPR * i) * VEC;
    if (c < a.D) st_codes<VEC>(a.y, base, c, a.D, f[i], q, a.code);
  }
}

// Rows longer than a workgroup's registers: read again from cache for each step.
template <int DT, int RT>
__global__ __launch_bounds__(256) void rms_fwd_long_kernel(RmsArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[4];
  __shared__ uint32_t redm[4];
  const long long r = blockIdx.x, base = r * a.D;
  float f[VEC], s = 0.f;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    ld_row<DT, VEC>(a.x, base, c, a.D, f);
    if (a.res) {
      float q[VEC];
      ld_row<RT, VEC>(a.res, base, c, a.D, q);
      add_row<DT, RT, VEC>(a, base, c, f, q);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += f[j] * f[j];
  }
  s = row_sum<256>(s, red);
  const float rstd = rstd_of(s, a.D, a.eps);
  // (a lane reads again what itself has written)
  auto load = [&](int c) {
    if (a.res) ld_row<RT, VEC>(a.h, base, c, a.D, f);
    else ld_row<DT, VEC>(a.x, base, c, a.D, f);
    scale_row<VEC>(a, c, rstd, f);
  };
  if (!a.scale) {
    for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
      load(c);
      st_row<DT, VEC>(a.y, base, c, a.D, f);
    }
    return;
  }
  uint32_t m = 0;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j < a.D) m = max(m, abs_bits(f[j]));
  }
  const Row8 q = row8(row_max<256>(m, redm), a.code, s);
  if (threadIdx.x == 0) a.scale[r] = q.scale;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
    st_codes<VEC>(a.y, base, c, a.D, f, q, a.code);
  }
}

struct RmsBwdArgs {
  const void* h;
  const void* w;
  const void* dy;
  const void* dh;
  void* dx;
  void* dr;
  float* pw;     // [parts][D] partial sums of dweight (NULL: not wanted, or no parts)
  void* dw;      // [D] dweight of the weight's type where one workgroup takes all rows (else NULL)
  float* rstd;   // rows longer than registers hold: [rows] (NULL: not wanted)
  long long rows;
  int D;
  float eps, offset;
  int wt, groups;   // groups walking the rows
};

// The gradients of VEC elements from element c of a row: e, hh in; stores.
template <int DT, int RT, int VEC>
__device__ __forceinline__ void st_grads(const RmsBwdArgs& a, long long base, int c, const float (&f)[VEC]) {
  st_row<DT, VEC>(a.dx, base, c, a.D, f);
  if (a.dr) st_row<RT, VEC>(a.dr, base, c, a.D, f);
}

// Element c of dweight, of type wt.
__device__ __forceinline__ void st_weight(void* dw, long long c, float s, int wt) {
  if (wt == GDN_DTYPE_F32) ste<GDN_DTYPE_F32>(dw, c, s);
  else if (wt == GDN_DTYPE_BF16) ste<GDN_DTYPE_BF16>(dw, c, s);
  else ste<GDN_DTYPE_F16>(dw, c, s);
}

// Two sums over the lanes of a row at once (as row_sum).
template <int LPR>
__device__ __forceinline__ void row_sum2(float& x, float& y, float (*red)[4]) {
#pragma unroll
  for (int off = 1; off < (LPR < 64 ? LPR : 64); off *= 2) {
    x += __shfl_xor(x, off);
    y += __shfl_xor(y, off);
  }
  if constexpr (LPR > 64) {
    if (threadIdx.x % 64 == 0) {
      red[0][threadIdx.x / 64] = x;
      red[1][threadIdx.x / 64] = y;
    }
    __syncthreads();
    x = red[0][0];
    y = red[1][0];
#pragma unroll
    for (int w = 1; w < LPR / 64; ++w) {
      x += red[0][w];
      y += red[1][w];
    }
  }
}

// A group of LPR lanes walks the rows gid, gid + groups, ..., its columns'
// weights and partial sums of dweight in registers, with the next row loaded
// while the current one is reduced; the groups of a workgroup are summed in LDS.
// (rstd is formed again with the other sum of the row, not read: nothing is kept
// of a forward but h.)
template <int DT, int RT, int LPR, int VPT>
__global__ __launch_bounds__(256) void rms_bwd_kernel(RmsBwdArgs a) {
  constexpr int VEC = Elt<DT>::VEC, RV = VEC / Elt<RT>::VEC;   // 16-byte loads of RT per one of DT
  constexpr int GPW = 256 / LPR;
  __shared__ float red[2][2][4];
  extern __shared__ float part[];   // [GPW][D] where groups are summed
  const int l = threadIdx.x % LPR, gi = threadIdx.x / LPR;
  const int gid = blockIdx.x * GPW + gi;
  const bool live = gid < a.groups;
  float w[VPT][VEC], dw[VPT][VEC];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (a.w) ld_par<VEC>(a.w, 0, (l + LPR * i) * VEC, a.D, a.wt, w[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = a.w ? w[i][j] + a.offset : 1.f;
      dw[i][j] = 0.f;
    }
  }
  // the next row's bits, on their way while this one is reduced
  u32x4e rx[VPT][RV], rh[VPT][RV], ry[VPT];
  auto load = [&](long long r) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (l + LPR * i) * VEC;
      ry[i] = ld_raw<DT>(a.dy, r * a.D, c, a.D);
#pragma unroll
      for (int u = 0; u < RV; ++u) {
        rx[i][u] = ld_raw<RT>(a.h, r * a.D, c + u * Elt<RT>::VEC, a.D);
        rh[i][u] = a.dh ? ld_raw<RT>(a.dh, r * a.D, c + u * Elt<RT>::VEC, a.D) : u32x4e{0, 0, 0, 0};
      }
    }
  };
  const float inv_d = 1.f / a.D;
  int ph = 0;
  if (live && gid < a.rows) load(gid);
  for (long long r = live ? gid : a.rows; r < a.rows; r += a.groups, ph ^= 1) {
    float x[VPT][VEC], dy[VPT][VEC], dh[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      unpack<DT>(ry[i], dy[i]);
#pragma unroll
      for (int u = 0; u < RV; ++u) {
        unpack<RT>(rx[i][u], x[i] + u * Elt<RT>::VEC);
        unpack<RT>(rh[i][u], dh[i] + u * Elt<RT>::VEC);
      }
    }
    if (r + a.groups < a.rows) load(r + a.groups);
    float ss = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ss += x[i][j] * x[i][j];
        s += dy[i][j] * w[i][j] * x[i][j];
      }
    row_sum2<LPR>(ss, s, red[ph]);
    const float rstd = rstd_of(ss, a.D, a.eps);
    s *= rstd * inv_d;   // mean(e hh)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[i][j] *= rstd;
        dw[i][j] += dy[i][j] * x[i][j];
        x[i][j] = rstd * (dy[i][j] * w[i][j] - x[i][j] * s) + dh[i][j];
      }
      const int c = (l + LPR * i) * VEC;
      if (c < a.D) st_grads<DT, RT, VEC>(a, r * a.D, c, x[i]);
    }
  }
  if (!a.pw && !a.dw) return;
  if constexpr (GPW > 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (l + LPR * i) * VEC + j;
        if (c < a.D) part[gi * a.D + c] = dw[i][j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += 256) {
      float s = part[c];
      for (int g = 1; g < GPW; ++g) s += part[g * a.D + c];
      if (a.dw) st_weight(a.dw, c, s, a.wt);
      else a.pw[(long long)blockIdx.x * a.D + c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (l + LPR * i) * VEC;
      if (a.dw) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (c + j < a.D) st_weight(a.dw, c + j, dw[i][j], a.wt);
      } else if (c < a.D) {
        st_row<GDN_DTYPE_F32, VEC>(a.pw, (long long)gid * a.D, c, a.D, dw[i]);
      }
    }
  }
}

// Rows longer than registers hold: dx and rstd; the sums by rms_cols_kernel.
template <int DT, int RT>
__global__ __launch_bounds__(256) void rms_bwd_long_kernel(RmsBwdArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[2][4];
  const long long r = blockIdx.x, base = r * a.D;
  float x[VEC], dy[VEC], w[VEC], ss = 0.f, s = 0.f;
  auto load = [&](int c) {
    ld_row<RT, VEC>(a.h, base, c, a.D, x);
    ld_row<DT, VEC>(a.dy, base, c, a.D, dy);
    if (a.w) ld_par<VEC>(a.w, 0, c, a.D, a.wt, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (a.w) dy[j] *= w[j] + a.offset;
  };
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ss += x[j] * x[j];
      s += dy[j] * x[j];
    }
  }
  row_sum2<256>(ss, s, red);
  const float rstd = rstd_of(ss, a.D, a.eps);
  s *= rstd / a.D;
  if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
    float dh[VEC];
    if (a.dh) ld_row<RT, VEC>(a.dh, base, c, a.D, dh);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = rstd * (dy[j] - x[j] * rstd * s) + (a.dh ? dh[j] : 0.f);
    st_grads<DT, RT, VEC>(a, base, c, x);
  }
}

// Partial sums of dweight over the rows [p, p + 1) * span: a lane per column.
template <int DT, int RT>
__global__ __launch_bounds__(256) void rms_cols_kernel(RmsBwdArgs a, long long span) {
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.D) return;
  const long long i0 = blockIdx.y * span, i1 = min(a.rows, i0 + span);
  float dw = 0.f;
  for (long long i = i0; i < i1; ++i)
    dw += lde<DT>(a.dy, i * a.D + c) * (lde<RT>(a.h, i * a.D + c) * a.rstd[i]);
  a.pw[blockIdx.y * (long long)a.D + c] = dw;
}

// dw[c] = sum over p < P of part[p][c], in a fixed order: 64 columns per
// workgroup, 16 lanes per column.
__global__ __launch_bounds__(1024) void rms_sum_kernel(const float* part, void* dw, int P, int D, int wt) {
  __shared__ float red[16][64];
  const int l = threadIdx.x % 64, sl = threadIdx.x / 64;
  const long long c = (long long)blockIdx.x * 64 + l;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int p = sl; p < P; p += 16) s += part[(long long)p * D + c];
  }
  red[sl][l] = s;
  __syncthreads();
  if (sl == 0 && c < D) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][l];
    st_weight(dw, c, s, wt);
  }
}

}  // namespace gdn

namespace {

// Groups that walk the rows of the backward, and the partial sums they leave (0:
// none): two workgroups per CU, no more groups than rows; a few rows take one
// workgroup, which writes the weight's gradient itself (replayed, 4 rows of 1024
// bf16: 4.4 us, with a second launch 6.2; 8, two to a group: 5.5 and 6.2; 16, four
// to a group: 7.6 and 6.3; a call's host time is 8 us less without).
struct RmsPlan {
  gdn::RowForm f;
  long long groups, parts, span;
};
constexpr int kRmsFew = 2;   // rows per group of that one
RmsPlan rms_plan(long long rows, int D, int dtype) {
  RmsPlan p{gdn::row_form(D, dtype), 0, 0, 0};
  if (!p.f.lpr) {
    p.parts = rows < 64 ? (rows ? rows : 1) : 64;
    p.span = (rows + p.parts - 1) / p.parts;
    return p;
  }
  const int gpw = 256 / p.f.lpr;
  p.groups = 2LL * gdn::device_cus() * gpw;
  if (p.groups > rows) p.groups = rows;
  if (rows <= (long long)kRmsFew * gpw) {
    if (p.groups > gpw) p.groups = gpw;
    return p;
  }
  p.parts = (p.groups + gpw - 1) / gpw;
  return p;
}

int check_rms(const char* name, long long rows, int D, int dtype, int r_dtype, int w_dtype) {
  if (rows < 0 || D < 1)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": rows must be >= 0 and D >= 1");
  if (!gdn::dtype_ok(dtype) || !gdn::dtype_ok(w_dtype) || (r_dtype != dtype && r_dtype != GDN_DTYPE_F32))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported dtype code");
  if (rows >= (1LL << 31) || D > (1 << 28))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  return GDN_OK;
}

}  // namespace

#define GDN_RMS_FORMS(CALL, TT, RR)                                                        \
  CALL(TT, RR, 16, 1) CALL(TT, RR, 32, 1) CALL(TT, RR, 64, 1) CALL(TT, RR, 64, 2)          \
      CALL(TT, RR, 64, 4) CALL(TT, RR, 256, 2) CALL(TT, RR, 256, 4)
#define GDN_RMS_TYPES(FORMS, LONG, CALL)                                                   \
  FORMS(CALL, GDN_DTYPE_BF16, GDN_DTYPE_BF16)                                              \
  FORMS(CALL, GDN_DTYPE_BF16, GDN_DTYPE_F32)                                               \
  FORMS(CALL, GDN_DTYPE_F16, GDN_DTYPE_F16)                                                \
  FORMS(CALL, GDN_DTYPE_F16, GDN_DTYPE_F32)                                                \
  FORMS(CALL, GDN_DTYPE_F32, GDN_DTYPE_F32)                                                \
  CALL(GDN_DTYPE_F32, GDN_DTYPE_F32, 256, 8)                                               \
  LONG(GDN_DTYPE_BF16, GDN_DTYPE_BF16)                                                     \
  LONG(GDN_DTYPE_BF16, GDN_DTYPE_F32)                                                      \
  LONG(GDN_DTYPE_F16, GDN_DTYPE_F16)                                                       \
  LONG(GDN_DTYPE_F16, GDN_DTYPE_F32)                                                       \
  LONG(GDN_DTYPE_F32, GDN_DTYPE_F32)

extern "C" int gdn_rms_norm_fwd(const void* x, const void* residual, const void* weight, void* y,
                                void* h, float* scale, long long rows, int D, float eps,
                                float offset, int dtype, int r_dtype, int w_dtype, int out_dtype,
                                void* stream) {
  const char* name = "gdn_rms_norm_fwd";
  if (const int rc = check_rms(name, rows, D, dtype, r_dtype, w_dtype)) return rc;
  const bool bits8 = out_dtype == GDN_DTYPE_E4M3 || out_dtype == GDN_DTYPE_I8;
  if (!bits8 && out_dtype != dtype)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": out_dtype must be dtype or an 8-bit type");
  if (rows == 0) return GDN_OK;
  if (!x || !y || (residual && !h) || (bits8 && !scale))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": x and y, h with a residual and scale with "
                                                            "8 bits must be non-NULL");
  const gdn::RowForm f = gdn::row_form(D, dtype);
  const int per = f.lpr ? 256 / f.lpr : 1;   // rows per workgroup
  if (const int fit = gdn_host::check_lanes(name, (rows + per - 1) / per, 256)) return fit;
  const size_t n = (size_t)rows * D, xb = dtype == GDN_DTYPE_F32 ? 4 : 2, rb = r_dtype == GDN_DTYPE_F32 ? 4 : 2;
  const size_t yb = bits8 ? 1 : xb, wb = (size_t)D * (w_dtype == GDN_DTYPE_F32 ? 4 : 2);
  // (a lane writes where it has read, of the same width)
  auto apart = [&](const void* out, size_t ob, const void* in, size_t ib) {
    return !in || (out == in && ob == ib) || !gdn_host::overlaps(out, n * ob, in, n * ib);
  };
  // (the weight is read behind h's stores; of a single row y may be the weight)
  auto over = [&](const void* out, size_t ob) { return weight && gdn_host::overlaps(out, n * ob, weight, wb); };
  if ((over(y, yb) && !(rows == 1 && y == weight && yb * D == wb)) || (residual && over(h, rb)))
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": outputs must not overlap the weight");
  if (!apart(y, yb, x, xb) || !apart(y, yb, residual, rb) ||
      (residual && (!apart(h, rb, x, xb) || !apart(h, rb, residual, rb) ||
                    gdn_host::overlaps(h, n * rb, y, n * yb))))
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": outputs must not overlap each other, or an input "
                                                             "but as a whole of the same element size");
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
  const gdn::RmsArgs a{x, residual, weight, y, h, bits8 ? scale : nullptr, rows, D, eps, offset, w_dtype, out_dtype};
#define GDN_RF(TT, RR, LL, VV)                                                                   \
  if (dtype == TT && r_dtype == RR && f.lpr == LL && f.vpt == VV) {                              \
    hipLaunchKernelGGL((gdn::rms_fwd_kernel<TT, RR, LL, VV>), dim3((unsigned)((rows + per - 1) / per)), \
                       dim3(256), 0, st, a);                                                     \
    return gdn_host::check_launch(name);                                                         \
  }
#define GDN_RFL(TT, RR)                                                                          \
  if (dtype == TT && r_dtype == RR) {                                                            \
    hipLaunchKernelGGL((gdn::rms_fwd_long_kernel<TT, RR>), dim3((unsigned)rows), dim3(256), 0, st, a); \
    return gdn_host::check_launch(name);                                                         \
  }
  GDN_RMS_TYPES(GDN_RMS_FORMS, GDN_RFL, GDN_RF)
#undef GDN_RF
#undef GDN_RFL
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported configuration");
}

extern "C" size_t gdn_rms_norm_bwd_workspace_bytes(long long rows, int D, int dtype) {
  if (check_rms("gdn_rms_norm_bwd_workspace_bytes", rows, D, dtype, dtype, GDN_DTYPE_F32) || rows == 0)
    return 0;
  const RmsPlan p = rms_plan(rows, D, dtype);
  return ((size_t)p.parts * D + (p.f.lpr ? 0 : rows)) * sizeof(float);
}

extern "C" int gdn_rms_norm_bwd(const void* h, const void* weight, const void* dy, const void* dh,
                                void* dx, void* dr, void* dweight, long long rows, int D, float eps,
                                float offset, int dtype, int h_dtype, int w_dtype, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* name = "gdn_rms_norm_bwd";
  if (const int rc = check_rms(name, rows, D, dtype, h_dtype, w_dtype)) return rc;
  if (rows > 0 && (!h || !dy || !dx))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": h, dy and dx must be non-NULL");
  if (dweight)
    if (const int fit = gdn_host::check_lanes(name, ((long long)D + 63) / 64, 1024)) return fit;
  RmsPlan p{};
  float* pw = nullptr;
  if (rows > 0) {
    const size_t n = (size_t)rows * D, xb = dtype == GDN_DTYPE_F32 ? 4 : 2, hb = h_dtype == GDN_DTYPE_F32 ? 4 : 2;
    const void* outs[2] = {dx, dr};
    const void* ins[3] = {h, dy, dh};
    for (int o = 0; o < 2; ++o)
      for (int i = 0; i < 3; ++i)
        if (outs[o] && ins[i] && gdn_host::overlaps(outs[o], n * (o ? hb : xb), ins[i], n * (i == 1 ? xb : hb)))
          return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": gradients must not overlap an input");
    if (dr && gdn_host::overlaps(dx, n * xb, dr, n * hb))
      return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": dx and dr must not overlap");
    p = rms_plan(rows, D, dtype);
    if (!p.f.lpr)
      if (const int fit = gdn_host::check_lanes(name, rows, 256)) return fit;
    if (dweight) {
      const size_t need = ((size_t)p.parts * D + (p.f.lpr ? 0 : rows)) * sizeof(float);
      if (need && (!workspace || workspace_bytes < need))
        return gdn_host::fail(GDN_ERR_WORKSPACE, std::string(name) + ": workspace needs " +
                                                     std::to_string(need) + " bytes, got " +
                                                     std::to_string(workspace_bytes));
      if (need) pw = static_cast<float*>(workspace);
    }
  }
  if (rows == 0 && !dweight) return GDN_OK;
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const gdn::RmsBwdArgs a{h, weight, dy, dh, dx, dr, pw, pw ? nullptr : dweight,
                            pw && !p.f.lpr ? pw + p.parts * D : nullptr, rows, D, eps, offset, w_dtype,
                            (int)p.groups};
    const int gpw = p.f.lpr ? 256 / p.f.lpr : 1;
    const size_t lds = gpw > 1 && dweight ? (size_t)gpw * D * sizeof(float) : 0;
#define GDN_RB(TT, RR, LL, VV)                                                                   \
  if (dtype == TT && h_dtype == RR && p.f.lpr == LL && p.f.vpt == VV)                            \
    hipLaunchKernelGGL((gdn::rms_bwd_kernel<TT, RR, LL, VV>),                                    \
                       dim3((unsigned)((p.groups + gpw - 1) / gpw)), dim3(256), lds, st, a);
#define GDN_RBL(TT, RR)                                                                          \
  if (dtype == TT && h_dtype == RR && !p.f.lpr) {                                                \
    hipLaunchKernelGGL((gdn::rms_bwd_long_kernel<TT, RR>), dim3((unsigned)rows), dim3(256), 0, st, a); \
    if (pw)                                                                                      \
      hipLaunchKernelGGL((gdn::rms_cols_kernel<TT, RR>),                                         \
                         dim3((unsigned)((D + 255) / 256), (unsigned)p.parts), dim3(256), 0, st, a, p.span); \
  }
    GDN_RMS_TYPES(GDN_RMS_FORMS, GDN_RBL, GDN_RB)
#undef GDN_RB
#undef GDN_RBL
  }
  // (no rows: the sum over nothing is zero)
  if (dweight && (pw || rows == 0))
    hipLaunchKernelGGL(gdn::rms_sum_kernel, dim3((unsigned)((D + 63) / 64)), dim3(1024), 0, st, pw,
                       dweight, (int)p.parts, D, w_dtype);
  return gdn_host::check_launch(name);
}
