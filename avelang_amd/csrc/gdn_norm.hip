// Layer norm over the last axis for gfx950, forward and backward (declared in
// gdn_linear.h):
//     xh = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  y = xh w + b
//     e  = dy w,  dx = rstd (e - mean(e) - xh mean(e xh))
//     dw = sum over rows of dy xh,  db = sum over rows of dy
// Every pass is bound by HBM: a row is read once into registers (16 bytes per
// lane and load), reduced there (the variance from the centred values), and
// written once.  A row takes 16, 32 or 64 lanes of a wave, or a workgroup of
// 256 lanes; longer rows than registers hold are re-read from cache.  Measured:
// forward 8192 x 4096 bf16 26.5 us (5.1 TB/s), 262144 rows of 128 27.7 us (4.8);
// backward 8192 x 4096 36.8 us (5.5 TB/s; 56 to 61 without the next row on its
// way) and 4.1 us for the sums of the partial weight gradients.
#include "gdn_chunk.h"
#include "../../include/gdn_linear.h"

namespace gdn {

// 16 bytes at an element-aligned address (rows of odd length, sliced bases)
typedef uint32_t u32x4e __attribute__((ext_vector_type(4), aligned(2)));

// the elements of 16 bytes, as floats
template <int DT>
__device__ __forceinline__ void unpack(u32x4e raw, float* f) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (DT == GDN_DTYPE_F32) {
      f[w] = __uint_as_float(raw[w]);
    } else {
      f[2 * w] = Elt<DT>::to_f(static_cast<uint16_t>(raw[w]));
      f[2 * w + 1] = Elt<DT>::to_f(static_cast<uint16_t>(raw[w] >> 16));
    }
  }
}
// N elements of type DT at p (element-aligned), as floats
template <int DT, int N>
__device__ __forceinline__ void ldn(const void* p, long long i, float (&f)[N]) {
  constexpr int VEC = Elt<DT>::VEC;
  static_assert(N % VEC == 0, "whole vectors");
#pragma unroll
  for (int u = 0; u < N / VEC; ++u)
    unpack<DT>(*reinterpret_cast<const u32x4e*>(static_cast<const typename Elt<DT>::T*>(p) + i + u * VEC),
               f + u * VEC);
}
template <int DT, int N>
__device__ __forceinline__ void stn(void* p, long long i, const float (&f)[N]) {
  constexpr int VEC = Elt<DT>::VEC;
#pragma unroll
  for (int u = 0; u < N / VEC; ++u) {
    u32x4e raw;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (DT == GDN_DTYPE_F32)
        raw[w] = __float_as_uint(f[u * VEC + w]);
      else
        raw[w] = Elt<DT>::from_f(f[u * VEC + 2 * w]) |
                 (static_cast<uint32_t>(Elt<DT>::from_f(f[u * VEC + 2 * w + 1])) << 16);
    }
    *reinterpret_cast<u32x4e*>(static_cast<typename Elt<DT>::T*>(p) + i + u * VEC) = raw;
  }
}

// N parameters from element i of a tensor of runtime type wt
template <int N>
__device__ __forceinline__ void ldw(const void* p, long long i, int wt, float (&f)[N]) {
  if (wt == GDN_DTYPE_F32) {
    ldn<GDN_DTYPE_F32, N>(p, i, f);
  } else if constexpr (N % 8 == 0) {
    if (wt == GDN_DTYPE_BF16) ldn<GDN_DTYPE_BF16, N>(p, i, f);
    else ldn<GDN_DTYPE_F16, N>(p, i, f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = ldp(p, i + j, wt);
  }
}

// Elements c .. c + VEC - 1 of a row of D at p + base (0 past its end).
template <int DT, int VEC>
__device__ __forceinline__ void ld_row(const void* p, long long base, int c, int D,
                                       float (&f)[VEC]) {
  if (c + VEC <= D) {
    ldn<DT, VEC>(p, base + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = c + j < D ? lde<DT>(p, base + c + j) : 0.f;
  }
}
// The same as raw bits.
template <int DT>
__device__ __forceinline__ u32x4e ld_raw(const void* p, long long base, int c, int D) {
  constexpr int VEC = Elt<DT>::VEC;
  const auto* src = static_cast<const typename Elt<DT>::T*>(p) + base + c;
  if (c + VEC <= D) return *reinterpret_cast<const u32x4e*>(src);
  u32x4e r = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if (c + j >= D) break;
    if constexpr (DT == GDN_DTYPE_F32) r[j] = __float_as_uint(src[j]);
    else r[j / 2] |= static_cast<uint32_t>(src[j]) << (16 * (j % 2));
  }
  return r;
}
template <int DT, int VEC>
__device__ __forceinline__ void st_row(void* p, long long base, int c, int D,
                                       const float (&f)[VEC]) {
  if (c + VEC <= D) {
    stn<DT, VEC>(p, base + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j < D) ste<DT>(p, base + c + j, f[j]);
  }
}
template <int VEC>
__device__ __forceinline__ void ld_par(const void* p, long long base, int c, int D, int wt,
                                       float (&f)[VEC]) {
  if (c + VEC <= D) {
    ldw<VEC>(p, base + c, wt, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = c + j < D ? ldp(p, base + c + j, wt) : 0.f;
  }
}

// Sum over the LPR lanes of a row: a wave's shuffles, and across the four
// waves of a 256-lane row through `red` (a buffer per call in flight).
template <int LPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
#pragma unroll
  for (int off = 1; off < (LPR < 64 ? LPR : 64); off *= 2) x += __shfl_xor(x, off);
  if constexpr (LPR > 64) {
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < LPR / 64; ++w) x += red[w];
  }
  return x;
}

struct NormArgs {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* stats;
  long long rows;
  int heads, D;
  float eps;
  int wt;
};

// One row per group of LPR lanes (256 / LPR groups), VPT 16-byte vectors per
// lane.
template <int DT, int LPR, int VPT>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[2][4];
  const int l = threadIdx.x % LPR;
  const long long r = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (LPR < 256 && r >= a.rows) return;
  const long long base = r * a.D;
  float f[VPT][VEC];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) ld_row<DT, VEC>(a.x, base, (l + LPR * i) * VEC, a.D, f[i]);
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += f[i][j];
  const float mean = row_sum<LPR>(s, red[0]) / a.D;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      f[i][j] -= mean;
      if ((l + LPR * i) * VEC + j < a.D) s += f[i][j] * f[i][j];
    }
  const float rstd = 1.f / sqrtf(row_sum<LPR>(s, red[1]) / a.D + a.eps);
  if (a.stats && l == 0) {
    a.stats[2 * r] = mean;
    a.stats[2 * r + 1] = rstd;
  }
  const long long pb = a.heads > 1 ? (r % a.heads) * a.D : 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (l + LPR * i) * VEC;
    if (c >= a.D) break;
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[i][j] *= rstd;
    float p[VEC];
    if (a.w) {
      ld_par<VEC>(a.w, pb, c, a.D, a.wt, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[i][j] *= p[j];
    }
    if (a.b) {
      ld_par<VEC>(a.b, pb, c, a.D, a.wt, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[i][j] += p[j];
    }
    st_row<DT, VEC>(a.y, base, c, a.D, f[i]);
  }
}

// Rows longer than a workgroup's registers: three passes, two of them from cache.
template <int DT>
__global__ __launch_bounds__(256) void norm_fwd_long_kernel(NormArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[2][4];
  const long long r = blockIdx.x, base = r * a.D;
  float f[VEC], s = 0.f;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    ld_row<DT, VEC>(a.x, base, c, a.D, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += f[j];
  }
  const float mean = row_sum<256>(s, red[0]) / a.D;
  s = 0.f;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    ld_row<DT, VEC>(a.x, base, c, a.D, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j < a.D) s += (f[j] - mean) * (f[j] - mean);
  }
  const float rstd = 1.f / sqrtf(row_sum<256>(s, red[1]) / a.D + a.eps);
  if (a.stats && threadIdx.x == 0) {
    a.stats[2 * r] = mean;
    a.stats[2 * r + 1] = rstd;
  }
  const long long pb = a.heads > 1 ? (r % a.heads) * a.D : 0;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    float w[VEC], b[VEC];
    ld_row<DT, VEC>(a.x, base, c, a.D, f);
    if (a.w) ld_par<VEC>(a.w, pb, c, a.D, a.wt, w);
    if (a.b) ld_par<VEC>(a.b, pb, c, a.D, a.wt, b);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      f[j] = (f[j] - mean) * rstd * (a.w ? w[j] : 1.f) + (a.b ? b[j] : 0.f);
    st_row<DT, VEC>(a.y, base, c, a.D, f);
  }
}

struct NormBwdArgs {
  const void* x;
  const void* w;
  const void* dy;
  const float* stats;
  void* dx;
  float* pw;   // [parts][heads * D] partial sums of dweight, of dbias (NULL: not wanted)
  float* pb;
  long long rows;
  int heads, D, wt;
  int groups;  // groups walking the rows (a multiple of heads)
};

// A group of LPR lanes walks the rows gid, gid + groups, ... -- all of one
// head, so its columns' weights and partial sums stay in registers -- with the
// next row loaded while the current one is reduced.  With one head the groups
// of a workgroup are summed in LDS first.
template <int DT, int LPR, int VPT>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  constexpr int GPW = 256 / LPR;
  __shared__ float red[2][2][4];
  extern __shared__ float part[];   // [GPW][D] where groups are summed
  const int l = threadIdx.x % LPR, gi = threadIdx.x / LPR;
  const int gid = blockIdx.x * GPW + gi;
  const bool live = gid < a.groups;
  const long long hb = a.heads > 1 ? (long long)(gid % a.heads) * a.D : 0;
  float w[VPT][VEC], dw[VPT][VEC], db[VPT][VEC];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (a.w) {
      ld_par<VEC>(a.w, hb, (l + LPR * i) * VEC, a.D, a.wt, w[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[i][j] = 1.f;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  // the next row's bits, on their way while this one is reduced
  u32x4e rx[VPT], ry[VPT];
  float nm = 0.f, nr = 0.f;
  auto load = [&](long long r) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      rx[i] = ld_raw<DT>(a.x, r * a.D, (l + LPR * i) * VEC, a.D);
      ry[i] = ld_raw<DT>(a.dy, r * a.D, (l + LPR * i) * VEC, a.D);
    }
    nm = a.stats[2 * r];
    nr = a.stats[2 * r + 1];
  };
  const float inv_d = 1.f / a.D;
  int ph = 0;
  if (live && gid < a.rows) load(gid);
  for (long long r = live ? gid : a.rows; r < a.rows; r += a.groups, ph ^= 1) {
    float x[VPT][VEC], dy[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      unpack<DT>(rx[i], x[i]);
      unpack<DT>(ry[i], dy[i]);
    }
    const float mean = nm, rstd = nr;
    if (r + a.groups < a.rows) load(r + a.groups);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        // (past the row's end 0, and so is dy: the mean of a near-constant row
        // times rstd may be infinite)
        x[i][j] = (l + LPR * i) * VEC + j < a.D ? (x[i][j] - mean) * rstd : 0.f;
        dw[i][j] += dy[i][j] * x[i][j];
        db[i][j] += dy[i][j];
        dy[i][j] *= w[i][j];
        s1 += dy[i][j];
        s2 += dy[i][j] * x[i][j];
      }
    s1 = row_sum<LPR>(s1, red[ph][0]) * inv_d;
    s2 = row_sum<LPR>(s2, red[ph][1]) * inv_d;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = rstd * (dy[i][j] - s1 - x[i][j] * s2);
      const int c = (l + LPR * i) * VEC;
      if (c < a.D) st_row<DT, VEC>(a.dx, r * a.D, c, a.D, x[i]);
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = which ? a.pb : a.pw;
    if (!out) continue;
    if (GPW > 1 && a.heads == 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int c = (l + LPR * i) * VEC + j;
          if (c < a.D) part[gi * a.D + c] = which ? db[i][j] : dw[i][j];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += 256) {
        float s = part[c];
        for (int g = 1; g < GPW; ++g) s += part[g * a.D + c];
        out[(long long)blockIdx.x * a.D + c] = s;
      }
    } else if (live) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = (l + LPR * i) * VEC;
        if (c < a.D) st_row<GDN_DTYPE_F32, VEC>(out, (long long)gid * a.D, c, a.D,
                                                which ? db[i] : dw[i]);
      }
    }
  }
}

// Rows longer than registers hold: dx alone; the sums by norm_cols_kernel.
template <int DT>
__global__ __launch_bounds__(256) void norm_bwd_long_kernel(NormBwdArgs a) {
  constexpr int VEC = Elt<DT>::VEC;
  __shared__ float red[2][4];
  const long long r = blockIdx.x, base = r * a.D;
  const long long hb = a.heads > 1 ? (r % a.heads) * a.D : 0;
  const float mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
  float x[VEC], dy[VEC], w[VEC], s1 = 0.f, s2 = 0.f;
  auto load = [&](int c) {
    ld_row<DT, VEC>(a.x, base, c, a.D, x);
    ld_row<DT, VEC>(a.dy, base, c, a.D, dy);
    if (a.w) ld_par<VEC>(a.w, hb, c, a.D, a.wt, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = c + j < a.D ? (x[j] - mean) * rstd : 0.f;   // (as above)
      if (a.w) dy[j] *= w[j];
    }
  };
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      s1 += dy[j];
      s2 += dy[j] * x[j];
    }
  }
  s1 = row_sum<256>(s1, red[0]) / a.D;
  s2 = row_sum<256>(s2, red[1]) / a.D;
  for (int c = threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
    load(c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = rstd * (dy[j] - s1 - x[j] * s2);
    st_row<DT, VEC>(a.dx, base, c, a.D, x);
  }
}

// Partial sums of dweight and dbias for the rows r of part p, r / heads in
// [p, p + 1) * span: a lane per column.
template <int DT>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormBwdArgs a, long long span) {
  const long long C = (long long)a.heads * a.D;
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const long long per = a.rows / a.heads + (c / a.D < a.rows % a.heads);
  const long long i0 = blockIdx.y * span, i1 = min(per, i0 + span);
  float dw = 0.f, db = 0.f;
  for (long long i = i0; i < i1; ++i) {
    const long long r = i * a.heads + c / a.D;
    const float dy = lde<DT>(a.dy, i * C + c);
    dw += dy * (lde<DT>(a.x, i * C + c) - a.stats[2 * r]) * a.stats[2 * r + 1];
    db += dy;
  }
  if (a.pw) a.pw[blockIdx.y * C + c] = dw;
  if (a.pb) a.pb[blockIdx.y * C + c] = db;
}

// out[c] = sum over p < P of part[p][c], in a fixed order: 64 columns per
// workgroup, 16 lanes per column.
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float* pw, const float* pb, void* dw,
                                                        void* db, int P, long long C, int wt) {
  __shared__ float red[16][64];
  const float* part = blockIdx.y ? pb : pw;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int l = threadIdx.x % 64, sl = threadIdx.x / 64;
  const long long c = (long long)blockIdx.x * 64 + l;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int p = sl; p < P; p += 16) s += part[p * C + c];
  }
  red[sl][l] = s;
  __syncthreads();
  if (sl == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][l];
    if (wt == GDN_DTYPE_F32) ste<GDN_DTYPE_F32>(out, c, s);
    else if (wt == GDN_DTYPE_BF16) ste<GDN_DTYPE_BF16>(out, c, s);
    else ste<GDN_DTYPE_F16>(out, c, s);
  }
}

}  // namespace gdn

namespace {

// Lanes and vectors per row: the fewest lanes that hold it, a workgroup from
// four vectors per lane of a wave on; lpr 0: longer than a workgroup holds.
struct RowForm {
  int lpr, vpt;
};
RowForm row_form(int D, int dtype) {
  const int vec = dtype == GDN_DTYPE_F32 ? 4 : 8;
  const int n = (D + vec - 1) / vec;
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return {64, 4};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  if (vec == 4 && n <= 2048) return {256, 8};
  return {0, 0};
}

// Groups that walk the rows of the backward, and the partial sums they leave:
// two workgroups per CU, a multiple of the heads, no more than rows.
struct BwdPlan {
  RowForm f;
  long long groups, parts, span;
};
BwdPlan bwd_plan(long long rows, int heads, int D, int dtype) {
  BwdPlan p{row_form(D, dtype), 0, 0, 0};
  const long long per = (rows + heads - 1) / heads;   // rows of a head at most
  if (!p.f.lpr) {
    p.parts = per < 64 ? (per ? per : 1) : 64;
    p.span = (per + p.parts - 1) / p.parts;
    return p;
  }
  const int gpw = 256 / p.f.lpr;
  const long long want = 2LL * gdn::device_cus() * gpw;
  long long m = (want + heads - 1) / heads;
  if (m > per) m = per;
  if (m < 1) m = 1;
  p.groups = m * heads;
  p.parts = heads == 1 ? (p.groups + gpw - 1) / gpw : m;
  return p;
}

int check_norm(const char* name, long long rows, int heads, int D, int dtype, int w_dtype) {
  if (rows < 0 || heads < 1 || D < 1)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": rows must be >= 0, heads and D >= 1");
  if (!gdn::dtype_ok(dtype) || !gdn::dtype_ok(w_dtype))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported dtype code");
  // (rows' workgroups and columns of a row are counted in int)
  if (rows >= (1LL << 31) || (long long)heads * D >= (1LL << 31) || D > (1 << 30))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  return GDN_OK;
}

// A launch has under 2^32 lanes in a dimension.
int check_lanes(const char* name, long long workgroups, int lanes) {
  if (workgroups * lanes < (1LL << 32)) return GDN_OK;
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large for one launch");
}

}  // namespace

#define GDN_NORM_FORMS(CALL, TT)                                                                 \
  CALL(TT, 16, 1) CALL(TT, 32, 1) CALL(TT, 64, 1) CALL(TT, 64, 2) CALL(TT, 64, 4) CALL(TT, 256, 2) \
      CALL(TT, 256, 4)

extern "C" int gdn_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y,
                                  float* stats, long long rows, int heads, int D, float eps,
                                  int dtype, int w_dtype, void* stream) {
  const char* name = "gdn_layer_norm_fwd";
  const int rc = check_norm(name, rows, heads, D, dtype, w_dtype);
  if (rc) return rc;
  if (rows == 0) return GDN_OK;
  if (!x || !y) return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": x and y must be non-NULL");
  const RowForm f = row_form(D, dtype);
  const int per = f.lpr ? 256 / f.lpr : 1;   // rows per workgroup
  if (const int fit = check_lanes(name, (rows + per - 1) / per, 256)) return fit;
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
  const gdn::NormArgs a{x, weight, bias, y, stats, rows, heads, D, eps, w_dtype};
#define GDN_NF(TT, LL, VV)                                                                      \
  if (dtype == TT && f.lpr == LL && f.vpt == VV) {                                              \
    constexpr int GPW = 256 / LL;                                                               \
    hipLaunchKernelGGL((gdn::norm_fwd_kernel<TT, LL, VV>), dim3((unsigned)((rows + GPW - 1) / GPW)), \
                       dim3(256), 0, st, a);                                                    \
    return gdn_host::check_launch(name);                                                        \
  }
  GDN_NORM_FORMS(GDN_NF, GDN_DTYPE_BF16)
  GDN_NORM_FORMS(GDN_NF, GDN_DTYPE_F16)
  GDN_NORM_FORMS(GDN_NF, GDN_DTYPE_F32)
  GDN_NF(GDN_DTYPE_F32, 256, 8)
#undef GDN_NF
  const dim3 grid((unsigned)rows);
  if (dtype == GDN_DTYPE_F32)
    hipLaunchKernelGGL(gdn::norm_fwd_long_kernel<GDN_DTYPE_F32>, grid, dim3(256), 0, st, a);
  else if (dtype == GDN_DTYPE_BF16)
    hipLaunchKernelGGL(gdn::norm_fwd_long_kernel<GDN_DTYPE_BF16>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(gdn::norm_fwd_long_kernel<GDN_DTYPE_F16>, grid, dim3(256), 0, st, a);
  return gdn_host::check_launch(name);
}

extern "C" size_t gdn_layer_norm_bwd_workspace_bytes(long long rows, int heads, int D, int dtype) {
  if (check_norm("gdn_layer_norm_bwd_workspace_bytes", rows, heads, D, dtype, GDN_DTYPE_F32) ||
      rows == 0)
    return 0;
  return (size_t)bwd_plan(rows, heads, D, dtype).parts * heads * D * 2 * sizeof(float);
}

extern "C" int gdn_layer_norm_bwd(const void* x, const void* weight, const void* dy,
                                  const float* stats, void* dx, void* dweight, void* dbias,
                                  long long rows, int heads, int D, int dtype, int w_dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "gdn_layer_norm_bwd";
  const int rc = check_norm(name, rows, heads, D, dtype, w_dtype);
  if (rc) return rc;
  if (rows > 0 && (!x || !dy || !stats || !dx))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": x, dy, stats and dx must be non-NULL");
  const long long C = (long long)heads * D;
  auto st = static_cast<hipStream_t>(stream);
  const bool sums = dweight || dbias;
  if (sums)
    if (const int fit = check_lanes(name, (C + 63) / 64, 1024)) return fit;
  BwdPlan p{};
  float* pw = nullptr;
  float* pb = nullptr;
  if (rows > 0) {
    p = bwd_plan(rows, heads, D, dtype);
    if (!p.f.lpr)
      if (const int fit = check_lanes(name, rows, 256)) return fit;
    if (sums) {
      const size_t need = (size_t)p.parts * C * 2 * sizeof(float);
      if (!workspace || workspace_bytes < need)
        return gdn_host::fail(GDN_ERR_WORKSPACE, std::string(name) + ": workspace needs " +
                                                     std::to_string(need) + " bytes, got " +
                                                     std::to_string(workspace_bytes));
      pw = dweight ? static_cast<float*>(workspace) : nullptr;
      pb = dbias ? static_cast<float*>(workspace) + p.parts * C : nullptr;
    }
  }
  if (rows == 0 && !sums) return GDN_OK;
  gdn_host::launch_begin();
  if (rows > 0) {
    const gdn::NormBwdArgs a{x,  weight, dy,    stats, dx, pw, pb,
                             rows, heads,  D, w_dtype, (int)p.groups};
    bool done = false;
#define GDN_NB(TT, LL, VV)                                                                     \
  if (dtype == TT && p.f.lpr == LL && p.f.vpt == VV) {                                         \
    constexpr int GPW = 256 / LL;                                                              \
    const size_t lds = GPW > 1 && heads == 1 && sums ? (size_t)GPW * D * sizeof(float) : 0;    \
    hipLaunchKernelGGL((gdn::norm_bwd_kernel<TT, LL, VV>),                                     \
                       dim3((unsigned)((p.groups + GPW - 1) / GPW)), dim3(256), lds, st, a);   \
    done = true;                                                                               \
  }
    GDN_NORM_FORMS(GDN_NB, GDN_DTYPE_BF16)
    GDN_NORM_FORMS(GDN_NB, GDN_DTYPE_F16)
    GDN_NORM_FORMS(GDN_NB, GDN_DTYPE_F32)
    GDN_NB(GDN_DTYPE_F32, 256, 8)
#undef GDN_NB
    if (!done) {
      const dim3 cols((unsigned)((C + 255) / 256), (unsigned)p.parts);
#define GDN_NL(TT)                                                                             \
  if (dtype == TT) {                                                                           \
    hipLaunchKernelGGL(gdn::norm_bwd_long_kernel<TT>, dim3((unsigned)rows), dim3(256), 0, st, a); \
    if (sums) hipLaunchKernelGGL(gdn::norm_cols_kernel<TT>, cols, dim3(256), 0, st, a, p.span); \
  }
      GDN_NL(GDN_DTYPE_F32) GDN_NL(GDN_DTYPE_BF16) GDN_NL(GDN_DTYPE_F16)
#undef GDN_NL
    }
  }
  // (no rows: the sums over nothing are zero)
  if (sums)
    hipLaunchKernelGGL(gdn::norm_sum_kernel, dim3((unsigned)((C + 63) / 64), 2), dim3(1024), 0, st,
                       pw, pb, dweight, dbias, (int)p.parts, C, w_dtype);
  return gdn_host::check_launch(name);
}
