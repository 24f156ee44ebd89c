// Rows of a norm in registers: element-aligned 16-byte loads and stores of a
// row's elements and parameters, sums over the lanes of a row, and the rule for
// how many lanes that is (gdn_norm.hip, gdn_rms.hip).
#pragma once

#include "gdn_chunk.h"

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
// The same of parameters of runtime type wt.  One branch for a whole vector, 32 or
// 16 bits, and the 16-bit types told apart behind their loads: with a branch per
// type around every element's load the compiler has formed fp16's addresses on
// another type's path alone.
template <int VEC>
__device__ __forceinline__ void ld_par(const void* p, long long base, int c, int D, int wt,
                                       float (&f)[VEC]) {
  if (wt == GDN_DTYPE_F32) {
    ld_row<GDN_DTYPE_F32, VEC>(p, base, c, D, f);
    return;
  }
  typedef uint16_t u16e __attribute__((ext_vector_type(VEC), aligned(2)));
  const uint16_t* src = static_cast<const uint16_t*>(p) + base + c;
  u16e raw;
  if (c + VEC <= D) {
    raw = *reinterpret_cast<const u16e*>(src);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      raw[j] = 0;
      if (c + j < D) raw[j] = src[j];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    f[j] = wt == GDN_DTYPE_BF16 ? bf2f(raw[j]) : Elt<GDN_DTYPE_F16>::to_f(raw[j]);
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

// Lanes and vectors per row: the fewest lanes that hold it, a workgroup from
// four vectors per lane of a wave on; lpr 0: longer than a workgroup holds.
struct RowForm {
  int lpr, vpt;
};
inline RowForm row_form(int D, int dtype) {
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

}  // namespace gdn

namespace gdn_host {

// A launch has under 2^32 lanes in a dimension.
inline int check_lanes(const char* name, long long workgroups, int lanes) {
  if (workgroups * lanes < (1LL << 32)) return GDN_OK;
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large for one launch");
}

}  // namespace gdn_host
