// A paged key-value cache for gfx950: rows written into pages, as they are or
// quantised to 8 bits with a scale per row, and read back (declared in
// gdn_attn.h).  A row of D elements takes D / 8 lanes, 8 elements each; both
// directions read and write every byte once and are bound by HBM (a decode
// batch's few rows by one round trip).
//
// Codes are round(x M / max), ties to even, of the exact quotient: M x is exact
// in fp32 for 16-bit x (M = 448 = 7 * 64, 127), the quotient is brought to the
// nearest fp32 value by one fused correction, and no 16-bit x and max bring it
// within 2^-16 of a border between codes but exactly onto it.
#include <type_traits>

#include "gdn_bits8.h"
#include "gdn_norm_rows.h"

namespace gdn {

struct PagedArgs {
  const void* in[2];   // write: k, v;  read: the caches
  void* out[2];
  float* scale[2];
  long long token[2], head[2];   // strides of k, v
  const void* slots;
  long long num_slots;
  int T, H, page, slots64;
};

__device__ __forceinline__ long long slot_at(const PagedArgs& a, long long t) {
  return a.slots64 ? static_cast<const long long*>(a.slots)[t]
                   : (long long)static_cast<const int*>(a.slots)[t];
}
// Row (slot, head) of the cache, in rows.  (64-bit divisions, 100 instructions each,
// only where a cache has that many slots.)
__device__ __forceinline__ long long cache_row(const PagedArgs& a, long long slot, int h) {
  const bool few = a.num_slots < (1LL << 31);
  const long long p = few ? (uint32_t)slot / (uint32_t)a.page : slot / a.page;
  return (p * a.H + h) * a.page + (slot - p * a.page);
}

// Eight codes of a row, x in fp32 (16-bit values): exact quotients, rounded.
template <int CT>
__device__ __forceinline__ u32x2b codes8(const float (&x)[8], float most) {
  // a power of two brings the maximum to [1, 2) (from 2^127 on to [2, 4))
  const float unit = __uint_as_float(max(254 - (int)(__float_as_uint(most) >> 23), 1) << 23);
  const float m = most * unit, inv = 1.f / m, mul = largest8(CT) * unit;
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float n = x[j] * mul;
    const float r = n * inv;
    q[j] = fmaf(fmaf(-r, m, n), inv, r);
  }
  if constexpr (CT == GDN_DTYPE_E4M3)
    return u32x2b{e4m3_4(q[0], q[1], q[2], q[3]), e4m3_4(q[4], q[5], q[6], q[7])};
  else
    return u32x2b{int8_4(q[0], q[1], q[2], q[3]), int8_4(q[4], q[5], q[6], q[7])};
}

// Largest value over the LPR lanes of a row (8, 16 or 32), without LDS.
template <int LPR>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
  auto dpp = [](uint32_t v, auto c) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(c)::value, 0xf, 0xf, true);
  };
  x = max(x, dpp(x, std::integral_constant<int, 0xb1>{}));    // lanes of a pair changed
  x = max(x, dpp(x, std::integral_constant<int, 0x4e>{}));    // pairs
  x = max(x, dpp(x, std::integral_constant<int, 0x141>{}));   // eight lanes mirrored
  if constexpr (LPR >= 16) x = max(x, dpp(x, std::integral_constant<int, 0x140>{}));   // sixteen
  if constexpr (LPR == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
  }
  return x;
}

// A workgroup takes U 256 / LPR tokens of one head (blockIdx.y) of k or v
// (blockIdx.z): what it writes of codes and scales is in one piece.  U rows are on
// their way to a group of lanes: with 8-bit rows 2 where there are workgroups by the
// dozen to a CU (their launch, and what each lane works out ahead of its row, shows:
// 40000 tokens of 8 heads of 128 in e4m3 are written in 58 us, 4.2 TB/s read and
// written, and read in 50, 4.9 TB/s; one row 64 and 58, four 61 and 51), else 1 (256
// tokens of 2 heads of 256 3.0 and 2.8 us, two rows 3.6 and 3.3; 20011 of 8 heads of
// 128 in bf16 34 and 30 either way).
template <int DT, int CT, int D, int U>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedArgs a) {
  constexpr int LPR = D / 8, GR = 256 / LPR;
  const int l = threadIdx.x % LPR, h = blockIdx.y, k = blockIdx.z;
  const long long t0 = (long long)blockIdx.x * (GR * U) + threadIdx.x / LPR;
  u32x4e raw[U];
  long long dst[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const long long t = t0 + i * GR;
    dst[i] = -1;
    if (t >= a.T) break;   // (the lanes of a row together, here and below)
    const long long slot = slot_at(a, t);
    raw[i] = *reinterpret_cast<const u32x4e*>(static_cast<const uint16_t*>(a.in[k]) + t * a.token[k] +
                                              h * a.head[k] + 8 * l);
    if (slot >= 0 && slot < a.num_slots) dst[i] = cache_row(a, slot, h);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (t0 + i * GR >= a.T) return;
    if (dst[i] < 0) continue;
    if constexpr (CT == DT) {
      reinterpret_cast<u32x4e*>(a.out[k])[dst[i] * LPR + l] = raw[i];
    } else {
      float x[8];
      unpack<DT>(raw[i], x);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(x[j]));
      m = lanes_max<LPR>(m);
      if (l == 0) a.scale[k][dst[i]] = row8(m, CT).scale;
      reinterpret_cast<u32x2b*>(a.out[k])[dst[i] * LPR + l] =
          codes8<CT>(x, fmaxf(__uint_as_float(m), 0x1p-100f));
    }
  }
}

// Four codes as floats.
template <int CT>
__device__ __forceinline__ void values4(uint32_t w, float* f) {
  if constexpr (CT == GDN_DTYPE_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo[0];
    f[1] = lo[1];
    f[2] = hi[0];
    f[3] = hi[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (float)(int8_t)(w >> (8 * j));
  }
}

template <int DT, int CT, int D, int U>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedArgs a) {
  constexpr int LPR = D / 8, GR = 256 / LPR;
  constexpr bool C8 = CT == GDN_DTYPE_E4M3 || CT == GDN_DTYPE_I8;
  const int l = threadIdx.x % LPR, h = blockIdx.y, k = blockIdx.z;
  const long long t0 = (long long)blockIdx.x * (GR * U) + threadIdx.x / LPR;
  u32x4e raw[U];
  u32x2b code[U];
  float scale[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const long long t = t0 + i * GR;
    raw[i] = u32x4e{0, 0, 0, 0};
    code[i] = u32x2b{0, 0};
    scale[i] = 0.f;
    if (t >= a.T) break;
    const long long slot = slot_at(a, t);
    if (slot < 0 || slot >= a.num_slots) continue;
    const long long src = cache_row(a, slot, h);
    if constexpr (C8) {
      code[i] = reinterpret_cast<const u32x2b*>(a.in[k])[src * LPR + l];
      scale[i] = a.scale[k][src];
    } else {
      raw[i] = reinterpret_cast<const u32x4e*>(a.in[k])[src * LPR + l];
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const long long t = t0 + i * GR, at = t * a.H + h;
    if (t >= a.T) return;
    if constexpr (C8) {
      float f[8];
      values4<CT>(code[i][0], f);
      values4<CT>(code[i][1], f + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] *= scale[i];
        asm("" : "+v"(f[j]));   // (rounded to fp32 first, not in one step with the conversion to fp16)
      }
      stn<DT, 8>(a.out[k], at * D + 8 * l, f);
    } else {
      static_assert(DT == CT, "16-bit rows as they are");
      reinterpret_cast<u32x4e*>(a.out[k])[at * LPR + l] = raw[i];
    }
  }
}

}  // namespace gdn

namespace gdn_host {

// Checks that the operators of a paged cache share.
int check_cache(const char* name, const void* k_cache, const void* v_cache, const float* k_scale,
                const float* v_scale, int H, int D, int num_pages, int page_size, int cache_dtype) {
  const bool bits8 = cache_dtype == GDN_DTYPE_E4M3 || cache_dtype == GDN_DTYPE_I8;
  if (!bits8 && cache_dtype != GDN_DTYPE_BF16 && cache_dtype != GDN_DTYPE_F16)
    return fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported cache dtype code");
  if (H < 1 || num_pages < 0 || page_size < 1)
    return fail(GDN_ERR_SHAPE, std::string(name) + ": H and page_size must be >= 1, num_pages >= 0");
  if (D != 64 && D != 128 && D != 256)
    return fail(GDN_ERR_SHAPE, std::string(name) + ": D must be 64, 128 or 256");
  if (H >= (1 << 16) || page_size > (1 << 20) || (long long)num_pages * page_size >= (1LL << 40))
    return fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  if (num_pages > 0 && (!k_cache || !v_cache || (bits8 && (!k_scale || !v_scale))))
    return fail(GDN_ERR_NULL, std::string(name) + ": caches, and scales with 8 bits, must be non-NULL");
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) % 16)
    return fail(GDN_ERR_SHAPE, std::string(name) + ": caches must be 16-byte aligned");
  return GDN_OK;
}

}  // namespace gdn_host

namespace {

int launch_paged(const char* name, bool write, const gdn::PagedArgs& a, int D, int dtype, int cache_dtype,
                 hipStream_t st) {
  const int per = 256 / (D / 8);
  const bool two = cache_dtype != dtype && (long long)a.T * a.H * 2 / per >= 32LL * gdn::device_cus();
  const int tokens = two ? 2 * per : per;
  const dim3 grid((unsigned)((a.T + (long long)tokens - 1) / tokens), (unsigned)a.H, 2);
  if (const int fit = gdn_host::check_lanes(name, grid.x, 256)) return fit;
  gdn_host::launch_begin();
#define GDN_PAGED_U(TT, CC, DD, UU)                                                                        \
  if (write) hipLaunchKernelGGL((gdn::paged_write_kernel<TT, CC, DD, UU>), grid, dim3(256), 0, st, a);     \
  else hipLaunchKernelGGL((gdn::paged_read_kernel<TT, CC, DD, UU>), grid, dim3(256), 0, st, a);
#define GDN_PAGED(TT, CC, DD)                                                                              \
  if (dtype == TT && cache_dtype == CC && D == DD) {                                                       \
    if constexpr (TT != CC) {                                                                              \
      if (two) {                                                                                           \
        GDN_PAGED_U(TT, CC, DD, 2)                                                                         \
        return gdn_host::check_launch(name);                                                               \
      }                                                                                                    \
    }                                                                                                      \
    GDN_PAGED_U(TT, CC, DD, 1)                                                                             \
    return gdn_host::check_launch(name);                                                                   \
  }
#define GDN_PAGED_D(TT, CC) GDN_PAGED(TT, CC, 64) GDN_PAGED(TT, CC, 128) GDN_PAGED(TT, CC, 256)
  GDN_PAGED_D(GDN_DTYPE_BF16, GDN_DTYPE_BF16) GDN_PAGED_D(GDN_DTYPE_BF16, GDN_DTYPE_E4M3)
  GDN_PAGED_D(GDN_DTYPE_BF16, GDN_DTYPE_I8) GDN_PAGED_D(GDN_DTYPE_F16, GDN_DTYPE_F16)
  GDN_PAGED_D(GDN_DTYPE_F16, GDN_DTYPE_E4M3) GDN_PAGED_D(GDN_DTYPE_F16, GDN_DTYPE_I8)
#undef GDN_PAGED_D
#undef GDN_PAGED
#undef GDN_PAGED_U
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": dtype must be bf16 or f16, and the cache's unless it "
                                                           "has 8 bits");
}

}  // namespace

extern "C" int gdn_paged_write(const void* k, const void* v, long long k_token, long long k_head,
                               long long v_token, long long v_head, const void* slots,
                               int slots_int64, void* k_cache, void* v_cache, float* k_scale,
                               float* v_scale, int T, int H, int D, int num_pages, int page_size,
                               int dtype, int cache_dtype, void* stream) {
  const char* name = "gdn_paged_write";
  if (const int rc = gdn_host::check_cache(name, k_cache, v_cache, k_scale, v_scale, H, D, num_pages, page_size,
                                           cache_dtype))
    return rc;
  if (T < 0 || k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": sizes and strides must be non-negative");
  if (T == 0 || num_pages == 0) return GDN_OK;
  if (!k || !v || !slots)
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": k, v and slots must be non-NULL");
  // (all four are written or read by workgroups of their own)
  const bool bits8 = cache_dtype == GDN_DTYPE_E4M3 || cache_dtype == GDN_DTYPE_I8;
  const size_t rows = (size_t)num_pages * H * page_size, cb = rows * D * (bits8 ? 1 : 2);
  auto bytes = [&](long long token, long long head) { return ((size_t)(T - 1) * token + (H - 1) * head + D) * 2; };
  bool apart = !gdn_host::overlaps(k_cache, cb, v_cache, cb) &&
               !(bits8 && gdn_host::overlaps(k_scale, rows * 4, v_scale, rows * 4));
  for (const void* c : {k_cache, v_cache})
    apart = apart && !gdn_host::overlaps(c, cb, k, bytes(k_token, k_head)) &&
            !gdn_host::overlaps(c, cb, v, bytes(v_token, v_head));
  if (!apart)
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": the caches must not overlap each other, k or v");
  const gdn::PagedArgs a{{k, v}, {k_cache, v_cache}, {k_scale, v_scale}, {k_token, v_token}, {k_head, v_head}, slots,
                         (long long)num_pages * page_size, T, H, page_size, slots_int64};
  return launch_paged(name, true, a, D, dtype, cache_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int gdn_paged_read(const void* k_cache, const void* v_cache, const float* k_scale,
                              const float* v_scale, const void* slots, int slots_int64, void* k,
                              void* v, int T, int H, int D, int num_pages, int page_size,
                              int dtype, int cache_dtype, void* stream) {
  const char* name = "gdn_paged_read";
  if (const int rc = gdn_host::check_cache(name, k_cache, v_cache, k_scale, v_scale, H, D, num_pages, page_size,
                                           cache_dtype))
    return rc;
  if (T < 0) return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": T must be non-negative");
  if (T == 0) return GDN_OK;
  if (!k || !v || !slots)
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": k, v and slots must be non-NULL");
  const gdn::PagedArgs a{{k_cache, v_cache}, {k, v}, {const_cast<float*>(k_scale), const_cast<float*>(v_scale)},
                         {0, 0}, {0, 0}, slots, (long long)num_pages * page_size, T, H, page_size, slots_int64};
  return launch_paged(name, false, a, D, dtype, cache_dtype, static_cast<hipStream_t>(stream));
}
