// Attention of a sequence's newest tokens over a paged key-value cache, for
// gfx950 (declared in gdn_attn.h): per kv-head and row (token, q-head of its
// group)
//     o = sum_t e^{s_t - m} v_t / sum_t e^{s_t - m},   s_t = scale q . k_t
// over the tokens t that the row sees, with the running maximum m, sum and o of
// one pass (in base 2).
//
// The path reads the cache once (2 D elements per token and kv-head against 4 D
// flops per row: up to 32 rows share a read) and is bound by HBM.  A wave takes
// 32 tokens at a time (64 where rows are short) straight from HBM into the registers
// of its MFMA operands, no LDS in between: S^T = K Q^T with tokens as rows leaves P^T in the layout in
// which it is the operand of O^T = V^T P^T, whose V^T a lane forms in its own
// registers from eight tokens' 16-byte pieces (one v_perm per word).  The next
// tokens' K is on its way while these' softmax and V are worked on, and the other
// way round.
//
// Work: every (sequence, kv-head) is as many units of 128 tokens (256 where a wave
// takes 64) as its length has; all units in a row are cut into equal shares, one per workgroup, whatever
// the lengths (read on the device: nothing here depends on a host copy of them).
// A share that holds a whole (sequence, kv-head) writes its output; parts leave
// m, the sum and o over it in the workspace and a second launch joins them.
//
// Measured, kernel and join: 256 sequences of 100 to 8192 tokens, 8 heads of 128 in
// e4m3 395 + 5 us, 5.7 TB/s; one of 131072, 2 heads of 256 in bf16 50 + 5, 5.4 TB/s;
// 48 of 1 to 6000, 4 heads of 128 in bf16, 4 newest tokens 67 + 5, 4.5 TB/s (the
// shares' starts and ends, and the last tokens' masks); one of 449 9.0 + 2.5: a chain
// of latencies, lengths, table, K, softmax, the waves' join.
//
// Many newest tokens are taken in groups of 64 rows, each of which reads all of the
// sequence for itself, tokens past its own rows included (they are masked): 512 of
// 8192, 8 q-heads to each of 4 kv-heads of 128 in bf16, 189 us, 2048 of them 626, where
// their products alone are 54 and 195 at a large product's rate.
#include <algorithm>

#include "gdn_bits8.h"
#include "gdn_norm_rows.h"

namespace gdn {

constexpr int kUnit = 128;   // least tokens of a unit of work

struct PagedAttnArgs {
  const void* q;
  long long sn, sl, sh;   // q's strides of sequence, token and head
  const void* kc;
  const void* vc;
  const float* ks;
  const float* vs;
  const int32_t* table;
  long long table_stride;
  const int32_t* lens;
  void* o;
  float* lse;
  float* part;
  int4* desc;
  int N, L, Hq, Hkv, G, R, RG, rows;   // R = L G rows per kv-head in RG groups of at most `rows`
  int part_size;  // floats of a part: o [rows][D], m, sums [rows], 16-byte aligned
  int num_pages, page, cap, window;
  int whole;      // every (sequence, kv-head) is one unit, however long (no second launch)
  int by_item;    // desc has an entry per (sequence, kv-head, group of rows), not per workgroup
  float scale2;   // scale log2(e)
};

// Tokens [lo, hi) that a sequence's rows see, and their units (one at least).
struct Span {
  int lo, hi, units;
};
template <int UNIT>
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, int n) {
  Span s;
  s.hi = min(max(a.lens[n], 0), a.cap);
  s.lo = a.window > 0 ? max(0, s.hi - a.L + 1 - a.window) & ~15 : 0;
  s.units = a.whole ? 1 : max(1, (s.hi - s.lo + UNIT - 1) / UNIT);
  return s;
}

// x and its value 16 (32) lanes further, in every lane of both: v_permlane swaps
// of two copies, no LDS.
typedef uint32_t u32x2s __attribute__((ext_vector_type(2)));
template <int OFF>
__device__ __forceinline__ void both(float x, float& a, float& b) {
  const uint32_t u = __float_as_uint(x);
  u32x2s r;
  if constexpr (OFF == 16) r = __builtin_bit_cast(u32x2s, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  else r = __builtin_bit_cast(u32x2s, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  const uint32_t lo = r[0], hi = r[1];
  a = __uint_as_float(lo);
  b = __uint_as_float(hi);
}
// Largest value, sum over the four groups of 16 lanes.
__device__ __forceinline__ float xmax16(float x) {
  float a, b;
  both<16>(x, a, b);
  both<32>(fmaxf(a, b), a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float xsum16(float x) {
  float a, b;
  both<16>(x, a, b);
  both<32>(a + b, a, b);
  return a + b;
}
// The value of lane R of each four.
template <int R>
__device__ __forceinline__ float of_four(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), R * 0x55, 0xf, 0xf, true));
}
__device__ __forceinline__ float of_four(float x, int r) {
  return r == 0 ? of_four<0>(x) : r == 1 ? of_four<1>(x) : r == 2 ? of_four<2>(x) : of_four<3>(x);
}
// 2^x in one instruction (results under 2^-126 are 0).
__device__ __forceinline__ float exp2i(float x) { return __builtin_amdgcn_exp2f(x); }

// What the MFMAs run in: bf16 over a bf16 cache; fp16 else (8-bit codes are
// exact there, and two conversions cheaper than in bf16).
template <bool BF>
__device__ __forceinline__ f32x4 mfma_t(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (BF) return mfma16(a, b, c);
  else return mfma16h(a, b, c);
}
template <bool BF>
__device__ __forceinline__ uint16_t from_f(float f) {
  if constexpr (BF) return f2bf(f);
  else return f2h(f);
}
// Eight values as an operand, and what it leaves of them as another.
template <bool BF, bool LO>
__device__ __forceinline__ void operands(f32x4 p, f32x4 q, u16x8& hi, u16x8& lo) {
  u16x4 h[2], l[2];
  if constexpr (BF) {
    split_bf4(p, h[0], l[0]);
    split_bf4(q, h[1], l[1]);
  } else {
    h[0] = f2h4(p);
    h[1] = f2h4(q);
    if constexpr (LO) {
      l[0] = f2h4(p - __builtin_convertvector(__builtin_bit_cast(f16x4, h[0]), f32x4));
      l[1] = f2h4(q - __builtin_convertvector(__builtin_bit_cast(f16x4, h[1]), f32x4));
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = h[i / 4][i % 4];
    if constexpr (LO) lo[i] = l[i / 4][i % 4];
  }
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4w __attribute__((ext_vector_type(4)));

// Two codes in the halves of a word as fp16.  Integers: the byte (biased by 128)
// as an fp16 denormal u 2^-24, times 2^15, less 128 2^-9: the value times 2^-9,
// exactly.
constexpr float kI8 = 512.f;
// What the largest product of a row and V's scale becomes in fp16, up to twice as much:
// 2^15 of 65504 at the top, 28 bits of normal values below it.
constexpr float kTop = 0x1p14f;
__device__ __forceinline__ uint32_t i8_pair(uint32_t u) {
  const f16x2 x = __builtin_bit_cast(f16x2, u);
  const f16x2 k = {(_Float16)32768.f, (_Float16)32768.f}, b = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, k, b));
}
template <bool HI>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
}

// A word's elements of cache type CT that are not finite: 1 at the lowest bit of each.
template <int CT>
__device__ __forceinline__ uint32_t broken(uint32_t w) {
  if constexpr (CT == GDN_DTYPE_E4M3) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u;   // (0x7f alone carries)
  } else {
    // (an exponent of ones carries into the sign's place)
    constexpr uint32_t exp = CT == GDN_DTYPE_BF16 ? 0x7f807f80u : 0x7c007c00u, one = CT == GDN_DTYPE_BF16 ? 0x00800080u : 0x04000400u;
    return ((w & exp) + one) >> 15 & 0x00010001u;
  }
}

// x, of which nothing computed before is kept.
__device__ __forceinline__ uint32_t again(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Eight codes as an operand.
template <int CT>
__device__ __forceinline__ u16x8 codes_operand(uint32_t w0, uint32_t w1) {
  u32x4w r;
  if constexpr (CT == GDN_DTYPE_E4M3) {
    r = u32x4w{e4m3_pair<false>(w0), e4m3_pair<true>(w0), e4m3_pair<false>(w1), e4m3_pair<true>(w1)};
  } else {
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    r = u32x4w{i8_pair(__builtin_amdgcn_perm(0, w0, 0x0c010c00u)), i8_pair(__builtin_amdgcn_perm(0, w0, 0x0c030c02u)),
               i8_pair(__builtin_amdgcn_perm(0, w1, 0x0c010c00u)), i8_pair(__builtin_amdgcn_perm(0, w1, 0x0c030c02u))};
  }
  return __builtin_bit_cast(u16x8, r);
}

// Sixteens of tokens that a wave takes at a time, by the bytes of a row and the row tiles
// (of 16) that it works on: 8 KiB of K and as much of V on their way at once where rows
// are 128 bytes of one tile, or 256 (4 KiB where they are 64 of one tile, or 128 of two; 2
// where 64 of two; 16 where 512).  An e4m3 cache of 8 heads of 128 elements, 256 ragged
// sequences to 8192 tokens: 398 us, 465 with two sixteens.
__host__ __device__ constexpr int sixteens(int row_bytes, int nt) { return row_bytes <= 128 && nt == 1 ? 4 : 2; }
// Tokens of a unit of work: a step of all the waves that take tokens apart.
__host__ __device__ constexpr int unit_of(int row_bytes, int nt, int rw) {
  const int t = 16 * sixteens(row_bytes, nt) * (4 / rw);
  return t > kUnit ? t : kUnit;
}

// Workgroups of a CU, all there are of a call: 256 elements take the registers of
// two (131072 tokens of bf16 in two rounds of half the length: 55 us, in one 50).
__host__ __device__ constexpr int resident(int D) { return D == 256 ? 1 : 2; }

// NT: tiles of 16 rows that a wave works on with the same K and V; RW: waves of a workgroup
// that take rows apart, the others take tokens apart.  (32 rows in two waves that both read
// K and V, or in one: 48 sequences of 125 to 6000 tokens of 128 elements 76 us either way; the
// one leaves the other registers' worth of loads on their way.)
template <int QT, int CT, int D, int NT, int RW>
__global__ __launch_bounds__(256, resident(D))
void paged_attn_kernel(PagedAttnArgs a) {
  constexpr bool BF = CT == GDN_DTYPE_BF16;                        // bf16 products
  constexpr bool C8 = CT == GDN_DTYPE_E4M3 || CT == GDN_DTYPE_I8;  // codes with scales
  constexpr int ES = C8 ? 1 : 2, ROW = D * ES;                     // bytes of an element, of a row
  constexpr bool EACH = RW == 0;                                   // every wave on its own
  constexpr int RWS = EACH ? 1 : RW, TW = EACH ? 1 : 4 / RW;       // waves that take tokens apart
  constexpr int UNIT = unit_of(ROW, NT, RWS);
  constexpr int KL = ROW / 64;                                     // 16-byte pieces of K per lane and 16 tokens
  constexpr int E = D / 16;                                        // elements of V per lane and token
  constexpr int VD = E * ES / 4;                                   // words of them
  constexpr int CH = E * ES > 16 ? 16 / ES : E;                    // elements of one piece
  constexpr int NS = sixteens(ROW, NT), TT = 16 * NS;              // tokens that a wave takes at a time
  constexpr float BACK = (CT == GDN_DTYPE_I8 ? kI8 : 1.f) / kTop;   // C8: of acc, beside its unit
  // P in two parts: 2^-8 (bf16), 2^-11 of one would show in o.  (bf16 queries over 8 bits
  // take one, an eighth of o's half step: 256 ragged sequences of e4m3 to 8192 tokens are
  // 1.671e-3 from 64 bits in the norm, with two 1.661e-3, and 395 us, with two 397; 300 of 8
  // heads of 64 in int8 to 4000 139 and 150.)
  constexpr bool LO = BF || QT == GDN_DTYPE_F16;
  __shared__ float buf[EACH ? 1 : 4][EACH ? 1 : 16 * NT][D + 4];
  __shared__ float sm[4][16 * NT], sl[4][16 * NT];
  __shared__ int wave_sum[4];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int c16 = lane % 16, g = lane / 16;
  const int ts = EACH ? 0 : wave / RWS, rw = EACH ? 0 : wave % RWS;
  const char* const kc = static_cast<const char*>(a.kc);
  const char* const vc = static_cast<const char*>(a.vc);

  // this workgroup's share of all units
  const int HG = a.Hkv * a.RG;
  int u0, u1, share = 1, n = 0, prefix = 0, extra = 0;
  if constexpr (EACH) {
    u0 = blockIdx.x * 4 + wave;
    u1 = a.N * HG;
  } else if (a.whole) {
    share = (a.N * HG + gridDim.x - 1) / gridDim.x;
    u0 = min((int)blockIdx.x * share, a.N * HG);
    u1 = min(u0 + share, a.N * HG);
    n = prefix = u0 / HG;
  } else {
    const int per = (a.N + 255) / 256, first = tid * per, last = min(first + per, a.N);
    int sum = 0;
    for (int i = first; i < last; ++i) sum += span_of<UNIT>(a, i).units;
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int x = __shfl_up(incl, off);
      if (lane >= off) incl += x;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int units = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) incl += wave_sum[w];
      units += wave_sum[w];
    }
    units = __builtin_amdgcn_readfirstlane(units);
    // a workgroup's queries, first loads and output take about a unit's time: where
    // shares are of several units each (sequence, kv-head) counts one more, ahead of
    // its own.  (256 ragged sequences to 8192 tokens of e4m3: 507 us, with it 398, with
    // two 400; 48 of 4 newest tokens to 6000 of bf16: 88, 77, 77.)
    extra = units * HG > (int)gridDim.x;
    const int total = (units + extra * a.N) * HG;
    share = (total + gridDim.x - 1) / gridDim.x;
    u0 = min((int)blockIdx.x * share, total);
    u1 = min(u0 + share, total);
    if (!a.by_item && tid == 0) a.desc[blockIdx.x] = int4{0, 0, 0, 0};
    if (u0 >= u1) return;
    int at = incl - sum + extra * min(first, a.N);
    if (at * HG <= u0 && u0 < (incl + extra * last) * HG) {
      int i = first;
      for (;; ++i) {
        const int un = span_of<UNIT>(a, i).units + extra;
        if (u0 < (at + un) * HG) break;
        at += un;
      }
      found[0] = i;
      found[1] = at;
    }
    __syncthreads();
    n = __builtin_amdgcn_readfirstlane(found[0]);
    prefix = __builtin_amdgcn_readfirstlane(found[1]);
  }

  for (int u = u0; u < u1;) {
    if constexpr (EACH) n = u / HG;
    const Span sp = span_of<UNIT>(a, n);
    const int cost = sp.units + extra;
    const int rel = u - prefix * HG, item = EACH ? u % HG : rel / cost, start = EACH ? 0 : rel % cost;
    const int len = EACH ? cost : min(cost - start, u1 - u);
    const int kvh = item / a.RG, rg = item % a.RG;
    const int t0 = sp.lo + max(start - extra, 0) * UNIT;
    const int t1 = a.whole ? sp.hi : min(sp.lo + (start + len - extra) * UNIT, sp.hi);

    // the rows' queries: column c16 of tile n's operand is row row_of(n)
    auto row_of = [&](int i) { return 16 * ((rg * RWS + rw) * NT + i) + c16; };
    int pos[NT];   // its own place in the sequence
    u16x8 qf[NT][D / 32];
    float qscale[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int rr = row_of(i), l = rr / a.G;
      pos[i] = sp.hi - a.L + l;
      qscale[i] = a.scale2;
      float f[D / 32][8];
      uint32_t m = 0;
      const long long base = n * a.sn + l * a.sl + (kvh * a.G + rr % a.G) * a.sh;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int d = C8 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 32 * k + 8 * g;
        if (rr < a.R) {
          if constexpr (C8) ldn<QT, 8>(a.q, base + d, f[k]);
          else qf[i][k] = *reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(a.q) + base + d);
        } else {
          qf[i][k] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j) f[k][j] = 0.f;
        }
        if constexpr (C8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) m = max(m, abs_bits(f[k][j]));
        }
      }
      if constexpr (C8) {
        // in fp16, with a power of two that brings the row's largest value to
        // [2^14, 2^15): a bf16 value down to 2^-31 of it stays exact
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        const int e = min(max((int)(m >> 23), 64), 254) - 127;
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) qf[i][k][j] = f2h(ldexpf(f[k][j], 14 - e));
        qscale[i] = ldexpf(a.scale2 * (CT == GDN_DTYPE_I8 ? kI8 : 1.f), e - 14);
      }
    }

    // rows (in the cache) of the next 64 sixteens of this wave's tokens, one per lane
    constexpr int step = TT * TW;
    const int begin = t0 + TT * ts;
    const int tiles = t1 > begin ? (t1 - begin + step - 1) / step : 0;
    long long row64 = 0;
    auto look_up = [&](int it) {
      int t = begin + (it + lane / NS) * step + 16 * (lane % NS);
      t = min(t, (t1 - 1) & ~15);
      const int pg = a.table[n * a.table_stride + t / a.page];
      const bool ok = pg >= 0 && pg < a.num_pages;
      row64 = ok ? ((long long)pg * a.Hkv + kvh) * a.page + t % a.page : -1;
    };
    auto row_at = [&](int it, int s) {
      const int i = NS * (it % (64 / NS)) + s;
      const uint32_t lo = __builtin_amdgcn_readlane((int)row64, i);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(row64 >> 32), i);
      return (long long)((uint64_t)hi << 32 | lo);
    };

    u32x4w kr[NS][KL];
    uint32_t vr[4 * NS][VD];
    float kscale[NS], vscale[NS];   // of token 4 g + c16 % 4 of a sixteen
    long long rows[NS];   // of the tile whose K is loaded
    auto valid = [&](int it, int s) {   // tokens of a sixteen that there are
      return min(max(t1 - (begin + it * step + 16 * s), 1), 16);
    };
    auto load_k = [&](int it) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        rows[s] = row_at(it, s);
        const long long row = max(rows[s], 0ll);
        const char* p = kc + row * ROW;
        const int off = min(c16, valid(it, s) - 1) * ROW + 16 * g;
#pragma unroll
        for (int k = 0; k < KL; ++k) kr[s][k] = *reinterpret_cast<const u32x4w*>(p + (off + 64 * k));
        if constexpr (C8) kscale[s] = *(a.ks + row + (4u * g + c16 % 4));
      }
    };
    auto load_v = [&](const long long (&rv)[NS], int it) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const long long row = max(rv[s], 0ll);
        const char* p = vc + row * ROW;
        const int most = valid(it, s) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int off = min(4 * g + i, most) * ROW + c16 * CH * ES;
          uint32_t* dst = vr[4 * s + i];
          if constexpr (VD == 1) {
            dst[0] = *reinterpret_cast<const uint32_t*>(p + off);
          } else if constexpr (VD == 2) {
            const u32x2p x = *reinterpret_cast<const u32x2p*>(p + off);
            dst[0] = x[0];
            dst[1] = x[1];
          } else {
#pragma unroll
            for (int j = 0; j < VD / 4; ++j) {
              const u32x4w x = *reinterpret_cast<const u32x4w*>(p + (off + 256 * j));
#pragma unroll
              for (int w = 0; w < 4; ++w) dst[4 * j + w] = x[w];
            }
          }
        }
        if constexpr (C8) vscale[s] = *(a.vs + row + (4u * g + c16 % 4));
      }
    };

    f32x4 acc[NT][E];
    float m[NT], sum[NT], unit[NT];   // C8: acc holds products with V in units of 2^m unit
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      m[i] = -INFINITY;
      sum[i] = unit[i] = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) acc[i][j] = zero4();
    }
    long long rv[NS];
    if (tiles > 0) {
      look_up(0);
      load_k(0);
#pragma unroll
      for (int s = 0; s < NS; ++s) rv[s] = rows[s];
      load_v(rv, 0);
    }
    for (int it = 0; it < tiles; ++it) {
      const int tb = begin + it * step;
      f32x4 S[NT][NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int i = 0; i < NT; ++i) S[i][s] = zero4();
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          u16x8 kf;
          if constexpr (C8) kf = codes_operand<CT>(kr[s][k / 2][2 * (k % 2)], kr[s][k / 2][2 * (k % 2) + 1]);
          else kf = __builtin_bit_cast(u16x8, kr[s][k]);
#pragma unroll
          for (int i = 0; i < NT; ++i) S[i][s] = mfma_t<BF>(kf, qf[i][k], S[i][s]);
          if (C8 && k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) S[i][s][r] *= C8 ? qscale[i] * of_four(kscale[s], r) : qscale[i];
      }
      bool bad = false, here[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        here[s] = rows[s] < 0;
        bad |= here[s];
      }
      // tokens that some row of this wave does not see
      const bool mixed = (a.L > 1 && tb + TT - 1 > sp.hi - a.L) || (a.window > 0 && tb <= sp.hi - 1 - a.window);
      const bool part = mixed || bad || tb + TT > t1;
      if (part) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = tb + 16 * s + 4 * g + r;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              if (here[s]) S[i][s][r] = __builtin_nanf("");
              if (t >= t1 || t > pos[i] || (a.window > 0 && t <= pos[i] - a.window)) S[i][s][r] = -INFINITY;
            }
          }
      }
      if constexpr (CT != GDN_DTYPE_I8) {
        // Where not all rows see all tokens a value of V that is not finite must reach
        // only those that do (its product with a weight of 0 is NaN): it is taken out, and
        // its column of theirs is NaN from here on.
        bool any = false;
        if (mixed) {
#pragma unroll
          for (int t = 0; t < 4 * NS; ++t)
#pragma unroll
            for (int w = 0; w < VD; ++w) any |= broken<CT>(vr[t][w]) != 0;
        }
        if (mixed && __any(any)) {
#pragma unroll
          for (int h = 0; h < NS / 2; ++h) {
            u16x8 ones[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int j = 0; j < 8; ++j)
                ones[i][j] = S[i][2 * h + j / 4][j % 4] == -INFINITY ? (uint16_t)0 : from_f<BF>(1.f);
#pragma unroll
            for (int j = 0; j < E; ++j) {
              constexpr int PER = 4 / ES;   // elements of a word
              u16x8 ind;
#pragma unroll
              for (int t = 0; t < 8; ++t) {
                const uint32_t x = broken<CT>(again(vr[8 * h + t][j / PER])) >> (8 * ES * (j % PER));
                ind[t] = x & 1 ? from_f<BF>(1.f) : (uint16_t)0;
              }
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                const f32x4 hit = mfma_t<BF>(ind, ones[i], zero4());
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (hit[r] > 0.f) acc[i][j][r] = __builtin_nanf("");
              }
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 8 * h; t < 8 * h + 8; ++t)
#pragma unroll
              for (int w = 0; w < VD; ++w) vr[t][w] &= ~(broken<CT>(again(vr[t][w])) * (ES == 1 ? 0xffu : 0xffffu));
          }
        }
      }
      if (it + 1 < tiles) {
        if ((it + 1) % (64 / NS) == 0) look_up(it + 1);
        load_k(it + 1);
      }
      u16x8 hi[NT][NS / 2], lo[NT][NS / 2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float mx = S[i][0][0];
#pragma unroll
        for (int j = 1; j < 4 * NS; ++j) mx = fmaxf(mx, S[i][j / 4][j % 4]);
        mx = xmax16(mx);
        // (P in fp16 as it is: up to 2^15, 29 bits of normal values; a score of 2^20 or more,
        // of which 15 is not exact, up to 1)
        if constexpr (CT == GDN_DTYPE_F16) mx -= fabsf(mx) < 0x1p20f ? 15.f : 0.f;
        mx = fmaxf(m[i], mx);
        const float ref = mx == -INFINITY ? 0.f : mx;
        if (__any(mx > m[i])) {
          const float f = exp2i(m[i] - ref);   // (m = -inf: 0)
          sum[i] *= f;
          if constexpr (C8) {
            unit[i] *= f;
          } else {
#pragma unroll
            for (int j = 0; j < E; ++j) acc[i][j] *= f;
          }
          m[i] = mx;
        }
        f32x4 p[NS];
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 4 * NS; ++j) {
          float x = exp2i(S[i][j / 4][j % 4] - ref);
          sum[i] += x;
          if constexpr (C8) {
            // (a token that is not seen may have any scale)
            const float y = x * of_four(vscale[j / 4], j % 4);
            x = x == 0.f ? 0.f : y;
            big = fmaxf(big, x);
          }
          p[j / 4][j % 4] = x;
        }
        if constexpr (C8) {
          // P times V's scale, over a unit of the row's own: within a factor of two of the
          // largest that it has formed, in units of 2^m, so that what other rows see, or what
          // has no weight, cannot push this row's products out of fp16's range.  2^-110 at
          // least (no row has a smaller scale): the quotient stays in fp32's.
          big = xmax16(big);
          big = big > 0.f ? fmaxf(big, 0x1p-110f) : 0.f;
          const float was = unit[i];
          const bool more = big > 2.f * was;
          const bool any = __any(more);
          if (any) unit[i] = more ? big : was;
          const float inv = __builtin_amdgcn_rcpf(fmaxf(unit[i], 0x1p-111f) * (1.f / kTop));
          if (any) {
            const float f = more ? was * (1.f / kTop) * inv : 1.f;
#pragma unroll
            for (int j = 0; j < E; ++j) acc[i][j] *= f;
          }
#pragma unroll
          for (int s = 0; s < NS; ++s) p[s] *= inv;
        }
#pragma unroll
        for (int h = 0; h < NS / 2; ++h) operands<BF, LO>(p[2 * h], p[2 * h + 1], hi[i][h], lo[i][h]);
      }
      // O^T += V^T P^T
#pragma unroll
      for (int j = 0; j < E; ++j) {
#pragma unroll
        for (int h = 0; h < NS / 2; ++h) {
          u32x4w vf;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t* x = vr[8 * h + 2 * t];
            const uint32_t* y = vr[8 * h + 2 * t + 1];
            if constexpr (CT == GDN_DTYPE_E4M3) {
              const uint32_t w = __builtin_amdgcn_perm(y[j / 4], x[j / 4], j % 4 < 2 ? 0x05010400u : 0x07030602u);
              vf[t] = j % 2 ? e4m3_pair<true>(w) : e4m3_pair<false>(w);
            } else if constexpr (CT == GDN_DTYPE_I8) {
              constexpr uint32_t sel[4] = {0x0c040c00u, 0x0c050c01u, 0x0c060c02u, 0x0c070c03u};
              vf[t] = i8_pair(__builtin_amdgcn_perm(y[j / 4] ^ 0x80808080u, x[j / 4] ^ 0x80808080u, sel[j % 4]));
            } else {
              vf[t] = __builtin_amdgcn_perm(y[j / 2], x[j / 2], j % 2 ? 0x07060302u : 0x05040100u);
            }
          }
          const u16x8 v = __builtin_bit_cast(u16x8, vf);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            acc[i][j] = mfma_t<BF>(v, hi[i][h], acc[i][j]);
            if constexpr (LO) acc[i][j] = mfma_t<BF>(v, lo[i][h], acc[i][j]);
          }
        }
        // (conversions beside their products, not all ahead of them: registers)
        if (j % 2) __builtin_amdgcn_sched_barrier(0);
      }
      if (it + 1 < tiles) {
#pragma unroll
        for (int s = 0; s < NS; ++s) rv[s] = rows[s];
        load_v(rv, it + 1);
      }
    }
    // D's element of lane (c16, g), r of acc[i][j] is (j / CH) 16 CH + (4 g + r) CH +
    // j % CH of row c16 of tile i
    if constexpr (EACH) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float s = xsum16(sum[i]);
        const float f = s == 0.f ? 0.f : 1.f / s * (C8 ? unit[i] * BACK : 1.f);
        const int orow = row_of(i);
        if (orow >= a.R) continue;
        const long long at = ((long long)n * a.L + orow / a.G) * a.Hq + kvh * a.G + orow % a.G;
#pragma unroll
        for (int j = 0; j < E; j += 4)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            u16x4 h;
#pragma unroll
            for (int x = 0; x < 4; ++x) h[x] = Elt<QT>::from_f(acc[i][j + x][r] * f);
            *reinterpret_cast<u16x4*>(static_cast<uint16_t*>(a.o) + at * D + (j / CH) * 16 * CH + (4 * g + r) * CH +
                                      j % CH) = h;
          }
        if (a.lse && g == 0) a.lse[at] = s == 0.f ? -INFINITY : (m[i] + log2f(s)) * 0.69314718055994530942f;
      }
      u += 4 * gridDim.x;
      continue;
    }
    // the waves' parts joined
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      sum[i] = xsum16(sum[i]);
      if (g == 0) {
        sm[wave][16 * i + c16] = m[i];
        sl[wave][16 * i + c16] = sum[i];
      }
      // (each divided by its own sum: values near fp32's largest do not leave its range when
      // they are added up)
      const float f = sum[i] == 0.f ? 0.f : 1.f / sum[i] * (C8 ? unit[i] * BACK : 1.f);
      if (row_of(i) < a.R) {
#pragma unroll
        for (int j = 0; j < E; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            buf[wave][16 * i + c16][(j / CH) * 16 * CH + (4 * g + r) * CH + j % CH] = acc[i][j][r] * f;
      }
    }
    __syncthreads();
    const bool whole = len == cost;
    const int slot = u == u0 ? 2 * blockIdx.x : 2 * blockIdx.x + 1;
    float* const part = a.part + (size_t)slot * a.part_size;
    const int group = 16 * RWS * NT, here = min(a.R - group * rg, group);   // rows of this group
    for (int i = tid; i < here * (D / 4); i += 256) {
      const int row = i / (D / 4), d = 4 * (i % (D / 4)), w0 = row / (16 * NT), c = row % (16 * NT);
      float M = sm[w0][c];
#pragma unroll
      for (int w = 1; w < TW; ++w) M = fmaxf(M, sm[w0 + w * RWS][c]);
      const float ref = M == -INFINITY ? 0.f : M;
      float s = 0.f, f[TW];
      f32x4 o = zero4();
#pragma unroll
      for (int w = 0; w < TW; ++w) {
        f[w] = exp2i(sm[w0 + w * RWS][c] - ref) * sl[w0 + w * RWS][c];
        s += f[w];
      }
      const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
      for (int w = 0; w < TW; ++w)
        o += f[w] * inv * *reinterpret_cast<const f32x4*>(&buf[w0 + w * RWS][c][d]);
      const int orow = group * rg + row;
      const long long at = ((long long)n * a.L + orow / a.G) * a.Hq + kvh * a.G + orow % a.G;
      if (whole) {
        u16x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = Elt<QT>::from_f(o[j]);
        *reinterpret_cast<u16x4*>(static_cast<uint16_t*>(a.o) + at * D + d) = h;
        if (a.lse && d == 0) a.lse[at] = s == 0.f ? -INFINITY : (M + log2f(s)) * 0.69314718055994530942f;
      } else {
        *reinterpret_cast<f32x4*>(part + row * D + d) = o;
        if (d == 0) {
          part[a.rows * D + row] = M;
          part[a.rows * (D + 1) + row] = s;
        }
      }
    }
    // what the joining launch has to do: {sequence, item, first part's slot, parts}
    if (!a.whole && start == 0 && tid == 0 && (!whole || a.by_item))
      a.desc[a.by_item ? n * HG + item : blockIdx.x] =
          int4{n, item, slot, whole ? 0 : 1 + (cost - len + share - 1) / share};
    u += len;
    if (item == HG - 1 && start + len == cost) {
      prefix += cost;
      ++n;
    }
    __syncthreads();
  }
}

// Parts of one (sequence, kv-head) joined: block (entry of desc, row, columns).  LP
// lanes hold 4 LP columns of a row of a part, NT / LP parts are added at a time.
constexpr int kMostParts = 1024;   // workgroups at most
constexpr int kFewParts = 6;
template <int QT, int D, int NT, int LP>
__global__ __launch_bounds__(NT) void paged_attn_join_kernel(PagedAttnArgs a) {
  constexpr int GR = NT / LP, NW = NT / 64;
  static_assert(LP <= 64, "a row's lanes are of one wave");
  __shared__ float w[kMostParts];
  __shared__ float red[2][NW];
  __shared__ f32x4 acc[NW][LP];
  const int4 ds = a.desc[blockIdx.x];
  const int parts = ds.w;
  if (parts == 0) return;
  const int kvh = ds.y / a.RG, rg = ds.y % a.RG, row = blockIdx.y;
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, grp = tid / LP;
  const int col = blockIdx.z * LP + tid % LP;
  // part p: its workgroup's first, but for the one that begins here
  const int wg = ds.z / 2;
  auto at = [&](int p) { return a.part + (size_t)(p == 0 ? ds.z : 2 * (wg + p)) * a.part_size; };
  auto put = [&](int orow, float M, float s, f32x4 o) {
    const long long out = ((long long)ds.x * a.L + orow / a.G) * a.Hq + kvh * a.G + orow % a.G;
    u16x4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = Elt<QT>::from_f(o[j]);
    *reinterpret_cast<u16x4*>(static_cast<uint16_t*>(a.o) + out * D + 4 * col) = h;
    if (a.lse && col == 0) a.lse[out] = s == 0.f ? -INFINITY : (M + log2f(s)) * 0.69314718055994530942f;
  };
  if (parts <= kFewParts) {
    // few parts: a row to each group of lanes, the groups' rows with the first one's block
    const int r = row + grp, orow = rg * a.rows + r;
    if (row % GR || r >= a.rows || orow >= a.R) return;
    float m[kFewParts], l[kFewParts], M = -INFINITY;
    f32x4 x[kFewParts];
#pragma unroll
    for (int p = 0; p < kFewParts; ++p) {
      if (p >= parts) break;
      m[p] = at(p)[a.rows * D + r];
      l[p] = at(p)[a.rows * (D + 1) + r];
      x[p] = *reinterpret_cast<const f32x4*>(at(p) + r * D + 4 * col);
    }
#pragma unroll
    for (int p = 0; p < kFewParts; ++p)
      if (p < parts) M = fmaxf(M, m[p]);
    const float ref = M == -INFINITY ? 0.f : M;
    float s = 0.f;
    f32x4 o = zero4();
#pragma unroll
    for (int p = 0; p < kFewParts; ++p) {
      if (p >= parts) break;
      l[p] *= exp2i(m[p] - ref);
      s += l[p];
    }
    const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
    for (int p = 0; p < kFewParts; ++p) {
      if (p >= parts) break;
      o += l[p] * inv * x[p];
    }
    put(orow, M, s, o);
    return;
  }
  const int orow = rg * a.rows + row;
  if (orow >= a.R) return;
  float M = -INFINITY;
  for (int p = tid; p < parts; p += NT) {
    const float m = at(p)[a.rows * D + row];
    w[p] = m;
    M = fmaxf(M, m);
  }
#pragma unroll
  for (int off = 1; off < 64; off *= 2) M = fmaxf(M, __shfl_xor(M, off));
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) M = fmaxf(M, red[0][i]);
  const float ref = M == -INFINITY ? 0.f : M;
  float s = 0.f;
  for (int p = tid; p < parts; p += NT) {
    const float f = exp2i(w[p] - ref) * at(p)[a.rows * (D + 1) + row];
    w[p] = f;
    s += f;
  }
#pragma unroll
  for (int off = 1; off < 64; off *= 2) s += __shfl_xor(s, off);
  if (lane == 0) red[1][wave] = s;
  __syncthreads();
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += red[1][i];
  const float inv = s == 0.f ? 0.f : 1.f / s;
  f32x4 o = zero4();
#pragma unroll 8
  for (int p = grp; p < parts; p += GR) o += w[p] * inv * *reinterpret_cast<const f32x4*>(at(p) + row * D + 4 * col);
#pragma unroll
  for (int off = LP; off < 64; off *= 2)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], off);
  if (lane < LP) acc[wave][lane] = o;
  __syncthreads();
  if (tid >= LP) return;
#pragma unroll
  for (int i = 1; i < NW; ++i) o += acc[i][tid];
  put(orow, M, s, o);
}

}  // namespace gdn

namespace gdn_host {
int check_cache(const char* name, const void* k_cache, const void* v_cache, const float* k_scale,
                const float* v_scale, int H, int D, int num_pages, int page_size, int cache_dtype);
}

namespace {

// Workgroups, and how the rows of a kv-head are laid over their waves.
struct AttnPlan {
  int nt, rw, rg, rows, part_size;
  long long wgs, grid, items;   // workgroups where work is cut, launched
  bool each;    // every wave on its own
  bool whole;   // every (sequence, kv-head) one unit: nothing is cut
  size_t desc, bytes;
};
int attn_plan(const char* name, int N, int L, int Hq, int Hkv, int D, int max_length, int row_bytes, AttnPlan& p) {
  if (N < 0 || L < 1 || Hq < 1 || Hkv < 1 || max_length < 0)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": sizes must be non-negative (L, Hq, Hkv > 0)");
  if (Hq % Hkv)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": Hq must be a multiple of Hkv");
  if (D != 64 && D != 128 && D != 256)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": D must be 64, 128 or 256");
  const long long R = (long long)L * (Hq / Hkv);
  if (R > (1 << 20) || max_length > (1 << 30) || Hq > (1 << 20))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  p.nt = R <= 16 ? 1 : 2;
  p.rw = R <= 32 ? 1 : 2;
  const int group = 16 * p.nt * p.rw;
  p.rg = (int)((R + group - 1) / group);
  p.rows = (int)(R < group ? R : group);
  const int unit = row_bytes ? gdn::unit_of(row_bytes, p.nt, p.rw) : gdn::kUnit;   // (0: the smallest)
  const long long units = ((long long)max_length + unit - 1) / unit;
  const long long most = (units ? units : 1) * N * Hkv * p.rg;
  if (most + (long long)N * Hkv * p.rg >= (1LL << 30))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  p.items = (long long)N * Hkv * p.rg;
  p.wgs = (long long)gdn::resident(D) * gdn::device_cus();
  if (p.wgs > gdn::kMostParts) p.wgs = gdn::kMostParts;
  // Short sequences in numbers: a wave to each (sequence, kv-head), nothing joined, up
  // to 64 KiB of K and V each for every `wgs` of them.  8 heads of 128, ragged, in us
  // (each a wave / each a workgroup / shares): 256 sequences of e4m3 to 250 tokens 20 /
  // 34 / 32, to 1000 68 / 71 / 75, to 2000 126 / 112 / 120; of bf16 to 250 27 / 33 / 35,
  // to 700 80 / 76 / 82; 85 of e4m3 to 250 14.9 / 16.6 / 16.8, to 1000 38 / 26 / 30.
  p.each = row_bytes && p.nt == 1 && (long long)max_length * row_bytes * p.wgs <= 32768 * p.items;
  // Else few units each are not cut: a join costs what two units do, and shares gain
  // the less the more workgroups there are without.  bf16 as above, in us: one sequence
  // of 250 tokens 6.8 (cut 8.6); 16 to 250, 700 6.9, 12.7 (9.1, 12.5); 60 to 449 13.9
  // (19.6; in e4m3 13.0, 20.0); 85 to 700, 3000 24, 111 (27, 111); 256 of 4 heads, 4 newest tokens, to 1000
  // 63 (76).  24 units at most: one long sequence among short ones is one workgroup's.
  p.whole = p.each || (row_bytes && units <= 24 && (units - 2) * p.wgs <= 6 * p.items);
  if (p.wgs > most) p.wgs = most;
  p.grid = p.each ? std::min(p.wgs, (p.items + 3) / 4) : p.whole ? std::min(p.items, 1LL << 20) : p.wgs;
  p.part_size = (p.rows * (D + 2) + 3) / 4 * 4;
  p.desc = (size_t)p.wgs * 16;
  p.bytes = p.desc + (size_t)p.wgs * 2 * p.part_size * sizeof(float);
  p.bytes = (p.bytes + 255) / 256 * 256;
  return GDN_OK;
}

}  // namespace

extern "C" size_t gdn_paged_attn_workspace_bytes(int N, int L, int Hq, int Hkv, int D, int max_length) {
  AttnPlan p{};
  if (attn_plan("gdn_paged_attn_workspace_bytes", N, L, Hq, Hkv, D, max_length, 0, p)) return 0;
  return p.bytes;
}

extern "C" int gdn_paged_attn_fwd(const void* q, long long q_seq, long long q_token, long long q_head,
                                  const void* k_cache, const void* v_cache, const float* k_scale,
                                  const float* v_scale, const int32_t* block_table,
                                  long long table_row, const int32_t* lengths, void* o, float* lse,
                                  int N, int L, int Hq, int Hkv, int D, int num_pages,
                                  int page_size, int max_length, int window, float scale,
                                  int dtype, int cache_dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* name = "gdn_paged_attn_fwd";
  AttnPlan p{};
  const bool bits8 = cache_dtype == GDN_DTYPE_E4M3 || cache_dtype == GDN_DTYPE_I8;
  if (const int rc = attn_plan(name, N, L, Hq, Hkv, D, max_length, D * (bits8 ? 1 : 2), p)) return rc;
  if (const int rc = gdn_host::check_cache(name, k_cache, v_cache, k_scale, v_scale, Hkv, D, num_pages, page_size,
                                           cache_dtype))
    return rc;
  if (page_size % 16)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": page_size must be a multiple of 16");
  if (num_pages < 1)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": the cache must have a page");
  if (window < 0 || table_row < 0 || (max_length && table_row < (max_length - 1) / page_size + 1))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": window must be >= 0, and a table's row hold the "
                                                             "pages of max_length tokens");
  if (dtype != GDN_DTYPE_BF16 && dtype != GDN_DTYPE_F16)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported dtype code");
  if (N == 0) return GDN_OK;
  if (!q || !o || !lengths || (max_length && !block_table))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": q, o, block_table and lengths must be non-NULL");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) % 16 || (q_seq | q_token | q_head) % 8 ||
      q_seq < 0 || q_token < 0 || q_head < 0)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": q and o must be 16-byte aligned, q's strides "
                                                             "non-negative multiples of 8");
  if ((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 16)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": scales must be 16-byte aligned");
  const size_t ob = (size_t)N * L * Hq * D * 2;
  const size_t qb = ((size_t)(N - 1) * q_seq + (size_t)(L - 1) * q_token + (size_t)(Hq - 1) * q_head + D) * 2;
  const size_t cb = (size_t)num_pages * Hkv * page_size * D * (bits8 ? 1 : 2);
  if (gdn_host::overlaps(o, ob, q, qb) || gdn_host::overlaps(o, ob, k_cache, cb) ||
      gdn_host::overlaps(o, ob, v_cache, cb))
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": o must not overlap q or the caches");
  if (!workspace || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16)
    return gdn_host::fail(GDN_ERR_WORKSPACE, std::string(name) + ": workspace needs " + std::to_string(p.bytes) +
                                                 " bytes, 16-byte aligned, got " + std::to_string(workspace_bytes));
  const long long R = (long long)L * (Hq / Hkv);
  gdn::PagedAttnArgs a{};
  a.q = q;
  a.sn = q_seq;
  a.sl = q_token;
  a.sh = q_head;
  a.kc = k_cache;
  a.vc = v_cache;
  a.ks = k_scale;
  a.vs = v_scale;
  a.table = block_table;
  a.table_stride = table_row;
  a.lens = lengths;
  a.o = o;
  a.lse = lse;
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.desc);
  a.N = N;
  a.L = L;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.R = (int)R;
  a.RG = p.rg;
  a.rows = p.rows;
  a.part_size = p.part_size;
  a.num_pages = num_pages;
  a.page = page_size;
  a.cap = max_length;
  a.whole = p.whole;
  a.by_item = p.items <= p.wgs;
  a.window = window > (1 << 30) ? 1 << 30 : window;
  a.scale2 = scale * 1.44269504088896340736f;
  auto st = static_cast<hipStream_t>(stream);
  gdn_host::launch_begin();
  bool done = false;
#define GDN_PA(QQ, CC, DD, TT, WW)                                                                \
  if (dtype == QQ && cache_dtype == CC && D == DD && p.nt == TT && (p.each ? 0 : p.rw) == WW) {   \
    hipLaunchKernelGGL((gdn::paged_attn_kernel<QQ, CC, DD, TT, WW>), dim3((unsigned)p.grid), dim3(256), 0, st, a); \
    done = true;                                                                                  \
  }
#define GDN_PA_W(QQ, CC, DD) GDN_PA(QQ, CC, DD, 1, 0) GDN_PA(QQ, CC, DD, 1, 1) GDN_PA(QQ, CC, DD, 2, 1) GDN_PA(QQ, CC, DD, 2, 2)
#define GDN_PA_D(QQ, CC) GDN_PA_W(QQ, CC, 64) GDN_PA_W(QQ, CC, 128) GDN_PA_W(QQ, CC, 256)
  GDN_PA_D(GDN_DTYPE_BF16, GDN_DTYPE_BF16)
  GDN_PA_D(GDN_DTYPE_F16, GDN_DTYPE_F16)
  GDN_PA_D(GDN_DTYPE_BF16, GDN_DTYPE_E4M3)
  GDN_PA_D(GDN_DTYPE_F16, GDN_DTYPE_E4M3)
  GDN_PA_D(GDN_DTYPE_BF16, GDN_DTYPE_I8)
  GDN_PA_D(GDN_DTYPE_F16, GDN_DTYPE_I8)
#undef GDN_PA_D
#undef GDN_PA_W
#undef GDN_PA
  if (!done)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": the cache must be of q's type or have 8 bits");
  if (p.whole) return gdn_host::check_launch(name);
  const dim3 grid((unsigned)(a.by_item ? p.items : p.wgs), (unsigned)p.rows);
  // few outputs of many parts each: a CU's worth of lanes to 64 columns of each
  // (131072 tokens of one sequence, 256 parts of 16 rows of 256: 4.8 us, 6.2 with a CU
  // to a whole row)
  const bool wide = (long long)grid.x * grid.y <= gdn::device_cus();
#define GDN_PJ(QQ, DD)                                                                            \
  if (dtype == QQ && D == DD) {                                                                   \
    if (wide) hipLaunchKernelGGL((gdn::paged_attn_join_kernel<QQ, DD, 1024, 16>), dim3(grid.x, grid.y, DD / 64), \
                                 dim3(1024), 0, st, a);                                           \
    else hipLaunchKernelGGL((gdn::paged_attn_join_kernel<QQ, DD, 256, DD / 4>), grid, dim3(256), 0, st, a); \
  }
  GDN_PJ(GDN_DTYPE_BF16, 64) GDN_PJ(GDN_DTYPE_BF16, 128) GDN_PJ(GDN_DTYPE_BF16, 256)
  GDN_PJ(GDN_DTYPE_F16, 64) GDN_PJ(GDN_DTYPE_F16, 128) GDN_PJ(GDN_DTYPE_F16, 256)
#undef GDN_PJ
  return gdn_host::check_launch(name);
}
