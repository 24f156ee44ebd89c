// Internal interface of linear attention's chunked form (gdn_linear.hip,
// gdn_linear_bwd.hip): the plan of segments, the swizzled LDS tiles and the
// fragments read from them.
#pragma once

#include "gdn_chunk.h"

namespace gdn {

// One segment of a sequence: tokens tok0 .. tok0 + ntok - 1, the global chunk
// its first token starts (chunk-start states), its sequence and place in it.
struct LinSeg {
  int tok0, ntok, chunk0, seq;
  int first, last;   // first / last segment of its sequence
  int before;        // chunks of its sequence before it
};

// A sequence of several segments (seq < 0: no more of them): s0 .. s1 - 1.
struct LinJoin {
  int seq, s0, s1;
};

// Where a segment's data comes from: equal lengths by arithmetic, cu_seqlens
// through the table the table kernel wrote.
struct LinGrid {
  const LinSeg* table;      // [nseg], NULL: equal lengths
  const int32_t* status;    // != 0: a cu_seqlens violation (with table)
  const int32_t* order;     // [nseg] segments, longest first (with table)
  const LinJoin* joins;     // [nlong] the sequences of several segments (with table)
  int T, L, nps;            // tokens and segments per sequence (without table), chunks per segment
  int nseg;                 // segments at most
  int nlong;                // sequences of several segments at most
  int N, total;             // sequences, tokens of all
  bool one;                 // one workgroup per CU
};

__device__ __forceinline__ LinSeg lin_seg(const LinGrid& g, int s) {
  if (g.table) return g.table[s];
  LinSeg r;
  r.seq = s / g.nps;
  const int i = s % g.nps;
  r.tok0 = r.seq * g.T + i * g.L * kChunk;
  r.ntok = min(g.T - i * g.L * kChunk, g.L * kChunk);
  r.chunk0 = r.seq * ((g.T + kChunk - 1) / kChunk) + i * g.L;
  r.first = i == 0;
  r.last = i == g.nps - 1;
  r.before = i * g.L;
  return r;
}

// Decays: element (token, head) of g, or one per head.
struct LinDecay {
  const void* g;
  int dt, per_token;   // per_token: Hv, or 0 for one per head
};
// A decay under e^-150 is e^-150: both are 0 in fp32, and -inf (a reset) stays
// out of the differences of prefix sums.
__device__ __forceinline__ float lin_clamp(float x) { return x < -150.f ? -150.f : x; }
__device__ __forceinline__ float lin_g(const LinDecay& d, long long tok, int h) {
  return lin_clamp(ldp(d.g, tok * d.per_token + h, d.dt));
}

// A [64][D] bf16 tile in LDS: rows of 2 D bytes, their 16-byte units permuted
// by XOR with swz(row), which puts both kinds of fragment reads on distinct
// banks: 16 rows at one unit, and the transposing reads' 4 rows x 4 units.
template <int D>
struct LinTile {
  static constexpr int RS = 2 * D;
  static constexpr int BYTES = 64 * RS;
  static constexpr int UNITS = D / 8;   // 16-byte units per row
  __device__ static constexpr int swz(int r) {
    return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
  }
  __device__ static constexpr int off(int r, int u) { return r * RS + 16 * (u ^ swz(r)); }
  // Fragment reads.  Each takes a lane's byte base within a tile; what is left
  // is a constant per call, in the instruction or one XOR (a kernel hides the
  // bases from the compiler once per chunk, or it would keep every XORed copy
  // in a register of its own).
  //
  // Operand fragment of 16 rows and 32 columns: lane (r16, grp) holds
  // X[16 tt + r16][32 kb + 8 grp + i].
  static __device__ __forceinline__ int row_base(int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    return r16 * RS + 16 * (grp ^ swz(r16));
  }
  static __device__ __forceinline__ u16x8 rows(const char* p, int base, int tt, int kb) {
    return *reinterpret_cast<const u16x8*>(p + (base ^ (kb * 64)) + tt * 16 * RS);
  }
  // The same rows, with the columns in the order in which two 16-row tiles of
  // accumulators hold theirs: element i < 4 is column 32 kb + 4 grp + i, the
  // others 16 further on (the operand that meets a state kept in accumulators).
  static __device__ __forceinline__ int row4_base(int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    return off(r16, grp >> 1) + (grp & 1) * 8;
  }
  static __device__ __forceinline__ u16x8 rows4(const char* p, int base, int tt, int kb) {
    const int b = base ^ (kb * 64);
    return cat8(*reinterpret_cast<const u16x4*>(p + b + tt * 16 * RS),
                *reinterpret_cast<const u16x4*>(p + (b ^ 32) + tt * 16 * RS));
  }
  // Operand fragment of X^T, 16 columns and 32 rows: lane (r16, grp) holds
  // X[32 kb + 8 grp + i][16 T + r16].
  static __device__ __forceinline__ int col_base(int T, int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    const int m4 = r16 >> 2, q4 = r16 & 3, r0 = 8 * grp + m4;
    return off(r0, 2 * T + (q4 >> 1)) + (q4 & 1) * 8;
  }
  // (base: of tile T0, for tile T0 ^ T)
  static __device__ __forceinline__ u16x8 cols(const char* p, int base, int kb, int T) {
    const int at = kb * 32 * RS;
    base ^= 32 * T;
    // (four rows on, the unit's lowest bit is the other one)
    const u16x4 lo = lds_tr16(reinterpret_cast<const uint16_t*>(p + base + at));
    const u16x4 hi = lds_tr16(reinterpret_cast<const uint16_t*>(p + (base ^ 16) + 4 * RS + at));
    return cat8(lo, hi);
  }
  // The same with the rows in rows4's order: i < 4 row 32 kb + 4 grp + i, the
  // others 16 further on.
  static __device__ __forceinline__ int col4_base(int T, int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    const int m4 = r16 >> 2, q4 = r16 & 3;
    return off(4 * grp + m4, 2 * T + (q4 >> 1)) + (q4 & 1) * 8;
  }
  static __device__ __forceinline__ u16x8 cols4(const char* p, int base, int kb, int T) {
    const char* x = p + (base ^ (32 * T)) + kb * 32 * RS;
    return cat8(lds_tr16(reinterpret_cast<const uint16_t*>(x)),
                lds_tr16(reinterpret_cast<const uint16_t*>(x + 16 * RS)));
  }
};

// The 64 rows of a chunk on their way from HBM to a tile, 16 bytes per lane
// and load, by NT threads: rows at and past `n` are zero.
template <int D, int NT>
struct LinStage {
  static constexpr int UNITS = D / 8, ALL = 64 * UNITS, PER = (ALL + NT - 1) / NT;
  static constexpr int STEP = NT / UNITS;   // rows between a lane's loads
  static_assert(STEP % 4 == 0, "swizzle by constant offsets");
  u32x4 r[PER];
  // bytes into the chunk's rows of a lane's first load; and into the tile
  static __device__ __forceinline__ int from(int row, int tid) {
    return ((tid / UNITS) * row + tid % UNITS * 8) * 2;
  }
  static __device__ __forceinline__ int at(int tid, int i) {
    return LinTile<D>::off(tid / UNITS + i * STEP, tid % UNITS);
  }
  // p: the head's columns of the chunk's first token; row: elements per token
  __device__ __forceinline__ void load(const uint16_t* p, int row, int n, int from) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(p), 0, n > 0 ? ((n - 1) * row + D) * 2 : 0, kBufferFlags);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
          rs, from + i * STEP * row * 2, 0, 0));
  }
  // base: at(tid, 0)
  __device__ __forceinline__ void store(char* tile, int base, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (ALL % NT && tid + i * NT >= ALL) break;   // (its load was past row 64: 0)
      const int to = STEP % 16 == 0 ? base + i * STEP * LinTile<D>::RS : at(tid, i);
      *reinterpret_cast<u32x4*>(tile + to) = r[i];
    }
  }
};

// Sum over 16 lanes (lane 15 of each 16 has it).
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                 0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float row16_sum(float x) {
  x = dpp_add<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  return dpp_add<0x118, 0xf>(x);
}

// The index of this wave, known to be the same in all its lanes.
__device__ __forceinline__ int wave_index() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
}
__device__ __forceinline__ void hide(int& x) { asm volatile("" : "+v"(x)); }

// Inclusive prefix sum over a wave, in its lanes' own adders (no LDS).
__device__ __forceinline__ float wave_prefix(float x) {
  x = row16_sum(x);             // (a prefix sum within the 16 lanes)
  x = dpp_add<0x142, 0xa>(x);   // lane 15 of a row to the next: rows 1 and 3
  return dpp_add<0x143, 0xc>(x);   // lane 31 to rows 2 and 3
}

__device__ __forceinline__ float lane63(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// Eight bf16 values times eight fp32 factors (in LDS) as a sum of NP bf16
// parts, 2^-8 per part.  Three where a state is returned or saved (its error
// then is fp32's, 2e-7 of it; two leave 3e-6 and cost 64 packed prompts 957 us
// in place of 1067, 8192 tokens 100 of 105), two where it serves bf16 outputs.
template <int NP>
__device__ __forceinline__ void lin_split(u16x8 y, const float* f, u16x8 (&part)[NP]) {
  const f32x4 f0 = *reinterpret_cast<const f32x4*>(f), f1 = *reinterpret_cast<const f32x4*>(f + 4);
  f32x4 x0 = f32x4{bf2f(y[0]), bf2f(y[1]), bf2f(y[2]), bf2f(y[3])} * f0;
  f32x4 x1 = f32x4{bf2f(y[4]), bf2f(y[5]), bf2f(y[6]), bf2f(y[7])} * f1;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const u16x4 h0 = f2bf4(x0), h1 = f2bf4(x1);
    part[p] = cat8(h0, h1);
    if (p + 1 < NP) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x0[i] -= bf2f(h0[i]);
        x1[i] -= bf2f(h1[i]);
      }
    }
  }
}

// A saved state, 16 bits per value: four neighbours of one key's row as fp16
// with nine bits after the leading one, under a common factor 2^(16 e - 126)
// whose e is in their lowest bits.  (In bf16, seven bits, its rounding was what
// was wrong with dg: 2.0e-3 of it where dg's own is 1.7e-3, three times that for
// a few tokens behind an initial state.)  The largest of the four lies in
// [2^-1, 2^15), so that one 2^15 times smaller still has bf16's precision.  What
// is cut off is 2^-10 on average, 0.7 of which the factor makes up for; values of
// nine bits and less stay what they are, and so do infinities and NaN.
__device__ __forceinline__ u16x4 lin_pack(f32x4 x) {
  constexpr uint32_t M = 0x00010001;
  const float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  const uint32_t e = __float_as_uint(m) & 0x78000000u;
  x *= __uint_as_float(0x7E800000u - e) * 1.000671f;
  const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[0], x[1]));
  const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[2], x[3]));
  const uint32_t u = (e >> 27) | (e >> 12);   // bits 0, 1 of e / 2^27 in 0 and 16, bits 2, 3 in 2 and 18
  return __builtin_bit_cast(u16x4, u32x2p{(u & M) | (a & ~M), ((u >> 2) & M) | (b & ~M)});
}
__device__ __forceinline__ f32x4 lin_unpack(u16x4 p) {
  constexpr uint32_t M = 0x00010001;
  const u32x2p d = __builtin_bit_cast(u32x2p, p);
  uint32_t u = (d[0] & M) | ((d[1] & M) << 2);
  u |= u >> 15;
  const float s = __uint_as_float((u << 27) + 0x00800000u);
  const u16x4 h = __builtin_bit_cast(u16x4, u32x2p{d[0] & ~M, d[1] & ~M});
  f32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h[i])));
  return x * s;
}

// The decays of a chunk on their way in, by two waves: wave 0's lane l has its
// own token, wave 1's the token 64 - l, so that the prefix sums and the sums
// of what follows a token (63 - l) are the same scan.  Loaded a chunk ahead,
// without a branch, and converted where they are used: a wait for them here
// would hold up the loads behind them.
struct LinGates {
  FlatRaw raw;
  int n;
  static __device__ __forceinline__ int token(int w, int lane) { return w == 0 ? lane : 64 - lane; }
  // tok: the chunk's first token; n: its tokens (0: none); i: token(w, lane)
  __device__ __forceinline__ void load(const LinDecay& d, size_t tok, int n_, int h, int Hv, int i) {
    n = n_;
    const int es = d.dt == GDN_DTYPE_F32 ? 4 : 2;
    const char* p = static_cast<const char*>(d.g) + tok * d.per_token * es;
    raw = ldp_flat_raw(p, i * d.per_token + h, d.dt, d.per_token ? n * Hv : (n > 0 ? Hv : 0));
  }
  __device__ __forceinline__ float prefix(const LinDecay& d, int i) const {
    const float x = lin_clamp(flat_value(raw, d.dt));
    return wave_prefix(i < n ? x : 0.f);
  }
};

// A [K][V] fp32 state: a lane's part in one register offset, the tiles' and
// rows' in scalars; without a state (NULL) the loads give 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t lin_state(const float* p, int KV) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, p ? KV * 4 : 0, kBufferFlags);
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Workgroup -> (segment, v-head): the v-heads of a qk-head run on one XCD
// (workgroups go round the 8 of them) one after another and share q and k in
// its L2; a segment's qk-heads, and so segments of different lengths, are
// spread over the XCDs.  Packed segments start longest first.  The grid is
// lin_items(...) workgroups; false: none for this one.
inline long long lin_items(int nseg, int Hqk, int Hv) {
  return ((long long)nseg * Hqk + 7) / 8 * 8 * (Hv / Hqk);
}
__device__ __forceinline__ bool lin_item(const LinGrid& g, int nseg, int Hqk, int Hv, int& s,
                                         int& h) {
  const int rep = Hv / Hqk, i = blockIdx.x / 8, u = i / rep * 8 + blockIdx.x % 8;
  s = u / Hqk;
  h = u % Hqk * rep + i % rep;
  return s < nseg;
}

// Host: how a call is cut (byte offsets into the workspace).
struct LinPlan {
  int L, nps, nseg;          // as LinGrid
  bool one;                  // as LinGrid
  long long chunks;          // chunks of all sequences at most (chunk-start states)
  int nlong;                 // sequences of several segments at most (0: no join)
  size_t table, status, order, joins, segs, decay, total;
  // backward
  size_t part;               // fp32 partial dq, dk (several per qk-head)
  size_t dgtok;              // fp32 dg per token and v-head (one decay per head)
};
// Whether the backward takes two v-heads of a qk-head at a time.
inline bool lin_pair(int Hqk, int Hv) { return Hv / Hqk % 2 == 0; }
LinPlan lin_plan(int B, int T, int Hqk, int Hv, int K, int V, int N, bool has_cu, bool bwd);
// The workspace that the caller is asked for.
size_t lin_bytes(int B, int T, int Hqk, int Hv, int K, int V, int N, bool has_cu, bool bwd);
LinGrid lin_grid(const LinPlan& p, unsigned char* ws, int T, int N, int total, bool has_cu);
void launch_lin_table(const int32_t* cu, const LinPlan& p, unsigned char* ws, int N, int total,
                      hipStream_t st);
// Contribution of every segment to the state that follows (or, reverse, to the
// gradient of the state before it), then the states at every segment's border.
template <int K, int V>
void launch_lin_segments(const uint16_t* x, int x_row, const uint16_t* y, int y_row,
                         const LinDecay& d, const LinGrid& g, int Hqk, int Hv, float scale,
                         bool reverse, bool full, const float* edge, float* segs,
                         float* decay, float* end, hipStream_t st);

}  // namespace gdn
