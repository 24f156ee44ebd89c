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
};

// Where a segment's data comes from: equal lengths by arithmetic, cu_seqlens
// through the table the table kernel wrote.
struct LinGrid {
  const LinSeg* table;      // [nseg], NULL: equal lengths
  const int32_t* soff;      // [N + 1] first segment of each sequence (with table)
  const int32_t* status;    // != 0: a cu_seqlens violation (with table)
  int T, L, nps;            // tokens and segments per sequence (without table), chunks per segment
  int nseg;                 // segments at most
  int N, total;             // sequences, tokens of all
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
  return r;
}

// Decays: element (token, head) of g, or one per head.
struct LinDecay {
  const void* g;
  int dt, per_token;   // per_token: Hv, or 0 for one per head
};
// A decay under e^-150 is e^-150: both are 0 in fp32, and -inf (a reset) stays
// out of the differences of prefix sums.
__device__ __forceinline__ float lin_g(const LinDecay& d, long long tok, int h) {
  const float x = ldp(d.g, tok * d.per_token + h, d.dt);
  return x < -150.f ? -150.f : x;
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
  // Operand fragment of 16 rows and 32 columns: lane (r16, grp) holds
  // X[16 tt + r16][32 kb + 8 grp + i].
  static __device__ __forceinline__ u16x8 rows(const char* p, int tt, int kb, int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    const int base = r16 * RS + 16 * (grp ^ swz(r16));
    return *reinterpret_cast<const u16x8*>(p + ((base ^ (kb * 64)) + tt * 16 * RS));
  }
  // Operand fragment of X^T: 16 columns and 32 rows, lane (r16, grp) holds
  // X[32 kb + 8 grp + i][c], c = rho_row of tile T: 32 (T / 2) + 8 (r16 / 4) +
  // 4 (T % 2) + r16 % 4.  Two tiles' accumulator rows then hold 8 adjacent
  // columns per lane.
  static __device__ __forceinline__ u16x8 cols(const char* p, int kb, int T, int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    const int m4 = r16 >> 2, q4 = r16 & 3;
    const int r0 = 8 * grp + m4, r1 = r0 + 4;
    const int b0 = (r0 * RS + 16 * (q4 ^ swz(r0))) ^ ((T >> 1) * 64);
    const int b1 = (r1 * RS + 16 * (q4 ^ swz(r1))) ^ ((T >> 1) * 64);
    const int at = kb * 32 * RS + (T & 1) * 8;
    const u16x4 lo = lds_tr16(reinterpret_cast<const uint16_t*>(p + b0 + at));
    const u16x4 hi = lds_tr16(reinterpret_cast<const uint16_t*>(p + b1 + at));
    return cat8(lo, hi);
  }
  // The same for 16 adjacent columns: lane (r16, grp) holds
  // X[32 kb + 8 grp + i][16 T + r16].
  static __device__ __forceinline__ u16x8 cols16(const char* p, int kb, int T, int lane) {
    const int r16 = lane % 16, grp = lane / 16;
    const int m4 = r16 >> 2, q4 = r16 & 3;
    const int r0 = 8 * grp + m4, r1 = r0 + 4, u = 2 * T + (q4 >> 1);
    const int at = kb * 32 * RS + (q4 & 1) * 8;
    const u16x4 lo = lds_tr16(reinterpret_cast<const uint16_t*>(p + off(r0, u) + at));
    const u16x4 hi = lds_tr16(reinterpret_cast<const uint16_t*>(p + off(r1, u) + at));
    return cat8(lo, hi);
  }
};

// The 64 rows of a chunk on their way from HBM to a tile, 16 bytes per lane
// and load, by NT threads: rows at and past `n` are zero.
template <int D, int NT>
struct LinStage {
  static constexpr int ALL = 64 * (D / 8);
  static constexpr int PER = (ALL + NT - 1) / NT;
  u32x4 r[PER];
  // p: the head's columns of the chunk's first token; row: elements per token
  __device__ __forceinline__ void load(const uint16_t* p, int row, int n, int tid) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(p), 0, n > 0 ? ((n - 1) * row + D) * 2 : 0, kBufferFlags);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * NT;
      r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
          rs, ((u / (D / 8)) * row + (u % (D / 8)) * 8) * 2, 0, 0));
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * NT;
      if (ALL % NT && u >= ALL) break;   // (its load was past row 64: out of range, 0)
      *reinterpret_cast<u32x4*>(tile + LinTile<D>::off(u / (D / 8), u % (D / 8))) = r[i];
    }
  }
};

// Inclusive prefix sum over a wave.
__device__ __forceinline__ float wave_prefix(float x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const float y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  return x;
}
// Exclusive suffix sum over a wave (sums of what follows a lane).
__device__ __forceinline__ float wave_suffix(float x, int lane) {
  float s = __shfl_down(x, 1);
  if (lane == 63) s = 0.f;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const float y = __shfl_down(s, off);
    if (lane + off < 64) s += y;
  }
  return s;
}

// Workgroup -> work item so that neighbouring items run on the same XCD
// (workgroups go round the 8 of them) and share its L2.  The grid is
// xcd_grid(n); items at and past n are for nobody.
inline unsigned xcd_grid(long long n) { return (unsigned)((n + 7) / 8 * 8); }
__device__ __forceinline__ int xcd_item() {
  return (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
}

// Host: how a call is cut (byte offsets into the workspace).
struct LinPlan {
  int L, nps, nseg;          // as LinGrid
  long long chunks;          // chunks of all sequences at most (chunk-start states)
  size_t table, soff, status, segs, decay, total;
  // backward
  size_t part;               // fp32 partial dq, dk per v-head (Hv > Hqk)
  size_t dgtok;              // fp32 dg per token and v-head (one decay per head)
};
LinPlan lin_plan(int B, int T, int Hqk, int Hv, int K, int V, int N, bool has_cu, bool bwd);
LinGrid lin_grid(const LinPlan& p, unsigned char* ws, int T, int N, int total, bool has_cu);
void launch_lin_table(const int32_t* cu, const LinPlan& p, unsigned char* ws, int N, int total,
                      hipStream_t st);
// Contribution of every segment to the state that follows (or, reverse, to the
// gradient of the state before it), then the states at every segment's border.
template <int K, int V>
void launch_lin_segments(const uint16_t* x, int x_row, const uint16_t* y, int y_row,
                         const LinDecay& d, const LinGrid& g, int Hqk, int Hv, float scale,
                         bool reverse, const float* edge, float* segs, float* decay,
                         hipStream_t st);

}  // namespace gdn
