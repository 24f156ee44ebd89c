// Linear attention with a decay for each head, chunked form for gfx950
// (declared in gdn_linear.h).  Per v-head, state S [K][V] in fp32:
//     S_t = e^{g_t} S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t
// In chunks of 64 tokens, G the chunk's prefix sums of g and R_j the sum of
// what follows token j in it:
//     P_ij = scale e^{G_i - G_j} (q_i . k_j)   (j <= i)
//     o_i  = sum_j P_ij v_j + scale e^{G_i} S^T q_i
//     S'   = e^{G_63} S + sum_j k_j (e^{R_j} v_j)^T
// all products on bf16 MFMA with fp32 accumulation.  e^{R_j} v_j enters as a
// sum of bf16 parts: three (2^-24) where a state is returned or saved, two
// (2^-16) where it serves o alone; P two; the state's copy that q reads is single
// bf16 (2^-8, the size of o's own rounding: over 110 shapes o is at 1.2 of that at
// the median, 1.4 at most; both parts cost 6 % at 8192 tokens, 15 % on packed
// prompts).  The states that the backward reads are lin_pack's.  R is summed from the chunk's
// end, not as G_63 - G_j: its error stays in proportion to the decay it gives.
//
// A sequence is cut into segments of L chunks that run at the same time: one
// launch forms every segment's own contribution to the state (from k, v and
// g), one joins them along each sequence, one walks every segment from its
// start state and writes o.  Where a whole sequence fits a segment, and where a
// few chunks are stepped through again faster, the first two are left out.
#include <initializer_list>

#include "gdn_linear.h"
#include "../../include/gdn_linear.h"

namespace gdn {

// ---------------------------------------------------------------- table ----
// Segments of packed sequences: an entry per segment, the sequences of several
// segments, and the check of the cu_seqlens contract (on a violation
// every sequence is one empty segment).
__global__ __launch_bounds__(1024) void lin_table_kernel(const int32_t* cu, LinSeg* table,
                                                         LinJoin* joins, int32_t* status,
                                                         int32_t* order, int N,
                                                         int total, int L, int nseg, int nlong) {
  constexpr int BINS = 256;   // of lengths, for the order
  __shared__ int wsum[2][16], bin[BINS], nj;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  int bad = 0;
  for (int n = tid; n < N; n += 1024) bad |= cu[n + 1] < cu[n];
  if (tid == 0) bad |= cu[0] != 0 || cu[N] != total;
  bad = __syncthreads_or(bad);
  if (tid == 0) {
    *status = bad;
    nj = 0;
  }
  if (tid < BINS) bin[tid] = 0;
  auto bin_of = [&](int ntok) {   // longer ones first
    return BINS - 1 - (int)((long long)(ntok + kChunk - 1) / kChunk * (BINS - 1) / L);
  };
  int seg0 = 0, chunk0 = 0;   // of these 1024 sequences' first
  for (int n0 = 0; n0 < N; n0 += 1024) {
    const int n = n0 + tid;
    const int s = n < N && !bad ? cu[n] : 0;
    const int len = n < N && !bad ? cu[n + 1] - s : 0;
    const int nc = (len + kChunk - 1) / kChunk;
    const int ns = n < N ? max(1, (nc + L - 1) / L) : 0;
    int a = ns, b = nc;
    for (int off = 1; off < 64; off *= 2) {
      const int x = __shfl_up(a, off), y = __shfl_up(b, off);
      if (lane >= off) {
        a += x;
        b += y;
      }
    }
    __syncthreads();
    if (lane == 63) {
      wsum[0][wave] = a;
      wsum[1][wave] = b;
    }
    __syncthreads();
    int sa = seg0, sb = chunk0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) {
        sa += wsum[0][w];
        sb += wsum[1][w];
      }
      seg0 += wsum[0][w];
      chunk0 += wsum[1][w];
    }
    sa += a - ns;
    sb += b - nc;
    if (n < N) {
      for (int i = 0; i < ns && sa + i < nseg; ++i) {
        const int ntok = min(len - i * L * kChunk, L * kChunk);
        table[sa + i] = LinSeg{s + i * L * kChunk, ntok, sb + i * L, n, i == 0, i == ns - 1, i * L};
        atomicAdd(&bin[bin_of(ntok)], 1);
      }
      if (ns > 1) {
        const int j = atomicAdd(&nj, 1);
        if (j < nlong) joins[j] = LinJoin{n, sa, min(sa + ns, nseg)};
      }
    }
  }
  for (int i = seg0 + tid; i < nseg; i += 1024) {
    table[i] = LinSeg{0, 0, 0, -1, 0, 0, 0};
    order[i] = i;
  }
  __syncthreads();
  for (int i = nj + tid; i < nlong; i += 1024) joins[i] = LinJoin{-1, 0, 0};
  if (wave == 0) {   // where each bin's segments start
    constexpr int PER = BINS / 64;
    int x[PER], sum = 0;
    for (int i = 0; i < PER; ++i) {
      x[i] = bin[PER * lane + i];
      sum += x[i];
    }
    int at = sum;
    for (int off = 1; off < 64; off *= 2) {
      const int y = __shfl_up(at, off);
      if (lane >= off) at += y;
    }
    at -= sum;
    for (int i = 0; i < PER; ++i) {
      bin[PER * lane + i] = at;
      at += x[i];
    }
  }
  __syncthreads();
  // (which of equal lengths comes first changes when a segment runs, nothing else)
  for (int i = tid; i < min(seg0, nseg); i += 1024) order[atomicAdd(&bin[bin_of(table[i].ntok)], 1)] = i;
}

// 16 columns (ct) of a state [K][V] as accumulators: tile t's lane holds rows
// 16 t + 4 grp + r of column 16 ct + r16.
template <int K, int V>
__device__ __forceinline__ void lin_load_state(f32x4 (&S)[K / 16], const float* p, int ct, int lane) {
  const __amdgpu_buffer_rsrc_t rs = lin_state(p, K * V);
  const int at = (4 * (lane / 16) * V + 16 * ct + lane % 16) * 4;
#pragma unroll
  for (int t = 0; t < K / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[t][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
          rs, at, (16 * t + r) * V * 4, 0));
}
template <int K, int V>
__device__ __forceinline__ void lin_store_state(const f32x4 (&S)[K / 16], float* p, int ct, int lane) {
  const __amdgpu_buffer_rsrc_t rs = lin_state(p, K * V);
  const int at = (4 * (lane / 16) * V + 16 * ct + lane % 16) * 4;
#pragma unroll
  for (int t = 0; t < K / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[t][r]), rs, at,
                                            (16 * t + r) * V * 4, 0);
}

// -------------------------------------------------------------- segments ----
// A chunk's step of the state: S' = eC S + X^T (f Y), X and Y the tiles in xs and
// ys (bases xb, yb), f per token in LDS.
template <int K, int V, int CT, int NP>
__device__ __forceinline__ void lin_step(f32x4 (&S)[CT][K / 16], const char* xs, int xb,
                                         const char* ys, int yb, const float* f, float eC,
                                         int grp) {
#pragma unroll
  for (int T = 0; T < CT; ++T)
#pragma unroll
    for (int t = 0; t < K / 16; ++t) S[T][t] *= eC;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    u16x8 part[CT][NP];
#pragma unroll
    for (int T = 0; T < CT; ++T)
      lin_split(LinTile<V>::cols(ys, yb, kb, T), f + 32 * kb + 8 * grp, part[T]);
#pragma unroll
    for (int t = 0; t < K / 16; ++t) {
      const u16x8 a = LinTile<K>::cols(xs, xb, kb, t);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int T = 0; T < CT; ++T) S[T][t] = mfma16(a, part[T][p], S[T][t]);
    }
  }
}

// Contribution of a segment to the state after it: sum over its chunks of
// X^T (f Y) with x = k, y = v, f = e^R; or (REV) to the gradient of the state
// before it, chunks last to first, x = q, y = dO, f = scale e^G.  A wave owns
// 16 CT columns of Y and all rows of the state.  8192 tokens, 32 v-heads, 100 MB:
// 35 us in three parts, 28 in two.
template <int K, int V, int CT, int NP, bool REV>
__global__ __launch_bounds__(4 * V / CT, 4 / CT) void lin_segment_kernel(
    const uint16_t* __restrict__ x, int x_row, const uint16_t* __restrict__ y, int y_row,
    LinDecay dec, LinGrid grid, int Hqk, int Hv, float scale, bool all,
    float* __restrict__ segs, float* __restrict__ decay) {
  constexpr int NT = 4 * V / CT;
  __shared__ __align__(16) char xs[LinTile<K>::BYTES];
  __shared__ __align__(16) char ys[LinTile<V>::BYTES];
  __shared__ __align__(16) float fac[64];
  __shared__ float tot;
  int sid, h;
  if (grid.table) {
    if (!lin_item(grid, grid.nseg, Hqk, Hv, sid, h)) return;
    sid = grid.order[sid];
  } else {   // every segment, or every one but one of each sequence
    const int per = all ? grid.nps : grid.nps - 1;
    if (!lin_item(grid, grid.N * per, Hqk, Hv, sid, h)) return;
    sid = sid / per * grid.nps + sid % per + (REV && !all ? 1 : 0);
  }
  const int hq = h / (Hv / Hqk);
  const LinSeg sg = lin_seg(grid, sid);
  if (sg.seq < 0 || (!all && (REV ? sg.first : sg.last))) return;
  const int tid = threadIdx.x, lane = tid % 64, w = wave_index();
  const int grp = lane / 16;
  const int nc = (sg.ntok + kChunk - 1) / kChunk;

  f32x4 S[CT][K / 16];
#pragma unroll
  for (int T = 0; T < CT; ++T)
#pragma unroll
    for (int t = 0; t < K / 16; ++t) S[T][t] = zero4();
  LinStage<K, NT> sx;
  LinStage<V, NT> sy;
  LinGates lg;
  int gi = LinGates::token(w, lane);
  float gsum = 0.f;
  int xf = LinStage<K, NT>::from(x_row, tid), yf = LinStage<V, NT>::from(y_row, tid);
  int xt = LinStage<K, NT>::at(tid, 0), yt = LinStage<V, NT>::at(tid, 0);
  auto load = [&](int c) {
    const int n = c >= 0 && c < nc ? sg.ntok - c * kChunk : 0;
    const size_t t = n > 0 ? (size_t)sg.tok0 + c * kChunk : 0;
    if (w < 2) lg.load(dec, t, min(n, 64), h, Hv, gi);
    sx.load(x + t * x_row + hq * K, x_row, min(n, 64), xf);
    sy.load(y + t * y_row + h * V, y_row, min(n, 64), yf);
  };
  const int c0 = REV ? nc - 1 : 0, step = REV ? -1 : 1;
  int xb = LinTile<K>::col_base(0, lane), yb = LinTile<V>::col_base(CT * w, lane);
  load(c0);
  for (int i = 0; i < nc; ++i) {
    hide(xb);
    hide(xf);
    hide(yf);
    hide(gi);
    sx.store(xs, xt, tid);
    sy.store(ys, yt, tid);
    if (w < 2) {
      const float pre = lg.prefix(dec, gi);
      if (w == 1) {
        if (!REV) fac[63 - lane] = __expf(pre);
      } else {
        if (REV) fac[lane] = scale * __expf(pre);
        if (lane == 63) tot = pre;
        gsum += lane63(pre);
      }
    }
    __syncthreads();
    load(c0 + (i + 1) * step);
    lin_step<K, V, CT, NP>(S, xs, xb, ys, yb, fac, __expf(tot), grp);
    __syncthreads();
  }
#pragma unroll
  for (int T = 0; T < CT; ++T)
    lin_store_state<K, V>(S[T], segs + ((size_t)sid * Hv + h) * K * V, CT * w + T, lane);
  if (tid == 0) decay[(size_t)sid * Hv + h] = __expf(gsum);
}

// The states at every segment's start (REV: the gradients of the state at
// every segment's end) in place of the contributions, from `edge` (h0 / dht,
// nullable); into `end` (nullable) the state after the last.  Bound by HBM: a
// lane per E adjacent elements, four where that still gives every CU two
// workgroups (calls of 32 v-heads: 1024 tokens 31.8 us against 35.2 with one,
// 8192 103.5 against 106.7), else one, with as many segments' loads in flight
// (4 v-heads: 4096 tokens 27.6 us against 28.9 with four, 20011 49.7 and 51.2).
template <bool REV, int E>
__global__ __launch_bounds__(256) void lin_join_kernel(LinGrid grid, int Hv, int KV,
                                                       const float* edge,
                                                       float* __restrict__ segs,
                                                       const float* __restrict__ decay,
                                                       float* end) {
  typedef float vec __attribute__((ext_vector_type(E)));
  const int per = KV / (256 * E);
  int n = blockIdx.x / (Hv * per);
  const int h = blockIdx.x / per % Hv, e = (blockIdx.x % per * 256 + threadIdx.x) * E;
  int s0, s1;
  if (grid.table) {
    const LinJoin j = grid.joins[n];
    if (j.seq < 0) return;
    n = j.seq;
    s0 = j.s0;
    s1 = j.s1;
  } else {
    s0 = n * grid.nps;
    s1 = s0 + grid.nps;
  }
  auto at = [&](size_t s) { return reinterpret_cast<vec*>(segs + (s * Hv + h) * KV + e); };
  vec S = {};
  if (edge) S = *reinterpret_cast<const vec*>(edge + ((size_t)n * Hv + h) * KV + e);
  const int first = REV ? s1 - 1 : s0, step = REV ? -1 : 1, cnt = s1 - s0 - 1;
  constexpr int U = E == 1 ? 16 : 8;   // loads in flight
  for (int i = 0; i < cnt; i += U) {
    vec c[U];
    float d[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const size_t s = first + min(i + j, cnt - 1) * step;
      c[j] = *at(s);
      d[j] = decay[s * Hv + h];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i + j < cnt) {
        *at(first + (i + j) * step) = S;
        S = d[j] * S + c[j];
      }
    }
  }
  const size_t last = REV ? s0 : s1 - 1;
  vec x = {};
  if (end) x = decay[last * Hv + h] * S + *at(last);
  *at(last) = S;
  if (end) *reinterpret_cast<vec*>(end + ((size_t)n * Hv + h) * KV + e) = x;
}

// ------------------------------------------------------------------ walk ----
// One segment and v-head from its start state, chunk by chunk: o (OUT), the
// state at every chunk's start (SAVE), ht.  A wave owns 16 CT columns of V, all
// of the state's rows for them in its accumulators, whose layout is that of
// the operand with which S^T q is formed: the state never leaves the registers.
// K, q and v come from HBM once (registers to swizzled LDS tiles, a chunk
// ahead); what bounds a walk is the sum of a chunk's latencies (LDS reads, three
// barriers) over the two workgroups that a CU holds: 8192 tokens, 32 v-heads
// 64 us for 204 MB, 3.2 TB/s; 64 packed prompts in three parts 1069 us, 3.3 TB/s.
//
// ALONE: no launch has formed the segments' start states; each segment first
// steps the state through the chunks before it.
// (Two waves per SIMD is what LDS, or V / 16 waves of 128 registers and more,
// leave all forms but the smallest.)
template <int K, int V, int CT, int NP, bool OUT, bool SAVE, bool ALONE>
__global__ __launch_bounds__(4 * V / CT, CT == 1 && K + V == 128 ? 3 : 2) void lin_walk_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, TokenStride ts, LinDecay dec, LinGrid grid, int Hqk, int Hv,
    float scale, const float* h0, float* ht, const float* __restrict__ segs,
    uint16_t* __restrict__ o, u16x4* __restrict__ states) {
  constexpr int NT = 4 * V / CT, NW = V / 16 / CT;
  __shared__ __align__(16) char qs[LinTile<K>::BYTES];
  __shared__ __align__(16) char ks[LinTile<K>::BYTES];
  __shared__ __align__(16) char vs[LinTile<V>::BYTES];
  __shared__ __align__(16) char ps[LinTile<64>::BYTES], pl[LinTile<64>::BYTES];   // P in two parts
  __shared__ __align__(16) float sG[64], sQ[64], sK[64];   // G log2(e), scale e^G, e^R
  const int tid = threadIdx.x, lane = tid % 64, w = wave_index();
  const int r16 = lane % 16, grp = lane / 16;
  if (grid.table && *grid.status) {
    // a cu_seqlens violation: no sequence has a token, o is zero
    if (OUT) {
      const size_t n = (size_t)grid.total * Hv * V / 8;
      for (size_t i = (size_t)blockIdx.x * NT + tid; i < n; i += (size_t)gridDim.x * NT)
        reinterpret_cast<u32x4*>(o)[i] = u32x4{0, 0, 0, 0};
    }
  }
  int sid, h;
  if (!lin_item(grid, grid.nseg, Hqk, Hv, sid, h)) return;
  if (grid.table) sid = grid.order[sid];
  const int hq = h / (Hv / Hqk);
  LinSeg sg = lin_seg(grid, sid);
  if (sg.seq < 0) return;
  int own = 0;   // the segment's first chunk
  if (ALONE) {
    own = sg.before;
    sg.tok0 -= own * kChunk;
    sg.ntok += own * kChunk;
    sg.chunk0 -= own;
  }
  const int nc = (sg.ntok + kChunk - 1) / kChunk;

  f32x4 S[CT][K / 16];   // rows 16 t + 4 grp + r, column 16 (CT w + T) + r16
  // (several segments: the first one's from the join too, since ht may be h0)
  const float* src = ALONE || (sg.first && sg.last) ? (h0 ? h0 + ((size_t)sg.seq * Hv + h) * K * V : nullptr)
                              : segs + ((size_t)sid * Hv + h) * K * V;
#pragma unroll
  for (int T = 0; T < CT; ++T) lin_load_state<K, V>(S[T], src, CT * w + T, lane);

  LinStage<K, NT> sq, sk;
  LinStage<V, NT> sv;
  LinGates lg;
  int gi = LinGates::token(w, lane);
  int qf = LinStage<K, NT>::from(ts.q, tid), kf = LinStage<K, NT>::from(ts.k, tid);
  int vr = LinStage<V, NT>::from(ts.v, tid);
  const int kt = LinStage<K, NT>::at(tid, 0), vt = LinStage<V, NT>::at(tid, 0);
  int oat = (r16 * Hv * V + 16 * CT * w + 4 * grp) * 2;   // bytes into the chunk's rows of o
  auto load = [&](int c) {
    const int n = c < nc ? sg.ntok - c * kChunk : 0;
    const size_t t = n > 0 ? (size_t)sg.tok0 + c * kChunk : 0;
    if (w < 2) lg.load(dec, t, min(n, 64), h, Hv, gi);
    if (OUT && c >= own) sq.load(q + t * ts.q + hq * K, ts.q, min(n, 64), qf);
    sk.load(k + t * ts.k + hq * K, ts.k, min(n, 64), kf);
    sv.load(v + t * ts.v + h * V, ts.v, min(n, 64), vr);
  };
  if (OUT) {
    // the tiles of P above the diagonal that share a 32-wide block with it
    for (int i = tid; i < 64; i += NT) {
      const int r = i / 2 % 16 + (i / 32) * 32, u = 4 * (i / 32) + 2 + i % 2;
      *reinterpret_cast<u32x4*>(ps + LinTile<64>::off(r, u)) = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4*>(pl + LinTile<64>::off(r, u)) = u32x4{0, 0, 0, 0};
    }
  }
  int rb = LinTile<K>::row_base(lane), r4b = LinTile<K>::row4_base(lane);
  int kcb = LinTile<K>::col_base(0, lane);
  int vb = LinTile<V>::col_base(CT * w, lane), pb = LinTile<64>::row_base(lane);
  int pw = LinTile<64>::off(r16, grp >> 1) + (grp & 1) * 8;
  auto decays = [&]() {   // two waves
    const float pre = lg.prefix(dec, gi) * kLog2e, e = exp2_(pre);
    if (w == 1) {
      sK[63 - lane] = e;
    } else {
      sG[lane] = pre;
      sQ[lane] = scale * e;
    }
  };
  load(0);
  if constexpr (ALONE) {
    for (int c = 0; c < own; ++c) {
      hide(kcb);
      hide(vb);
      sk.store(ks, kt, tid);
      sv.store(vs, vt, tid);
      if (w < 2) decays();
      __syncthreads();
      load(c + 1);
      lin_step<K, V, CT, NP>(S, ks, kcb, vs, vb, sK, exp2_(sG[63]), grp);
      __syncthreads();
    }
  }
  for (int c = own; c < nc; ++c) {
    // (nothing derived from these is kept from one chunk for the next)
    int ln = lane;
    hide(ln);
    const int r16 = ln % 16, grp = ln / 16;
    hide(vb);
    hide(pb);
    hide(pw);
    hide(rb);
    hide(r4b);
    hide(kcb);
    hide(qf);
    hide(gi);
    hide(kf);
    hide(vr);
    hide(oat);
    if (OUT) sq.store(qs, kt, tid);
    sk.store(ks, kt, tid);
    sv.store(vs, vt, tid);
    if (w < 2) decays();
    __syncthreads();
    if (!OUT) load(c + 1);

    if (OUT) {
      // P, tile by tile (token block it, source block jt), as rows of two bf16 parts:
      // one's rounding is the same for all of a value's columns, which the first
      // token after an empty state shows in full (1.73 of o's own; 449 tokens 1 %
      // more, 8192 2 %, 64 packed prompts 4 %)
      for (int n = w; n < 10; n += NW) {
        const int it = tmat_block_row(n), jt = n - tmat_block(it, 0);
        f32x4 p = zero4();
#pragma unroll
        for (int kb = 0; kb < K / 32; ++kb)
          p = mfma16(LinTile<K>::rows(ks, rb, jt, kb), LinTile<K>::rows(qs, rb, it, kb), p);
        const int i = 16 * it + r16, j = 16 * jt + 4 * grp;
        const f32x4 gj = *reinterpret_cast<const f32x4*>(&sG[j]);
        const float gi = sG[i];
        // (a select on each side of the product: no branch around the exponential,
        // and what is masked may be infinite or NaN)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = j + r <= i;
          p[r] = (in ? p[r] * scale : 0.f) * exp2_(in ? gi - gj[r] : 0.f);
        }
        u16x4 hi, lo;
        split_bf4(p, hi, lo);
        *reinterpret_cast<u16x4*>(ps + (pw ^ (32 * jt)) + it * 2048) = hi;
        *reinterpret_cast<u16x4*>(pl + (pw ^ (32 * jt)) + it * 2048) = lo;
      }
    }
    if (OUT) load(c + 1);
    // the state as bf16 operands, by rows of 32 keys
    f32x4 O[4][CT];   // columns 16 (CT w + T) + 4 grp + r of token 16 tt + r16
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int T = 0; T < CT; ++T) O[tt][T] = zero4();
#pragma unroll
    for (int b = 0; b < K / 32; ++b) {
      u16x8 sb[CT], sl[CT];   // (sl: what sb leaves, for the saved copy)
#pragma unroll
      for (int T = 0; T < CT; ++T) {
        if constexpr (SAVE) {
          u16x4 h0, h1, l0, l1;
          split_bf4(S[T][2 * b], h0, l0);
          split_bf4(S[T][2 * b + 1], h1, l1);
          sb[T] = cat8(h0, h1);
          sl[T] = cat8(l0, l1);
        } else {
          sb[T] = cat8(f2bf4(S[T][2 * b]), f2bf4(S[T][2 * b + 1]));
        }
      }
      if (OUT) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const u16x8 f = LinTile<K>::rows4(qs, r4b, tt, b);
#pragma unroll
          for (int T = 0; T < CT; ++T) O[tt][T] = mfma16(sb[T], f, O[tt][T]);
        }
      }
      if (SAVE) {
        // transposed through products with a selection matrix (exact): lane
        // (r16, grp) gets key 16 t + r16, values 16 ct + 4 grp + r, half of its
        // share of the backward's fragment (rows4's order)
        u16x4* dst = states + ((size_t)(sg.chunk0 + c) * Hv + h) * (K / 16) * (V / 32) * 128 +
                     ((CT * w) >> 1) * 128 + lane * 2 + (CT * w & 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u16x8 sel;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sel[i] = grp == r16 >> 2 && i == 4 * e + (r16 & 3) ? 0x3F80 : 0;
          u16x4* at = dst + (2 * b + e) * (V / 32) * 128;
          const u16x4 x = lin_pack(mfma16(sl[0], sel, mfma16(sb[0], sel, zero4())));
          if constexpr (CT == 2)
            *reinterpret_cast<u16x8*>(at) =
                cat8(x, lin_pack(mfma16(sl[1], sel, mfma16(sb[1], sel, zero4()))));
          else
            *at = x;
        }
      }
    }
    if (OUT) {
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float eq = sQ[16 * tt + r16];
#pragma unroll
        for (int T = 0; T < CT; ++T) O[tt][T] *= eq;
      }
      __syncthreads();   // P
    }
    // (the matrix products go ahead of the other workgroup's P: 8192 tokens 106 us
    // against 111 without)
    __builtin_amdgcn_s_setprio(1);
    const float eC = exp2_(sG[63]);
    const u16x8 ones = {0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80};
#pragma unroll
    for (int T = 0; T < CT; ++T)
#pragma unroll
      for (int t = 0; t < K / 16; ++t) S[T][t] *= eC;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      u16x8 vf[CT], part[CT][NP];
#pragma unroll
      for (int T = 0; T < CT; ++T) {
        vf[T] = LinTile<V>::cols(vs, vb, kb, T);
        lin_split(vf[T], sK + 32 * kb + 8 * grp, part[T]);
      }
      if (OUT) {
        // The block's sums show a value that is not finite.  It must not
        // meet the zeros of P before its token: it is left out of the product, and
        // its column is NaN from its token on.
        f32x4 sum = mfma16(vf[0], ones, zero4());
        if constexpr (CT == 2) sum = mfma16(vf[1], ones, sum);
        const bool clean = __all(fabsf((sum[0] + sum[1]) + (sum[2] + sum[3])) < INFINITY);
        u16x8 vm[CT];
        int from[CT];   // the first such token of column r16 (64: none)
#pragma unroll
        for (int T = 0; T < CT; ++T) {
          vm[T] = vf[T];
          from[T] = 64;
          if (!clean) {
#pragma unroll
            for (int i = 7; i >= 0; --i)
              if ((vf[T][i] & 0x7F80) == 0x7F80) {
                vm[T][i] = 0;
                from[T] = 32 * kb + 8 * grp + i;
              }
            from[T] = min(from[T], __shfl_xor(from[T], 16));
            from[T] = min(from[T], __shfl_xor(from[T], 32));
          }
        }
#pragma unroll
        for (int tt = 2 * kb; tt < 4; ++tt) {
          const u16x8 f = LinTile<64>::rows(ps, pb, tt, kb);
#pragma unroll
          for (int T = 0; T < CT; ++T) O[tt][T] = mfma16(vm[T], f, O[tt][T]);
          const u16x8 fl = LinTile<64>::rows(pl, pb, tt, kb);
#pragma unroll
          for (int T = 0; T < CT; ++T) O[tt][T] = mfma16(vm[T], fl, O[tt][T]);
        }
        if (!clean) {
#pragma unroll
          for (int T = 0; T < CT; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = __shfl(from[T], 4 * grp + r);
#pragma unroll
              for (int tt = 2 * kb; tt < 4; ++tt)
                if (16 * tt + r16 >= at) O[tt][T][r] = NAN;
            }
        }
      }
#pragma unroll
      for (int t = 0; t < K / 16; ++t) {
        const u16x8 f = LinTile<K>::cols(ks, kcb, kb, t);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int T = 0; T < CT; ++T) S[T][t] = mfma16(f, part[T][p], S[T][t]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (OUT) {
      // (stores past the segment's last token are dropped)
      const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(
          o + ((size_t)(sg.tok0 + c * kChunk) * Hv + h) * V, 0,
          ((min(sg.ntok - c * kChunk, 64) - 1) * Hv + 1) * V * 2, kBufferFlags);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int T = 0; T < CT; ++T)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2p, f2bf4(O[tt][T])), ro,
                                                oat + (tt * 16 * Hv * V + 16 * T) * 2, 0, 0);
    }
    __syncthreads();
  }
  if (ht && sg.last) {
#pragma unroll
    for (int T = 0; T < CT; ++T)
      lin_store_state<K, V>(S[T], ht + ((size_t)sg.seq * Hv + h) * K * V, CT * w + T, lane);
  }
}

__global__ __launch_bounds__(256) void lin_copy_kernel(const f32x4* __restrict__ from,
                                                       f32x4* __restrict__ to, size_t n) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from[i];
}

// 16-column tiles per wave.  Two in the walk of a 128-column state read half of
// what one reads from LDS (64 packed prompts 1082 us against 1297, 8192 tokens
// 113 against 123); a walk of 64 columns has room for twice the waves with one,
// and where a workgroup has a CU to itself one is better for both (100 tokens of
// 32 v-heads 10.1 us against 11.4, 3000 54.1 against 56.9).
// In the segments both take the same time, and one leaves registers for four
// waves per SIMD.
template <int V>
constexpr int kColTiles = V == 128 ? 2 : 1;
constexpr int kSegTiles = 1;
// Whether each chunk's workgroup steps through those before it by itself (packed
// sequences: nps is of one that had all tokens).  One
// launch of 7 us and 1.7 per chunk stands against three of 15 (4 v-heads) to 18
// us and up to 0.9 per chunk (32 v-heads): 16 -> 32 heads, 256 tokens 13.7 us
// against 22.2, 449 20.7 against 24.4; 8 -> 16, 500 20.1 against 24.4; 16 -> 16,
// 768 26.9 against 24.4; 2 -> 4, 384 16.4 both, 449 19.4 against 16.8; packed, 16
// -> 32, two of 100 tokens 16.1 against 27.0.
inline bool lin_alone(const LinGrid& g, int Hv) {
  return g.nps > 1 && g.L == 1 &&
         (g.nps <= 6 || (g.nps <= 10 && 2LL * g.nseg * Hv >= device_cus()));
}

// ------------------------------------------------------------------ host ----
// Chunks per segment: as many as give every workgroup that the CUs hold one
// segment.
//
// Forward: one workgroup per CU, of a wave per 16 columns, against two of a wave
// per 32 (V = 64: 16), which has fewer contributions to write, join and read, but
// also fewer latencies side by side.  K = V = 128 (us): 20011 tokens of 4
// v-heads, 4.9 chunks per CU, 49.7 against 59.4; of 32 v-heads 1024 tokens, 2 per
// CU, 30.0 and 38.8, 4096, 8 per CU, 67.4 and 71.0, 6000, 12 per CU, 87.0 and
// 88.2, 8192, 16 per CU, 113 and 107.  K = 64, V = 128: 2048 tokens 32.9 and 36.3,
// 4096 50.8 and 50.5, 6000 67.7 and 64.4.  V = 64: 8192 tokens of 4 v-heads, 2 per
// CU, 29.5 and 33.3, 2048 of 32, 4 per CU, 34.0 and 33.5, 3000 43.2 and 40.5.
//
// Backward: a workgroup of the gradients has a CU to itself, or half (K = V = 64),
// and one or two v-heads.  (Training steps in us: 16 -> 16 heads of 128, 4096
// tokens 119, with twice the segments 132; 16 -> 32 of 64, 8192 tokens 153, with
// half 180; 16 -> 32 of 128, 8192 tokens 333, with half 467.)
long long lin_slots(int Hqk, int Hv, int K, int V, bool bwd, bool one) {
  if (bwd) return (long long)device_cus() * (K + V == 128 ? 2 : 1) * (lin_pair(Hqk, Hv) ? 2 : 1);
  return (long long)device_cus() * (one ? 1 : 2);
}
LinPlan lin_plan(int B, int T, int Hqk, int Hv, int K, int V, int N, bool has_cu, bool bwd) {
  LinPlan p{};
  const long long tokens = (long long)B * T;
  const long long per = ((long long)T + kChunk - 1) / kChunk;   // chunks of the longest sequence
  p.chunks = has_cu ? tokens / kChunk + N : B * per;
  p.one = !bwd && p.chunks * Hv < (V == 64 ? 4 : K == 64 ? 8 : 12) * (long long)device_cus();
  const long long slots = lin_slots(Hqk, Hv, K, V, bwd, p.one);
  long long L = (p.chunks * Hv + slots - 1) / slots;
  if (L < 1) L = 1;
  if (L > per) L = per > 0 ? per : 1;
  p.L = (int)L;
  p.nps = (int)(per > 0 ? (per + L - 1) / L : 1);
  p.nseg = (int)(has_cu ? N + tokens / (L * kChunk) : (long long)N * p.nps);
  // a sequence of several segments has more than L chunks
  p.nlong = (int)(p.nps < 2 ? 0 : has_cu ? tokens / (L * kChunk) : N);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  if (has_cu) {
    p.table = take((size_t)p.nseg * sizeof(LinSeg));
    p.status = take(4);
    p.order = take((size_t)p.nseg * 4);
    p.joins = take((size_t)p.nlong * sizeof(LinJoin));
  }
  if (p.nlong > 0) {
    p.segs = take((size_t)p.nseg * Hv * K * V * 4);
    p.decay = take((size_t)p.nseg * Hv * 4);
  }
  const int parts = Hv / Hqk / (lin_pair(Hqk, Hv) ? 2 : 1);
  if (bwd && parts > 1) p.part = take((size_t)tokens * Hqk * parts * K * 8);
  if (bwd) p.dgtok = take((size_t)tokens * Hv * 4);
  p.total = at;
  return p;
}

// Bytes that hold this call and every other of these heads whose B, T and N are
// no larger.  (lin_plan's own need is not monotone: 16 -> 32 heads of 128, 512
// tokens are 8 segments, 576 tokens 5.)  Of n sequences that are cut there are
// at most c = slots / Hv segments more than n less one (packed: c more than n),
// and none is cut where n * Hv reaches the slots (packed: where (chunks + n) *
// Hv / slots reaches the chunks).
size_t lin_bytes(int B, int T, int Hqk, int Hv, int K, int V, int N, bool has_cu, bool bwd) {
  const long long tokens = (long long)B * T, full = T / kChunk;
  const long long per = ((long long)T + kChunk - 1) / kChunk;
  const long long slots = lin_slots(Hqk, Hv, K, V, bwd, false), c = (slots + Hv - 1) / Hv;
  long long rows = 0;   // segments whose states are kept
  size_t at = 0;
  auto take = [&](long long bytes) { at += (size_t)(bytes + 255) / 256 * 256; };
  if (has_cu) {
    const long long more = full < c ? full : c;
    take((N + more) * (long long)sizeof(LinSeg));
    take(4);
    take((N + more) * 4LL);
    take(more * (long long)sizeof(LinJoin));
    const long long most = slots > Hv ? (per - 1) * (slots - Hv) / Hv : 0;
    const long long n = N < most ? N : most;
    rows = n > 0 ? n + more : 0;
  } else if (per > 1) {
    const long long n = N < (slots - 1) / Hv ? N : (slots - 1) / Hv;
    rows = n > 0 ? (n * per < c + n - 1 ? n * per : c + n - 1) : 0;
  }
  take(rows * Hv * K * V * 4);
  take(rows * Hv * 4);
  const int parts = Hv / Hqk / (lin_pair(Hqk, Hv) ? 2 : 1);
  if (bwd && parts > 1) take(tokens * Hqk * parts * K * 8);
  if (bwd) take(tokens * Hv * 4);
  return at;
}

LinGrid lin_grid(const LinPlan& p, unsigned char* ws, int T, int N, int total, bool has_cu) {
  LinGrid g{};
  if (has_cu) {
    g.table = reinterpret_cast<const LinSeg*>(ws + p.table);
    g.status = reinterpret_cast<const int32_t*>(ws + p.status);
    g.order = reinterpret_cast<const int32_t*>(ws + p.order);
    g.joins = reinterpret_cast<const LinJoin*>(ws + p.joins);
  }
  g.T = T;
  g.L = p.L;
  g.nps = p.nps;
  g.one = p.one;
  g.nseg = p.nseg;
  g.nlong = p.nlong;
  g.N = N;
  g.total = total;
  return g;
}

void launch_lin_table(const int32_t* cu, const LinPlan& p, unsigned char* ws, int N, int total,
                      hipStream_t st) {
  hipLaunchKernelGGL(lin_table_kernel, dim3(1), dim3(1024), 0, st, cu,
                     reinterpret_cast<LinSeg*>(ws + p.table),
                     reinterpret_cast<LinJoin*>(ws + p.joins),
                     reinterpret_cast<int32_t*>(ws + p.status),
                     reinterpret_cast<int32_t*>(ws + p.order), N, total, p.L, p.nseg, p.nlong);
}

template <int K, int V>
void launch_lin_segments(const uint16_t* x, int x_row, const uint16_t* y, int y_row,
                         const LinDecay& d, const LinGrid& g, int Hqk, int Hv, float scale,
                         bool reverse, bool full, const float* edge, float* segs, float* decay,
                         float* end, hipStream_t st) {
  const dim3 items((unsigned)lin_items(g.table ? g.nseg : g.N * (g.nps - (end ? 0 : 1)), Hqk, Hv));
  const long long waves = (long long)g.nlong * Hv * (K * V / 256);   // workgroups of one per lane
  const bool four = waves >= 8LL * device_cus();
  const dim3 elems((unsigned)(four ? waves / 4 : waves));
#define GDN_SEG(NP, REV)                                                                        \
  hipLaunchKernelGGL((lin_segment_kernel<K, V, kSegTiles, NP, REV>), items,                     \
                     dim3(4 * V / kSegTiles), 0, st, x, x_row, y, y_row, d, g, Hqk, Hv, scale,  \
                     end != nullptr, segs, decay);                                              \
  if (four)                                                                                     \
    hipLaunchKernelGGL((lin_join_kernel<REV, 4>), elems, dim3(256), 0, st, g, Hv, K * V, edge,   \
                       segs, decay, end);                                                       \
  else                                                                                          \
    hipLaunchKernelGGL((lin_join_kernel<REV, 1>), elems, dim3(256), 0, st, g, Hv, K * V, edge,   \
                       segs, decay, end)
  if (reverse) {
    if (full) { GDN_SEG(3, true); } else { GDN_SEG(2, true); }
  } else {
    if (full) { GDN_SEG(3, false); } else { GDN_SEG(2, false); }
  }
#undef GDN_SEG
}
#define GDN_LS(KK, VV)                                                                        \
  template void launch_lin_segments<KK, VV>(const uint16_t*, int, const uint16_t*, int,       \
                                            const LinDecay&, const LinGrid&, int, int, float, \
                                            bool, bool, const float*, float*, float*, float*,  \
                                            hipStream_t);
GDN_LS(128, 128) GDN_LS(128, 64) GDN_LS(64, 128) GDN_LS(64, 64)
#undef GDN_LS

namespace {
template <int K, int V>
void launch_walk(const uint16_t* q, const uint16_t* k, const uint16_t* v, TokenStride ts,
                 const LinDecay& d, const LinGrid& g, int Hqk, int Hv, float scale,
                 const float* h0, float* ht, float* segs, float* decay, uint16_t* o, u16x4* states,
                 hipStream_t st) {
  // (the saved states have the same bits whether they are formed with o and ht
  // or again)
  const bool full = ht || states;
  // (ht over h0, which the other workgroups still read: they read a copy)
  const bool alone = lin_alone(g, Hv);
  if (alone && ht && ht == h0) {
    const size_t n = (size_t)g.N * Hv * K * V / 4;
    hipLaunchKernelGGL(lin_copy_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st,
                       reinterpret_cast<const f32x4*>(h0), reinterpret_cast<f32x4*>(segs), n);
    h0 = segs;
  }
  if (g.nlong > 0 && !alone) {
    // equal lengths without saved states: the final states come from the segments'
    // contributions, and the walk, for o alone, takes two parts
    const bool end = ht && !states && !g.table;
    launch_lin_segments<K, V>(k, ts.k, v, ts.v, d, g, Hqk, Hv, 1.f, false, full, h0, segs, decay,
                              end ? ht : nullptr, st);
    if (end) ht = nullptr;
  }
  const dim3 items((unsigned)lin_items(g.nseg, Hqk, Hv));
#define GDN_LW(CT, NP, OUT, SAVE, ALONE)                                                     \
  hipLaunchKernelGGL((lin_walk_kernel<K, V, CT, NP, OUT, SAVE, ALONE>), items,               \
                     dim3(4 * V / CT), 0, st, q, k, v, ts, d, g, Hqk, Hv, scale, h0, ht, segs, \
                     o, states)
#define GDN_LWS(CT, ALONE)                         \
  if (o && states) GDN_LW(CT, 3, true, true, ALONE); \
  else if (!o) GDN_LW(CT, 3, false, true, ALONE);  \
  else if (ht) GDN_LW(CT, 3, true, false, ALONE);  \
  else GDN_LW(CT, 2, true, false, ALONE)
  if (alone) {
    GDN_LWS(1, true);
  } else if (g.one) {
    GDN_LWS(1, false);
  } else {
    GDN_LWS(kColTiles<V>, false);
  }
#undef GDN_LWS
#undef GDN_LW
}
}  // namespace

}  // namespace gdn

namespace gdn_host {
int validate_common(const void* q, const void* k, const void* v, const float* g, const float* beta,
                    const float* h0, const float* ht, const void* o, const int32_t* cu, int B,
                    int T, int Hqk, int Hv, int K, int V, int N);
int validate_rows(const char* name, const void* q, const void* k, const void* v, long long q_row,
                  long long k_row, long long v_row, const void* o, long long tokens, int Hqk,
                  int Hv, int K, int V, gdn::TokenStride& ts);

int lin_validate(const char* name, const void* q, const void* k, const void* v, long long q_row,
                 long long k_row, long long v_row, const void* g, int g_dtype, const float* h0,
                 const float* ht, const void* o, const int32_t* cu, int B, int T, int Hqk, int Hv,
                 int K, int V, int N, gdn::TokenStride& ts) {
  const float* gf = static_cast<const float*>(g);
  int rc = validate_common(q, k, v, gf, gf, h0, ht, o, cu, B, T, Hqk, Hv, K, V, N);
  if (rc) return rc;
  if (!gdn::dtype_ok(g_dtype)) return fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported dtype code");
  // (tokens, segments x heads and join workgroups are counted in 32 bits, and so
  // are the bytes of a chunk's rows; the lanes of a launch: lin_lanes)
  const long long tokens = (long long)B * T;
  if (tokens >= (1LL << 31) - 64 || (tokens / 64 + N) * (long long)Hv >= (1LL << 24) * 64 ||
      (long long)N * Hv * (K * V / 256) >= (1LL << 31) || Hv >= (1 << 15))
    return fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  if (tokens > 0)
    return validate_rows(name, q, k, v, q_row, k_row, v_row, o, tokens, Hqk, Hv, K, V, ts);
  ts = gdn::TokenStride{Hqk * K, Hqk * K, Hv * V};
  return GDN_OK;
}
// 16-byte aligned (rows are read and written in vectors).
int lin_aligned(const char* name, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return fail(GDN_ERR_SHAPE, std::string(name) + ": tensors must be 16-byte aligned");
  return GDN_OK;
}
// A launch has under 2^32 lanes in a dimension.
int lin_lanes(const char* name, long long lanes) {
  if (lanes < (1LL << 32)) return GDN_OK;
  return fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large for one launch");
}
bool lin_sizes_ok(int B, int T, int Hqk, int Hv, int K, int V, int N) {
  return B >= 0 && T >= 0 && Hqk > 0 && Hv > 0 && Hv % Hqk == 0 && N >= 0 &&
         (K == 64 || K == 128) && (V == 64 || V == 128);
}
}  // namespace gdn_host

extern "C" size_t gdn_linear_chunk_workspace_bytes(int B, int T, int Hqk, int Hv, int K, int V,
                                                   int N, int has_cu_seqlens) {
  if (!gdn_host::lin_sizes_ok(B, T, Hqk, Hv, K, V, N)) return 0;
  return gdn::lin_bytes(B, T, Hqk, Hv, K, V, N, has_cu_seqlens != 0, false);
}

extern "C" size_t gdn_linear_states_bytes(int B, int T, int Hv, int K, int V, int N,
                                          int has_cu_seqlens) {
  if (!gdn_host::lin_sizes_ok(B, T, Hv, Hv, K, V, N)) return 0;
  return (size_t)gdn::lin_plan(B, T, Hv, Hv, K, V, N, has_cu_seqlens != 0, false).chunks * Hv * K *
         V * 2;
}

extern "C" int gdn_linear_chunk_fwd(const void* q, const void* k, const void* v, long long q_row,
                                    long long k_row, long long v_row, const void* g, int g_dtype,
                                    int g_per_head, const float* h0, float* ht, void* o,
                                    const int32_t* cu_seqlens, int B, int T, int Hqk, int Hv,
                                    int K, int V, int N, float scale, void* states,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "gdn_linear_chunk_fwd";
  gdn::TokenStride ts;
  // (without o its checks look at the states, which are larger)
  int rc = gdn_host::lin_validate(name, q, k, v, q_row, k_row, v_row, g, g_dtype, h0, ht,
                                  o ? o : states, cu_seqlens, B, T, Hqk, Hv, K, V, N, ts);
  if (!rc) rc = gdn_host::lin_aligned(name, {o, h0, ht, states, workspace});
  if (rc) return rc;
  const bool has_cu = cu_seqlens != nullptr;
  const gdn::LinPlan p = gdn::lin_plan(B, T, Hqk, Hv, K, V, N, has_cu, false);
  rc = gdn_host::lin_lanes(name, gdn::lin_items(p.nseg, Hqk, Hv) * (p.nlong > 0 || p.one ? 4 * V : 256));
  if (rc) return rc;
  if (p.total > 0 && (!workspace || workspace_bytes < p.total))
    return gdn_host::fail(GDN_ERR_WORKSPACE, std::string(name) + ": workspace needs " +
                                                 std::to_string(p.total) + " bytes, got " +
                                                 std::to_string(workspace_bytes));
  if (N == 0 || ((long long)B * T == 0 && !ht)) return GDN_OK;
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  const gdn::LinGrid grid = gdn::lin_grid(p, ws, T, N, B * T, has_cu);
  if (has_cu) gdn::launch_lin_table(cu_seqlens, p, ws, N, B * T, st);
  const gdn::LinDecay d{g, g_dtype, g_per_head ? 0 : Hv};
  auto* segs = reinterpret_cast<float*>(ws + p.segs);
  auto* decay = reinterpret_cast<float*>(ws + p.decay);
#define GDN_LIN(KK, VV)                                                                        \
  if (K == KK && V == VV) {                                                                    \
    gdn::launch_walk<KK, VV>(static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), \
                             static_cast<const uint16_t*>(v), ts, d, grid, Hqk, Hv, scale, h0, \
                             ht, segs, decay, static_cast<uint16_t*>(o),                       \
                             static_cast<gdn::u16x4*>(states), st);                            \
    return gdn_host::check_launch(name);                                                       \
  }
  GDN_LIN(128, 128) GDN_LIN(128, 64) GDN_LIN(64, 128) GDN_LIN(64, 64)
#undef GDN_LIN
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported K/V");
}
