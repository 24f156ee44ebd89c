// Backward of linear attention's chunked form for gfx950 (declared in
// gdn_linear.h).  With S the state at a chunk's start (saved by the forward),
// D the gradient of the state at its end, G and R as in the forward and
// gamma_ij = scale e^{G_i - G_j} (j <= i):
//     P_ij = gamma_ij (q_i . k_j)      dP_ij = gamma_ij (do_i . v_j)
//     dv_j = sum_i P_ij do_i + e^{R_j} D^T k_j
//     dk_j = sum_i dP_ij q_i + e^{R_j} D v_j
//     dq_i = sum_j dP_ij k_j + scale e^{G_i} S do_i
//     D'   = e^{G_63} D + sum_i q_i (scale e^{G_i} do_i)^T
// and, from the parts a_i = q_i . (S's part of dq_i), b_j = k_j . (D's part of
// dk_j), M_ij = P_ij (do_i . v_j),
//     dg_t = e^{G_63} <S, D> + sum_{i >= t} a_i + sum_{j < t} b_j
//            + sum_{i >= t > j} M_ij,
// the last as row sums less column sums of the same fp32 numbers, so nothing
// but their own rounding is lost where it cancels: dg of a head whose memory
// is short is as good as that of a long one.  The saved states enter dq and dg
// whole (they are two bf16 parts), D in two parts.
//
// Segments as in the forward, walked last chunk to first: a launch for every
// segment's contribution to D, one that joins them, one for the gradients.
#include <initializer_list>
#include <type_traits>

#include "gdn_linear.h"
#include "../../include/gdn_linear.h"

namespace gdn {

struct LinBwdArgs {
  const uint16_t *q, *k, *v, *dO;
  TokenStride ts;
  LinDecay dec;
  LinGrid grid;
  int Hqk, Hv;
  float scale;
  const float* dht;
  float* dh0;
  const float* segs;
  const u16x8* states;   // lin_pack's
  uint16_t *dq, *dk, *dv;
  float *pq, *pk;      // [tokens][Hv / HP][K] partial dq, dk (NULL: none needed)
  void* dg;            // [tokens][Hv], of type dgt
  int dgt;
};

__device__ __forceinline__ void lin_put(void* p, size_t i, float x, int dt) {
  if (dt == GDN_DTYPE_F32) ste<GDN_DTYPE_F32>(p, i, x);
  else if (dt == GDN_DTYPE_BF16) ste<GDN_DTYPE_BF16>(p, i, x);
  else ste<GDN_DTYPE_F16>(p, i, x);
}

template <int K, int V>
struct LinGradLds {
  char qs[LinTile<K>::BYTES], ks[LinTile<K>::BYTES];
  char vs[LinTile<V>::BYTES], os[LinTile<V>::BYTES];
  char ps[LinTile<64>::BYTES], dps[LinTile<64>::BYTES];
  char pd[4][512], dpd[4][512];   // what bf16 leaves of their tiles on the diagonal, rows of 16
  char ds[2][2 * V * K];          // D^T in two bf16 parts, rows of K
  float sG[64], sQ[64], sK[64];   // G log2(e), scale e^G, e^R
  // (slots that their writers own and the reader adds up: M's row sums by source
  // block and pair of lane groups, its column sums by token block; a and b by wave
  // and group)
  float rowM[8][64], colM[4][64], asum[K / 8][64], bsum[K / 8][64];
  float csum[K / 32];
};

// What one wave of lin_grad_kernel does (see there).
template <int K, int V, int HP, int NP, bool VW>
__device__ __forceinline__ void lin_grad_walk(const LinBwdArgs& a, const LinSeg& sg, int sid, int hp,
                                              int w, LinGradLds<K, V>& lds) {
  constexpr int NT = 2 * (K + V), NV = V / 32, NK = K / 32;
  // who brings the tiles in: with four waves of each kind the key waves (two
  // heads' D leave the V waves few registers), but q the V waves; else all
  constexpr bool SPLIT = NK == 4 && NV == 4, KEYS = NK == 4 && NV == 2;
  constexpr bool BRINGS = !SPLIT && (!KEYS || !VW);   // all of them
  constexpr int NS = SPLIT || KEYS ? 256 : NT;
  char *qs = lds.qs, *ks = lds.ks, *vs = lds.vs, *os = lds.os, *ps = lds.ps, *dps = lds.dps;
  char *ds = lds.ds[0], *dl = lds.ds[1];
  float *sG = lds.sG, *sQ = lds.sQ, *sK = lds.sK;
  const int tid = threadIdx.x, lane = tid % 64;
  const int h0 = hp * HP, hq = h0 / (a.Hv / a.Hqk);
  const int nc = (sg.ntok + kChunk - 1) / kChunk;
  const int wk = VW ? 0 : w - NV, wv = VW ? w : 0;   // the wave's 32 columns

  // V waves: D of each head, rows (keys) 16 t + 4 grp + r, columns 32 wv + 16 T + r16
  f32x4 ST[HP][K / 16][2];
  auto state_at = [&](int lane, int T) {
    return (4 * (lane / 16) * V + 32 * wv + 16 * T + lane % 16) * 4;
  };
  if constexpr (VW) {
#pragma unroll
    for (int hh = 0; hh < HP; ++hh) {
      const int h = h0 + hh;
      const float* src =
          sg.first && sg.last ? (a.dht ? a.dht + ((size_t)sg.seq * a.Hv + h) * K * V : nullptr)
                              : a.segs + ((size_t)sid * a.Hv + h) * K * V;
      const __amdgpu_buffer_rsrc_t rst = lin_state(src, K * V);
#pragma unroll
      for (int t = 0; t < K / 16; ++t)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            ST[hh][t][T][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                rst, state_at(lane, T), (16 * t + r) * V * 4, 0));
    }
  }

  LinStage<K, NS> sq, sk;
  LinStage<V, NS> sv, so;
  LinGates lg;
  const int st = (SPLIT || KEYS) && !VW ? tid - 64 * NV : tid;
  int gi = LinGates::token(w, lane);
  int qf = LinStage<K, NS>::from(a.ts.q, st), kf = LinStage<K, NS>::from(a.ts.k, st);
  int vf = LinStage<V, NS>::from(a.ts.v, st), of = LinStage<V, NS>::from(a.Hv * V, st);
  const int kt = LinStage<K, NS>::at(st, 0), vt = LinStage<V, NS>::at(st, 0);
  auto load = [&](int c, int hh) {
    const int n = c >= 0 ? sg.ntok - c * kChunk : 0, h = h0 + hh;
    const size_t t = n > 0 ? (size_t)sg.tok0 + c * kChunk : 0;
    if (w < 2) lg.load(a.dec, t, min(n, 64), h, a.Hv, gi);
    if (hh == 0) {
      if (BRINGS || (SPLIT && VW)) sq.load(a.q + t * a.ts.q + hq * K, a.ts.q, min(n, 64), qf);
      if (BRINGS || (SPLIT && !VW)) sk.load(a.k + t * a.ts.k + hq * K, a.ts.k, min(n, 64), kf);
    }
    if (BRINGS || (SPLIT && !VW)) {
      sv.load(a.v + t * a.ts.v + h * V, a.ts.v, min(n, 64), vf);
      so.load(a.dO + (t * a.Hv + h) * V, a.Hv * V, min(n, 64), of);
    }
  };
  // the tiles above the diagonal that share a 32-wide block with it, and the
  // sums that no tile writes
  for (int i = tid; i < 64; i += NT) {
    const int r = i / 2 % 16 + (i / 32) * 32, u = 4 * (i / 32) + 2 + i % 2;
    *reinterpret_cast<u32x4*>(ps + LinTile<64>::off(r, u)) = u32x4{0, 0, 0, 0};
    *reinterpret_cast<u32x4*>(dps + LinTile<64>::off(r, u)) = u32x4{0, 0, 0, 0};
  }
  for (int i = tid; i < 512; i += NT) lds.rowM[i / 64][i % 64] = 0.f;
  for (int i = tid; i < 256; i += NT) lds.colM[i / 64][i % 64] = 0.f;
  __syncthreads();

  // A chunk's gradients leave ahead of the loads issued after it: the wait for
  // loads counts stores too.
  f32x4 X[4][2], Y[4][2];   // dv; or dk and dq, over the heads (by token tile)
  auto store_grads = [&](int c, int h) {
    int ln = lane;
    hide(ln);
    const int r16 = ln % 16, grp = ln / 16;
    const int n = min(sg.ntok - c * kChunk, 64);
    const size_t tok = (size_t)sg.tok0 + c * kChunk;
    // columns 16 T + 4 grp + r of the wave's 32, token 16 tt + r16 (stores past
    // the segment's last token are dropped)
    auto put = [&](void* p, int heads, int hd, int es, int width, const f32x4 (&x)[4][2]) {
      const int row = heads * width * es, at = r16 * row + (32 * (VW ? wv : wk) + 4 * grp) * es;
      const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc(
          static_cast<char*>(p) + (tok * heads + hd) * width * es, 0, (n - 1) * row + width * es,
          kBufferFlags);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          if (es == 4)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x[tt][T]), rd,
                                                   at + tt * 16 * row + 64 * T, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2p, f2bf4(x[tt][T])), rd,
                                                  at + tt * 16 * row + 32 * T, 0, 0);
        }
    };
    if constexpr (VW) {
      put(a.dv, a.Hv, h, 2, V, X);
    } else if (a.pq) {
      put(a.pq, a.Hv / HP, hp, 4, K, Y);
      put(a.pk, a.Hv / HP, hp, 4, K, X);
    } else {
      put(a.dq, a.Hqk, hq, 2, K, Y);
      put(a.dk, a.Hqk, hq, 2, K, X);
    }
  };
  // key waves: the saved state's fragments of their keys, an iteration ahead
  u16x8 SF[2][V / 32];
  auto load_states = [&](int c, int hh) {
    const u16x8* sp = a.states + (((size_t)(sg.chunk0 + max(c, 0)) * a.Hv + h0 + hh) * (K / 16) +
                                  2 * wk) * (V / 32) * 64 + lane;
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int b = 0; b < V / 32; ++b) SF[T][b] = sp[(T * (V / 32) + b) * 64];
  };
  auto zero = [](f32x4 (&x)[4][2]) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) x[tt][0] = x[tt][1] = zero4();
  };

  auto iterate = [&](int c, auto head) {
    constexpr int hh = decltype(head)::value;
    const int h = h0 + hh;
    // (nothing derived from these is kept from one iteration for the next)
    int ln = lane;
    hide(ln);
    const int lane = ln, r16 = ln % 16, grp = ln / 16;
    const int krb = LinTile<K>::row_base(lane), vrb = LinTile<V>::row_base(lane);
    const int kr4 = LinTile<K>::row4_base(lane), vr4 = LinTile<V>::row4_base(lane);
    const int kcb = LinTile<K>::col_base(0, lane), vcb = LinTile<V>::col_base(0, lane);
    const int pb = LinTile<64>::row_base(lane), pcb = LinTile<64>::col_base(0, lane);
    const int pw = LinTile<64>::off(r16, grp >> 1) + (grp & 1) * 8;
    const int dcb = LinTile<K>::col4_base(2 * wk, lane);   // key waves: D^T read
    const int dwb = kr4 + 32 * wv * 2 * K;                 // V waves: D^T written
    const int kc4 = LinTile<K>::col4_base(0, lane), vc4 = LinTile<V>::col4_base(0, lane);
    const int dtr = (4 * grp + (r16 >> 2)) * 32 + (r16 & 3) * 8;   // pd, dpd transposed
    hide(qf);
    hide(kf);
    hide(vf);
    hide(of);
    hide(gi);
    if (hh == 0) {
      if (BRINGS || (SPLIT && VW)) sq.store(qs, kt, st);
      if (BRINGS || (SPLIT && !VW)) sk.store(ks, kt, st);
    }
    if (BRINGS || (SPLIT && !VW)) {
      sv.store(vs, vt, st);
      so.store(os, vt, st);
    }
    if (w < 2) {
      const float pre = lg.prefix(a.dec, gi) * kLog2e, e = exp2_(pre);
      if (w == 1) {
        sK[63 - lane] = e;
      } else {
        sG[lane] = pre;
        sQ[lane] = a.scale * e;
      }
    }
    if constexpr (VW) {
#pragma unroll
      for (int t = 0; t < K / 16; ++t)
#pragma unroll
        for (int T = 0; T < 2; ++T)
        {
          u16x4 hi, lo;
          split_bf4(ST[hh][t][T], hi, lo);
          *reinterpret_cast<u16x4*>(ds + (dwb ^ (32 * t)) + T * 16 * 2 * K) = hi;
          *reinterpret_cast<u16x4*>(dl + (dwb ^ (32 * t)) + T * 16 * 2 * K) = lo;
        }
    }
    __syncthreads();
    if (VW ? c < nc - 1 || hh > 0 : c < nc - 1 && hh == 0)
      store_grads(hh > 0 ? c : c + 1, VW ? (hh > 0 ? h - 1 : h0 + HP - 1) : h0);
    // the next iteration's tiles: on their way through the products behind the
    // next barrier alone, long enough (from the start of the iteration on they
    // took 48 registers, which two heads' gradients do not leave: scratch)
    auto load_next = [&]() {
      if (hh + 1 < HP) load(c, hh + 1);
      else load(c - 1, 0);
    };
    const float eC = exp2_(sG[63]);
    if constexpr (VW) {
      // dv's part of D, then D of the chunk before
      zero(X);
#pragma unroll
      for (int b = 0; b < K / 32; ++b) {
        // (both parts as they lie in LDS for the key waves: formed again they take
        // registers that two heads' D does not leave, 212 us against 207)
        u16x8 df[2], dlo[2];
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          df[T] = LinTile<K>::rows4(ds, kr4, 2 * wv + T, b);
          dlo[T] = LinTile<K>::rows4(dl, kr4, 2 * wv + T, b);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const u16x8 f = LinTile<K>::rows4(ks, kr4, tt, b);
#pragma unroll
          for (int T = 0; T < 2; ++T) X[tt][T] = mfma16(dlo[T], f, mfma16(df[T], f, X[tt][T]));
        }
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float f = sK[16 * tt + r16];
        X[tt][0] *= f;
        X[tt][1] *= f;
      }
#pragma unroll
      for (int t = 0; t < K / 16; ++t) {
        ST[hh][t][0] *= eC;
        ST[hh][t][1] *= eC;
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        u16x8 part[2][NP];
#pragma unroll
        for (int T = 0; T < 2; ++T)
          lin_split(LinTile<V>::cols(os, vcb, kb, 2 * wv + T), sQ + 32 * kb + 8 * grp, part[T]);
#pragma unroll
        for (int t = 0; t < K / 16; ++t) {
          const u16x8 f = LinTile<K>::cols(qs, kcb, kb, t);
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int T = 0; T < 2; ++T) ST[hh][t][T] = mfma16(f, part[T][p], ST[hh][t][T]);
        }
      }
      load_next();
    } else {
      // P and dP, tile by tile, as bf16 rows, what these leave of the tiles on the
      // diagonal, and the sums of M
      for (int m = wk; m < 10; m += NK) {
        const int it = tmat_block_row(m), jt = m - tmat_block(it, 0);
        f32x4 p = zero4(), d = zero4();
#pragma unroll
        for (int kb = 0; kb < K / 32; ++kb)
          p = mfma16(LinTile<K>::rows(ks, krb, jt, kb), LinTile<K>::rows(qs, krb, it, kb), p);
#pragma unroll
        for (int kb = 0; kb < V / 32; ++kb)
          d = mfma16(LinTile<V>::rows(vs, vrb, jt, kb), LinTile<V>::rows(os, vrb, it, kb), d);
        const int i = 16 * it + r16, j = 16 * jt + 4 * grp;
        const f32x4 gj = *reinterpret_cast<const f32x4*>(&sG[j]);
        const float gi = sG[i];
        f32x4 M;
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = j + r <= i;
          const float gam = a.scale * exp2_(in ? gi - gj[r] : 0.f);
          d[r] = in ? d[r] : 0.f;
          p[r] = (in ? p[r] : 0.f) * gam;
          M[r] = p[r] * d[r];
          d[r] *= gam;
          rs += M[r];
        }
        u16x4 ph, pl, dh, dl;
        split_bf4(p, ph, pl);
        split_bf4(d, dh, dl);
        *reinterpret_cast<u16x4*>(ps + (pw ^ (32 * jt)) + it * 2048) = ph;
        *reinterpret_cast<u16x4*>(dps + (pw ^ (32 * jt)) + it * 2048) = dh;
        if (it == jt) {
          *reinterpret_cast<u16x4*>(lds.pd[it] + r16 * 32 + grp * 8) = pl;
          *reinterpret_cast<u16x4*>(lds.dpd[it] + r16 * 32 + grp * 8) = dl;
        }
        rs += __shfl_xor(rs, 16);
        if (grp % 2 == 0) lds.rowM[2 * jt + grp / 2][i] = rs;
#pragma unroll
        for (int r = 0; r < 4; ++r) M[r] = row16_sum(M[r]);
        if (r16 == 15) *reinterpret_cast<f32x4*>(&lds.colM[it][j]) = M;
      }
      if (hh == 0) {
        zero(X);
        zero(Y);
      }
      // the parts of dk from D and of dq from S: products, then the tokens' factors
      auto inter = [&](f32x4 (&out)[4][2], const float* fac, const char* own, auto sums,
                       auto&& op, auto&& rows) {
        f32x4 Z[4][2];
        zero(Z);
#pragma unroll
        for (int b = 0; b < V / 32; ++b) {
          u16x8 f[2][2];
#pragma unroll
          for (int T = 0; T < 2; ++T) op(T, b, f[T]);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            const u16x8 x = rows(tt, b);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int T = 0; T < 2; ++T) Z[tt][T] = mfma16(f[T][p], x, Z[tt][T]);
          }
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int i = 16 * tt + r16;
          const float e = fac[i];
          float s = 0.f;
#pragma unroll
          for (int T = 0; T < 2; ++T) {
            Z[tt][T] *= e;
            out[tt][T] += Z[tt][T];
            const u16x4 x = *reinterpret_cast<const u16x4*>(
                own + LinTile<K>::off(i, 4 * wk + 2 * T + (grp >> 1)) + (grp & 1) * 8);
#pragma unroll
            for (int r = 0; r < 4; ++r) s += bf2f(x[r]) * Z[tt][T][r];
          }
          sums[4 * wk + grp][i] = s;
        }
      };
      inter(X, sK, ks, lds.bsum,
            [&](int T, int b, u16x8 (&out)[2]) {
              out[0] = LinTile<K>::cols4(ds, dcb, b, T);
              out[1] = LinTile<K>::cols4(dl, dcb, b, T);
            },
            [&](int tt, int b) { return LinTile<V>::rows4(vs, vr4, tt, b); });
      // both parts of S and of D: <S, D>, a and b are sums of random signs in dg,
      // which show every rounding in full.  <S, D> of 16 keys is the trace of a
      // product of fragments.
      f32x4 SD = zero4();
      inter(Y, sQ, qs, lds.asum,
            [&](int T, int b, u16x8 (&out)[2]) {
              u16x4 h0, h1, l0, l1;
              split_bf4(lin_unpack(u16x4{SF[T][b][0], SF[T][b][1], SF[T][b][2], SF[T][b][3]}), h0, l0);
              split_bf4(lin_unpack(u16x4{SF[T][b][4], SF[T][b][5], SF[T][b][6], SF[T][b][7]}), h1, l1);
              out[0] = cat8(h0, h1);
              out[1] = cat8(l0, l1);
              const u16x8 f = LinTile<K>::cols4(ds, dcb, b, T);
              SD = mfma16(f, out[0], SD);
              SD = mfma16(f, out[1], SD);
              SD = mfma16(LinTile<K>::cols4(dl, dcb, b, T), out[0], SD);
            },
            [&](int tt, int b) { return LinTile<V>::rows4(os, vr4, tt, b); });
      float cs = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) cs += 4 * grp + r == r16 ? SD[r] : 0.f;
      load_next();
      if (hh + 1 < HP) load_states(c, hh + 1);
      else load_states(c - 1, 0);
      cs = wave_prefix(cs);
      if (lane == 63) lds.csum[wk] = cs;
    }
    __syncthreads();   // P, dP and the sums

    if (VW && w == 0) {
      float x = 0.f, y = 0.f, cs = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) x += lds.rowM[u][lane];
#pragma unroll
      for (int u = 0; u < 4; ++u) x -= lds.colM[u][lane];
#pragma unroll
      for (int u = 0; u < 4 * NK; ++u) {
        x += lds.asum[u][lane];
        y += lds.bsum[u][lane];
      }
#pragma unroll
      for (int u = 0; u < NK; ++u) cs += lds.csum[u];
      // prefix sums of y before the token, and of x from it on (the total less
      // what is before it)
      const float px = wave_prefix(x);
      const float dg = eC * cs + (lane63(px) - px + x) + (wave_prefix(y) - y);
      const int n = sg.ntok - c * kChunk;
      if (lane < n) lin_put(a.dg, ((size_t)sg.tok0 + c * kChunk + lane) * a.Hv + h, dg, a.dgt);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      u16x8 f[2];
#pragma unroll
      for (int T = 0; T < 2; ++T)
        f[T] = VW ? LinTile<V>::cols(os, vcb, kb, 2 * wv + T) : LinTile<K>::cols(qs, kcb, kb, 2 * wk + T);
#pragma unroll
      for (int tt = 0; tt < 2 * kb + 2; ++tt) {
        const u16x8 pf = LinTile<64>::cols(VW ? ps : dps, pcb, kb, tt);
#pragma unroll
        for (int T = 0; T < 2; ++T) X[tt][T] = mfma16(f[T], pf, X[tt][T]);
      }
      // what bf16 leaves of P's (dP's) diagonal tiles: where a gradient is a few
      // tokens' sum their rounding is the same for all of its columns and shows in
      // full
      auto diagonal = [&](f32x4 (&out)[4][2], auto&& columns, auto&& tile) {
        const u16x4 none = {0, 0, 0, 0};
        const u16x8 x0 = columns(0), x1 = columns(1);
#pragma unroll
        for (int t = 2 * kb; t < 2 * kb + 2; ++t) {
          const u16x4 lo = tile(t);
          const u16x8 y = t % 2 ? cat8(none, lo) : cat8(lo, none);
          out[t][0] = mfma16(x0, y, out[t][0]);
          out[t][1] = mfma16(x1, y, out[t][1]);
        }
      };
      diagonal(X, [&](int T) { return VW ? LinTile<V>::cols4(os, vc4, kb, 2 * wv + T)
                                         : LinTile<K>::cols4(qs, kc4, kb, 2 * wk + T); },
               [&](int t) { return lds_tr16(reinterpret_cast<const uint16_t*>((VW ? lds.pd : lds.dpd)[t] + dtr)); });
      if constexpr (!VW)
        diagonal(Y, [&](int T) { return LinTile<K>::cols4(ks, kc4, kb, 2 * wk + T); },
                 [&](int t) { return *reinterpret_cast<const u16x4*>(lds.dpd[t] + r16 * 32 + grp * 8); });
      if constexpr (!VW) {
#pragma unroll
        for (int T = 0; T < 2; ++T) f[T] = LinTile<K>::cols(ks, kcb, kb, 2 * wk + T);
#pragma unroll
        for (int tt = 2 * kb; tt < 4; ++tt) {
          const u16x8 pf = LinTile<64>::rows(dps, pb, tt, kb);
#pragma unroll
          for (int T = 0; T < 2; ++T) Y[tt][T] = mfma16(f[T], pf, Y[tt][T]);
        }
      }
    }
    __syncthreads();
  };

  if constexpr (!VW) {
    if (nc > 0) load_states(nc - 1, 0);
  }
  load(nc - 1, 0);
  for (int c = nc - 1; c >= 0; --c) {
    iterate(c, std::integral_constant<int, 0>{});
    if constexpr (HP == 2) iterate(c, std::integral_constant<int, 1>{});
  }
  if (nc > 0) store_grads(0, VW ? h0 + HP - 1 : h0);
  if constexpr (VW) {
    if (a.dh0 && sg.first) {
#pragma unroll
      for (int hh = 0; hh < HP; ++hh) {
        const __amdgpu_buffer_rsrc_t rd =
            lin_state(a.dh0 + ((size_t)sg.seq * a.Hv + h0 + hh) * K * V, K * V);
#pragma unroll
        for (int t = 0; t < K / 16; ++t)
#pragma unroll
          for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(ST[hh][t][T][r]), rd,
                                                    state_at(lane, T), (16 * t + r) * V * 4, 0);
      }
    }
  }
}

// A workgroup walks one segment of HP v-heads of one qk-head, chunk by chunk
// and in each chunk head by head: q and k are staged once, dk and dq add up
// over the heads in registers.  V / 32 waves own 32 columns of every D (dv,
// dh0) and leave it in LDS, in two bf16 parts, for the K / 32 waves that own 32 key columns
// (dk, dq, P, dP and with the saved states' fragments <S, D>, all of which
// reduce over V).  NP: the parts of dO's products on the way to dh0 (three
// where it is wanted).  8192 tokens, 16 -> 32 heads: 188 us (178 at the highest
// clock) for 403 MB read and written at least (one head at a time, with fp32 parts of
// dq and dk summed by a launch of their own, 226 + 59 where two at a time took 175).
// Bound by latencies: registers (up to 256, none in scratch) and LDS (160 KiB)
// leave one workgroup, two waves per SIMD, whose waves wait half of their time,
// at three barriers per head and chunk and for LDS; MFMA is busy a quarter of it.
template <int K, int V, int HP, int NP>
__global__ __launch_bounds__(2 * (K + V), 2) void lin_grad_kernel(LinBwdArgs a) {
  constexpr int NT = 2 * (K + V);
  __shared__ __align__(16) LinGradLds<K, V> lds;
  if (a.grid.table && *a.grid.status) {
    // a cu_seqlens violation: every gradient over the tokens is zero
    const size_t nv = (size_t)a.grid.total * a.Hv * V / 8, nk = (size_t)a.grid.total * a.Hqk * K / 8;
    const size_t ng = (size_t)a.grid.total * a.Hv, st = (size_t)gridDim.x * NT;
    const size_t i0 = (size_t)blockIdx.x * NT + threadIdx.x;
    for (size_t i = i0; i < nv; i += st) reinterpret_cast<u32x4*>(a.dv)[i] = u32x4{0, 0, 0, 0};
    for (size_t i = i0; i < nk; i += st) {
      reinterpret_cast<u32x4*>(a.dq)[i] = u32x4{0, 0, 0, 0};
      reinterpret_cast<u32x4*>(a.dk)[i] = u32x4{0, 0, 0, 0};
    }
    for (size_t i = i0; i < ng; i += st) lin_put(a.dg, i, 0.f, a.dgt);
  }
  int sid, hp;
  if (!lin_item(a.grid, a.grid.nseg, a.Hqk, a.Hv / HP, sid, hp)) return;
  if (a.grid.table) sid = a.grid.order[sid];
  const LinSeg sg = lin_seg(a.grid, sid);
  if (sg.seq < 0) return;
  const int w = wave_index();
  if (w < V / 32) lin_grad_walk<K, V, HP, NP, true>(a, sg, sid, hp, w, lds);
  else lin_grad_walk<K, V, HP, NP, false>(a, sg, sid, hp, w, lds);
}

// dq, dk of a qk-head: the sum of its rep parts, 8 elements per lane.
__global__ __launch_bounds__(256) void lin_group_sum_kernel(const float* __restrict__ pq,
                                                            const float* __restrict__ pk,
                                                            uint16_t* __restrict__ dq,
                                                            uint16_t* __restrict__ dk,
                                                            const int32_t* status, long long rows,
                                                            int rep, int K) {
  const long long u = (long long)blockIdx.x * 256 + threadIdx.x;
  if (u * 8 >= rows * K) return;
  const long long row = u * 8 / K;
  const int c = u * 8 % K;
  const float* p = blockIdx.y ? pk : pq;
  f32x4 s0 = zero4(), s1 = zero4();
  if (!status || !*status) {
    for (int r = 0; r < rep; ++r) {
      const f32x4* x = reinterpret_cast<const f32x4*>(p + (row * rep + r) * K + c);
      s0 += x[0];
      s1 += x[1];
    }
  }
  *reinterpret_cast<u16x8*>((blockIdx.y ? dk : dq) + u * 8) = cat8(f2bf4(s0), f2bf4(s1));
}

// One decay per head: its gradient, the sum over all tokens (a workgroup per
// head, a fixed order).
__global__ __launch_bounds__(1024) void lin_head_sum_kernel(const float* __restrict__ x,
                                                            void* __restrict__ out, int tokens,
                                                            int Hv, int dt) {
  __shared__ float red[16];
  float s = 0.f;
#pragma unroll 4
  for (int t = threadIdx.x; t < tokens; t += 1024) s += x[(size_t)t * Hv + blockIdx.x];
#pragma unroll
  for (int o = 1; o < 64; o *= 2) s += __shfl_xor(s, o);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i];
    lin_put(out, blockIdx.x, s, dt);
  }
}

namespace {
template <int K, int V>
void launch_grad(const LinBwdArgs& a, float* segs, float* decay, hipStream_t st) {
  if (a.grid.nlong > 0)
    launch_lin_segments<K, V>(a.q, a.ts.q, a.dO, a.Hv * V, a.dec, a.grid, a.Hqk, a.Hv, a.scale,
                              true, a.dh0 != nullptr, a.dht, segs, decay, nullptr, st);
#define GDN_LG(HP, NP)                                                                       \
  hipLaunchKernelGGL((lin_grad_kernel<K, V, HP, NP>),                                        \
                     dim3((unsigned)lin_items(a.grid.nseg, a.Hqk, a.Hv / HP)), dim3(2 * (K + V)), 0, st, a)
  if (lin_pair(a.Hqk, a.Hv)) {
    if (a.dh0) GDN_LG(2, 3);
    else GDN_LG(2, 2);
  } else {
    if (a.dh0) GDN_LG(1, 3);
    else GDN_LG(1, 2);
  }
#undef GDN_LG
}
}  // namespace

}  // namespace gdn

namespace gdn_host {
int lin_validate(const char* name, const void* q, const void* k, const void* v, long long q_row,
                 long long k_row, long long v_row, const void* g, int g_dtype, const float* h0,
                 const float* ht, const void* o, const int32_t* cu, int B, int T, int Hqk, int Hv,
                 int K, int V, int N, gdn::TokenStride& ts);
bool lin_sizes_ok(int B, int T, int Hqk, int Hv, int K, int V, int N);
int lin_lanes(const char* name, long long lanes);
int lin_aligned(const char* name, std::initializer_list<const void*> ptrs);
}  // namespace gdn_host

extern "C" size_t gdn_linear_chunk_bwd_workspace_bytes(int B, int T, int Hqk, int Hv, int K, int V,
                                                       int N, int has_cu_seqlens) {
  if (!gdn_host::lin_sizes_ok(B, T, Hqk, Hv, K, V, N)) return 0;
  return gdn::lin_bytes(B, T, Hqk, Hv, K, V, N, has_cu_seqlens != 0, true);
}

extern "C" int gdn_linear_chunk_bwd(const void* q, const void* k, const void* v, long long q_row,
                                    long long k_row, long long v_row, const void* g, int g_dtype,
                                    int g_per_head, const void* dO, const float* dht,
                                    const void* states, void* dq, void* dk, void* dv, void* dg,
                                    float* dh0, const int32_t* cu_seqlens, int B, int T, int Hqk,
                                    int Hv, int K, int V, int N, float scale, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* name = "gdn_linear_chunk_bwd";
  gdn::TokenStride ts;
  int rc = gdn_host::lin_validate(name, q, k, v, q_row, k_row, v_row, g, g_dtype, dht, dh0, dv,
                                  cu_seqlens, B, T, Hqk, Hv, K, V, N, ts);
  if (!rc) rc = gdn_host::lin_aligned(name, {dO, dht, states, dq, dk, dv, dh0, workspace});
  if (rc) return rc;
  const long long tokens = (long long)B * T;
  if ((tokens > 0 && (!dO || !states || !dq || !dk)) || ((tokens > 0 || g_per_head) && !dg))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": dO, states, dq, dk and dg must be non-NULL");
  // the gradients leave while the inputs (whole rows where they are slices) are read
  auto span = [&](int row, int width) { return tokens > 0 ? (size_t)((tokens - 1) * row + width) * 2 : 0; };
  const int es = g_dtype == GDN_DTYPE_F32 ? 4 : 2;
  const size_t nqk = (size_t)tokens * Hqk * K * 2, nvo = (size_t)tokens * Hv * V * 2;
  const size_t ng = (size_t)(g_per_head ? 1 : tokens) * Hv * es, nst = (size_t)N * Hv * K * V * 4;
  const void* in[] = {q, k, v, g, dO, states, cu_seqlens};
  const size_t nin[] = {span(ts.q, Hqk * K), span(ts.k, Hqk * K), span(ts.v, Hv * V), ng, nvo,
                        gdn_linear_states_bytes(B, T, Hv, K, V, N, cu_seqlens != nullptr), (N + 1) * 4ull};
  const void* out[] = {dq, dk, dv, dg, dh0};
  const size_t nout[] = {nqk, nqk, nvo, ng, nst};
  auto meet = [](const void* a, size_t na, const void* b, size_t nb) {
    return a && b && na && nb && gdn_host::overlaps(a, na, b, nb);
  };
  for (int i = 0; i < 5; ++i) {
    bool bad = i < 4 && meet(out[i], nout[i], dht, nst);   // (dh0 may be dht)
    for (int j = 0; j < 7; ++j) bad |= meet(out[i], nout[i], in[j], nin[j]);
    for (int j = i + 1; j < 5; ++j) bad |= meet(out[i], nout[i], out[j], nout[j]);
    if (bad)
      return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": a gradient overlaps an input or another gradient");
  }
  const bool has_cu = cu_seqlens != nullptr;
  const gdn::LinPlan p = gdn::lin_plan(B, T, Hqk, Hv, K, V, N, has_cu, true);
  const int hp = gdn::lin_pair(Hqk, Hv) ? 2 : 1;
  rc = gdn_host::lin_lanes(name, gdn::lin_items(p.nseg, Hqk, Hv / hp) * 2 * (K + V));
  if (!rc && p.nlong > 0) rc = gdn_host::lin_lanes(name, gdn::lin_items(p.nseg, Hqk, Hv) * 4 * V);
  if (!rc && Hv / Hqk / hp > 1) rc = gdn_host::lin_lanes(name, tokens * Hqk * K / 8 + 255);
  if (rc) return rc;
  if (p.total > 0 && (!workspace || workspace_bytes < p.total))
    return gdn_host::fail(GDN_ERR_WORKSPACE, std::string(name) + ": workspace needs " +
                                                 std::to_string(p.total) + " bytes, got " +
                                                 std::to_string(workspace_bytes));
  const bool walk = N > 0 && (tokens > 0 || dh0);
  if (!walk && !g_per_head) return GDN_OK;
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  void* dgt = g_per_head ? ws + p.dgtok : dg;   // (one decay per head: fp32, summed below)
  if (walk) {
    const gdn::LinGrid grid = gdn::lin_grid(p, ws, T, N, B * T, has_cu);
    if (has_cu) gdn::launch_lin_table(cu_seqlens, p, ws, N, B * T, st);
    gdn::LinBwdArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.dO = static_cast<const uint16_t*>(dO);
    a.ts = ts;
    a.dec = gdn::LinDecay{g, g_dtype, g_per_head ? 0 : Hv};
    a.grid = grid;
    a.Hqk = Hqk;
    a.Hv = Hv;
    a.scale = scale;
    a.dht = dht;
    a.dh0 = dh0;
    a.states = static_cast<const gdn::u16x8*>(states);
    a.dq = static_cast<uint16_t*>(dq);
    a.dk = static_cast<uint16_t*>(dk);
    a.dv = static_cast<uint16_t*>(dv);
    a.dg = dgt;
    a.dgt = g_per_head ? GDN_DTYPE_F32 : g_dtype;
    const int parts = Hv / Hqk / hp;   // of a qk-head's gradients
    if (parts > 1) {
      a.pq = reinterpret_cast<float*>(ws + p.part);
      a.pk = a.pq + tokens * Hqk * parts * K;
    }
    float* segs = reinterpret_cast<float*>(ws + p.segs);
    float* decay = reinterpret_cast<float*>(ws + p.decay);
    a.segs = segs;
    if (K == 128 && V == 128) gdn::launch_grad<128, 128>(a, segs, decay, st);
    else if (K == 128) gdn::launch_grad<128, 64>(a, segs, decay, st);
    else if (V == 128) gdn::launch_grad<64, 128>(a, segs, decay, st);
    else gdn::launch_grad<64, 64>(a, segs, decay, st);
    if (a.pq && tokens > 0)
      hipLaunchKernelGGL(gdn::lin_group_sum_kernel,
                         dim3((unsigned)((tokens * Hqk * K / 8 + 255) / 256), 2), dim3(256), 0, st,
                         a.pq, a.pk, a.dq, a.dk, grid.status, tokens * Hqk, parts, K);
  }
  if (g_per_head)
    hipLaunchKernelGGL(gdn::lin_head_sum_kernel, dim3(Hv), dim3(1024), 0, st,
                       static_cast<const float*>(dgt), dg, (int)tokens, Hv, g_dtype);
  return gdn_host::check_launch(name);
}
