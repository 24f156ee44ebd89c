// Linear attention with a decay for each head, token by token (decode), for
// gfx950 (declared in gdn_linear.h).  Per token and v-head
//     S' = e^g S + k v^T,   o = scale (e^g S^T q + (k . q) v)
// so one pass over the old state gives o and the new state.
//
// The path streams fp32 states (64 KiB per v-head at K = V = 128: 0.4 flop/B)
// and is bound by HBM, or for a few sequences by one round trip.  A
// workgroup advances a tile of all K rows and CW columns of one state; columns
// do not depend on each other, so where whole states would not fill the GPU
// they are cut into tiles of 16 columns.  A lane holds float4 columns of K /
// ROWG rows; a persistent grid walks the tiles, the next tile's state loaded
// while the current one is advanced, in 16-byte streaming loads.
#include <initializer_list>

#include "gdn_linear.h"
#include "../../include/gdn_linear.h"

namespace gdn {

struct LinRecArgs {
  const uint16_t *q, *k, *v;
  TokenStride ts;
  LinDecay dec;
  const float* h0;
  float* ht;
  uint16_t* o;
  const int32_t* cu;
  const int32_t* slots;
  int T, total, Hqk, Hv, N, num_slots, ntiles;
  float scale;
};

template <int K, int V, int CW, int NT>
__global__ __launch_bounds__(NT) void lin_recurrent_kernel(LinRecArgs a) {
  constexpr int COLG = CW / 4, ROWG = NT / COLG, RPT = K / ROWG, NW = NT / 64, CT = V / CW;
  static_assert(ROWG * COLG == NT && RPT * ROWG == K && COLG <= 64, "tile shape");
  __shared__ float kq_s[2][K];
  __shared__ f32x4 red[NW][COLG];
  __shared__ float redk[NW];
  const int tid = threadIdx.x, cg = tid % COLG, rg = tid / COLG, lane = tid % 64, wave = tid / 64;
  const int G = gridDim.x;

  // a cu_seqlens violation: no sequence has a token, o is zero.  (The check is
  // 0.5 us of a single sequence's 5.0, 1.7 of 177 at 256.)
  bool bad = false;
  if (a.cu) {
    int b = tid == 0 && (a.cu[0] != 0 || a.cu[a.N] != a.total);
    for (int n = tid; n < a.N; n += NT) b |= a.cu[n + 1] < a.cu[n];
    bad = __syncthreads_or(b);
    if (bad) {
      const size_t all = (size_t)a.total * a.Hv * V / 8;
      for (size_t i = (size_t)blockIdx.x * NT + tid; i < all; i += (size_t)G * NT)
        reinterpret_cast<u32x4*>(a.o)[i] = u32x4{0, 0, 0, 0};
    }
  }

  auto slot_of = [&](int n) {
    if (!a.slots) return n;
    const int s = a.slots[n];
    return s < 0 || s >= a.num_slots ? -1 : s;
  };
  auto load_state = [&](f32x4 (&S)[RPT], int tile) {
    const int tl = min(tile, a.ntiles - 1), sh = tl / CT, n = sh / a.Hv;
    const int slot = slot_of(n);
    const bool live = a.h0 && tile < a.ntiles && slot >= 0;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(a.h0) + (live ? ((size_t)slot * a.Hv + sh % a.Hv) * (size_t)(K * V) : 0),
        0, live ? K * V * 4 : 0, kBufferFlags);
#pragma unroll
    for (int i = 0; i < RPT; ++i)
      S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
          rs, ((rg + ROWG * i) * V + (tl % CT) * CW + 4 * cg) * 4, 0, kStoreStream));
  };
  auto run_tile = [&](f32x4 (&S)[RPT], int tile) {
    const int sh = tile / CT, n = sh / a.Hv, h = sh % a.Hv, hq = h / (a.Hv / a.Hqk);
    const int col = (tile % CT) * CW + 4 * cg;
    const int slot = slot_of(n);
    if (slot < 0) return;
    int s, e;
    seq_bounds(a.cu, n, a.T, a.total, s, e);
    if (bad) e = s;
    if (a.slots) {
      // a slot that another sequence names too: neither advances it, and the
      // output rows are NaN so that the caller's error shows
      int hit = 0;
      for (int m = tid; m < a.N; m += NT) hit |= m != n && a.slots[m] == slot;
      if (__syncthreads_or(hit)) {
        if (rg == 0)
          for (int t = s; t < e; ++t)
            *reinterpret_cast<u16x4*>(a.o + ((size_t)t * a.Hv + h) * V + col) =
                u16x4{0x7FC0, 0x7FC0, 0x7FC0, 0x7FC0};
        return;
      }
    }
    for (int t = s; t < e; ++t) {
      for (int j = tid; j < 2 * K; j += NT) {
        const uint16_t* p = j < K ? a.k + (size_t)t * a.ts.k : a.q + (size_t)t * a.ts.q;
        kq_s[j / K][j % K] = bf2f(p[hq * K + j % K]);
      }
      const u16x4 vb = *reinterpret_cast<const u16x4*>(a.v + (size_t)t * a.ts.v + h * V + col);
      const float eg = __expf(lin_g(a.dec, t, h));
      __syncthreads();
      f32x4 sq = zero4();
      float kq = 0.f, kr[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        kr[i] = kq_s[0][rg + ROWG * i];
        const float qr = kq_s[1][rg + ROWG * i];
        sq += S[i] * qr;
        kq += kr[i] * qr;
      }
#pragma unroll
      for (int off = COLG; off < 64; off *= 2) {
#pragma unroll
        for (int c = 0; c < 4; ++c) sq[c] += __shfl_xor(sq[c], off);
        kq += __shfl_xor(kq, off);
      }
      if (lane < COLG) red[wave][cg] = sq;
      if (lane == 0) redk[wave] = kq;
      const f32x4 vf = {bf2f(vb[0]), bf2f(vb[1]), bf2f(vb[2]), bf2f(vb[3])};
#pragma unroll
      for (int i = 0; i < RPT; ++i) S[i] = eg * S[i] + kr[i] * vf;
      __syncthreads();
      if (rg == 0) {
        sq = red[0][cg];
        kq = redk[0];
#pragma unroll
        for (int ww = 1; ww < NW; ++ww) {
          sq += red[ww][cg];
          kq += redk[ww];
        }
        *reinterpret_cast<u16x4*>(a.o + ((size_t)t * a.Hv + h) * V + col) =
            f2bf4(a.scale * (eg * sq + kq * vf));
      }
    }
    if (a.ht) {
      float* dst = a.ht + ((size_t)slot * a.Hv + h) * (size_t)(K * V) + col;
#pragma unroll
      for (int i = 0; i < RPT; ++i)
        __builtin_nontemporal_store(S[i], reinterpret_cast<f32x4*>(dst + (rg + ROWG * i) * V));
    }
  };

  // (ping-pong by name: the state stays in registers)
  f32x4 A[RPT], B[RPT];
  int tile = blockIdx.x;
  load_state(A, tile);
  while (tile < a.ntiles) {
    load_state(B, tile + G);
    run_tile(A, tile);
    tile += G;
    if (tile >= a.ntiles) break;
    __syncthreads();   // red / kq_s of the last token
    load_state(A, tile + G);
    run_tile(B, tile);
    tile += G;
    __syncthreads();
  }
}

template <int K, int V>
void launch_lin_recurrent(LinRecArgs a, hipStream_t st) {
  const int states = a.N * a.Hv;
  // whole states where they give every CU two workgroups (256 sequences of 32
  // v-heads: 170 us, 6.4 TB/s; in tiles of 16 columns 385), else 16 columns
  if (states >= 2 * device_cus()) {
    a.ntiles = states;
    hipLaunchKernelGGL((lin_recurrent_kernel<K, V, V, 512>),
                       dim3((unsigned)min(a.ntiles, 4 * device_cus())), dim3(512), 0, st, a);
  } else {
    a.ntiles = states * (V / 16);
    hipLaunchKernelGGL((lin_recurrent_kernel<K, V, 16, 256>),
                       dim3((unsigned)min(a.ntiles, 8 * device_cus())), dim3(256), 0, st, a);
  }
}

}  // namespace gdn

namespace gdn_host {
int lin_validate(const char* name, const void* q, const void* k, const void* v, long long q_row,
                 long long k_row, long long v_row, const void* g, int g_dtype, const float* h0,
                 const float* ht, const void* o, const int32_t* cu, int B, int T, int Hqk, int Hv,
                 int K, int V, int N, gdn::TokenStride& ts);
int lin_aligned(const char* name, std::initializer_list<const void*> ptrs);
}

extern "C" int gdn_linear_recurrent_fwd(const void* q, const void* k, const void* v,
                                        long long q_row, long long k_row, long long v_row,
                                        const void* g, int g_dtype, int g_per_head,
                                        const float* h0, float* ht, void* o,
                                        const int32_t* cu_seqlens, const int32_t* state_indices,
                                        int B, int T, int Hqk, int Hv, int K, int V, int N,
                                        int num_slots, float scale, void* stream) {
  const char* name = "gdn_linear_recurrent_fwd";
  gdn::TokenStride ts;
  int rc = gdn_host::lin_validate(name, q, k, v, q_row, k_row, v_row, g, g_dtype,
                                        state_indices ? nullptr : h0, state_indices ? nullptr : ht,
                                        o, cu_seqlens, B, T, Hqk, Hv, K, V, N, ts);
  if (!rc) rc = gdn_host::lin_aligned(name, {o, h0, ht});
  if (rc) return rc;
  if (num_slots < 0 || (!state_indices && num_slots != N))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": num_slots must be >= 0, and N without state_indices");
  if (state_indices && h0 && ht && h0 != ht &&
      gdn_host::overlaps(h0, (size_t)num_slots * Hv * K * V * 4, ht, (size_t)num_slots * Hv * K * V * 4))
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": ht must equal h0 exactly or not overlap it");
  if (N == 0 || num_slots == 0 || ((long long)B * T == 0 && !ht)) return GDN_OK;
  gdn_host::launch_begin();
  const gdn::LinRecArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                          static_cast<const uint16_t*>(v), ts,
                          gdn::LinDecay{g, g_dtype, g_per_head ? 0 : Hv}, h0, ht,
                          static_cast<uint16_t*>(o), cu_seqlens, state_indices, T, B * T, Hqk, Hv,
                          N, num_slots, 0, scale};
  auto st = static_cast<hipStream_t>(stream);
  if (K == 128 && V == 128) gdn::launch_lin_recurrent<128, 128>(a, st);
  else if (K == 128) gdn::launch_lin_recurrent<128, 64>(a, st);
  else if (V == 128) gdn::launch_lin_recurrent<64, 128>(a, st);
  else gdn::launch_lin_recurrent<64, 64>(a, st);
  return gdn_host::check_launch(name);
}
