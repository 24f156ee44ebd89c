// Rotary positions for gfx950 (declared in gdn_attn.h):
//     (a, b) -> m (a cos t - b sin t, b cos t + a sin t),  t = p f_j
// of the pairs of a head's first R elements, the rest copied.
//
// The path reads and writes every element once and is bound by HBM.  A lane
// owns a unit of 2 VEC elements of a head (VEC pairs, or 2 VEC elements of the
// copied part), forms its pairs' sines and cosines once and turns that unit of
// several heads.  There is no table of angles: a position's turns p f / 2 pi are
// formed in 64 bits and reduced there, so far positions lose nothing, and no
// position is out of a table's range.
//
// bf16: 8192 tokens of 40 heads of 128, neighbours, 38 us, 4.4 TB/s read and written (a
// lane's two pieces lie side by side, so that the lanes of one instruction take 16 bytes of
// every 32); 256 tokens of 18 heads of 256, a quarter turned, 5.3 us: a round trip behind
// the angles.
#include <algorithm>

#include "gdn_norm_rows.h"
#include "../../include/gdn_attn.h"

namespace gdn {

struct RotaryArgs {
  const void* x[2];
  void* y[2];
  long long xs[2][3], ys[2][3];
  const void* pos;
  const double* freq;
  long long pos_batch;
  int heads[2];
  int T, R, units, per_wg, rows, split, inplace;   // rows: B T;  split: lanes' groups per token
  float mag, sign;
  int pos64;
};

// VEC elements at p + i: 16 bytes, or fewer where VEC is not a whole vector.
template <int DT, int VEC>
__device__ __forceinline__ void ld_unit(const void* p, long long i, float (&f)[VEC]) {
  if constexpr (VEC % Elt<DT>::VEC == 0) {
    ldn<DT, VEC>(p, i, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = lde<DT>(p, i + j);
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void st_unit(void* p, long long i, const float (&f)[VEC]) {
  if constexpr (VEC % Elt<DT>::VEC == 0) {
    stn<DT, VEC>(p, i, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) ste<DT>(p, i + j, f[j]);
  }
}

constexpr int kRotaryBatch = 4;   // heads whose loads a lane has on their way

template <int DT, int VEC, bool NEAR>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr int U = kRotaryBatch;
  const int slot = threadIdx.x / a.units, u = threadIdx.x % a.units;
  const long long id = (long long)blockIdx.x * a.per_wg + slot;
  if (slot >= a.per_wg || id >= (long long)a.rows * a.split) return;
  const int row = (int)(id / a.split), h0 = (int)(id % a.split);
  const int b = row / a.T, t = row % a.T;
  const bool turn = 2 * VEC * u < a.R;
  if (!turn && a.inplace) return;
  // offsets of the unit's two halves in a head
  const int lo = NEAR || !turn ? 2 * VEC * u : VEC * u;
  const int hi = NEAR || !turn ? lo + VEC : lo + a.R / 2;
  const int total = a.heads[0] + a.heads[1];
  long long in[2], out[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    in[k] = b * a.xs[k][0] + t * a.xs[k][1];
    out[k] = b * a.ys[k][0] + t * a.ys[k][1];
  }
  float x[U][VEC], y[U][VEC];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int head = h + i * a.split;
      if (head >= total) break;
      const int k = head >= a.heads[0], hh = k ? head - a.heads[0] : head;
      const long long at = in[k] + hh * a.xs[k][2];
      ld_unit<DT, VEC>(a.x[k], at + lo, x[i]);
      ld_unit<DT, VEC>(a.x[k], at + hi, y[i]);
    }
  };
  load(h0);
  float c[VEC], s[VEC];
  if (turn) {
    const long long pi = b * a.pos_batch + t;
    const double p = a.pos64 ? (double)static_cast<const long long*>(a.pos)[pi]
                             : (double)static_cast<const int*>(a.pos)[pi];
    double f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = a.freq[VEC * u + j];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      double w = p * f[j] * 0.15915494309189533577;   // turns: 1 / (2 pi)
      w -= rint(w);
      sincospif(2.f * (float)w, &s[j], &c[j]);
      c[j] *= a.mag;
      s[j] *= a.mag * a.sign;
    }
  }
  for (int h = h0; h < total; h += U * a.split) {
    if (h != h0) load(h);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int head = h + i * a.split;
      if (head >= total) break;
      if (turn) {
        if constexpr (NEAR) {
          // neighbours: pair j is elements 2 j and 2 j + 1 of x and y together
          float z[2 * VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            z[j] = x[i][j];
            z[VEC + j] = y[i][j];
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float p = z[2 * j], q = z[2 * j + 1];
            z[2 * j] = p * c[j] - q * s[j];
            z[2 * j + 1] = q * c[j] + p * s[j];
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            x[i][j] = z[j];
            y[i][j] = z[VEC + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float p = x[i][j], q = y[i][j];
            x[i][j] = p * c[j] - q * s[j];
            y[i][j] = q * c[j] + p * s[j];
          }
        }
      }
      const int k = head >= a.heads[0], hh = k ? head - a.heads[0] : head;
      const long long at = out[k] + hh * a.ys[k][2];
      st_unit<DT, VEC>(a.y[k], at + lo, x[i]);
      st_unit<DT, VEC>(a.y[k], at + hi, y[i]);
    }
  }
}

}  // namespace gdn

namespace {

// Whether sum x_i stride_i = rem has a solution with lo_i <= x_i <= hi_i, strides falling: of
// each only the x that leave what the rest can reach (one or two where strides nest; `steps`
// bounds what others may take, and what is not settled by then counts as a solution).
struct Term {
  long long stride, lo, hi;
};
bool solvable(const Term* t, int n, long long rem, int& steps) {
  if (n == 0) return rem == 0;
  if (--steps < 0) return true;
  long long least = 0, most = 0;   // of the rest
  for (int i = 1; i < n; ++i) {
    least += t[i].lo * t[i].stride;
    most += t[i].hi * t[i].stride;
  }
  auto floor_div = [](long long a, long long b) { return a >= 0 ? a / b : -((b - 1 - a) / b); };
  const long long from = std::max(t->lo, -floor_div(most - rem, t->stride));
  const long long to = std::min(t->hi, floor_div(rem - least, t->stride));
  for (long long x = from; x <= to; ++x)
    if (solvable(t + 1, n - 1, rem - x * t->stride, steps)) return true;
  return false;
}

// Whether two tensors [n0, n1, n2, D] (strides in elements of es bytes, the last 1) share a byte.
bool share(const void* a, const long long* as, const long long (&an)[3], const void* b, const long long* bs,
           const long long (&bn)[3], int D, int es) {
  Term t[7];
  int n = 0;
  auto add = [&](long long stride, long long lo, long long hi) {
    if (stride == 0 || lo == hi) return;
    int i = 0;
    while (i < n && t[i].stride > stride) ++i;
    if (i == n || t[i].stride != stride) {
      for (int j = n++; j > i; --j) t[j] = t[j - 1];
      t[i] = Term{stride, 0, 0};
    }
    t[i].lo += lo;
    t[i].hi += hi;
  };
  for (int j = 0; j < 3; ++j) {
    add(as[j] * es, 0, an[j] - 1);
    add(bs[j] * es, 1 - bn[j], 0);
  }
  add(1, 1 - D * es, D * es - 1);
  int steps = 1 << 16;
  return solvable(t, n, (long long)(reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a)), steps);
}

}  // namespace

extern "C" int gdn_rotary(const void* q, const void* k, void* q_out, void* k_out,
                          const long long* strides, int B, int T, int Hq, int Hk, int D,
                          const void* positions, int pos_int64, long long pos_batch,
                          const double* inv_freq, int R, float magnitude, int interleaved,
                          int inverse, int dtype, void* stream) {
  const char* name = "gdn_rotary";
  if (!k) Hk = 0;
  if (B < 0 || T < 0 || Hq < 1 || Hk < 0)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": sizes must be non-negative (Hq > 0)");
  if (D < 2 || D > 512 || D % 2 || R < 2 || R > D || R % 2)
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": D and R must be even, 2 <= R <= D <= 512");
  if (!gdn::dtype_ok(dtype))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported dtype code");
  if (Hq > (1 << 20) || Hk > (1 << 20) || (long long)B * T >= (1LL << 31))
    return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": problem too large");
  if ((long long)B * T == 0) return GDN_OK;
  if (!positions || !inv_freq || !strides || !q || !q_out || (Hk && !k_out))
    return gdn_host::fail(GDN_ERR_NULL, std::string(name) + ": q, its output, strides, positions and inv_freq must be "
                                                            "non-NULL, and k's output with k");
  const void* x[2] = {q, k};
  void* y[2] = {q_out, k_out};
  const int heads[2] = {Hq, Hk}, two = Hk > 0 ? 2 : 1;
  const long long *xs = strides, *ys = strides + 6;
  const bool inplace = q == q_out;
  for (int i = 0; i < two; ++i) {
    for (int j = 0; j < 3; ++j) {
      if (xs[3 * i + j] < 0 || ys[3 * i + j] < 0)
        return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": strides must be non-negative");
      if (inplace && xs[3 * i + j] != ys[3 * i + j])
        return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": in place both must have the same strides");
    }
    if (inplace != (x[i] == y[i]))
      return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": both tensors in place, or none");
  }
  const int es = dtype == GDN_DTYPE_F32 ? 4 : 2;
  auto bytes = [&](const long long* st, int h) {
    return (size_t)((B - 1) * st[0] + (T - 1) * st[1] + (h - 1) * st[2] + D) * es;
  };
  if (two == 2 && share(y[0], ys, {B, T, Hq}, y[1], ys + 3, {B, T, Hk}, D, es))
    return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": the two outputs must share no element");
  if (!inplace)
    for (int i = 0; i < two; ++i)
      for (int j = 0; j < two; ++j)
        if (gdn_host::overlaps(y[i], bytes(ys + 3 * i, heads[i]), x[j], bytes(xs + 3 * j, heads[j])))
          return gdn_host::fail(GDN_ERR_ALIAS, std::string(name) + ": outputs must not overlap an input, but in place");
  // the widest units that divide both parts of a head: 16 bytes of each half, 2
  // elements, or 1
  const int full = dtype == GDN_DTYPE_F32 ? 4 : 8;
  int vec = 1;
  for (const int v : {full, 2})
    if (vec == 1 && R % (2 * v) == 0 && D % (2 * v) == 0) vec = v;
  gdn::RotaryArgs a{};
  for (int i = 0; i < two; ++i) {
    a.x[i] = x[i];
    a.y[i] = y[i];
    a.heads[i] = heads[i];
    for (int j = 0; j < 3; ++j) {
      a.xs[i][j] = xs[3 * i + j];
      a.ys[i][j] = ys[3 * i + j];
    }
  }
  a.pos = positions;
  a.pos64 = pos_int64;
  a.pos_batch = pos_batch;
  a.freq = inv_freq;
  a.T = T;
  a.R = R;
  a.units = D / (2 * vec);
  a.per_wg = 256 / a.units;
  a.rows = B * T;
  a.inplace = inplace;
  a.mag = magnitude;
  a.sign = inverse ? -1.f : 1.f;
  // groups of lanes per token: as many heads to a group as leave every CU four
  // workgroups, eight at most
  const int total = Hq + Hk;
  const long long want = 4LL * gdn::device_cus() * a.per_wg;
  long long split = (want + a.rows - 1) / a.rows;
  if (split < (total + 7) / 8) split = (total + 7) / 8;
  a.split = (int)(split < total ? split : total);
  const long long wgs = ((long long)a.rows * a.split + a.per_wg - 1) / a.per_wg;
  if (const int fit = gdn_host::check_lanes(name, wgs, 256)) return fit;
  gdn_host::launch_begin();
  auto st = static_cast<hipStream_t>(stream);
#define GDN_ROT(TT, VV, NN)                                                                   \
  if (dtype == TT && vec == VV && !interleaved == !NN) {                                      \
    hipLaunchKernelGGL((gdn::rotary_kernel<TT, VV, NN>), dim3((unsigned)wgs), dim3(256), 0, st, a); \
    return gdn_host::check_launch(name);                                                      \
  }
#define GDN_ROT_V(TT, FULL)                                                                   \
  GDN_ROT(TT, FULL, false) GDN_ROT(TT, FULL, true) GDN_ROT(TT, 2, false) GDN_ROT(TT, 2, true) \
  GDN_ROT(TT, 1, false) GDN_ROT(TT, 1, true)
  GDN_ROT_V(GDN_DTYPE_BF16, 8)
  GDN_ROT_V(GDN_DTYPE_F16, 8)
  GDN_ROT_V(GDN_DTYPE_F32, 4)
#undef GDN_ROT
#undef GDN_ROT_V
  return gdn_host::fail(GDN_ERR_SHAPE, std::string(name) + ": unsupported configuration");
}
