// RMS norm of every query and key head with the position rotation in the same pass.  Per head
// row x of K elements, with s = 1 / sqrt(mean x^2 + eps):
//   n_i = x_i s w_i;   the first R elements are rotated in pairs (i, i') by the row's angle,
//   y_i = n_i cos - n_i' sin,  y_i' = n_i sin + n_i' cos     (i' = i + R/2, or i' = i + 1, i even)
// Backward: dn = the rotation by the opposite angle of dy, e = w dn, dw = sum dn x s,
//   dx = s (e - x s^2 mean(e x)).
//
// Nothing is reused between rows but the token's cosines and the weights, so HBM bounds it:
// a group of lanes owns a token, keeps V weights a lane in registers and walks the token's heads.
// A rotated element's partner lies in another lane's vector: it is loaded once more (the line is
// in L1) rather than passed through shuffles whose register index would be dynamic.
#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace qkn {

struct P {
  int64_t tokens;
  int T, H, HK, K, R, pairs, wdtype, pos64, table;
  int lanes, hg, nhg;  // lanes of a row, heads of a unit, units of a token
  int wvec;            // the weights start on a vector
  float eps;
  const void *q, *k, *qw, *kw;
  int64_t qs[3], ks[3];  // strides (batch, row, head) of q and k in elements
  const float *cos, *sin;
  const void* pos;
  int64_t pb;  // batch stride of positions (row stride 1)
  void *yq, *yk;
  // backward
  const void *dyq, *dyk;
  int64_t dqs[3], dks[3];
  void *dq, *dk;
  float* part;  // [blocks][2][K]
};

// What a lane needs of one vector (elements e0 .. e0 + V): where the partners are and the angle's
// cosine and signed sine (y_i = n_i c_i + n_partner s_i).
template <int V>
struct Rot {
  int p0;  // first partner's element (half-split); interleaved partners are inside the vector
  bool on;
  float c[V], s[V];
};

template <int V>
__device__ __forceinline__ Rot<V> rotation(const P& p, int e0, int64_t pos, float sign) {
  Rot<V> r;
  r.on = e0 < p.R;
  r.p0 = e0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    r.c[i] = 1.f;
    r.s[i] = 0.f;
  }
  if (!r.on) return r;
  const int half = p.R >> 1;
  const bool inside = pos >= 0 && pos < p.table;
  const float* ct = p.cos + (inside ? pos : 0) * half;
  const float* st = p.sin + (inside ? pos : 0) * half;
  const float bad = __int_as_float(0x7fffffff);  // a position outside the table gives NaN
  if (p.pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = e0 + i;
      r.c[i] = inside ? ct[e >> 1] : bad;
      r.s[i] = inside ? ((e & 1) ? sign : -sign) * st[e >> 1] : bad;
    }
    r.p0 = V == 1 ? (e0 ^ 1) : e0;
  } else {
    const bool low = e0 < half;
    const int a = low ? e0 : e0 - half;
    r.p0 = low ? e0 + half : e0 - half;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      r.c[i] = inside ? ct[a + i] : bad;
      r.s[i] = inside ? (low ? -sign : sign) * st[a + i] : bad;
    }
  }
  return r;
}

// V weights from element e0 (ones without weights); e0 is a multiple of V
template <typename T, int V>
__device__ __forceinline__ void weights(const void* w, const P& p, int e0, float (&r)[V]) {
  if (w == nullptr || e0 >= p.K) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = 1.f;
  } else if (p.wvec && p.wdtype == TOPS_F32) {
    Vx<float, V>::load(static_cast<const float*>(w) + e0, r);
  } else if (p.wvec) {
    Vx<T, V>::load(static_cast<const T*>(w) + e0, r);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = load_param(w, p.wdtype, e0 + i);
  }
}

// The heads h0 .. h1 of q (or of k) of one token, HB at a time: their loads are issued before the first sum.
// Every lane of a warp takes the same turns, since the sums are full-warp exchanges; `live` says whose rows exist.
template <typename T, int V, int J, int HB>
__device__ __forceinline__ void heads_fwd(const P& p, const T* x, int64_t hs, T* y, const void* weight, int h0, int h1,
                                          int turns, bool live, int l, const Rot<V> (&rot)[J]) {
  float w[J][V], pw[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    weights<T, V>(weight, p, (l + j * p.lanes) * V, w[j]);
    weights<T, V>(weight, p, rot[j].p0, pw[j]);
  }
  for (int i = 0; i < turns; i += HB) {
    Raw<T, V> own[HB][J], par[HB][J];
#pragma unroll
    for (int u = 0; u < HB; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (live && h0 + i + u < h1 && e0 < p.K) {
          own[u][j].load(x + (h0 + i + u) * hs + e0);
          if (rot[j].on && !(p.pairs && V > 1)) par[u][j].load(x + (h0 + i + u) * hs + rot[j].p0);
        }
      }
    float ss[HB];
#pragma unroll
    for (int u = 0; u < HB; ++u) {
      ss[u] = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (live && h0 + i + u < h1 && (l + j * p.lanes) * V < p.K) {
          float v[V];
          own[u][j].get(v);
#pragma unroll
          for (int c = 0; c < V; ++c) ss[u] = fmaf(v[c], v[c], ss[u]);
        }
      }
    }
    for (int o = p.lanes >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < HB; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
#pragma unroll
    for (int u = 0; u < HB; ++u) {
      const float s = rsqrtf(ss[u] / (float)p.K + p.eps);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (live && h0 + i + u < h1 && e0 < p.K) {
          float out[V];
          own[u][j].get(out);
#pragma unroll
          for (int c = 0; c < V; ++c) out[c] *= s * w[j][c];
          if (rot[j].on) {
            float o[V];
            if (p.pairs && V > 1) {
#pragma unroll
              for (int c = 0; c < V; ++c) o[c] = out[c ^ (V > 1 ? 1 : 0)];
            } else {
              par[u][j].get(o);
#pragma unroll
              for (int c = 0; c < V; ++c) o[c] *= s * pw[j][c];
            }
#pragma unroll
            for (int c = 0; c < V; ++c) out[c] = fmaf(out[c], rot[j].c[c], o[c] * rot[j].s[c]);
          }
          Vx<T, V>::store(y + (h0 + i + u) * p.K + e0, out);
        }
      }
    }
  }
}

__device__ __forceinline__ int64_t position(const P& p, int b, int t) {
  if (!p.R || !p.pos) return t;
  return p.pos64 ? static_cast<const int64_t*>(p.pos)[b * p.pb + t] : static_cast<const int32_t*>(p.pos)[b * p.pb + t];
}

template <typename T, int V, int J>
__global__ void __launch_bounds__(256) k_qk_fwd(const P p) {
  constexpr int HB = J == 1 ? 4 : 1;
  const int lane = threadIdx.x & 31, l = lane & (p.lanes - 1);
  const int rpw = 32 / p.lanes;
  const int64_t unit = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * rpw + lane / p.lanes;
  const bool live = unit < p.tokens * p.nhg;
  const int64_t tok = live ? unit / p.nhg : 0;
  const int h0 = live ? (int)(unit - tok * p.nhg) * p.hg : 0, h1 = h0 + p.hg;
  const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
  const int64_t pos = position(p, b, t);
  Rot<V> rot[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e0 = (l + j * p.lanes) * V;
    rot[j] = rotation<V>(p, e0 < p.K ? e0 : p.K, pos, 1.f);
  }
  // units of a warp may lie on both sides of the border between q and k: each side's turns are the warp's most
  const int q1 = min(h1, p.H), k0 = max(h0, p.H) - p.H, k1 = min(h1, p.H + p.HK) - p.H;
  const int qn = __reduce_max_sync(0xffffffffu, live ? max(q1 - h0, 0) : 0);
  const int kn = __reduce_max_sync(0xffffffffu, live ? max(k1 - k0, 0) : 0);
  if (qn > 0)
    heads_fwd<T, V, J, HB>(p, static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1], p.qs[2],
                           static_cast<T*>(p.yq) + tok * p.H * p.K, p.qw, h0, q1, qn, live, l, rot);
  if (kn > 0)
    heads_fwd<T, V, J, HB>(p, static_cast<const T*>(p.k) + b * p.ks[0] + t * p.ks[1], p.ks[2],
                           static_cast<T*>(p.yk) + tok * p.HK * p.K, p.kw, k0, k1, kn, live, l, rot);
}

// As heads_fwd: both sums of a row (x^2 and e x) come from the same loads; the rows' dw terms are kept.
template <typename T, int V, int J, int HB>
__device__ __forceinline__ void heads_bwd(const P& p, const T* x, int64_t hs, const T* dy, int64_t gs, T* dx,
                                          const void* weight, int h0, int h1, int turns, bool live, int l,
                                          const Rot<V> (&rot)[J], float (&dw)[J][V]) {
  float w[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) weights<T, V>(weight, p, (l + j * p.lanes) * V, w[j]);
  for (int i = 0; i < turns; i += HB) {
    Raw<T, V> xr[HB][J], gr[HB][J], pr[HB][J];
#pragma unroll
    for (int u = 0; u < HB; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (live && h0 + i + u < h1 && e0 < p.K) {
          xr[u][j].load(x + (h0 + i + u) * hs + e0);
          gr[u][j].load(dy + (h0 + i + u) * gs + e0);
          if (rot[j].on && !(p.pairs && V > 1)) pr[u][j].load(dy + (h0 + i + u) * gs + rot[j].p0);
        }
      }
    float ss[HB], ex[HB];
    float e[HB][J][V];
#pragma unroll
    for (int u = 0; u < HB; ++u) {
      ss[u] = ex[u] = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (live && h0 + i + u < h1 && (l + j * p.lanes) * V < p.K) {
          float v[V];
          xr[u][j].get(v);
          gr[u][j].get(e[u][j]);
          if (rot[j].on) {
            float o[V];
            if (p.pairs && V > 1) {
#pragma unroll
              for (int c = 0; c < V; ++c) o[c] = e[u][j][c ^ (V > 1 ? 1 : 0)];
            } else {
              pr[u][j].get(o);
            }
#pragma unroll
            for (int c = 0; c < V; ++c) e[u][j][c] = fmaf(e[u][j][c], rot[j].c[c], o[c] * rot[j].s[c]);
          }
#pragma unroll
          for (int c = 0; c < V; ++c) {
            ss[u] = fmaf(v[c], v[c], ss[u]);
            ex[u] = fmaf(e[u][j][c] * w[j][c], v[c], ex[u]);
          }
        }
      }
    }
    for (int o = p.lanes >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < HB; ++u) {
        ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
        ex[u] += __shfl_xor_sync(0xffffffffu, ex[u], o);
      }
#pragma unroll
    for (int u = 0; u < HB; ++u) {
      const float s = rsqrtf(ss[u] / (float)p.K + p.eps);
      const float m = s * s * ex[u] / (float)p.K;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (live && h0 + i + u < h1 && e0 < p.K) {
          float v[V], out[V];
          xr[u][j].get(v);
#pragma unroll
          for (int c = 0; c < V; ++c) {
            out[c] = s * (e[u][j][c] * w[j][c] - v[c] * m);
            dw[j][c] = fmaf(e[u][j][c] * v[c], s, dw[j][c]);
          }
          Vx<T, V>::store(dx + (h0 + i + u) * p.K + e0, out);
        }
      }
    }
  }
}

// Each block keeps its rows' dw terms and writes one partial row per weight.
template <typename T, int V, int J>
__global__ void __launch_bounds__(256) k_qk_bwd(const P p) {
  constexpr int HB = J == 1 ? 2 : 1;
  const int lane = threadIdx.x & 31, l = lane & (p.lanes - 1), warp = threadIdx.x >> 5;
  const int rpw = 32 / p.lanes;
  const int64_t units = p.tokens * p.nhg, step = (int64_t)gridDim.x * 8 * rpw;
  const int64_t first = ((int64_t)blockIdx.x * 8 + warp) * rpw;
  float dw[2][J][V];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int c = 0; c < V; ++c) dw[g][j][c] = 0.f;
  for (int64_t u0 = first; u0 < units; u0 += step) {  // the same turns for every lane of a warp
    const int64_t unit = u0 + lane / p.lanes;
    const bool live = unit < units;
    const int64_t tok = live ? unit / p.nhg : 0;
    const int h0 = live ? (int)(unit - tok * p.nhg) * p.hg : 0, h1 = h0 + p.hg;
    const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
    const int64_t pos = position(p, b, t);
    Rot<V> rot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e0 = (l + j * p.lanes) * V;
      rot[j] = rotation<V>(p, e0 < p.K ? e0 : p.K, pos, -1.f);
    }
    const int q1 = min(h1, p.H), k0 = max(h0, p.H) - p.H, k1 = min(h1, p.H + p.HK) - p.H;
    const int qn = __reduce_max_sync(0xffffffffu, live ? max(q1 - h0, 0) : 0);
    const int kn = __reduce_max_sync(0xffffffffu, live ? max(k1 - k0, 0) : 0);
    if (qn > 0)
      heads_bwd<T, V, J, HB>(p, static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1], p.qs[2],
                             static_cast<const T*>(p.dyq) + b * p.dqs[0] + t * p.dqs[1], p.dqs[2],
                             static_cast<T*>(p.dq) + tok * p.H * p.K, p.qw, h0, q1, qn, live, l, rot, dw[0]);
    if (kn > 0)
      heads_bwd<T, V, J, HB>(p, static_cast<const T*>(p.k) + b * p.ks[0] + t * p.ks[1], p.ks[2],
                             static_cast<const T*>(p.dyk) + b * p.dks[0] + t * p.dks[1], p.dks[2],
                             static_cast<T*>(p.dk) + tok * p.HK * p.K, p.kw, k0, k1, kn, live, l, rot, dw[1]);
  }
  if (p.part == nullptr) return;
  // rows of the block: fold the groups of a warp, then the warps, in a fixed order
  __shared__ float red[8][2][256];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int c = 0; c < V; ++c) {
        float a = dw[g][j][c];
        for (int o = p.lanes; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        const int el = (l + j * p.lanes) * V + c;
        if (lane < p.lanes && el < p.K) red[warp][g][el] = a;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.K; i += 256) {
    const int g = i / p.K, el = i - g * p.K;
    float a = 0.f;
    for (int w8 = 0; w8 < 8; ++w8) a += red[w8][g][el];
    p.part[(int64_t)blockIdx.x * 2 * p.K + i] = a;
  }
}

__global__ void __launch_bounds__(1024) k_qk_dw(int blocks, int K, int wdtype, const float* __restrict__ part, void* dqw,
                                                void* dkw) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < 2 * K)
    for (int i = threadIdx.y; i < blocks; i += 32) s += part[(int64_t)i * 2 * K + c];
  __shared__ float red[32][33];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < 2 * K) {
    float t = 0.f;
    for (int y = 0; y < 32; ++y) t += red[y][threadIdx.x];
    void* o = c < K ? dqw : dkw;
    if (o) store_param(o, wdtype, c < K ? c : c - K, t);
  }
}

int check(const tops_gla_qk_norm_args* a) {
  TOPS_CHECK_ARG(a != nullptr, "qk_norm: args is NULL");
  TOPS_CHECK_ARG(a->B >= 0 && a->T >= 0 && a->H >= 0 && a->HK >= 0, "qk_norm: negative dimension");
  if (a->K < 1 || a->K > 256) return fail(TOPS_ERR_UNSUPPORTED, "qk_norm: heads must have 1 to 256 elements");
  TOPS_CHECK_ARG(dtype_known(a->dtype), "qk_norm: unknown dtype");
  TOPS_CHECK_ARG(a->w_dtype == a->dtype || a->w_dtype == TOPS_F32, "qk_norm: w_dtype must be dtype or TOPS_F32");
  TOPS_CHECK_ARG(a->R >= 0 && a->R <= a->K && a->R % 2 == 0, "qk_norm: the rotated part must be even and fit the head");
  TOPS_CHECK_ARG(a->R == 0 || (a->cos_table && a->sin_table && a->table_rows > 0), "qk_norm: a rotation needs its tables");
  TOPS_CHECK_ARG(a->R == 0 || a->positions || a->T <= a->table_rows, "qk_norm: more rows than the tables have");
  return TOPS_OK;
}

P params(const tops_gla_qk_norm_args* a) {
  P p{};
  p.tokens = (int64_t)a->B * a->T;
  p.T = a->T; p.H = a->H; p.HK = a->HK; p.K = a->K; p.R = a->R;
  p.pairs = a->interleaved; p.wdtype = a->w_dtype; p.pos64 = a->positions_int64; p.table = a->table_rows;
  p.eps = a->eps;
  p.q = a->q; p.k = a->k; p.qw = a->q_weight; p.kw = a->k_weight;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_strides[i];
    p.ks[i] = a->k_strides[i];
  }
  p.cos = a->cos_table; p.sin = a->sin_table;
  p.pos = a->positions; p.pb = a->positions_stride_b;
  p.yq = a->q_out; p.yk = a->k_out;
  p.wvec = aligned_to(a->q_weight, 16) && aligned_to(a->k_weight, 16);
  return p;
}

// The widest vector that divides the head, the partner's offset and every stride and base.
int vector_of(const P& p, int es, bool bwd) {
  const int unit = (p.R && !p.pairs) ? p.R / 2 : (p.R ? p.R : p.K);
  for (int v : {8, 4}) {
    const int bytes = std::min(16, v * es);
    bool ok = p.K % v == 0 && unit % v == 0;
    const int ev = bytes / es;
    auto strides = [&](const int64_t (&s)[3]) { return s[0] % ev == 0 && s[1] % ev == 0 && s[2] % ev == 0; };
    ok = ok && strides(p.qs) && strides(p.ks) && aligned_to(p.q, bytes) && aligned_to(p.k, bytes);
    if (bwd)
      ok = ok && strides(p.dqs) && strides(p.dks) && aligned_to(p.dyq, bytes) && aligned_to(p.dyk, bytes) &&
           aligned_to(p.dq, bytes) && aligned_to(p.dk, bytes);
    else
      ok = ok && aligned_to(p.yq, bytes) && aligned_to(p.yk, bytes);
    if (ok) return v;
  }
  return 1;
}

// lanes of a row and heads of a unit: a unit walks several heads with one load of the angles
// while there are tokens enough for every SM, else every head is its own unit
void split(P& p, int v, int64_t want) {
  const int chunks = (p.K + v - 1) / v;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < chunks) p.lanes *= 2;
  const int heads = p.H + p.HK;
  const int64_t per = std::max<int64_t>(1, (int64_t)heads * p.tokens * p.lanes / want);
  p.hg = (int)std::min<int64_t>(heads, per);
  p.nhg = (heads + p.hg - 1) / p.hg;
}

template <typename F>
int by_type(int dtype, int v, F f) {
  auto go = [&](auto t) {
    if (v == 8) return f(t, std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    if (v == 4) return f(t, std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
    return f(t, std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
  };
  if (dtype == TOPS_F32) return go(float());
  if (dtype == TOPS_BF16) return go(__nv_bfloat16());
  return go(__half());
}

constexpr int64_t kWant = 148 * 2048;
constexpr int kBwdBlocks = 148 * 2;

}  // namespace qkn
}  // namespace tops

using namespace tops;
using namespace tops::qkn;

extern "C" {

TOPS_API int tops_gla_qk_norm_rotary_fwd(const tops_gla_qk_norm_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if ((int64_t)a->B * a->T == 0 || a->H + a->HK == 0) return TOPS_OK;
  TOPS_CHECK_ARG((!a->H || (a->q && a->q_out)) && (!a->HK || (a->k && a->k_out)), "qk_norm_fwd: q, k and their outputs are required");
  P p = params(a);
  const int v = vector_of(p, dtype_bytes(a->dtype), false);
  split(p, v, kWant);
  const int64_t units = p.tokens * p.nhg, per_block = 8 * (32 / p.lanes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "qk_norm_fwd");
  by_type(a->dtype, v, [&](auto t, auto vv, auto jj) {
    k_qk_fwd<decltype(t), decltype(vv)::value, decltype(jj)::value>
        <<<(unsigned)((units + per_block - 1) / per_block), 256, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("qk_norm_fwd");
  return TOPS_OK;
}

TOPS_API size_t tops_gla_qk_norm_rotary_bwd_workspace_size(const tops_gla_qk_norm_bwd_args* a) {
  if (a == nullptr || check(&a->f) != TOPS_OK || (!a->dq_weight && !a->dk_weight)) return 0;
  return (size_t)kBwdBlocks * 2 * a->f.K * sizeof(float);
}

TOPS_API int tops_gla_qk_norm_rotary_bwd(const tops_gla_qk_norm_bwd_args* a, void* stream) {
  TOPS_CHECK_ARG(a != nullptr, "qk_norm_bwd: args is NULL");
  if (int rc = check(&a->f)) return rc;
  const tops_gla_qk_norm_args& f = a->f;
  const bool rows = (int64_t)f.B * f.T > 0 && f.H + f.HK > 0;
  TOPS_CHECK_ARG(!rows || ((!f.H || (f.q && a->dq_out && a->dq)) && (!f.HK || (f.k && a->dk_out && a->dk))),
                 "qk_norm_bwd: q, k, their output gradients and dq, dk are required");
  const size_t need = tops_gla_qk_norm_rotary_bwd_workspace_size(a);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "qk_norm_bwd: workspace smaller than tops_gla_qk_norm_rotary_bwd_workspace_size()");
  P p = params(&f);
  p.dyq = a->dq_out; p.dyk = a->dk_out; p.dq = a->dq; p.dk = a->dk;
  for (int i = 0; i < 3; ++i) {
    p.dqs[i] = a->dq_out_strides[i];
    p.dks[i] = a->dk_out_strides[i];
  }
  p.part = need ? static_cast<float*>(a->workspace) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int blocks = 0;
  if (rows) {
    const int v = vector_of(p, dtype_bytes(f.dtype), true);
    split(p, v, kWant);
    const int64_t units = p.tokens * p.nhg, per_block = 8 * (32 / p.lanes);
    blocks = (int)std::min<int64_t>(kBwdBlocks, (units + per_block - 1) / per_block);
    LaunchTimer lt(st, "qk_norm_bwd");
    by_type(f.dtype, v, [&](auto t, auto vv, auto jj) {
      k_qk_bwd<decltype(t), decltype(vv)::value, decltype(jj)::value><<<blocks, 256, 0, st>>>(p);
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("qk_norm_bwd");
  }
  if (need) {
    LaunchTimer lt(st, "qk_norm_dw");
    k_qk_dw<<<(2 * f.K + 31) / 32, dim3(32, 32), 0, st>>>(blocks, f.K, f.w_dtype, static_cast<const float*>(a->workspace),
                                                          a->dq_weight, a->dk_weight);
    TOPS_CUDA_LAUNCH_CHECK("qk_norm_dw");
  }
  return TOPS_OK;
}

}  // extern "C"
