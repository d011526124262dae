// RMS norm of every query and key head with the position rotation in the same pass.  Per head
// row x of K elements, with s = 1 / sqrt(mean x^2 + eps):
//   n_i = x_i s w_i;   the first R elements are rotated in pairs (i, i') by the row's angle,
//   y_i = n_i cos - n_i' sin,  y_i' = n_i sin + n_i' cos     (i' = i + R/2, or i' = i + 1, i even)
// Backward: dn = the rotation by the opposite angle of dy, e = w dn, dw = sum dn x s,
//   dx = s (e - x s^2 mean(e x)).
//
// Nothing is reused between rows but the token's cosines and the weights, so HBM bounds it: a group of lanes owns a
// token and walks its heads, V elements a lane.  The heads' vectors come through a ring in shared memory, several heads
// ahead of their use and without registers; a rotated element's partner is read there from the other lane's column.
// 32768 tokens, 16 + 4 heads of 128 bf16, calls in a row: forward 70 us = 4.8 TB/s (issue 76 %), backward 120 us =
// 4.2 TB/s and 128 with the weights' sums (issue 65 %, HBM 48 %: 112 registers leave it 15 warps an SM).
#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace qkn {

struct P {
  int64_t tokens;
  int T, H, HK, K, R, pairs, wdtype, pos64, table;
  int lanes, hg, nhg;  // lanes of a row, heads of a unit, units of a token
  int wvec, tvec;      // the weights and the tables start on a vector
  float eps, inv_k;
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
  int p0;  // first partner's element (half-split); interleaved partners are inside the vector (V > 1)
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
    float c[V], s[V];
    if (p.tvec) {  // half is a multiple of V
      Vx<float, V>::load(ct + a, c);
      Vx<float, V>::load(st + a, s);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = ct[a + i];
        s[i] = st[a + i];
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      r.c[i] = inside ? c[i] : bad;
      r.s[i] = inside ? (low ? -sign : sign) * s[i] : bad;
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

// the sum of a b over V elements, two at a time
template <int V>
__device__ __forceinline__ float dot_n(const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    return a[0] * b[0];
  } else {
    float2 s = mul2(make_float2(a[0], a[1]), make_float2(b[0], b[1]));
#pragma unroll
    for (int i = 2; i < V; i += 2) s = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
    return s.x + s.y;
  }
}
template <int V>
__device__ __forceinline__ void fill(float (&r)[V], float v) {
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = v;
}

__device__ __forceinline__ int64_t position(const P& p, int b, int t) {
  if (!p.R || !p.pos) return t;
  return p.pos64 ? static_cast<const int64_t*>(p.pos)[b * p.pb + t] : static_cast<const int32_t*>(p.pos)[b * p.pb + t];
}

// A ring of head vectors: kThreads columns of J vectors for each of kSlots heads and each of M tensors.
constexpr int kThreads = 128, kAhead = 3, kSlots = kAhead + 1, kWarps = kThreads / 32;
template <typename T, int V, int J, int M>
struct Ring {
  Raw<T, V> v[kSlots][M][J][kThreads];
};

// The heads of a unit, one a turn: every lane of a warp takes every turn, since the sums are full-warp exchanges.  A walk
// goes over the heads of q, then of k, in one tensor (pointers, no products in the loop).
template <typename T>
struct Walk {
  const T *at, *k;
  int64_t qs, ks;
  int h;  // head of q, then of k behind them
  __device__ __forceinline__ Walk(const P& p, const void* q_, const int64_t (&sq)[3], const void* k_, const int64_t (&sk)[3],
                                  int b, int t, int h0)
      : k(static_cast<const T*>(k_) + b * sk[0] + t * sk[1]), qs(sq[2]), ks(sk[2]), h(h0) {
    at = h0 < p.H ? static_cast<const T*>(q_) + b * sq[0] + t * sq[1] + h0 * qs : k + (h0 - p.H) * ks;
  }
  __device__ __forceinline__ void next(const P& p) {
    at += h < p.H ? qs : ks;
    if (++h == p.H) at = k;
  }
};
template <typename T>
struct Out {
  T *at, *k;
  int h;
  __device__ __forceinline__ Out(const P& p, void* q_, void* k_, int64_t tok, int h0)
      : k(static_cast<T*>(k_) + tok * p.HK * p.K), h(h0) {
    at = h0 < p.H ? static_cast<T*>(q_) + (tok * p.H + h0) * p.K : k + (h0 - p.H) * p.K;
  }
  __device__ __forceinline__ void next(const P& p) {
    at += p.K;
    if (++h == p.H) at = k;
  }
};
__device__ __forceinline__ float group_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {  // selected, not branched over: the branch would cost a convergence each
    const float r = __shfl_xor_sync(0xffffffffu, v, o);
    v += lanes > o ? r : 0.f;
  }
  return v;
}

template <typename T, int V, int J>
__global__ void __launch_bounds__(kThreads) k_qk_fwd(const P p) {
  __shared__ Ring<T, V, J, 1> ring;
  const int tid = threadIdx.x, lane = tid & 31, l = lane & (p.lanes - 1), base = tid - l;
  const int rpw = 32 / p.lanes;
  const int64_t unit = ((int64_t)blockIdx.x * kWarps + (tid >> 5)) * rpw + lane / p.lanes;
  const bool live = unit < p.tokens * p.nhg;
  const int64_t tok = live ? unit / p.nhg : 0;
  const int h0 = live ? (int)(unit - tok * p.nhg) * p.hg : 0;
  const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
  const int turns = live ? min(p.hg, p.H + p.HK - h0) : 0;
  Walk<T> in(p, p.q, p.qs, p.k, p.ks, b, t, h0);
  Out<T> out_at(p, p.yq, p.yk, tok, h0);
  auto ask = [&](int i) {
    if (i < turns) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (e0 < p.K) {
          Raw<T, V>& to = ring.v[i % kSlots][0][j][tid];
          if constexpr (V == 1) to.load(in.at + e0);
          else copy_async<Raw<T, V>::B>(&to, in.at + e0);
        }
      }
      in.next(p);
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ask(i);
  const int64_t pos = position(p, b, t);
  Rot<V> rot[J];
  float w[J][V], pw[J][V];  // the weight times the cosine, and the partner's times the sine
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e0 = (l + j * p.lanes) * V;
    rot[j] = rotation<V>(p, e0 < p.K ? e0 : p.K, pos, 1.f);
  }
  int of = -1;  // whose weights they are
  for (int i = 0; i < p.hg; ++i) {
    copies_wait<kAhead - 1>();
    __syncwarp();  // the other lanes' copies too, and nobody reads the slot that is filled next
    ask(i + kAhead);
    const bool on = i < turns, isq = out_at.h < p.H;
    if (of != (int)isq) {
      of = isq;
      const void* wt = isq ? p.qw : p.kw;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        weights<T, V>(wt, p, (l + j * p.lanes) * V, w[j]);
        if (p.pairs && V > 1) {
#pragma unroll
          for (int c = 0; c < V; ++c) pw[j][c] = w[j][c ^ (V > 1 ? 1 : 0)];
        } else {
          weights<T, V>(wt, p, rot[j].p0, pw[j]);
        }
        mul_n<V>(w[j], w[j], rot[j].c);
        mul_n<V>(pw[j], pw[j], rot[j].s);
      }
    }
    float v[J][V], ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      fill<V>(v[j], 0.f);
      if (on && (l + j * p.lanes) * V < p.K) ring.v[i % kSlots][0][j][tid].get(v[j]);
      ss += dot_n<V>(v[j], v[j]);
    }
    ss = group_sum(ss, p.lanes);
    if (!on) continue;
    const float s = rsqrtf(fmaf(ss, p.inv_k, p.eps));
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e0 = (l + j * p.lanes) * V;
      if (e0 < p.K) {
        float out[V], o[V];
        mul_n<V>(out, v[j], w[j]);
        if (rot[j].on) {
          if (p.pairs && V > 1) {
#pragma unroll
            for (int c = 0; c < V; ++c) o[c] = v[j][c ^ (V > 1 ? 1 : 0)];
          } else {
            const int pc = rot[j].p0 / V;  // the partner's vector: lane pc % lanes, slot pc / lanes
            ring.v[i % kSlots][0][J == 1 ? 0 : pc / p.lanes][base + (J == 1 ? pc : pc & (p.lanes - 1))].get(o);
          }
          fma_n<V>(out, o, pw[j]);
        }
        float s_n[V];
        fill<V>(s_n, s);
        mul_n<V>(out, out, s_n);
        Vx<T, V>::store(out_at.at + e0, out);
      }
    }
    out_at.next(p);
  }
}

// Both sums of a row (x^2 and e x) come from the same loads.  Each block keeps its rows' dw terms and writes one partial
// row per weight.
template <typename T, int V, int J>
__global__ void __launch_bounds__(kThreads) k_qk_bwd(const P p) {
  __shared__ Ring<T, V, J, 2> ring;
  const int tid = threadIdx.x, lane = tid & 31, l = lane & (p.lanes - 1), base = tid - l, warp = tid >> 5;
  const int rpw = 32 / p.lanes;
  const int64_t units = p.tokens * p.nhg, step = (int64_t)gridDim.x * kWarps * rpw;
  const int64_t first = ((int64_t)blockIdx.x * kWarps + warp) * rpw;
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
    const int h0 = live ? (int)(unit - tok * p.nhg) * p.hg : 0;
    const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
    const int turns = live ? min(p.hg, p.H + p.HK - h0) : 0;
    Walk<T> in(p, p.q, p.qs, p.k, p.ks, b, t, h0), gin(p, p.dyq, p.dqs, p.dyk, p.dks, b, t, h0);
    Out<T> out_at(p, p.dq, p.dk, tok, h0);
    auto ask = [&](int i) {
      if (i < turns) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int e0 = (l + j * p.lanes) * V;
          if (e0 < p.K) {
            Raw<T, V>&tx = ring.v[i % kSlots][0][j][tid], &tg = ring.v[i % kSlots][1][j][tid];
            if constexpr (V == 1) {
              tx.load(in.at + e0);
              tg.load(gin.at + e0);
            } else {
              copy_async<Raw<T, V>::B>(&tx, in.at + e0);
              copy_async<Raw<T, V>::B>(&tg, gin.at + e0);
            }
          }
        }
        in.next(p);
        gin.next(p);
      }
      copies_commit();
    };
    __syncwarp();  // the unit before it has been read
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ask(i);
    const int64_t pos = position(p, b, t);
    Rot<V> rot[J];
    float w[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e0 = (l + j * p.lanes) * V;
      rot[j] = rotation<V>(p, e0 < p.K ? e0 : p.K, pos, -1.f);
    }
    int of = -1;
    for (int i = 0; i < p.hg; ++i) {
      copies_wait<kAhead - 1>();
      __syncwarp();
      ask(i + kAhead);
      const bool on = i < turns, isq = out_at.h < p.H;
      if (of != (int)isq) {
        of = isq;
#pragma unroll
        for (int j = 0; j < J; ++j) weights<T, V>(isq ? p.qw : p.kw, p, (l + j * p.lanes) * V, w[j]);
      }
      float v[J][V], e[J][V], ew[J][V], ss = 0.f, ex = 0.f;  // x, the gradient turned back, and that times the weight
#pragma unroll
      for (int j = 0; j < J; ++j) {
        fill<V>(v[j], 0.f);
        fill<V>(e[j], 0.f);
        if (on && (l + j * p.lanes) * V < p.K) {
          ring.v[i % kSlots][0][j][tid].get(v[j]);
          ring.v[i % kSlots][1][j][tid].get(e[j]);
          if (rot[j].on) {
            float o[V];
            if (p.pairs && V > 1) {
#pragma unroll
              for (int c = 0; c < V; ++c) o[c] = e[j][c ^ (V > 1 ? 1 : 0)];
            } else {
              const int pc = rot[j].p0 / V;
              ring.v[i % kSlots][1][J == 1 ? 0 : pc / p.lanes][base + (J == 1 ? pc : pc & (p.lanes - 1))].get(o);
            }
            mul_n<V>(e[j], e[j], rot[j].c);
            fma_n<V>(e[j], o, rot[j].s);
          }
        }
        mul_n<V>(ew[j], e[j], w[j]);
        ss += dot_n<V>(v[j], v[j]);
        ex += dot_n<V>(ew[j], v[j]);
      }
      ss = group_sum(ss, p.lanes);
      ex = group_sum(ex, p.lanes);
      if (!on) continue;
      const float s = rsqrtf(fmaf(ss, p.inv_k, p.eps));
      const float m = s * (s * (s * ex)) * p.inv_k;  // in this order every product is in range: x s is of order 1
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e0 = (l + j * p.lanes) * V;
        if (e0 < p.K) {
          float out[V], c[V];
          fill<V>(c, -m);
          mul_n<V>(out, v[j], c);
          fill<V>(c, s);
          fma_n<V>(out, ew[j], c);
          mul_n<V>(v[j], v[j], c);
          Vx<T, V>::store(out_at.at + e0, out);
        }
        if (isq) fma_n<V>(dw[0][j], e[j], v[j]);
        else fma_n<V>(dw[1][j], e[j], v[j]);
      }
      out_at.next(p);
    }
  }
  if (p.part == nullptr) return;
  // rows of the block: fold the groups of a warp, then the warps, in a fixed order
  __syncthreads();
  float(*red)[2][256] = reinterpret_cast<float(*)[2][256]>(&ring);  // [kWarps]
  static_assert(sizeof(ring) >= kWarps * 2 * 256 * sizeof(float), "the ring holds the partial sums");
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
  for (int i = threadIdx.x; i < 2 * p.K; i += kThreads) {
    const int g = i / p.K, el = i - g * p.K;
    float a = 0.f;
    for (int w = 0; w < kWarps; ++w) a += red[w][g][el];
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
  if (a->B > kMaxRows || a->T > kMaxRows || a->H > kMaxChannels || a->HK > kMaxChannels)
    return fail(TOPS_ERR_UNSUPPORTED, "qk_norm: too many rows or heads");
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
  p.eps = a->eps; p.inv_k = 1.f / (float)a->K;
  p.q = a->q; p.k = a->k; p.qw = a->q_weight; p.kw = a->k_weight;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_strides[i];
    p.ks[i] = a->k_strides[i];
  }
  p.cos = a->cos_table; p.sin = a->sin_table;
  p.pos = a->positions; p.pb = a->positions_stride_b;
  p.yq = a->q_out; p.yk = a->k_out;
  p.tvec = aligned_to(a->cos_table, 16) && aligned_to(a->sin_table, 16);
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
constexpr int kBwdBlocks = 148 * 4;

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
  const int64_t units = p.tokens * p.nhg, per_block = kWarps * (32 / p.lanes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "qk_norm_fwd");
  by_type(a->dtype, v, [&](auto t, auto vv, auto jj) {
    k_qk_fwd<decltype(t), decltype(vv)::value, decltype(jj)::value>
        <<<(unsigned)((units + per_block - 1) / per_block), kThreads, 0, st>>>(p);
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
    const int64_t units = p.tokens * p.nhg, per_block = kWarps * (32 / p.lanes);
    blocks = (int)std::min<int64_t>(kBwdBlocks, (units + per_block - 1) / per_block);
    LaunchTimer lt(st, "qk_norm_bwd");
    by_type(f.dtype, v, [&](auto t, auto vv, auto jj) {
      k_qk_bwd<decltype(t), decltype(vv)::value, decltype(jj)::value><<<blocks, kThreads, 0, st>>>(p);
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
