// Selective state space scan.  Per channel d with N states, delta = softplus(dt + bias) or dt + bias:
//   h_t[n] = exp(delta_t A[d, n]) h_{t-1}[n] + delta_t x_t B_t[n],   y_t = sum_n C_t[n] h_t[n] + D x_t,
//   out = y silu(z)          (B, C shared by the D / G channels of a group)
// Backward, with dy = dout silu(z) and g_t = C_t dy_t + a_{t+1} g_{t+1} (the gradient of h_t):
//   dC_t = sum_d dy h,  dB_t = sum_d g delta x,  dx = delta sum_n g B + D dy,
//   ddelta = x sum_n g B + sum_n A a g h_{t-1},  dA = sum_t delta a g h_{t-1},  dh0 = a_1 g_1
#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace ssm {

constexpr int CK = 16;  // rows between saved states

struct P {
  int B, T, D, N, G, S, softplus;
  const int32_t* cu;
  const void *x, *dt, *z, *bm, *cm;
  int64_t xs[2], ds[2], zs[2], bs[2], cs[2];
  const float *A, *skip, *bias, *h0;
  void* y;
  float *ht, *states;
  // backward
  const void* dout;
  int64_t os[2];
  const float* dht;
  void *dx, *ddt, *dz;
  float* pbc;   // [G][parts][B T][2][N]: dB, dC of one part of a group's channels
  int parts;
  float* pa;    // [B][D][N] dA of one batch row
  float* pd;    // [B][2][D] dD, dbias of one batch row
  float* dh0;
};

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(__expf(v)); }

template <typename T, int NP>
__global__ void __launch_bounds__(128) k_scan_fwd(const P p) {
  const int rep = p.D / p.G, nblk = (rep + 127) / 128, grp = blockIdx.x / nblk, b = blockIdx.y;
  const int dg = (blockIdx.x - grp * nblk) * 128 + threadIdx.x;  // channel of the group
  if (dg >= rep) return;
  const int d = grp * rep + dg;
  float A[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A[n] = n < p.N ? p.A[(int64_t)d * p.N + n] : 0.f;
    h[n] = 0.f;
  }
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  SeqAt q{b, 0, p.T};
  if (p.cu) q.e = 0;
  if (!p.cu && p.h0)
    for (int n = 0; n < NP; ++n) h[n] = n < p.N ? p.h0[((int64_t)b * p.D + d) * p.N + n] : 0.f;
  const int nck = (p.T + CK - 1) / CK;
  for (int t = 0; t < p.T; ++t) {
    const int64_t yo = ((int64_t)b * p.T + t) * p.D + d;
    if (p.cu && (t >= q.e || q.n < 0)) {
      q = seq_at(p.cu, p.S, p.T, t);
      for (int n = 0; n < NP; ++n)
        h[n] = (q.n >= 0 && p.h0 && n < p.N) ? p.h0[((int64_t)q.n * p.D + d) * p.N + n] : 0.f;
    }
    if (p.states && t % CK == 0)
      for (int n = 0; n < NP; ++n)
        if (n < p.N) p.states[(((int64_t)b * nck + t / CK) * p.D + d) * p.N + n] = h[n];
    if (q.n < 0) {
      static_cast<T*>(p.y)[yo] = from_f<T>(0.f);
      continue;
    }
    const float x = to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + t * p.xs[1] + d]);
    float dl = to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + t * p.ds[1] + d]) + bias;
    if (p.softplus) dl = softplus(dl);
    const T* Bt = static_cast<const T*>(p.bm) + b * p.bs[0] + t * p.bs[1] + grp * p.N;
    const T* Ct = static_cast<const T*>(p.cm) + b * p.cs[0] + t * p.cs[1] + grp * p.N;
    float y = 0.f;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      if (n < p.N) {
        h[n] = fmaf(__expf(dl * A[n]), h[n], dl * x * to_f<T>(Bt[n]));
        y = fmaf(to_f<T>(Ct[n]), h[n], y);
      }
    }
    y = fmaf(skip, x, y);
    if (p.z) {
      const float z = to_f<T>(static_cast<const T*>(p.z)[b * p.zs[0] + t * p.zs[1] + d]);
      y *= z * fast_sigmoid(z);
    }
    static_cast<T*>(p.y)[yo] = from_f<T>(y);
    if (p.cu && p.ht && t == q.e - 1)
      for (int n = 0; n < NP; ++n)
        if (n < p.N) p.ht[((int64_t)q.n * p.D + d) * p.N + n] = h[n];
  }
  if (!p.cu && p.ht)
    for (int n = 0; n < NP; ++n)
      if (n < p.N) p.ht[((int64_t)b * p.D + d) * p.N + n] = h[n];
}

// Packed sequences without rows: their final state is their initial one (and its gradient the
// final state's).
__global__ void k_scan_empty(int S, int T, int64_t DN, const int32_t* __restrict__ cu, const float* __restrict__ from,
                             float* __restrict__ to) {
  const int n = blockIdx.y;
  if (min(cu[n + 1], T) > max(cu[n], 0)) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < DN; i += (int64_t)gridDim.x * blockDim.x)
    to[n * DN + i] = from ? from[n * DN + i] : 0.f;
}

template <typename T, int NP>
__global__ void __launch_bounds__(128) k_scan_bwd(const P p) {
  const int rep = p.D / p.G, nblk = (rep + 127) / 128, grp = blockIdx.x / nblk, b = blockIdx.y;
  const int dg = (blockIdx.x - grp * nblk) * 128 + threadIdx.x;
  const bool on = dg < rep;
  const int d = grp * rep + dg;
  const int lane = threadIdx.x & 31;
  const int nck = (p.T + CK - 1) / CK;
  float A[NP], g[NP], dA[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A[n] = on && n < p.N ? p.A[(int64_t)d * p.N + n] : 0.f;
    g[n] = dA[n] = 0.f;
    if (!p.cu && p.dht && on && n < p.N) g[n] = p.dht[((int64_t)b * p.D + d) * p.N + n];
  }
  const float bias = on && p.bias ? p.bias[d] : 0.f, skip = on && p.skip ? p.skip[d] : 0.f;
  float dskip = 0.f, dbias = 0.f;
  float hb[CK][NP], hs[CK + 1][NP];  // the state before and after each row (a sequence's first row starts anew)
  for (int c = nck - 1; c >= 0; --c) {
    const int s = c * CK, e = min(s + CK, p.T);
    for (int n = 0; n < NP; ++n)
      hs[0][n] = on && n < p.N ? p.states[(((int64_t)b * nck + c) * p.D + d) * p.N + n] : 0.f;
    for (int t = s; t < e; ++t) {  // the states of the chunk again
      SeqAt q{b, 0, p.T};
      if (p.cu) q = seq_at(p.cu, p.S, p.T, t);
      float x = 0.f, dl = 0.f;
      if (on && q.n >= 0) {
        x = to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + t * p.xs[1] + d]);
        dl = to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + t * p.ds[1] + d]) + bias;
        if (p.softplus) dl = softplus(dl);
      }
      const T* Bt = static_cast<const T*>(p.bm) + b * p.bs[0] + t * p.bs[1] + grp * p.N;
      for (int n = 0; n < NP; ++n) {
        float h = hs[t - s][n];
        if (p.cu && t == q.s) h = (on && q.n >= 0 && p.h0 && n < p.N) ? p.h0[((int64_t)q.n * p.D + d) * p.N + n] : 0.f;
        hb[t - s][n] = h;
        hs[t - s + 1][n] = q.n >= 0 && n < p.N ? fmaf(__expf(dl * A[n]), h, dl * x * to_f<T>(Bt[n])) : 0.f;
      }
    }
    for (int t = e - 1; t >= s; --t) {
      SeqAt q{b, 0, p.T};
      if (p.cu) q = seq_at(p.cu, p.S, p.T, t);
      const bool row = q.n >= 0;
      const int64_t yo = ((int64_t)b * p.T + t) * p.D + d;
      float x = 0.f, v = 0.f, dl = 0.f, dy = 0.f, dout = 0.f, z = 0.f, zs = 1.f;
      if (on && row) {
        x = to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + t * p.xs[1] + d]);
        v = to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + t * p.ds[1] + d]) + bias;
        dl = p.softplus ? softplus(v) : v;
        dout = dy = to_f<T>(static_cast<const T*>(p.dout)[b * p.os[0] + t * p.os[1] + d]);
        if (p.z) {
          z = to_f<T>(static_cast<const T*>(p.z)[b * p.zs[0] + t * p.zs[1] + d]);
          zs = fast_sigmoid(z);
          dy = dout * z * zs;
        }
      }
      if (p.cu && t == q.e - 1)
        for (int n = 0; n < NP; ++n)
          g[n] = (on && row && p.dht && n < p.N) ? p.dht[((int64_t)q.n * p.D + d) * p.N + n] : 0.f;
      const T* Bt = static_cast<const T*>(p.bm) + b * p.bs[0] + t * p.bs[1] + grp * p.N;
      const T* Ct = static_cast<const T*>(p.cm) + b * p.cs[0] + t * p.cs[1] + grp * p.N;
      float gB = 0.f, aw = 0.f, y = skip * x;
      for (int n = 0; n < NP; ++n) {
        float vb = 0.f, vc = 0.f;
        if (on && row && n < p.N) {
          const float Bn = to_f<T>(Bt[n]), Cn = to_f<T>(Ct[n]), h = hs[t - s + 1][n], hp = hb[t - s][n];
          const float gt = fmaf(Cn, dy, g[n]);
          const float r = __expf(dl * A[n]) * gt, w = r * hp;
          gB = fmaf(gt, Bn, gB);
          y = fmaf(Cn, h, y);
          aw = fmaf(A[n], w, aw);
          dA[n] = fmaf(dl, w, dA[n]);
          g[n] = r;
          vb = gt * dl * x;
          vc = dy * h;
        }
        for (int o = 16; o > 0; o >>= 1) {
          vb += __shfl_xor_sync(0xffffffffu, vb, o);
          vc += __shfl_xor_sync(0xffffffffu, vc, o);
        }
        if (lane == 0 && n < p.N) {
          float* o = p.pbc + ((((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * p.B + b) * p.T + t) * 2 * p.N;
          o[n] = vb;
          o[p.N + n] = vc;
        }
      }
      if (on) {
        float dv = x * gB + aw;
        if (p.softplus) dv *= 1.f / (1.f + __expf(-v));
        dskip = fmaf(dy, x, dskip);
        if (!row) dv = 0.f;
        dbias += dv;
        static_cast<T*>(p.dx)[yo] = from_f<T>(row ? fmaf(dl, gB, skip * dy) : 0.f);
        static_cast<T*>(p.ddt)[yo] = from_f<T>(dv);
        if (p.dz) static_cast<T*>(p.dz)[yo] = from_f<T>(dout * y * zs * fmaf(z, 1.f - zs, 1.f));
        if (p.cu && p.dh0 && row && t == q.s)
          for (int n = 0; n < NP; ++n)
            if (n < p.N) p.dh0[((int64_t)q.n * p.D + d) * p.N + n] = g[n];
      }
    }
  }
  if (!on) return;
  for (int n = 0; n < NP; ++n)
    if (n < p.N) {
      p.pa[((int64_t)b * p.D + d) * p.N + n] = dA[n];
      if (!p.cu && p.dh0) p.dh0[((int64_t)b * p.D + d) * p.N + n] = g[n];
    }
  p.pd[((int64_t)b * 2) * p.D + d] = dskip;
  p.pd[((int64_t)b * 2 + 1) * p.D + d] = dbias;
}

// dB, dC [B, T, G, N] = the parts' sums, in a fixed order
template <typename T>
__global__ void k_scan_bc(const P p, T* __restrict__ dB, T* __restrict__ dC) {
  const int64_t rows = (int64_t)p.B * p.T, per = rows * 2 * p.N;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int grp = blockIdx.y;
  if (i >= per) return;
  float s = 0.f;
  for (int k = 0; k < p.parts; ++k) s += p.pbc[((int64_t)grp * p.parts + k) * per + i];
  const int64_t row = i / (2 * p.N);
  const int c = (int)(i - row * 2 * p.N);
  T* o = c < p.N ? dB : dC;
  o[(row * p.G + grp) * p.N + (c < p.N ? c : c - p.N)] = from_f<T>(s);
}

// out[i] = sum over parts of part[k][i], in a fixed order
__global__ void k_scan_sum(int parts, int64_t n, int64_t stride, const float* __restrict__ part, float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += part[k * stride + i];
  out[i] = s;
}

// One token of each of B rows: the state is read and written once (HBM bounds it).
template <typename T>
__global__ void __launch_bounds__(128) k_scan_step(const P p) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (id >= (int64_t)p.B * p.D) return;
  const int b = (int)(id / p.D), d = (int)(id - (int64_t)b * p.D), grp = d / (p.D / p.G);
  const float x = to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + d]);
  float dl = to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + d]) + (p.bias ? p.bias[d] : 0.f);
  if (p.softplus) dl = softplus(dl);
  const T* Bt = static_cast<const T*>(p.bm) + b * p.bs[0] + grp * p.N;
  const T* Ct = static_cast<const T*>(p.cm) + b * p.cs[0] + grp * p.N;
  float y = p.skip ? p.skip[d] * x : 0.f;
  for (int n = 0; n < p.N; ++n) {
    const float h = fmaf(__expf(dl * p.A[(int64_t)d * p.N + n]), p.h0[id * p.N + n], dl * x * to_f<T>(Bt[n]));
    p.ht[id * p.N + n] = h;
    y = fmaf(to_f<T>(Ct[n]), h, y);
  }
  if (p.z) {
    const float z = to_f<T>(static_cast<const T*>(p.z)[b * p.zs[0] + d]);
    y *= z * fast_sigmoid(z);
  }
  static_cast<T*>(p.y)[id] = from_f<T>(y);
}

int check(const tops_gla_scan_args* a) {
  TOPS_CHECK_ARG(a != nullptr, "ssm_scan: args is NULL");
  TOPS_CHECK_ARG(a->B >= 0 && a->T >= 0 && a->D > 0 && a->S >= 0, "ssm_scan: negative or zero dimension");
  TOPS_CHECK_ARG(a->G > 0 && a->D % a->G == 0, "ssm_scan: D must be a multiple of G");
  if (a->N < 1 || a->N > 64) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: a channel must have 1 to 64 states");
  TOPS_CHECK_ARG(dtype_known(a->dtype), "ssm_scan: unknown dtype");
  if (a->B > 65535) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: at most 65535 batch rows");
  if (a->cu_seqlens) {
    TOPS_CHECK_ARG(a->B == 1, "ssm_scan: cu_seqlens requires B == 1");
    TOPS_CHECK_ARG(a->S >= 1 && a->S <= 65535, "ssm_scan: cu_seqlens requires 1 to 65535 sequences");
  } else {
    TOPS_CHECK_ARG(a->S == a->B, "ssm_scan: S must equal B without cu_seqlens");
  }
  return TOPS_OK;
}

P params(const tops_gla_scan_args* a) {
  P p{};
  p.B = a->B; p.T = a->T; p.D = a->D; p.N = a->N; p.G = a->G; p.S = a->S; p.softplus = a->softplus;
  p.cu = a->cu_seqlens;
  p.x = a->x; p.dt = a->dt; p.z = a->z; p.bm = a->Bm; p.cm = a->Cm;
  for (int i = 0; i < 2; ++i) {
    p.xs[i] = a->x_strides[i];
    p.ds[i] = a->dt_strides[i];
    p.zs[i] = a->z_strides[i];
    p.bs[i] = a->b_strides[i];
    p.cs[i] = a->c_strides[i];
  }
  p.A = a->A; p.skip = a->skip; p.bias = a->dt_bias; p.h0 = a->h0;
  p.y = a->y; p.ht = a->ht; p.states = a->states;
  return p;
}

// bump allocator over the caller's workspace (dry run when base == nullptr)
struct Carve {
  char* base;
  size_t used = 0;
  float* take(size_t count) {
    used = (used + 255) & ~size_t(255);
    float* p = base ? reinterpret_cast<float*>(base + used) : nullptr;
    used += count * sizeof(float);
    return p;
  }
};

size_t carve_bwd(P& p, void* ws) {
  Carve c{static_cast<char*>(ws)};
  p.parts = (p.D / p.G + 127) / 128 * 4;
  p.pbc = c.take((size_t)p.G * p.parts * p.B * p.T * 2 * p.N);
  p.pa = c.take((size_t)p.B * p.D * p.N);
  p.pd = c.take((size_t)p.B * 2 * p.D);
  return c.used;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == TOPS_F32) return f(float());
  if (dtype == TOPS_BF16) return f(__nv_bfloat16());
  return f(__half());
}

int empty_states(const P& p, const float* from, float* to, cudaStream_t st) {
  if (!p.cu || !to) return TOPS_OK;
  LaunchTimer lt(st, "ssm_scan_empty");
  const int64_t dn = (int64_t)p.D * p.N;
  k_scan_empty<<<dim3((unsigned)std::min<int64_t>((dn + 255) / 256, 64), p.S), 256, 0, st>>>(p.S, p.T, dn, p.cu, from, to);
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_empty");
  return TOPS_OK;
}

}  // namespace ssm
}  // namespace tops

using namespace tops;
using namespace tops::ssm;

extern "C" {

TOPS_API size_t tops_gla_ssm_scan_states_size(const tops_gla_scan_args* a) {
  if (check(a) != TOPS_OK) return 0;
  return (size_t)a->B * ((a->T + CK - 1) / CK) * a->D * a->N * sizeof(float);
}

TOPS_API size_t tops_gla_ssm_scan_fwd_workspace_size(const tops_gla_scan_args* a) {
  if (check(a) != TOPS_OK) return 0;
  return 0;
}

TOPS_API int tops_gla_ssm_scan_fwd(const tops_gla_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  const bool rows = (int64_t)a->B * a->T > 0;
  TOPS_CHECK_ARG(!rows || (a->x && a->dt && a->Bm && a->Cm && a->A && a->y), "ssm_scan_fwd: x, dt, B, C, A and y are required");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const P p = params(a);
  if (int rc = empty_states(p, p.h0, p.ht, st)) return rc;
  if (p.B == 0 || (!rows && !p.ht)) return TOPS_OK;
  LaunchTimer lt(st, "ssm_scan_fwd");
  const dim3 grid((p.D / p.G + 127) / 128 * p.G, p.B);
  by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if (p.N <= 16) k_scan_fwd<T, 16><<<grid, 128, 0, st>>>(p);
    else k_scan_fwd<T, 64><<<grid, 128, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_fwd");
  return TOPS_OK;
}

TOPS_API size_t tops_gla_ssm_scan_bwd_workspace_size(const tops_gla_scan_bwd_args* a) {
  if (a == nullptr || check(&a->f) != TOPS_OK) return 0;
  P p = params(&a->f);
  return carve_bwd(p, nullptr);
}

TOPS_API int tops_gla_ssm_scan_bwd(const tops_gla_scan_bwd_args* a, void* stream) {
  TOPS_CHECK_ARG(a != nullptr, "ssm_scan_bwd: args is NULL");
  if (int rc = check(&a->f)) return rc;
  const tops_gla_scan_args& f = a->f;
  const bool rows = (int64_t)f.B * f.T > 0;
  TOPS_CHECK_ARG(!rows || (f.x && f.dt && f.Bm && f.Cm && f.A && f.states && a->dout && a->dx && a->ddt && a->dB && a->dC),
                 "ssm_scan_bwd: x, dt, B, C, A, states, dout and the gradients of x, dt, B and C are required");
  TOPS_CHECK_ARG(!rows || !f.z || a->dz, "ssm_scan_bwd: z needs dz");
  P p = params(&f);
  const size_t need = carve_bwd(p, a->workspace);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "ssm_scan_bwd: workspace smaller than tops_gla_ssm_scan_bwd_workspace_size()");
  p.dout = a->dout; p.os[0] = a->dout_strides[0]; p.os[1] = a->dout_strides[1];
  p.dht = a->dht; p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz; p.dh0 = a->dh0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = empty_states(p, p.dht, p.dh0, st)) return rc;
  if (p.B > 0) {
    LaunchTimer lt(st, "ssm_scan_bwd");
    const dim3 grid((p.D / p.G + 127) / 128 * p.G, p.B);
    by_type(f.dtype, [&](auto t) {
      using T = decltype(t);
      if (p.N <= 16) k_scan_bwd<T, 16><<<grid, 128, 0, st>>>(p);
      else k_scan_bwd<T, 64><<<grid, 128, 0, st>>>(p);
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_bwd");
  }
  if (rows) {
    LaunchTimer lt(st, "ssm_scan_bc");
    const int64_t per = (int64_t)p.B * p.T * 2 * p.N;
    by_type(f.dtype, [&](auto t) {
      using T = decltype(t);
      k_scan_bc<T><<<dim3((unsigned)((per + 255) / 256), p.G), 256, 0, st>>>(p, static_cast<T*>(a->dB), static_cast<T*>(a->dC));
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_bc");
  }
  const struct { int64_t n, stride; const float* part; float* out; } sums[] = {
      {(int64_t)p.D * p.N, (int64_t)p.D * p.N, p.pa, a->dA}, {p.D, 2 * (int64_t)p.D, p.pd, a->dskip},
      {p.D, 2 * (int64_t)p.D, p.pd + p.D, a->ddt_bias}};
  for (const auto& s : sums) {
    if (!s.out) continue;
    LaunchTimer lt(st, "ssm_scan_sum");
    k_scan_sum<<<(unsigned)((s.n + 255) / 256), 256, 0, st>>>(p.B, s.n, s.stride, s.part, s.out);
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_sum");
  }
  return TOPS_OK;
}

TOPS_API int tops_gla_ssm_scan_step(const tops_gla_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  TOPS_CHECK_ARG(a->T == 1 && !a->cu_seqlens, "ssm_scan_step: T must be 1, without cu_seqlens");
  if (a->B == 0) return TOPS_OK;
  TOPS_CHECK_ARG(a->x && a->dt && a->Bm && a->Cm && a->A && a->h0 && a->y && a->ht,
                 "ssm_scan_step: x, dt, B, C, A, h0, y and ht are required");
  const P p = params(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "ssm_scan_step");
  by_type(a->dtype, [&](auto t) {
    k_scan_step<decltype(t)><<<(unsigned)(((int64_t)p.B * p.D + 127) / 128), 128, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_step");
  return TOPS_OK;
}

}  // extern "C"
