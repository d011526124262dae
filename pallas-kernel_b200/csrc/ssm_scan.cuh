// Selective state space scan.  Per channel d with N states, delta = softplus(dt + bias) or dt + bias:
//   h_t[n] = exp(delta_t A[d, n]) h_{t-1}[n] + delta_t x_t B_t[n],   y_t = sum_n C_t[n] h_t[n] + D x_t,
//   out = y silu(z)          (B, C shared by the D / G channels of a group)
// Backward, with dy = dout silu(z) and g_t = C_t dy_t + a_{t+1} g_{t+1} (the gradient of h_t):
//   dC_t = sum_d dy h,  dB_t = sum_d g delta x,  dx = delta sum_n g B + D dy,
//   ddelta = x sum_n g B + sum_n A a g h_{t-1},  dA = sum_t delta a g h_{t-1},  dh0 = a_1 g_1
//
// One exponential per (row, channel, state): at N = 16 the exponential unit (16 a clock and SM) takes the
// forward almost three times the time of its bytes; the backward fills no single unit (issue 55 %, shared
// memory 60 %).  So:
//  * a thread owns NT states of one channel and keeps them, A and their gradients in registers over all rows; LN
//    lanes share a channel and the other lanes are other channels;
//  * what a row needs once per channel (delta, delta x, dy) or once per state (B, C) is computed once per
//    block, a tile of rows ahead, into shared memory; the tile's elementwise work (softplus, gates,
//    rounding, 8- or 16-byte accesses) is spread over all threads, its loads issued one tile early;
//  * sums over the lanes of a channel (y, and the backward's) and over channels (dB, dC) are folded for
//    several rows at a time, so that each exchange halves the values that a lane still carries;
//  * arithmetic on state pairs is packed (fma.rn.f32x2), which halves its issue slots.
// Where B x D is too small for all SMs, the rows are split into segments: a first pass gives each segment's
// decay and its state from zero, a small kernel chains them, and the main pass starts every segment from its
// own state.  That costs the exponentials twice.
#pragma once

#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace ssm {

// Rows between saved states: 4 N / 8 bytes a row and channel, as much as two fp32 values at N = 16.  The backward
// computes the states between them again; with 16 rows between them an earlier form of it swept more rows twice (1112
// against 1088 us; not measured again on the present form).
constexpr int CK = 8;

struct P {
  int B, T, D, N, G, S, softplus;
  const int32_t* cu;
  const void *x, *dt, *z, *bm, *cm;
  int64_t xs[2], ds[2], zs[2], bs[2], cs[2];
  const float *A, *skip, *bias, *h0;
  void* y;
  float *ht, *states;
  int vx, vd, vz, vb, vc, vy, vo, vg;  // four elements of that tensor may be read (written) at once
  // segments of the rows
  int seg, nseg;
  float* carry;   // [B][nseg][D][N]: state (gradient) of a segment from zero, then the one it starts from
  float* sdelta;  // [B][nseg][D]: sum of delta over a segment
  int* broken;    // [nseg]: a sequence begins (ends) in the segment: nothing passes through it
  // backward
  const void* dout;
  int64_t os[2];
  const float* dht;
  void *dx, *ddt, *dz;
  float* pbc;   // [G][parts][B T][2][N]: dB, dC of one part of a group's channels
  int parts;
  float* pa;    // [B nseg][D][N]: dA of one segment
  float* pd;    // [B nseg][2][D]: dD, dbias of one segment
  float* dh0;
};

constexpr float kLn2 = 0.69314718055994531f;
// ex2.approx errs by -2e-8 on average where decays lie (against 64 bits, arguments -1 .. -0.002), and a state's
// error is that times the rows it remembers: the exponent's multiply-add takes the mean error back.  dA of states that
// remember 60 to 200 rows: 1.7 .. 2.8e-6 off without it, 0.4 .. 0.7e-6 with it; states that remember 1000 rows lie
// outside that range and gain nothing (1.0e-6 without, 1.8e-6 with it); outputs 0.93e-6 and 0.65e-6.
constexpr float kEx2Mean = 2.0e-8f * kLog2e;

// exp(delta A) of a pair, A given times log2(e)
__device__ __forceinline__ float2 decay2(float delta, float2 A) {
  const float2 e = fma2(dup(delta), A, dup(kEx2Mean));
  return make_float2(ex2(e.x), ex2(e.y));
}

// softplus(v) = max(v, 0) + log1p(w), w = exp(-|v|) in (0, 1], of a pair.  log1p(w) = w q(w) with q the interpolant of
// log1p(w) / w in ten Chebyshev nodes of [0, 1]: off by 1e-7 relative (in fp32, also for the smallest w), nine packed
// multiply-adds for two channels and no second use of the exponential unit.
__device__ __forceinline__ float2 softplus2(float2 v) {
  const float2 w = make_float2(ex2(-kLog2e * fabsf(v.x)), ex2(-kLog2e * fabsf(v.y)));
  float2 q = dup(-3.176057013e-03f);
  q = fma2(q, w, dup(1.954252832e-02f));
  q = fma2(q, w, dup(-5.637361482e-02f));
  q = fma2(q, w, dup(1.054362357e-01f));
  q = fma2(q, w, dup(-1.526966691e-01f));
  q = fma2(q, w, dup(1.966327429e-01f));
  q = fma2(q, w, dup(-2.495161593e-01f));
  q = fma2(q, w, dup(3.332971036e-01f));
  q = fma2(q, w, dup(-4.999989271e-01f));
  q = fma2(q, w, dup(1.f));
  return fma2(w, q, make_float2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
}
__device__ __forceinline__ float softplus(float v) { return softplus2(make_float2(v, v)).x; }

// Sums of V values over the L lanes that differ in bits m0, 2 m0, ... of the lane: as long as a lane carries
// several, an exchange halves them.  Returns the first index of the V >> log2(L) (at least one) that this lane holds.
template <int V, int L, int M0>
__device__ __forceinline__ int fold(float (&v)[V], int lane) {
  int off = 0;
  int cnt = V;
#pragma unroll
  for (int m = M0; m < L * M0; m <<= 1) {
    const bool up = lane & m;
    if (cnt > 1) {
      cnt >>= 1;
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        if (i < cnt) {
          const float send = up ? v[i] : v[i + cnt], keep = up ? v[i + cnt] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m);
        }
      if (up) off += cnt;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    }
  }
  return off;
}

// Four elements of T as they lie in memory (those at `valid` and beyond are zero).  They are taken apart where they
// are used, a tile later: a load's registers may not be touched before.
template <typename T>
struct Quad {
  uint32_t w[sizeof(T)];  // 4 sizeof(T) bytes
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t h = (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]);
      if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(h));
      else return __uint_as_float((uint32_t)h << 16);
    }
  }
};
template <typename T>
__device__ __forceinline__ void quad_load(const T* p, bool vec, int valid, Quad<T>& q) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) q.w[i] = 0;
  if (vec) {
    if (valid >= 4) {
      if constexpr (sizeof(T) == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        q.w[0] = v.x; q.w[1] = v.y; q.w[2] = v.z; q.w[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        q.w[0] = v.x; q.w[1] = v.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < valid) {
        if constexpr (sizeof(T) == 4) q.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        else q.w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ void quad_store(T* p, bool vec, int valid, const float (&r)[4]) {
  if (vec && valid >= 4) {
    Vx<T, 4>::store(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = from_f<T>(r[i]);
  }
}

// NT states of one channel in global memory (those at N and beyond are not there)
template <int NT>
__device__ __forceinline__ void states_load(const float* p, int n0, int N, float2 (&h)[NT / 2]) {
#pragma unroll
  for (int i = 0; i < NT / 2; ++i)
    h[i] = make_float2(n0 + 2 * i < N ? p[n0 + 2 * i] : 0.f, n0 + 2 * i + 1 < N ? p[n0 + 2 * i + 1] : 0.f);
}
template <int NT>
__device__ __forceinline__ void states_store(float* p, int n0, int N, const float2 (&h)[NT / 2]) {
  if (NT == 4 && N % 4 == 0) {
    if (n0 < N) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0].x, h[0].y, h[NT / 2 - 1].x, h[NT / 2 - 1].y);
    return;
  }
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) {
    if (n0 + 2 * i < N) p[n0 + 2 * i] = h[i].x;
    if (n0 + 2 * i + 1 < N) p[n0 + 2 * i + 1] = h[i].y;
  }
}
template <int NT>
__device__ __forceinline__ void pairs_load(const float* p, float2 (&v)[NT / 2]) {
  if constexpr (NT == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(f.x, f.y);
    v[1] = make_float2(f.z, f.w);
  } else {
    v[0] = *reinterpret_cast<const float2*>(p);
  }
}

// what a row is to packed sequences
enum { kFirst = 1, kLast = 2, kNone = 4 };
__device__ __forceinline__ int row_flags(const P& p, int t, int& n) {
  const SeqAt q = seq_at(p.cu, p.S, p.T, t);
  n = q.n;
  return q.n < 0 ? kNone : (t == q.s ? kFirst : 0) | (t == q.e - 1 ? kLast : 0);
}

// own + 2^e c.  Decays grow where A and delta have one sign; over a segment 2^e alone may pass fp32 there: a state of
// zero stays zero, and a small one is multiplied by the root twice.
__device__ __forceinline__ float carried(float e, float c, float own) {
  if (e <= 126.f) return fmaf(ex2(e), c, own);
  const float root = ex2(0.5f * e);
  return c == 0.f ? own : fmaf(root, root * c, own);
}

// Chains the segments: slot k becomes what segment k starts from.  Forward: slot 0 is not read by the main pass
// (segment 0's own pass began with h0).  Backward: from the last segment, which starts from dht (packed: zero).
template <bool BACK>
__global__ void __launch_bounds__(128) k_scan_chain(const P p) {
  const int64_t dn = (int64_t)p.D * p.N, i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int b = blockIdx.y;
  if (i >= dn) return;
  const float A = p.A[i] * kLog2e;
  const int ch = (int)(i / p.N);
  float c = BACK && p.dht && !p.cu ? p.dht[b * dn + i] : 0.f;
  constexpr int U = 8;  // segments whose loads are in flight together
  for (int s0 = 0; s0 < p.nseg; s0 += U) {
    float own[U], e[U];
    bool cut[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u, k = BACK ? p.nseg - 1 - s : s;
      if (s >= p.nseg - 1) continue;  // the last segment passes nothing on
      own[u] = p.carry[((int64_t)b * p.nseg + k) * dn + i];
      e[u] = A * p.sdelta[((int64_t)b * p.nseg + k) * p.D + ch];
      cut[u] = (p.cu && p.broken[k]) || (!BACK && s == 0);  // segment 0 forward began with h0 itself
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u, k = BACK ? p.nseg - 1 - s : s;
      if (s >= p.nseg) break;
      p.carry[((int64_t)b * p.nseg + k) * dn + i] = c;
      if (s < p.nseg - 1) c = cut[u] ? own[u] : carried(e[u], c, own[u]);
    }
  }
}

// Packed sequences without rows: their final state is their initial one (and its gradient the final state's).  So is
// that of a sequence whose last (first) row falling offsets give to another one: nobody else would write it.
static __global__ void k_scan_empty(int S, int T, int64_t DN, const int32_t* __restrict__ cu, const float* __restrict__ from,
                                    float* __restrict__ to, bool back) {
  const int n = blockIdx.y, s = max(cu[n], 0), e = min(cu[n + 1], T);
  if (e > s && seq_at(cu, S, T, back ? s : e - 1).n == n) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < DN; i += (int64_t)gridDim.x * blockDim.x)
    to[n * DN + i] = from ? from[n * DN + i] : 0.f;
}

// A block walks its rows alone.  Measured at T = 2048, N = 16 (us, one segment against split): forward blocks of 128
// threads 128: 148 / 115, 192: 190 / 165, 256: 190 / 220; backward blocks of 256 threads 128: 711 / 530, 192: 960 / 785,
// 256: 961 / 1046.  So rows are split below 1.5 (1.6) blocks an SM.
constexpr int kSms = 148, kFwdBlocks = kSms * 3 / 2, kBwdBlocks = kSms * 8 / 5, kMinSegment = 64;

inline int check(const tops_gla_scan_args* a) {
  TOPS_CHECK_ARG(a != nullptr, "ssm_scan: args is NULL");
  TOPS_CHECK_ARG(a->B >= 0 && a->T >= 0 && a->D > 0 && a->S >= 0, "ssm_scan: negative or zero dimension");
  TOPS_CHECK_ARG(a->G > 0 && a->D % a->G == 0, "ssm_scan: D must be a multiple of G");
  if (a->T > kMaxRows || a->D > kMaxChannels) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: too many rows or channels");
  if (a->G > 65535) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: at most 65535 groups");
  if (a->N < 1 || a->N > 64) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: a channel must have 1 to 64 states");
  TOPS_CHECK_ARG(dtype_known(a->dtype), "ssm_scan: unknown dtype");
  if (a->B > 65535) return fail(TOPS_ERR_UNSUPPORTED, "ssm_scan: at most 65535 batch rows");
  if (a->cu_seqlens) {
    TOPS_CHECK_ARG(a->B == 1, "ssm_scan: cu_seqlens requires B == 1");
    TOPS_CHECK_ARG(a->S >= 1 && a->S <= 65535, "ssm_scan: cu_seqlens requires 1 to 65535 sequences");
  } else {
    TOPS_CHECK_ARG(a->S == a->B, "ssm_scan: S must equal B without cu_seqlens");
  }
  TOPS_CHECK_ARG(aligned_to(a->workspace, 16), "ssm_scan: workspace must be 16-byte aligned");
  return TOPS_OK;
}

inline P params(const tops_gla_scan_args* a) {
  P p{};
  p.B = a->B; p.T = a->T; p.D = a->D; p.N = a->N; p.G = a->G; p.S = a->S; p.softplus = a->softplus;
  p.cu = a->cu_seqlens;
  p.x = a->x; p.dt = a->dt; p.z = a->z; p.bm = a->Bm; p.cm = a->Cm;
  p.xs[0] = a->x_stride_b; p.xs[1] = a->x_stride_t;
  p.ds[0] = a->dt_stride_b; p.ds[1] = a->dt_stride_t;
  p.zs[0] = a->z_stride_b; p.zs[1] = a->z_stride_t;
  p.bs[0] = a->b_stride_b; p.bs[1] = a->b_stride_t;
  p.cs[0] = a->c_stride_b; p.cs[1] = a->c_stride_t;
  p.A = a->A; p.skip = a->skip; p.bias = a->dt_bias; p.h0 = a->h0;
  p.y = a->y; p.ht = a->ht; p.states = a->states;
  const int es = dtype_bytes(a->dtype);
  const bool ch4 = p.D / p.G % 4 == 0;
  auto quads = [&](const void* t, const int64_t (&s)[2], bool ok) {
    return ok && aligned_to(t, 4 * es) && s[0] % 4 == 0 && s[1] % 4 == 0;
  };
  p.vx = quads(p.x, p.xs, ch4);
  p.vd = quads(p.dt, p.ds, ch4);
  p.vz = quads(p.z, p.zs, ch4);
  p.vb = quads(p.bm, p.bs, p.N % 4 == 0);
  p.vc = quads(p.cm, p.cs, p.N % 4 == 0);
  p.vy = ch4 && aligned_to(p.y, 4 * es);
  return p;
}

// calls f with (T, LN, NT, VAR)
template <typename F>
int by_shape(const P& p, int dtype, F f) {
  auto states = [&](auto t, auto var) {
    if (p.N <= 8) return f(t, std::integral_constant<int, 4>(), std::integral_constant<int, 2>(), var);
    if (p.N <= 16) return f(t, std::integral_constant<int, 4>(), std::integral_constant<int, 4>(), var);
    if (p.N <= 32) return f(t, std::integral_constant<int, 8>(), std::integral_constant<int, 4>(), var);
    return f(t, std::integral_constant<int, 16>(), std::integral_constant<int, 4>(), var);
  };
  auto packed = [&](auto t) { return p.cu ? states(t, std::true_type()) : states(t, std::false_type()); };
  if (dtype == TOPS_F32) return packed(float());
  if (dtype == TOPS_BF16) return packed(__nv_bfloat16());
  return packed(__half());
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

// Segments of the rows: none where there are `wanted` blocks, else two to four waves of the blocks that fit (`resident`
// on an SM), so that the fullest SM walks few rows one after another: waves x rows of a segment (backward B1 T4096 D4096
// with 5, 10, 19 segments: 2, 3, 5 waves, 1664, 1248, 1120 rows and 639, 498, 426 us).  One wave leaves the first pass
// without blocks; where two counts are within 3 %, the greater balances better (packed prompts 201 -> 193 us).
inline void split(P& p, int blocks_per_row, int wanted, int resident) {
  p.seg = std::max(p.T, 1);
  p.nseg = 1;
  const int64_t blocks = (int64_t)blocks_per_row * p.B, slots = kSms * resident;
  if (blocks == 0 || blocks >= wanted || p.T < 2 * kMinSegment) return;
  int64_t best = INT64_MAX;
  for (int waves = 2; waves <= 4; ++waves) {
    const int want = (int)std::min<int64_t>(waves * slots / blocks, p.T / kMinSegment);
    if (want < 2) continue;
    const int seg = ((p.T + want - 1) / want + 31) / 32 * 32, n = (p.T + seg - 1) / seg;
    const int64_t walked = (n * blocks + slots - 1) / slots * seg;
    if (best != INT64_MAX && walked * 32 > best * 33) continue;
    best = std::min(best, walked);
    p.seg = seg;
    p.nseg = n;
  }
}

inline int lanes_of(int N) { return N <= 16 ? 4 : N <= 32 ? 8 : 16; }
inline int blocks_of(const P& p, int db) { return (p.D / p.G + db - 1) / db * p.G; }

inline size_t carve_segments(P& p, Carve& c) {
  if (p.nseg > 1) {
    p.carry = c.take((size_t)p.B * p.nseg * p.D * p.N);
    p.sdelta = c.take((size_t)p.B * p.nseg * p.D);
    p.broken = reinterpret_cast<int*>(c.take(p.nseg));
  }
  return c.used;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == TOPS_F32) return f(float());
  if (dtype == TOPS_BF16) return f(__nv_bfloat16());
  return f(__half());
}

inline int empty_states(const P& p, const float* from, float* to, bool back, cudaStream_t st) {
  if (!p.cu || !to) return TOPS_OK;
  LaunchTimer lt(st, "ssm_scan_empty");
  const int64_t dn = (int64_t)p.D * p.N;
  k_scan_empty<<<dim3((unsigned)std::min<int64_t>((dn + 255) / 256, 64), p.S), 256, 0, st>>>(p.S, p.T, dn, p.cu, from, to, back);
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_empty");
  return TOPS_OK;
}

}  // namespace ssm
}  // namespace tops
