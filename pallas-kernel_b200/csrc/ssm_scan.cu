// Selective state space scan.  Per channel d with N states, delta = softplus(dt + bias) or dt + bias:
//   h_t[n] = exp(delta_t A[d, n]) h_{t-1}[n] + delta_t x_t B_t[n],   y_t = sum_n C_t[n] h_t[n] + D x_t,
//   out = y silu(z)          (B, C shared by the D / G channels of a group)
// Backward, with dy = dout silu(z) and g_t = C_t dy_t + a_{t+1} g_{t+1} (the gradient of h_t):
//   dC_t = sum_d dy h,  dB_t = sum_d g delta x,  dx = delta sum_n g B + D dy,
//   ddelta = x sum_n g B + sum_n A a g h_{t-1},  dA = sum_t delta a g h_{t-1},  dh0 = a_1 g_1
//
// One exponential per (row, channel, state): at N = 16 the exponential unit (16 a clock and SM) bounds the
// forward at twice the time that its bytes take, and instruction issue the backward.  So:
//  * a thread owns CH channels x NT states and keeps their states, A and gradients in registers over all
//    rows; LN lanes share a channel and the other lanes are other channels;
//  * what a row needs once per channel (delta, delta x, dy) or once per state (B, C) is computed once per
//    block, a tile of rows ahead, into shared memory; the tile's elementwise work (softplus, gates,
//    rounding, 8- or 16-byte accesses) is spread over all threads, its loads issued one tile early;
//  * sums over the lanes of a channel (y, and the backward's) and over channels (dB, dC) are folded for
//    several rows at a time, so that each exchange halves the values that a lane still carries;
//  * arithmetic on state pairs is packed (fma.rn.f32x2), which halves its issue slots.
// Where B x D is too small for all SMs, the rows are split into segments: a first pass gives each segment's
// decay and its state from zero, a small kernel chains them, and the main pass starts every segment from its
// own state.  That costs the exponentials twice.
#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace ssm {

constexpr int CK = 16;  // rows between saved states = rows of a backward tile

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

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
// ex2.approx errs by -2e-8 on average where decays lie (against 64 bits, arguments -1 .. -0.002), and a state's
// error is that times the rows it remembers: the exponent's multiply-add takes the mean error back.
constexpr float kEx2Mean = 2.0e-8f * kLog2e;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 dup(float v) { return make_float2(v, v); }
// exp(delta A) of a pair, A given times log2(e)
__device__ __forceinline__ float2 decay2(float delta, float2 A) {
  const float2 e = fma2(dup(delta), A, dup(kEx2Mean));
  return make_float2(ex2(e.x), ex2(e.y));
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(__expf(v)); }

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

// four elements of T (those at `valid` and beyond are zero)
template <typename T>
struct Quad {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void quad_load(const T* p, bool vec, int valid, Quad<T>& q) {
  if (vec && valid >= 4) {
    alignas(16) T raw[4];
    Vx<T, 4>::load_raw(p, raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = i < valid ? p[i] : from_f<T>(0.f);
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

// SUM: the first pass over a segment (its state from zero and the sum of delta) instead of its output.
template <typename T, int LN, int NT, int CH, bool VAR, bool SUM>
__global__ void __launch_bounds__(128) k_scan_fwd(const P p) {
  constexpr int TS = 32, DB = 128 / LN * CH, NP = LN * NT, QC = DB / 4, RPP = 128 / QC, QN = RPP >= TS ? 1 : TS / RPP;
  constexpr int BQ = TS * NP / 4, BN = (BQ + 127) / 128;           // quads of B (of C) in a tile
  constexpr int RG = LN / CH < 4 ? LN / CH : 4, V = RG * CH;       // rows whose sums are folded at once
  __shared__ __align__(16) float2 su[TS][DB];
  __shared__ __align__(16) float sb[TS][NP], sc[TS][NP], sy[TS][DB];
  __shared__ int sflag[TS], sseq[TS];
  const int tid = threadIdx.x, lane = tid & 31, nl = lane % LN, b = blockIdx.y, k = blockIdx.z;
  const int rep = p.D / p.G, nblk = (rep + DB - 1) / DB, grp = blockIdx.x / nblk;
  const int c0 = (blockIdx.x - grp * nblk) * DB;                   // first channel of the block in its group
  const int cb = tid / 32 * (32 / LN * CH) + lane / LN * CH;       // first channel of the thread in the block
  const int n0 = nl * NT;
  const int64_t dbase = (int64_t)grp * rep + c0;
  const int t_first = k * p.seg, t_end = min(t_first + p.seg, p.T);

  float2 A[CH][NT / 2], h[CH][NT / 2];
  float dsum[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    dsum[i] = 0.f;
    const bool on = c0 + cb + i < rep;
    states_load<NT>(p.A + (dbase + cb + i) * p.N, n0, on ? p.N : 0, A[i]);
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      A[i][j] = mul2(A[i][j], dup(kLog2e));
      h[i][j] = dup(0.f);
    }
    if (on && !SUM) {
      if (k > 0) states_load<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
      else if (!VAR && p.h0) states_load<NT>(p.h0 + ((int64_t)b * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
    }
    if (on && SUM && !VAR && k == 0 && p.h0)
      states_load<NT>(p.h0 + ((int64_t)b * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
  }

  // staging: this thread's quads of channels are column qc of rows qr, qr + RPP, ...
  const int qc = tid % QC, qr = tid / QC;
  const int valid = min(max(rep - c0 - qc * 4, 0), 4);
  const T* xp = static_cast<const T*>(p.x) + b * p.xs[0] + dbase + qc * 4;
  const T* dp = static_cast<const T*>(p.dt) + b * p.ds[0] + dbase + qc * 4;
  const T* zp = static_cast<const T*>(p.z) + b * p.zs[0] + dbase + qc * 4;
  const T* bp = static_cast<const T*>(p.bm) + b * p.bs[0] + grp * p.N;
  const T* cp = static_cast<const T*>(p.cm) + b * p.cs[0] + grp * p.N;
  float bias[4], skip[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = p.bias && i < valid ? p.bias[dbase + qc * 4 + i] : 0.f;
    skip[i] = p.skip && i < valid ? p.skip[dbase + qc * 4 + i] : 0.f;
  }
  Quad<T> xr[QN], dr[QN], zr[QN], br[BN], cr[BN];
  int flag = 0, seq = 0;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int t = t0 + qr + j * RPP;
      const int v = (qr + j * RPP < TS && t < t_end) ? valid : 0;
      quad_load<T>(xp + t * p.xs[1], p.vx, v, xr[j]);
      quad_load<T>(dp + t * p.ds[1], p.vd, v, dr[j]);
      if (!SUM) quad_load<T>(zp + t * p.zs[1], p.vz, p.z ? v : 0, zr[j]);
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * 128, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4, t = t0 + row;
      const int v = (q < BQ && t < t_end) ? min(max(p.N - n, 0), 4) : 0;
      quad_load<T>(bp + t * p.bs[1] + n, p.vb, v, br[j]);
      if (!SUM) quad_load<T>(cp + t * p.cs[1] + n, p.vc, v, cr[j]);
    }
    if (VAR && tid < TS) flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
  };

  fetch(t_first);
  int broken = 0;
  for (int t0 = t_first; t0 < t_end; t0 += TS) {
    if (VAR) {
      if (tid < TS) {
        sflag[tid] = flag;
        sseq[tid] = seq;
      }
      broken |= __syncthreads_or(flag & (kFirst | kNone));
    }
    Quad<T> xc[QN], zc[QN];
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int row = qr + j * RPP;
      xc[j] = xr[j];
      if (!SUM) zc[j] = zr[j];
      if (row < TS) {
        const bool gone = t0 + row >= t_end || (VAR && (sflag[row] & kNone));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float dl = to_f<T>(dr[j].v[i + e]) + bias[i + e];
            if (p.softplus) dl = softplus(dl);
            f[2 * e] = gone ? 0.f : dl;
            f[2 * e + 1] = gone ? 0.f : dl * to_f<T>(xr[j].v[i + e]);
          }
          *reinterpret_cast<float4*>(&su[row][qc * 4 + i]) = make_float4(f[0], f[1], f[2], f[3]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * 128, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      if (q < BQ) {
        const bool gone = VAR && (sflag[row] & kNone);
        float fb[4], fc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fb[i] = gone ? 0.f : to_f<T>(br[j].v[i]);
          fc[i] = SUM || gone ? 0.f : to_f<T>(cr[j].v[i]);
        }
        *reinterpret_cast<float4*>(&sb[row][n]) = make_float4(fb[0], fb[1], fb[2], fb[3]);
        if (!SUM) *reinterpret_cast<float4*>(&sc[row][n]) = make_float4(fc[0], fc[1], fc[2], fc[3]);
      }
    }
    __syncthreads();
    if (t0 + TS < t_end) fetch(t0 + TS);
    const int rows = min(TS, t_end - t0);

    for (int r0 = 0; r0 < rows; r0 += RG) {  // rows at t_end and beyond: delta = 0, nothing moves
      if (!SUM && p.states != nullptr && (r0 & (CK - 1)) == 0) {
        const int nck = (p.T + CK - 1) / CK;
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (c0 + cb + i < rep)
            states_store<NT>(p.states + (((int64_t)b * nck + (t0 + r0) / CK) * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
      }
      float ys[V];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        const int r = r0 + rr;
        int f = 0;
        if (VAR) {
          f = sflag[r];
          if (f & (kFirst | kNone)) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
#pragma unroll
              for (int j = 0; j < NT / 2; ++j) h[i][j] = dup(0.f);
              if ((f & kFirst) && p.h0 && c0 + cb + i < rep)
                states_load<NT>(p.h0 + ((int64_t)sseq[r] * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
            }
          }
        }
        float2 Bv[NT / 2], Cv[NT / 2];
        pairs_load<NT>(&sb[r][n0], Bv);
        if (!SUM) pairs_load<NT>(&sc[r][n0], Cv);
        float du[2 * CH];
        if constexpr (CH == 2) {
          const float4 q = *reinterpret_cast<const float4*>(&su[r][cb]);
          du[0] = q.x; du[1] = q.y; du[2] = q.z; du[3] = q.w;
        } else {
          const float2 q = su[r][cb];
          du[0] = q.x; du[1] = q.y;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          float2 acc = dup(0.f);
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) {
            h[i][j] = fma2(decay2(du[2 * i], A[i][j]), h[i][j], mul2(dup(du[2 * i + 1]), Bv[j]));
            if (!SUM) acc = j ? fma2(Cv[j], h[i][j], acc) : mul2(Cv[j], h[i][j]);
          }
          if (SUM) dsum[i] += du[2 * i];
          else ys[rr * CH + i] = acc.x + acc.y;
        }
        if (VAR && !SUM && (f & kLast) && p.ht) {
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if (c0 + cb + i < rep) states_store<NT>(p.ht + ((int64_t)sseq[r] * p.D + dbase + cb + i) * p.N, n0, p.N, h[i]);
        }
      }
      if (!SUM) {
        const int at = fold<V, LN, 1>(ys, lane);
#pragma unroll
        for (int i = 0; i < (V > LN ? V / LN : 1); ++i) sy[r0 + (at + i) / CH][cb + (at + i) % CH] = ys[i];
      }
    }
    __syncthreads();
    if (!SUM) {
#pragma unroll
      for (int j = 0; j < QN; ++j) {
        const int row = qr + j * RPP, t = t0 + row;
        if (row < TS && t < t_end) {
          const float4 s4 = *reinterpret_cast<const float4*>(&sy[row][qc * 4]);
          float o[4] = {s4.x, s4.y, s4.z, s4.w};
          const bool gone = VAR && (sflag[row] & kNone);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[i] = fmaf(skip[i], to_f<T>(xc[j].v[i]), o[i]);
            if (p.z) {
              const float z = to_f<T>(zc[j].v[i]);
              o[i] *= z * fast_sigmoid(z);
            }
            if (gone) o[i] = 0.f;
          }
          quad_store<T>(static_cast<T*>(p.y) + ((int64_t)b * p.T + t) * p.D + dbase + qc * 4, p.vy, valid, o);
        }
      }
      if (VAR) __syncthreads();  // sflag is read above
    }
  }

#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (c0 + cb + i >= rep) continue;
    const int64_t d = dbase + cb + i;
    if (SUM) {
      states_store<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, h[i]);
      if (nl == 0) p.sdelta[((int64_t)b * p.nseg + k) * p.D + d] = dsum[i];
    } else if (!VAR && p.ht && k == p.nseg - 1) {
      states_store<NT>(p.ht + ((int64_t)b * p.D + d) * p.N, n0, p.N, h[i]);
    }
  }
  if (SUM && VAR && blockIdx.x == 0 && tid == 0) p.broken[k] = broken != 0;
}

// Chains the segments: slot k becomes what segment k starts from.  Forward: slot 0 is not read by the main pass
// (segment 0's own pass began with h0).  Backward: from the last segment, which starts from dht (packed: zero).
template <bool BACK>
__global__ void __launch_bounds__(128) k_scan_chain(const P p) {
  const int64_t dn = (int64_t)p.D * p.N, i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int b = blockIdx.y;
  if (i >= dn) return;
  const float A = p.A[i] * kLog2e;
  float c = BACK && p.dht && !p.cu ? p.dht[b * dn + i] : 0.f;
  for (int s = 0; s < p.nseg; ++s) {
    const int k = BACK ? p.nseg - 1 - s : s;
    if (s == p.nseg - 1) {
      p.carry[((int64_t)b * p.nseg + k) * dn + i] = c;
      break;
    }
    const int64_t at = ((int64_t)b * p.nseg + k) * dn + i;
    const float own = p.carry[at];
    p.carry[at] = c;
    // segment 0 forward began with h0 itself
    if ((p.cu && p.broken[k]) || (!BACK && s == 0)) c = own;
    else c = fmaf(ex2(A * p.sdelta[((int64_t)b * p.nseg + k) * p.D + i / p.N]), c, own);
  }
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

constexpr int kBwdThreads = 256;
template <int LN, int NT>
constexpr size_t bwd_smem() {
  return sizeof(float) * CK * ((kBwdThreads / LN) * 6 + 2 * LN * NT + 8 * 2 * LN * NT);
}

// One segment, tile by tile from its end.  A tile's states are computed again from the saved state before it:
// its first half once more than its second, so that only 8 rows of states and decays are in registers.
template <typename T, int LN, int NT, bool VAR>
__global__ void __launch_bounds__(kBwdThreads, 2) k_scan_bwd(const P p) {
  constexpr int TS = CK, HALF = 8, DB = kBwdThreads / LN, NP = LN * NT, QC = DB / 4, NH = NT / 2;
  extern __shared__ __align__(16) float smem[];
  float2(*su)[DB] = reinterpret_cast<float2(*)[DB]>(smem);                    // delta, delta x
  float(*sdy)[DB] = reinterpret_cast<float(*)[DB]>(smem + TS * DB * 2);
  float(*sq)[TS][DB] = reinterpret_cast<float(*)[TS][DB]>(smem + TS * DB * 3);  // sum g B, sum A a g h, sum C h
  float(*sb)[NP] = reinterpret_cast<float(*)[NP]>(smem + TS * DB * 6);
  float(*sc)[NP] = reinterpret_cast<float(*)[NP]>(smem + TS * DB * 6 + TS * NP);
  float(*sr)[TS][2 * NP] = reinterpret_cast<float(*)[TS][2 * NP]>(smem + TS * DB * 6 + TS * NP * 2);  // a warp's dB, dC
  __shared__ int sflag[TS], sseq[TS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nl = lane % LN, b = blockIdx.y, k = blockIdx.z;
  const int rep = p.D / p.G, nblk = (rep + DB - 1) / DB, grp = blockIdx.x / nblk, blk = blockIdx.x - grp * nblk;
  const int c0 = blk * DB, cb = warp * (32 / LN) + lane / LN, n0 = nl * NT;
  const int64_t dbase = (int64_t)grp * rep + c0;
  const bool on = c0 + cb < rep;
  const int64_t d = dbase + cb;
  const int t_first = k * p.seg, t_end = min(t_first + p.seg, p.T);
  const int nck = (p.T + CK - 1) / CK;

  float2 A[NH], g[NH], dA[NH];
  states_load<NT>(p.A + d * p.N, n0, on ? p.N : 0, A);
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    A[j] = mul2(A[j], dup(kLog2e));
    g[j] = dA[j] = dup(0.f);
  }
  if (on) {
    if (k < p.nseg - 1) states_load<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, g);
    else if (!VAR && p.dht) states_load<NT>(p.dht + ((int64_t)b * p.D + d) * p.N, n0, p.N, g);
  }

  // staging: one quad of channels of one row a thread
  const int qc = tid % QC, qr = tid / QC;
  const int valid = min(max(rep - c0 - qc * 4, 0), 4);
  const int64_t qd = dbase + qc * 4;
  float bias[4], skip[4], dskip[4], dbias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = p.bias && i < valid ? p.bias[qd + i] : 0.f;
    skip[i] = p.skip && i < valid ? p.skip[qd + i] : 0.f;
    dskip[i] = dbias[i] = 0.f;
  }
  constexpr int BQ = TS * NP / 4, BN = (BQ + kBwdThreads - 1) / kBwdThreads;
  Quad<T> xr, dr, zr, gr, br[BN], cr[BN];
  float2 hr[NH];
  int flag = 0, seq = 0;
  auto fetch = [&](int t0) {
    const int t = t0 + qr;
    const int v = (qr < TS && t < t_end) ? valid : 0;
    quad_load<T>(static_cast<const T*>(p.x) + b * p.xs[0] + t * p.xs[1] + qd, p.vx, v, xr);
    quad_load<T>(static_cast<const T*>(p.dt) + b * p.ds[0] + t * p.ds[1] + qd, p.vd, v, dr);
    quad_load<T>(static_cast<const T*>(p.dout) + b * p.os[0] + t * p.os[1] + qd, p.vo, v, gr);
    quad_load<T>(static_cast<const T*>(p.z) + b * p.zs[0] + t * p.zs[1] + qd, p.vz, p.z ? v : 0, zr);
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * kBwdThreads, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      const int w = (q < BQ && t0 + row < t_end) ? min(max(p.N - n, 0), 4) : 0;
      quad_load<T>(static_cast<const T*>(p.bm) + b * p.bs[0] + (t0 + row) * p.bs[1] + grp * p.N + n, p.vb, w, br[j]);
      quad_load<T>(static_cast<const T*>(p.cm) + b * p.cs[0] + (t0 + row) * p.cs[1] + grp * p.N + n, p.vc, w, cr[j]);
    }
    states_load<NT>(p.states + (((int64_t)b * nck + t0 / CK) * p.D + d) * p.N, n0, on ? p.N : 0, hr);
    if (VAR && tid < TS) flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
  };

  const int last = t_first + (t_end - t_first - 1) / TS * TS;
  if (t_first < t_end) fetch(last);
  for (int t0 = last; t0 >= t_first; t0 -= TS) {
    if (VAR) {
      if (tid < TS) {
        sflag[tid] = flag;
        sseq[tid] = seq;
      }
      __syncthreads();
    }
    const bool gone = qr >= TS || t0 + qr >= t_end || (VAR && (sflag[qr] & kNone));
    float xf[4], vf[4], zf[4], gf[4], dl[4], dy[4], zs[4];  // kept for the tile's outputs
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xf[i] = gone ? 0.f : to_f<T>(xr.v[i]);
      vf[i] = to_f<T>(dr.v[i]) + bias[i];
      dl[i] = gone ? 0.f : p.softplus ? softplus(vf[i]) : vf[i];
      gf[i] = gone ? 0.f : to_f<T>(gr.v[i]);
      zf[i] = gone ? 0.f : to_f<T>(zr.v[i]);
      zs[i] = fast_sigmoid(zf[i]);
      dy[i] = p.z ? gf[i] * zf[i] * zs[i] : gf[i];
    }
    if (qr < TS) {
      *reinterpret_cast<float4*>(&su[qr][qc * 4]) = make_float4(dl[0], dl[0] * xf[0], dl[1], dl[1] * xf[1]);
      *reinterpret_cast<float4*>(&su[qr][qc * 4 + 2]) = make_float4(dl[2], dl[2] * xf[2], dl[3], dl[3] * xf[3]);
      *reinterpret_cast<float4*>(&sdy[qr][qc * 4]) = make_float4(dy[0], dy[1], dy[2], dy[3]);
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * kBwdThreads, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      if (q < BQ) {
        const bool none = VAR && (sflag[row] & kNone);
        float fb[4], fc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fb[i] = none ? 0.f : to_f<T>(br[j].v[i]);
          fc[i] = none ? 0.f : to_f<T>(cr[j].v[i]);
        }
        *reinterpret_cast<float4*>(&sb[row][n]) = make_float4(fb[0], fb[1], fb[2], fb[3]);
        *reinterpret_cast<float4*>(&sc[row][n]) = make_float4(fc[0], fc[1], fc[2], fc[3]);
      }
    }
    float2 hs[NH];
#pragma unroll
    for (int j = 0; j < NH; ++j) hs[j] = hr[j];
    __syncthreads();
    if (t0 > t_first) fetch(t0 - TS);

    // the state before row r (a sequence's first row starts anew)
    auto enter = [&](int r, float2(&h)[NH]) {
      if (VAR && (sflag[r] & (kFirst | kNone))) {
#pragma unroll
        for (int j = 0; j < NH; ++j) h[j] = dup(0.f);
        if ((sflag[r] & kFirst) && p.h0 && on) states_load<NT>(p.h0 + ((int64_t)sseq[r] * p.D + d) * p.N, n0, p.N, h);
      }
    };
#pragma unroll 1
    for (int half = 1; half >= 0; --half) {
      float2 h[NH];
#pragma unroll
      for (int j = 0; j < NH; ++j) h[j] = hs[j];
      if (half == 1) {
#pragma unroll
        for (int r = 0; r < HALF; ++r) {
          enter(r, h);
          float2 Bv[NH];
          pairs_load<NT>(&sb[r][n0], Bv);
          const float2 q = su[r][cb];
#pragma unroll
          for (int j = 0; j < NH; ++j) h[j] = fma2(decay2(q.x, A[j]), h[j], mul2(dup(q.y), Bv[j]));
        }
      }
      const int r0 = half * HALF;
      float2 a[HALF][NH], hp[HALF + 1][NH];
#pragma unroll
      for (int r = 0; r < HALF; ++r) {
        enter(r0 + r, h);
        float2 Bv[NH];
        pairs_load<NT>(&sb[r0 + r][n0], Bv);
        const float2 q = su[r0 + r][cb];
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          hp[r][j] = h[j];
          a[r][j] = decay2(q.x, A[j]);
          h[j] = fma2(a[r][j], h[j], mul2(dup(q.y), Bv[j]));
        }
      }
#pragma unroll
      for (int j = 0; j < NH; ++j) hp[HALF][j] = h[j];
#pragma unroll
      for (int r4 = HALF - 4; r4 >= 0; r4 -= 4) {
        float s1[4], s2[4], s3[4];
#pragma unroll
        for (int rr = 3; rr >= 0; --rr) {
          const int r = r4 + rr;
          if (VAR && (sflag[r0 + r] & (kLast | kNone))) {
#pragma unroll
            for (int j = 0; j < NH; ++j) g[j] = dup(0.f);
            if ((sflag[r0 + r] & kLast) && p.dht && on)
              states_load<NT>(p.dht + ((int64_t)sseq[r0 + r] * p.D + d) * p.N, n0, p.N, g);
          }
          float2 Bv[NH], Cv[NH], w1 = dup(0.f), w2 = dup(0.f), w3 = dup(0.f);
          pairs_load<NT>(&sb[r0 + r][n0], Bv);
          pairs_load<NT>(&sc[r0 + r][n0], Cv);
          const float2 q = su[r0 + r][cb];
          const float dyv = sdy[r0 + r][cb];
          float bc[2 * NT];
#pragma unroll
          for (int j = 0; j < NH; ++j) {
            float2 ht = hp[r + 1][j];
            if (VAR) ht = fma2(a[r][j], hp[r][j], mul2(dup(q.y), Bv[j]));  // the next row may have started anew
            g[j] = fma2(Cv[j], dup(dyv), g[j]);
            w1 = j ? fma2(g[j], Bv[j], w1) : mul2(g[j], Bv[j]);
            w3 = j ? fma2(Cv[j], ht, w3) : mul2(Cv[j], ht);
            const float2 vb = mul2(g[j], dup(q.y)), vc = mul2(ht, dup(dyv));
            bc[2 * j] = vb.x; bc[2 * j + 1] = vb.y;
            bc[NT + 2 * j] = vc.x; bc[NT + 2 * j + 1] = vc.y;
            g[j] = mul2(a[r][j], g[j]);
            const float2 w = mul2(g[j], hp[r][j]);
            w2 = j ? fma2(A[j], w, w2) : mul2(A[j], w);
            dA[j] = fma2(dup(q.x), w, dA[j]);
          }
          s1[rr] = w1.x + w1.y;
          s2[rr] = w2.x + w2.y;
          s3[rr] = w3.x + w3.y;
          const int at = fold<2 * NT, 32 / LN, LN>(bc, lane);  // over the warp's channels
          constexpr int KEEP = 2 * NT / (32 / LN) > 1 ? 2 * NT / (32 / LN) : 1;
#pragma unroll
          for (int i = 0; i < KEEP; ++i)
            sr[warp][r0 + r][((at + i) / NT) * NP + n0 + (at + i) % NT] = bc[i];
          if (VAR && (sflag[r0 + r] & kFirst) && p.dh0 && on)
            states_store<NT>(p.dh0 + ((int64_t)sseq[r0 + r] * p.D + d) * p.N, n0, p.N, g);
        }
        const int o1 = fold<4, LN, 1>(s1, lane);  // over the lanes of a channel
        fold<4, LN, 1>(s2, lane);
        fold<4, LN, 1>(s3, lane);
        sq[0][r0 + r4 + o1][cb] = s1[0];
        sq[1][r0 + r4 + o1][cb] = s2[0];
        sq[2][r0 + r4 + o1][cb] = s3[0];
      }
    }
    __syncthreads();

    const int t = t0 + qr;
    if (qr < TS && t < t_end) {
      const bool none = VAR && (sflag[qr] & kNone);
      float odx[4], oddt[4], odz[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gB = sq[0][qr][qc * 4 + i], aw = sq[1][qr][qc * 4 + i] * kLn2;
        const float y = fmaf(skip[i], xf[i], sq[2][qr][qc * 4 + i]);
        odx[i] = none ? 0.f : fmaf(dl[i], gB, skip[i] * dy[i]);
        float dv = fmaf(xf[i], gB, aw);
        if (p.softplus) dv *= fast_sigmoid(vf[i]);
        oddt[i] = none ? 0.f : dv;
        odz[i] = none ? 0.f : gf[i] * y * zs[i] * fmaf(zf[i], 1.f - zs[i], 1.f);
        dbias[i] += oddt[i];
        dskip[i] = fmaf(dy[i], xf[i], dskip[i]);
      }
      const int64_t o = ((int64_t)b * p.T + t) * p.D + qd;
      quad_store<T>(static_cast<T*>(p.dx) + o, p.vg, valid, odx);
      quad_store<T>(static_cast<T*>(p.ddt) + o, p.vg, valid, oddt);
      if (p.dz) quad_store<T>(static_cast<T*>(p.dz) + o, p.vg, valid, odz);
    }
    float* part = p.pbc + (((int64_t)blockIdx.x * p.B + b) * p.T + t0) * 2 * p.N;
    for (int i = tid; i < TS * 2 * NP; i += kBwdThreads) {
      const int row = i / (2 * NP), c = i - row * 2 * NP, n = c % NP;
      if (t0 + row < t_end && n < p.N) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kBwdThreads / 32; ++w) s += sr[w][row][c];
        part[(int64_t)row * 2 * p.N + (c / NP) * p.N + n] = s;
      }
    }
    if (VAR) __syncthreads();
  }

  const int64_t sg = (int64_t)b * p.nseg + k;
  if (on) {
    states_store<NT>(p.pa + (sg * p.D + d) * p.N, n0, p.N, dA);
    if (!VAR && p.dh0 && k == 0) states_store<NT>(p.dh0 + ((int64_t)b * p.D + d) * p.N, n0, p.N, g);
  }
  // dD and dbias: the rows' threads of a quad, in a fixed order
  __syncthreads();
  float* red = smem;  // [2][TS][DB]
  if (qr < TS)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[qr * DB + qc * 4 + i] = dskip[i];
      red[(TS + qr) * DB + qc * 4 + i] = dbias[i];
    }
  __syncthreads();
  for (int i = tid; i < 2 * DB; i += kBwdThreads) {
    const int which = i / DB, c = i - which * DB;
    if (c0 + c >= rep) continue;
    float s = 0.f;
    for (int r = 0; r < (kBwdThreads / QC < TS ? kBwdThreads / QC : TS); ++r) s += red[(which * TS + r) * DB + c];
    p.pd[(sg * 2 + which) * p.D + dbase + c] = s;
  }
}

// The backward's first pass over a segment: the gradient that leaves it with nothing coming in, and the sum of delta.
template <typename T, int LN, int NT, bool VAR>
__global__ void __launch_bounds__(128) k_scan_bwd_sum(const P p) {
  constexpr int TS = 32, DB = 128 / LN, NP = LN * NT, QC = DB / 4, RPP = 128 / QC, QN = RPP >= TS ? 1 : TS / RPP;
  constexpr int NH = NT / 2, BQ = TS * NP / 4, BN = (BQ + 127) / 128;
  __shared__ __align__(16) float2 su[TS][DB];  // delta, dy
  __shared__ __align__(16) float sc[TS][NP];
  __shared__ int sflag[TS], sseq[TS];
  const int tid = threadIdx.x, lane = tid & 31, nl = lane % LN, b = blockIdx.y, k = blockIdx.z + 1;  // segment 0 passes nothing on
  const int rep = p.D / p.G, nblk = (rep + DB - 1) / DB, grp = blockIdx.x / nblk;
  const int c0 = (blockIdx.x - grp * nblk) * DB, cb = tid / 32 * (32 / LN) + lane / LN, n0 = nl * NT;
  const int64_t dbase = (int64_t)grp * rep + c0, d = dbase + cb;
  const bool on = c0 + cb < rep;
  const int t_first = k * p.seg, t_end = min(t_first + p.seg, p.T);
  float2 A[NH], g[NH];
  states_load<NT>(p.A + d * p.N, n0, on ? p.N : 0, A);
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    A[j] = mul2(A[j], dup(kLog2e));
    g[j] = dup(0.f);
  }
  float dsum = 0.f;
  const int qc = tid % QC, qr = tid / QC;
  const int valid = min(max(rep - c0 - qc * 4, 0), 4);
  const int64_t qd = dbase + qc * 4;
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = p.bias && i < valid ? p.bias[qd + i] : 0.f;
  int broken = 0;
  const int last = t_first + (t_end - t_first - 1) / TS * TS;
  for (int t0 = last; t0 >= t_first; t0 -= TS) {
    int flag = 0, seq = 0;
    if (VAR) {
      if (tid < TS) {
        flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
        sflag[tid] = flag;
        sseq[tid] = seq;
      }
      broken |= __syncthreads_or(flag & (kLast | kNone));
    }
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int row = qr + j * RPP, t = t0 + row;
      if (row >= TS) continue;
      const bool gone = t >= t_end || (VAR && (sflag[row] & kNone));
      Quad<T> dr, gr, zr;
      const int v = gone ? 0 : valid;
      quad_load<T>(static_cast<const T*>(p.dt) + b * p.ds[0] + t * p.ds[1] + qd, p.vd, v, dr);
      quad_load<T>(static_cast<const T*>(p.dout) + b * p.os[0] + t * p.os[1] + qd, p.vo, v, gr);
      quad_load<T>(static_cast<const T*>(p.z) + b * p.zs[0] + t * p.zs[1] + qd, p.vz, p.z ? v : 0, zr);
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float dl = to_f<T>(dr.v[i]) + bias[i];
        if (p.softplus) dl = softplus(dl);
        const float z = to_f<T>(zr.v[i]);
        const float dy = p.z ? to_f<T>(gr.v[i]) * z * fast_sigmoid(z) : to_f<T>(gr.v[i]);
        f[2 * i] = gone ? 0.f : dl;
        f[2 * i + 1] = gone ? 0.f : dy;
      }
      *reinterpret_cast<float4*>(&su[row][qc * 4]) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(&su[row][qc * 4 + 2]) = make_float4(f[4], f[5], f[6], f[7]);
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * 128, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      if (q >= BQ) continue;
      const bool gone = t0 + row >= t_end || (VAR && (sflag[row] & kNone));
      Quad<T> cr;
      quad_load<T>(static_cast<const T*>(p.cm) + b * p.cs[0] + (t0 + row) * p.cs[1] + grp * p.N + n, p.vc,
                   gone ? 0 : min(max(p.N - n, 0), 4), cr);
      *reinterpret_cast<float4*>(&sc[row][n]) =
          make_float4(to_f<T>(cr.v[0]), to_f<T>(cr.v[1]), to_f<T>(cr.v[2]), to_f<T>(cr.v[3]));
    }
    __syncthreads();
    for (int r = min(TS, t_end - t0) - 1; r >= 0; --r) {
      if (VAR && (sflag[r] & (kLast | kNone))) {
#pragma unroll
        for (int j = 0; j < NH; ++j) g[j] = dup(0.f);
        if ((sflag[r] & kLast) && p.dht && on) states_load<NT>(p.dht + ((int64_t)sseq[r] * p.D + d) * p.N, n0, p.N, g);
      }
      float2 Cv[NH];
      pairs_load<NT>(&sc[r][n0], Cv);
      const float2 q = su[r][cb];
#pragma unroll
      for (int j = 0; j < NH; ++j) g[j] = mul2(decay2(q.x, A[j]), fma2(Cv[j], dup(q.y), g[j]));
      dsum += q.x;
    }
    __syncthreads();
  }
  if (on) {
    states_store<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, g);
    if (nl == 0) p.sdelta[((int64_t)b * p.nseg + k) * p.D + d] = dsum;
  }
  if (VAR && blockIdx.x == 0 && tid == 0) p.broken[k] = broken != 0;
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

constexpr int kMinSegment = 128, kFwdBlocks = 148, kBwdBlocks = 148;

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

// Rows of a segment.  A block walks its rows alone, so without enough blocks the SMs idle; every split costs the
// exponentials of a first pass.
void split(P& p, int blocks_per_row, int blocks_wanted) {
  p.seg = std::max(p.T, 1);
  p.nseg = 1;
  const int64_t blocks = (int64_t)blocks_per_row * p.B;
  if (blocks >= blocks_wanted || p.T < 2 * kMinSegment) return;
  const int want = (int)std::min<int64_t>((2 * blocks_wanted + blocks - 1) / blocks, p.T / kMinSegment);
  if (want < 2) return;
  p.seg = ((p.T + want - 1) / want + 31) / 32 * 32;
  p.nseg = (p.T + p.seg - 1) / p.seg;
}

int lanes_of(int N) { return N <= 16 ? 4 : N <= 32 ? 8 : 16; }
int blocks_of(const P& p, int db) { return (p.D / p.G + db - 1) / db * p.G; }

size_t carve_segments(P& p, Carve& c) {
  if (p.nseg > 1) {
    p.carry = c.take((size_t)p.B * p.nseg * p.D * p.N);
    p.sdelta = c.take((size_t)p.B * p.nseg * p.D);
    p.broken = reinterpret_cast<int*>(c.take(p.nseg));
  }
  return c.used;
}

// channels of a forward thread: two share the loads of B and C
int fwd_channels(const P& p) { return (int64_t)blocks_of(p, 128 / lanes_of(p.N) * 2) * p.B >= kFwdBlocks ? 2 : 1; }

size_t plan_fwd(P& p, void* ws) {
  split(p, blocks_of(p, 128 / lanes_of(p.N)), kFwdBlocks);
  Carve c{static_cast<char*>(ws)};
  return carve_segments(p, c);
}

size_t plan_bwd(P& p, void* ws) {
  p.parts = blocks_of(p, kBwdThreads / lanes_of(p.N)) / p.G;
  split(p, p.parts * p.G, kBwdBlocks);
  Carve c{static_cast<char*>(ws)};
  p.pbc = c.take((size_t)p.G * p.parts * p.B * p.T * 2 * p.N);
  p.pa = c.take((size_t)p.B * p.nseg * p.D * p.N);
  p.pd = c.take((size_t)p.B * p.nseg * 2 * p.D);
  return carve_segments(p, c);
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
  P p = params(a);
  return plan_fwd(p, nullptr);
}

TOPS_API int tops_gla_ssm_scan_fwd(const tops_gla_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  const bool rows = (int64_t)a->B * a->T > 0;
  TOPS_CHECK_ARG(!rows || (a->x && a->dt && a->Bm && a->Cm && a->A && a->y), "ssm_scan_fwd: x, dt, B, C, A and y are required");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  P p = params(a);
  const size_t need = plan_fwd(p, a->workspace);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "ssm_scan_fwd: workspace smaller than tops_gla_ssm_scan_fwd_workspace_size()");
  if (int rc = empty_states(p, p.h0, p.ht, st)) return rc;
  if (p.B == 0 || (!rows && !p.ht)) return TOPS_OK;
  if (p.nseg > 1) {
    LaunchTimer lt(st, "ssm_scan_sum");
    by_shape(p, a->dtype, [&](auto t, auto ln, auto nt, auto var) {
      constexpr int LN = decltype(ln)::value;
      k_scan_fwd<decltype(t), LN, decltype(nt)::value, 1, decltype(var)::value, true>
          <<<dim3(blocks_of(p, 128 / LN), p.B, p.nseg - 1), 128, 0, st>>>(p);
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_sum");
    k_scan_chain<false><<<dim3((unsigned)(((int64_t)p.D * p.N + 127) / 128), p.B), 128, 0, st>>>(p);
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_chain");
  }
  LaunchTimer lt(st, "ssm_scan_fwd");
  const int ch = p.nseg > 1 ? 1 : fwd_channels(p);
  by_shape(p, a->dtype, [&](auto t, auto ln, auto nt, auto var) {
    using T = decltype(t);
    constexpr int LN = decltype(ln)::value, NT = decltype(nt)::value;
    constexpr bool VAR = decltype(var)::value;
    if (ch == 2) k_scan_fwd<T, LN, NT, 2, VAR, false><<<dim3(blocks_of(p, 256 / LN), p.B, p.nseg), 128, 0, st>>>(p);
    else k_scan_fwd<T, LN, NT, 1, VAR, false><<<dim3(blocks_of(p, 128 / LN), p.B, p.nseg), 128, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_fwd");
  return TOPS_OK;
}

TOPS_API size_t tops_gla_ssm_scan_bwd_workspace_size(const tops_gla_scan_bwd_args* a) {
  if (a == nullptr || check(&a->f) != TOPS_OK) return 0;
  P p = params(&a->f);
  return plan_bwd(p, nullptr);
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
  const size_t need = plan_bwd(p, a->workspace);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "ssm_scan_bwd: workspace smaller than tops_gla_ssm_scan_bwd_workspace_size()");
  p.dout = a->dout; p.os[0] = a->dout_strides[0]; p.os[1] = a->dout_strides[1];
  p.dht = a->dht; p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz; p.dh0 = a->dh0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = empty_states(p, p.dht, p.dh0, st)) return rc;
  if (p.B > 0) {
    const int es = dtype_bytes(f.dtype);
    const bool ch4 = p.D / p.G % 4 == 0;
    p.vo = ch4 && aligned_to(p.dout, 4 * es) && p.os[0] % 4 == 0 && p.os[1] % 4 == 0;
    p.vg = ch4 && aligned_to(p.dx, 4 * es) && aligned_to(p.ddt, 4 * es) && aligned_to(p.dz, 4 * es);
    if (p.nseg > 1) {
      LaunchTimer lt(st, "ssm_scan_bwd_sum");
      by_shape(p, f.dtype, [&](auto t, auto ln, auto nt, auto var) {
        constexpr int LN = decltype(ln)::value;
        k_scan_bwd_sum<decltype(t), LN, decltype(nt)::value, decltype(var)::value>
            <<<dim3(blocks_of(p, 128 / LN), p.B, p.nseg - 1), 128, 0, st>>>(p);
        return 0;
      });
      TOPS_CUDA_LAUNCH_CHECK("ssm_scan_bwd_sum");
      k_scan_chain<true><<<dim3((unsigned)(((int64_t)p.D * p.N + 127) / 128), p.B), 128, 0, st>>>(p);
      TOPS_CUDA_LAUNCH_CHECK("ssm_scan_chain");
    }
    LaunchTimer lt(st, "ssm_scan_bwd");
    const int rc = by_shape(p, f.dtype, [&](auto t, auto ln, auto nt, auto var) {
      constexpr int LN = decltype(ln)::value, NT = decltype(nt)::value;
      auto kernel = k_scan_bwd<decltype(t), LN, NT, decltype(var)::value>;
      constexpr size_t bytes = bwd_smem<LN, NT>();
      if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return cuda_status(e, "ssm_scan_bwd");
      }
      kernel<<<dim3(p.parts * p.G, p.B, p.nseg), kBwdThreads, bytes, st>>>(p);
      return 0;
    });
    if (rc) return rc;
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
    k_scan_sum<<<(unsigned)((s.n + 255) / 256), 256, 0, st>>>(p.B * p.nseg, s.n, s.stride, s.part, s.out);
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
