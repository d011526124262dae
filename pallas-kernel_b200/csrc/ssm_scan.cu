// Selective state space scan: the forward and the single-token step (ssm_scan.cuh has the mathematics).
#include "ssm_scan.cuh"

namespace tops {
namespace ssm {

// SUM: the first pass over a segment (its state from zero and the sum of delta) instead of its output.
template <typename T, int LN, int NT, int CH, bool VAR, bool SUM>
__global__ void __launch_bounds__(128) k_scan_fwd(const P p) {
  constexpr int TS = 32, DB = 128 / LN * CH, NP = LN * NT, QC = DB / 4, RPP = 128 / QC, QN = RPP >= TS ? 1 : TS / RPP;
  constexpr int BQ = TS * NP / 4, BN = (BQ + 127) / 128;           // quads of B (of C) in a tile
  constexpr int RG = 4, V = RG * CH;                               // rows in flight, whose sums are folded at once
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
          float2 dl = make_float2(dr[j].get(i) + bias[i], dr[j].get(i + 1) + bias[i + 1]);
          if (p.softplus) dl = softplus2(dl);
          if (gone) dl = dup(0.f);
          *reinterpret_cast<float4*>(&su[row][qc * 4 + i]) =
              make_float4(dl.x, gone ? 0.f : dl.x * xr[j].get(i), dl.y, gone ? 0.f : dl.y * xr[j].get(i + 1));
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
          fb[i] = gone ? 0.f : br[j].get(i);
          fc[i] = SUM || gone ? 0.f : cr[j].get(i);
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
      // the decays and inputs of all rows first: nothing of them waits for a state
      float2 a[RG][CH][NT / 2], ub[RG][CH][NT / 2];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float2 Bv[NT / 2];
        pairs_load<NT>(&sb[r0 + rr][n0], Bv);
        float du[2 * CH];
        if constexpr (CH == 2) {
          const float4 q = *reinterpret_cast<const float4*>(&su[r0 + rr][cb]);
          du[0] = q.x; du[1] = q.y; du[2] = q.z; du[3] = q.w;
        } else {
          const float2 q = su[r0 + rr][cb];
          du[0] = q.x; du[1] = q.y;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          if (SUM) dsum[i] += du[2 * i];
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) {
            a[rr][i][j] = decay2(du[2 * i], A[i][j]);
            ub[rr][i][j] = mul2(dup(du[2 * i + 1]), Bv[j]);
          }
        }
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
        float2 Cv[NT / 2];
        if (!SUM) pairs_load<NT>(&sc[r][n0], Cv);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          float2 acc = dup(0.f);
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) {
            h[i][j] = fma2(a[rr][i][j], h[i][j], ub[rr][i][j]);
            if (!SUM) acc = j ? fma2(Cv[j], h[i][j], acc) : mul2(Cv[j], h[i][j]);
          }
          if (!SUM) ys[rr * CH + i] = acc.x + acc.y;
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
            o[i] = fmaf(skip[i], xc[j].get(i), o[i]);
            if (p.z) {
              const float z = zc[j].get(i);
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

// One token of each of B rows: the state is read and written once (HBM bounds it).  Q lanes share a channel, four
// states each (16 bytes of the state), and take R rows of the batch one after another, their states loaded together:
// A, the bias and the skip weight are read once for them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_scan_step(const P p, int Q, int R) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, ch = id / Q;
  const int nq = (int)(id - ch * Q), n0 = nq * 4;
  const bool on = ch < p.D;
  const int d = on ? (int)ch : 0, grp = d / (p.D / p.G), cnt = min(4, p.N - n0);
  float A[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] = on && i < cnt ? p.A[(int64_t)d * p.N + n0 + i] * kLog2e : 0.f;
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  const int b0 = blockIdx.y * R;
  constexpr int U = 4;
  for (int bb = b0; bb < min(b0 + R, p.B); bb += U) {
    float h[U][4];
    float x[U], dt[U], z[U], Bv[U][4], Cv[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = bb + u;
      const bool row = on && cnt > 0 && b < min(b0 + R, p.B);
      const float* hp = p.h0 + ((int64_t)b * p.D + d) * p.N + n0;
      if (VEC) {
        const float4 v = row ? *reinterpret_cast<const float4*>(hp) : make_float4(0.f, 0.f, 0.f, 0.f);
        h[u][0] = v.x; h[u][1] = v.y; h[u][2] = v.z; h[u][3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[u][i] = row && i < cnt ? hp[i] : 0.f;
      }
      x[u] = row ? to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + d]) : 0.f;
      dt[u] = row ? to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + d]) : 0.f;
      z[u] = row && p.z ? to_f<T>(static_cast<const T*>(p.z)[b * p.zs[0] + d]) : 0.f;
      Quad<T> bq, cq;
      quad_load<T>(static_cast<const T*>(p.bm) + b * p.bs[0] + grp * p.N + n0, p.vb, row ? cnt : 0, bq);
      quad_load<T>(static_cast<const T*>(p.cm) + b * p.cs[0] + grp * p.N + n0, p.vc, row ? cnt : 0, cq);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Bv[u][i] = bq.get(i);
        Cv[u][i] = cq.get(i);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = bb + u;
      const bool row = on && cnt > 0 && b < min(b0 + R, p.B);
      float dl = dt[u] + bias;
      if (p.softplus) dl = softplus(dl);
      const float du = dl * x[u];
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[u][i] = fmaf(ex2(fmaf(dl, A[i], kEx2Mean)), h[u][i], du * Bv[u][i]);
        y = fmaf(Cv[u][i], h[u][i], y);
      }
      for (int o = 1; o < Q; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (!row) continue;
      float* ho = p.ht + ((int64_t)b * p.D + d) * p.N + n0;
      if (VEC) {
        *reinterpret_cast<float4*>(ho) = make_float4(h[u][0], h[u][1], h[u][2], h[u][3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < cnt) ho[i] = h[u][i];
      }
      if (nq == 0) {
        y = fmaf(skip, x[u], y);
        if (p.z) y *= z[u] * fast_sigmoid(z[u]);
        static_cast<T*>(p.y)[(int64_t)b * p.D + d] = from_f<T>(y);
      }
    }
  }
}

// channels of a forward thread: two share the loads of B and C
int fwd_channels(const P& p) { return (int64_t)blocks_of(p, 128 / lanes_of(p.N) * 2) * p.B >= kFwdBlocks ? 2 : 1; }

size_t plan_fwd(P& p, void* ws) {
  split(p, blocks_of(p, 128 / lanes_of(p.N)), kFwdBlocks);
  Carve c{static_cast<char*>(ws)};
  return carve_segments(p, c);
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

TOPS_API int tops_gla_ssm_scan_step(const tops_gla_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  TOPS_CHECK_ARG(a->T == 1 && !a->cu_seqlens, "ssm_scan_step: T must be 1, without cu_seqlens");
  if (a->B == 0) return TOPS_OK;
  TOPS_CHECK_ARG(a->x && a->dt && a->Bm && a->Cm && a->A && a->h0 && a->y && a->ht,
                 "ssm_scan_step: x, dt, B, C, A, h0, y and ht are required");
  const P p = params(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "ssm_scan_step");
  int Q = 1;  // lanes of a channel: a power of two, so that a channel lies in one warp
  while (Q * 4 < p.N) Q *= 2;
  const int blocks = (int)(((int64_t)p.D * Q + 255) / 256);
  // rows of a thread: all loads of four are in flight at once; fewer where the grid would not fill the SMs
  int R = 4;
  while (R > 1 && (int64_t)blocks * ((p.B + R - 1) / R) < 148 * 4) R /= 2;
  R = std::max(R, (p.B + 65534) / 65535);
  const bool vec = p.N % 4 == 0 && aligned_to(p.h0, 16) && aligned_to(p.ht, 16);
  by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid(blocks, (p.B + R - 1) / R);
    if (vec) k_scan_step<T, true><<<grid, 256, 0, st>>>(p, Q, R);
    else k_scan_step<T, false><<<grid, 256, 0, st>>>(p, Q, R);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_step");
  return TOPS_OK;
}

}  // extern "C"
