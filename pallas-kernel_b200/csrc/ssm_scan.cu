// Selective state space scan: the forward and the single-token step (ssm_scan.cuh has the mathematics).
#include "ssm_scan.cuh"

namespace tops {
namespace ssm {

// SUM: the first pass over a segment (its state from zero and the sum of delta) instead of its output.
// B4 T2048 D4096 N16 bf16: 286 us at 512 blocks = 1.9e12 exponentials a second of 4.6e12 (266 where no states are
// saved); B1 T8191 in segments 230 us and 155 us for the first pass.  64 or 256 threads a block: 295, 320 us; 4 rows in
// flight: 311.
constexpr int kFwdThreads = 128;

template <typename T, int LN, int NT, bool VAR, bool SUM>
__global__ void __launch_bounds__(kFwdThreads) k_scan_fwd(const P p) {
  constexpr int TS = 32, DB = kFwdThreads / LN, NP = LN * NT, QC = DB / 4, RPP = kFwdThreads / QC;
  constexpr int QN = RPP >= TS ? 1 : TS / RPP, NH = NT / 2;
  constexpr int BQ = TS * NP / 4, BN = (BQ + kFwdThreads - 1) / kFwdThreads;           // quads of B (of C) in a tile
  constexpr int RG = 8;                                            // rows in flight, whose sums are folded at once
  __shared__ __align__(16) float2 su[TS][DB];
  __shared__ __align__(16) float sb[TS][NP], sc[TS][NP], sy[TS][DB];
  __shared__ int sflag[TS], sseq[TS];
  __shared__ unsigned smark;
  const int tid = threadIdx.x, lane = tid & 31, nl = lane % LN, b = blockIdx.y, k = blockIdx.z;
  const int rep = p.D / p.G, nblk = (rep + DB - 1) / DB, grp = blockIdx.x / nblk;
  const int c0 = (blockIdx.x - grp * nblk) * DB;                   // first channel of the block in its group
  const int cb = tid / 32 * (32 / LN) + lane / LN;                 // channel of the thread in the block
  const int n0 = nl * NT;
  const int64_t dbase = (int64_t)grp * rep + c0;
  const int t_first = k * p.seg, t_end = min(t_first + p.seg, p.T);

  const bool on = c0 + cb < rep;
  const int64_t d = dbase + cb;
  float2 A[NH], h[NH];
  float dsum = 0.f;
  states_load<NT>(p.A + d * p.N, n0, on ? p.N : 0, A);
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    A[j] = mul2(A[j], dup(kLog2e));
    h[j] = dup(0.f);
  }
  if (on) {
    if (k > 0 && !SUM) states_load<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, h);
    else if (k == 0 && !VAR && p.h0) states_load<NT>(p.h0 + ((int64_t)b * p.D + d) * p.N, n0, p.N, h);
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
      const int q = tid + j * kFwdThreads, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4, t = t0 + row;
      const int v = (q < BQ && t < t_end) ? min(max(p.N - n, 0), 4) : 0;
      quad_load<T>(bp + t * p.bs[1] + n, p.vb, v, br[j]);
      if (!SUM) quad_load<T>(cp + t * p.cs[1] + n, p.vc, v, cr[j]);
    }
    if (VAR && tid < TS) flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
  };

  fetch(t_first);
  int broken = 0;
  for (int t0 = t_first; t0 < t_end; t0 += TS) {
    unsigned marks = 0;  // a bit for every row of the tile that begins or ends a sequence, or belongs to none
    if (VAR) {
      static_assert(TS == 32, "one warp marks a tile's rows");
      if (tid < TS) {
        sflag[tid] = flag;
        sseq[tid] = seq;
        marks = __ballot_sync(0xffffffffu, flag);
        if (tid == 0) smark = marks;
        if (SUM) broken |= __ballot_sync(0xffffffffu, flag & (kFirst | kNone));
      }
      __syncthreads();
      marks = smark;
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
      const int q = tid + j * kFwdThreads, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
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

    auto save = [&](int r) {
      static_assert(CK % RG == 0, "states are saved where a group of rows begins");
      if (!SUM && p.states != nullptr && on && (r & (CK - 1)) == 0) {
        const int nck = (p.T + CK - 1) / CK;
        states_store<NT>(p.states + (((int64_t)b * nck + (t0 + r) / CK) * p.D + d) * p.N, n0, p.N, h);
      }
    };
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += RG) {  // rows at t_end and beyond: delta = 0, nothing moves
      save(r0);
      if (VAR && (marks >> r0 & ((1u << RG) - 1))) {  // one by one: few rows of a packed batch
#pragma unroll 1
        for (int r = r0; r < min(r0 + RG, rows); ++r) {
          const int f = sflag[r];
          if (f & (kFirst | kNone)) {
#pragma unroll
            for (int j = 0; j < NH; ++j) h[j] = dup(0.f);
            if ((f & kFirst) && p.h0 && on) states_load<NT>(p.h0 + ((int64_t)sseq[r] * p.D + d) * p.N, n0, p.N, h);
          }
          float2 Bv[NH], Cv[NH], acc = dup(0.f);
          pairs_load<NT>(&sb[r][n0], Bv);
          if (!SUM) pairs_load<NT>(&sc[r][n0], Cv);
          const float2 q = su[r][cb];
          if (SUM) dsum += q.x;
#pragma unroll
          for (int j = 0; j < NH; ++j) {
            h[j] = fma2(decay2(q.x, A[j]), h[j], mul2(dup(q.y), Bv[j]));
            if (!SUM) acc = j ? fma2(Cv[j], h[j], acc) : mul2(Cv[j], h[j]);
          }
          if (!SUM) {
            float y[1] = {acc.x + acc.y};
            fold<1, LN, 1>(y, lane);
            sy[r][cb] = y[0];
            if ((f & kLast) && p.ht && on) states_store<NT>(p.ht + ((int64_t)sseq[r] * p.D + d) * p.N, n0, p.N, h);
          }
        }
        continue;
      }
      // the decays and inputs of all rows first: nothing of them waits for a state
      float2 a[RG][NH], ub[RG][NH];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float2 Bv[NH];
        pairs_load<NT>(&sb[r0 + rr][n0], Bv);
        const float2 q = su[r0 + rr][cb];
        if (SUM) dsum += q.x;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          a[rr][j] = decay2(q.x, A[j]);
          ub[rr][j] = mul2(dup(q.y), Bv[j]);
        }
      }
      float ys[RG];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float2 Cv[NH], acc = dup(0.f);
        if (!SUM) pairs_load<NT>(&sc[r0 + rr][n0], Cv);
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          h[j] = fma2(a[rr][j], h[j], ub[rr][j]);
          if (!SUM) acc = j ? fma2(Cv[j], h[j], acc) : mul2(Cv[j], h[j]);
        }
        if (!SUM) ys[rr] = acc.x + acc.y;
      }
      if (!SUM) {
        const int at = fold<RG, LN, 1>(ys, lane);
#pragma unroll
        for (int i = 0; i < (RG > LN ? RG / LN : 1); ++i) sy[r0 + at + i][cb] = ys[i];
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

  if (on) {
    if (SUM) {
      states_store<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, h);
      if (nl == 0) p.sdelta[((int64_t)b * p.nseg + k) * p.D + d] = dsum;
    } else if (!VAR && p.ht && k == p.nseg - 1) {
      states_store<NT>(p.ht + ((int64_t)b * p.D + d) * p.N, n0, p.N, h);
    }
  }
  if (SUM && VAR && blockIdx.x == 0 && tid == 0) p.broken[k] = broken != 0;
}

// One token of each of B rows: the state is read and written once (HBM bounds it).  Q lanes share a channel, four
// states each (16 bytes of the state), and take four rows of the batch at a time, whose loads are in flight together; A
// is read once for them.  What a row needs once per channel (delta, the gate, the output) is one lane's work: the lane
// that the fold of the four rows' sums leaves that row with.  States are read and written as streams (first to leave L2):
// 256 rows D4096 N16: 28.3 us = 5.0 TB/s.
template <typename T, int Q, bool VEC>
__global__ void __launch_bounds__(256) k_scan_step(const P p, int R) {
  constexpr int U = 4, OWN = Q >= U ? 1 : U / Q;  // rows at a time, and of them a lane's own
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, ch = id / Q;
  const int lane = threadIdx.x & 31, nq = lane % Q, n0 = nq * 4;
  const bool on = ch < p.D;
  const int d = on ? (int)ch : 0, grp = d / (p.D / p.G), cnt = min(4, p.N - n0);
  // own rows begin at `mine`, as fold() leaves them; the owner of row u is lane owner(u) of the channel
  const int mine = Q == 1 ? 0 : Q == 2 ? nq * 2 : (nq & 1) * 2 + (nq >> 1 & 1);
  auto owner = [](int u) { return Q == 1 ? 0 : Q == 2 ? u >> 1 : (u >> 1) + (u & 1) * 2; };
  float A[4];
  if (VEC) {
    const float4 v = on && cnt > 0 ? *reinterpret_cast<const float4*>(p.A + (int64_t)d * p.N + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
    A[0] = v.x; A[1] = v.y; A[2] = v.z; A[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] = on && i < cnt ? p.A[(int64_t)d * p.N + n0 + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] *= kLog2e;
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  const int b0 = blockIdx.y * R, b1 = min(b0 + R, p.B);
  for (int bb = b0; bb < b1; bb += U) {
    float h[U][4], x[OWN], z[OWN], dl[OWN];
    Quad<T> bq[U], cq[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = bb + u;
      const bool row = on && cnt > 0 && b < b1;
      const float* hp = p.h0 + ((int64_t)b * p.D + d) * p.N + n0;
      if (VEC) {
        const float4 v = row ? __ldcs(reinterpret_cast<const float4*>(hp)) : make_float4(0.f, 0.f, 0.f, 0.f);
        h[u][0] = v.x; h[u][1] = v.y; h[u][2] = v.z; h[u][3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[u][i] = row && i < cnt ? hp[i] : 0.f;
      }
      quad_load<T>(static_cast<const T*>(p.bm) + b * p.bs[0] + grp * p.N + n0, p.vb, row ? cnt : 0, bq[u]);
      quad_load<T>(static_cast<const T*>(p.cm) + b * p.cs[0] + grp * p.N + n0, p.vc, row ? cnt : 0, cq[u]);
    }
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int b = bb + mine + o;
      const bool row = on && b < b1;
      x[o] = row ? to_f<T>(static_cast<const T*>(p.x)[b * p.xs[0] + d]) : 0.f;
      dl[o] = row ? to_f<T>(static_cast<const T*>(p.dt)[b * p.ds[0] + d]) : 0.f;
      z[o] = row && p.z ? to_f<T>(static_cast<const T*>(p.z)[b * p.zs[0] + d]) : 0.f;
    }
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      dl[o] += bias;
      if (p.softplus) dl[o] = softplus(dl[o]);
    }
    float ys[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = bb + u;
      float delta = dl[u % OWN], du = dl[u % OWN] * x[u % OWN];
      if (Q > 1) {
        delta = __shfl_sync(0xffffffffu, delta, owner(u), Q);
        du = __shfl_sync(0xffffffffu, du, owner(u), Q);
      }
      ys[u] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[u][i] = fmaf(ex2(fmaf(delta, A[i], kEx2Mean)), h[u][i], du * bq[u].get(i));
        ys[u] = fmaf(cq[u].get(i), h[u][i], ys[u]);
      }
      if (on && cnt > 0 && b < b1) {
        float* ho = p.ht + ((int64_t)b * p.D + d) * p.N + n0;
        if (VEC) {
          __stcs(reinterpret_cast<float4*>(ho), make_float4(h[u][0], h[u][1], h[u][2], h[u][3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < cnt) ho[i] = h[u][i];
        }
      }
    }
    fold<U, Q, 1>(ys, lane);
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int b = bb + mine + o;
      if (!on || b >= b1 || nq >= U) continue;
      float y = fmaf(skip, x[o], ys[o]);
      if (p.z) y *= z[o] * fast_sigmoid(z[o]);
      static_cast<T*>(p.y)[(int64_t)b * p.D + d] = from_f<T>(y);
    }
  }
}

size_t plan_fwd(P& p, void* ws) {
  split(p, blocks_of(p, kFwdThreads / lanes_of(p.N)), kFwdBlocks, p.cu ? 5 : 4);
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
  TOPS_CHECK_ARG(a->N <= 8 || a->N % 4 || (aligned_to(a->ht, 16) && aligned_to(a->states, 16)),
                 "ssm_scan_fwd: ht and states must be 16-byte aligned (their four states a thread are one store)");
  TOPS_CHECK_ARG(rows || a->B == 0 || !a->ht || a->A, "ssm_scan_fwd: the final state needs A");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  P p = params(a);
  const size_t need = plan_fwd(p, a->workspace);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "ssm_scan_fwd: workspace smaller than tops_gla_ssm_scan_fwd_workspace_size()");
  if (int rc = empty_states(p, p.h0, p.ht, false, st)) return rc;
  if (p.B == 0 || (!rows && !p.ht)) return TOPS_OK;
  if (p.nseg > 1) {
    LaunchTimer lt(st, "ssm_scan_sum");
    by_shape(p, a->dtype, [&](auto t, auto ln, auto nt, auto var) {
      constexpr int LN = decltype(ln)::value;
      k_scan_fwd<decltype(t), LN, decltype(nt)::value, decltype(var)::value, true>
          <<<dim3(blocks_of(p, kFwdThreads / LN), p.B, p.nseg - 1), kFwdThreads, 0, st>>>(p);
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_sum");
    k_scan_chain<false><<<dim3((unsigned)(((int64_t)p.D * p.N + 127) / 128), p.B), 128, 0, st>>>(p);
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_chain");
  }
  LaunchTimer lt(st, "ssm_scan_fwd");
  by_shape(p, a->dtype, [&](auto t, auto ln, auto nt, auto var) {
    constexpr int LN = decltype(ln)::value;
    k_scan_fwd<decltype(t), LN, decltype(nt)::value, decltype(var)::value, false>
        <<<dim3(blocks_of(p, kFwdThreads / LN), p.B, p.nseg), kFwdThreads, 0, st>>>(p);
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
  // Lanes of a channel: a power of two, so that a channel lies in one warp.  Eight rows a thread (28.3 us at 256 rows D4096
  // N16; four: 30.3, sixteen: 29.0) where that still leaves four blocks an SM.
  const bool vec = p.N % 4 == 0 && aligned_to(p.h0, 16) && aligned_to(p.ht, 16) && aligned_to(p.A, 16);
  by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto lanes) {
      constexpr int Q = decltype(lanes)::value;
      const int blocks = (int)(((int64_t)p.D * Q + 255) / 256);
      const int R = (int64_t)blocks * (p.B / 8) >= kSms * 4 ? 8 : 4;
      const dim3 grid(blocks, (p.B + R - 1) / R);
      if (vec) k_scan_step<T, Q, true><<<grid, 256, 0, st>>>(p, R);
      else k_scan_step<T, Q, false><<<grid, 256, 0, st>>>(p, R);
      return 0;
    };
    if (p.N <= 4) return go(std::integral_constant<int, 1>());
    if (p.N <= 8) return go(std::integral_constant<int, 2>());
    if (p.N <= 16) return go(std::integral_constant<int, 4>());
    if (p.N <= 32) return go(std::integral_constant<int, 8>());
    return go(std::integral_constant<int, 16>());
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_step");
  return TOPS_OK;
}

}  // extern "C"
