// Selective state space scan: the backward (ssm_scan.cuh has the mathematics).
#include "ssm_scan.cuh"

namespace tops {
namespace ssm {

constexpr int kBwdThreads = 256, kBwdRows = 16, kBwdPart = 4;  // rows of a tile, and of what is in registers at once

// The sums of dB and dC over a warp's channels halve what a lane carries with every exchange.  Which half a lane keeps
// follows its number; instead of selecting, a lane holds its NT states in an order of its own, register j for state
// n0 + (j ^ order), so that it always keeps the lower registers.  B and C lie in shared memory in each order, so that a
// row is still one load.
template <int LN, int NT>
struct Order {
  static constexpr int BITS = NT == 2 ? 1 : LN <= 8 ? 2 : 1;  // exchanges that halve the states
  static constexpr int COPIES = 1 << BITS;
  static __device__ __forceinline__ int of(int lane) {
    int o = lane & LN ? NT / 2 : 0;
    if (BITS == 2 && (lane & (2 * LN))) o |= 1;
    return o;
  }
  // the place of an order's copy: the two orders of a quarter warp lie side by side (no bank conflict)
  static constexpr __device__ __forceinline__ int slot(int order) {
    return NT == 2 ? order : BITS == 2 ? (order & 1) << 1 | order >> 1 : order >> 1;
  }
  static constexpr __device__ __forceinline__ int order_at(int slot) {
    return NT == 2 ? slot : BITS == 2 ? (slot & 1) << 1 | slot >> 1 : slot << 1;
  }
};
template <int NT>
__device__ __forceinline__ void ordered_load(const float* p, int n0, int order, int N, float2 (&h)[NT / 2]) {
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) {
    const int a = n0 + ((2 * i) ^ order), b = n0 + ((2 * i + 1) ^ order);
    h[i] = make_float2(a < N ? p[a] : 0.f, b < N ? p[b] : 0.f);
  }
}
template <int NT>
__device__ __forceinline__ void ordered_store(float* p, int n0, int order, int N, const float2 (&h)[NT / 2]) {
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) {
    const int a = n0 + ((2 * i) ^ order), b = n0 + ((2 * i + 1) ^ order);
    if (a < N) p[a] = h[i].x;
    if (b < N) p[b] = h[i].y;
  }
}

template <int LN, int NT>
constexpr size_t bwd_smem() {
  return sizeof(float) * kBwdRows *
         ((kBwdThreads / LN) * 6 + 2 * Order<LN, NT>::COPIES * LN * NT + kBwdThreads / 32 * 2 * LN * NT);
}

// One segment, tile by tile from its end.  The states of kBwdPart rows at a time are computed again from the saved state
// before them and kept in registers with their decays (eight rows spilled: 1088 against 1004 us); what the tile's outputs
// need of the inputs stays packed as it came, the rest is read back from shared memory.  B4 T2048 D4096 N16 bf16: 930 us
// at 256 blocks, 800 us for the same work in many more blocks.  No unit is full: issue 55 %, the shared-memory pipe 60 %
// (33 instructions and 0.28 wavefronts an element, of which the folds are 10 and 0.08), 14 warps an SM.
template <typename T, int LN, int NT, bool VAR>
__global__ void __launch_bounds__(kBwdThreads, 2) k_scan_bwd(const P p) {
  constexpr int TS = kBwdRows, HALF = kBwdPart, DB = kBwdThreads / LN, NP = LN * NT, QC = DB / 4, NH = NT / 2;
  extern __shared__ __align__(16) float smem[];
  float2(*su)[DB] = reinterpret_cast<float2(*)[DB]>(smem);                    // delta, delta x
  float(*sdy)[DB] = reinterpret_cast<float(*)[DB]>(smem + TS * DB * 2);
  float(*sq)[TS][DB] = reinterpret_cast<float(*)[TS][DB]>(smem + TS * DB * 3);  // sum g B, sum A a g h, sum C h
  using O = Order<LN, NT>;
  constexpr int NC = O::COPIES * NP;
  float(*sb)[NC] = reinterpret_cast<float(*)[NC]>(smem + TS * DB * 6);
  float(*sc)[NC] = reinterpret_cast<float(*)[NC]>(smem + TS * DB * 6 + TS * NC);
  float(*sr)[TS][2 * NP] = reinterpret_cast<float(*)[TS][2 * NP]>(smem + TS * DB * 6 + TS * NC * 2);  // a warp's dB, dC
  __shared__ int sflag[TS], sseq[TS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nl = lane % LN, b = blockIdx.y, k = blockIdx.z;
  const int rep = p.D / p.G, nblk = (rep + DB - 1) / DB, grp = blockIdx.x / nblk, blk = blockIdx.x - grp * nblk;
  const int c0 = blk * DB, cb = warp * (32 / LN) + lane / LN, n0 = nl * NT;
  const int order = O::of(lane), m0 = O::slot(order) * NP + n0;  // its states' order and where its B and C begin
  const int64_t dbase = (int64_t)grp * rep + c0;
  const bool on = c0 + cb < rep;
  const int64_t d = dbase + cb;
  const int t_first = k * p.seg, t_end = min(t_first + p.seg, p.T);
  const int nck = (p.T + CK - 1) / CK;

  float2 A[NH], g[NH], dA[NH];
  ordered_load<NT>(p.A + d * p.N, n0, order, on ? p.N : 0, A);
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    A[j] = mul2(A[j], dup(kLog2e));
    g[j] = dA[j] = dup(0.f);
  }
  if (on) {
    if (k < p.nseg - 1) ordered_load<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, order, p.N, g);
    else if (!VAR && p.dht) ordered_load<NT>(p.dht + ((int64_t)b * p.D + d) * p.N, n0, order, p.N, g);
  }

  // staging: one quad of channels of one row a thread
  const int qc = tid % QC, qr = tid / QC;
  const int valid = min(max(rep - c0 - qc * 4, 0), 4);
  const int64_t qd = dbase + qc * 4;
  float bias[4], dskip[4], dbias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = p.bias && i < valid ? p.bias[qd + i] : 0.f;
    dskip[i] = dbias[i] = 0.f;
  }
  constexpr int BQ = TS * NP / 4, BN = (BQ + kBwdThreads - 1) / kBwdThreads;
  Quad<T> xr, dr, zr, gr, br[BN], cr[BN];
  float2 hr[NH];
  int flag = 0, seq = 0;
  auto saved = [&](int t, float2(&h)[NH]) {  // the state before row t
    ordered_load<NT>(p.states + (((int64_t)b * nck + t / CK) * p.D + d) * p.N, n0, order, on && t < t_end ? p.N : 0, h);
  };
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
    saved(t0 + TS - CK, hr);
    if (VAR && tid < TS) flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
  };

  const int last = t_end > t_first ? t_first + (t_end - t_first - 1) / TS * TS : t_first - TS;
  if (last >= t_first) fetch(last);
  for (int t0 = last; t0 >= t_first; t0 -= TS) {
    bool flagged = false;  // a row of the tile begins or ends a sequence, or belongs to none
    if (VAR) {
      if (tid < TS) {
        sflag[tid] = flag;
        sseq[tid] = seq;
      }
      flagged = __syncthreads_or(flag);
    }
    const bool gone = qr >= TS || t0 + qr >= t_end || (VAR && (sflag[qr] & kNone));
    const Quad<T> xc = xr, dc = dr, zc = zr, gc = gr;  // for the tile's outputs
    if (qr < TS) {
      float dl[4], dy[4];
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float2 v = make_float2(dc.get(i) + bias[i], dc.get(i + 1) + bias[i + 1]);
        if (p.softplus) v = softplus2(v);
        dl[i] = gone ? 0.f : v.x;
        dl[i + 1] = gone ? 0.f : v.y;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = zc.get(i);
        dy[i] = gone ? 0.f : p.z ? gc.get(i) * z * fast_sigmoid(z) : gc.get(i);
      }
      const float x0 = gone ? 0.f : xc.get(0), x1 = gone ? 0.f : xc.get(1), x2 = gone ? 0.f : xc.get(2),
                  x3 = gone ? 0.f : xc.get(3);
      *reinterpret_cast<float4*>(&su[qr][qc * 4]) = make_float4(dl[0], dl[0] * x0, dl[1], dl[1] * x1);
      *reinterpret_cast<float4*>(&su[qr][qc * 4 + 2]) = make_float4(dl[2], dl[2] * x2, dl[3], dl[3] * x3);
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
          fb[i] = none ? 0.f : br[j].get(i);
          fc[i] = none ? 0.f : cr[j].get(i);
        }
#pragma unroll
        for (int c = 0; c < O::COPIES; ++c) {
          const int o = O::order_at(c);
          *reinterpret_cast<float4*>(&sb[row][c * NP + n]) = make_float4(fb[o], fb[1 ^ o], fb[2 ^ o], fb[3 ^ o]);
          *reinterpret_cast<float4*>(&sc[row][c * NP + n]) = make_float4(fc[o], fc[1 ^ o], fc[2 ^ o], fc[3 ^ o]);
        }
      }
    }
    float2 h[NH], hc[NH], hs[NH];  // the state, the saved one of this part, and of the part before it
#pragma unroll
    for (int j = 0; j < NH; ++j) hc[j] = hr[j];
    __syncthreads();
    if (t0 > t_first) fetch(t0 - TS);

    auto rows = [&](auto with_flags) {
      constexpr bool FLAG = decltype(with_flags)::value;
      // the state before row r (a sequence's first row starts anew)
      auto enter = [&](int r, float2(&h)[NH]) {
        if (FLAG && (sflag[r] & (kFirst | kNone))) {
#pragma unroll
          for (int j = 0; j < NH; ++j) h[j] = dup(0.f);
          if ((sflag[r] & kFirst) && p.h0 && on) ordered_load<NT>(p.h0 + ((int64_t)sseq[r] * p.D + d) * p.N, n0, order, p.N, h);
        }
      };
#pragma unroll 1
      for (int part = TS / HALF - 1; part >= 0; --part) {
        const int r0 = part * HALF;
        if (HALF == CK || part % (CK / HALF) == CK / HALF - 1) {  // a new saved state; the one before it is on its way
          if (part != TS / HALF - 1)
#pragma unroll
            for (int j = 0; j < NH; ++j) hc[j] = hs[j];
          if (r0 - (CK - HALF) >= CK) saved(t0 + r0 - (CK - HALF) - CK, hs);
        }
#pragma unroll
        for (int j = 0; j < NH; ++j) h[j] = hc[j];
        if (HALF < CK && part % (CK / HALF) != 0) {
#pragma unroll
          for (int rr = 0; rr < CK - HALF; ++rr) {
            const int r = r0 - (CK - HALF) + rr;
            enter(r, h);
            float2 Bv[NH];
            pairs_load<NT>(&sb[r][m0], Bv);
            const float2 q = su[r][cb];
#pragma unroll
            for (int j = 0; j < NH; ++j) h[j] = fma2(decay2(q.x, A[j]), h[j], mul2(dup(q.y), Bv[j]));
          }
        }
        float2 a[HALF][NH], hp[HALF + 1][NH];
#pragma unroll
        for (int r = 0; r < HALF; ++r) {
          enter(r0 + r, h);
          float2 Bv[NH];
          pairs_load<NT>(&sb[r0 + r][m0], Bv);
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
            if (FLAG && (sflag[r0 + r] & (kLast | kNone))) {
#pragma unroll
              for (int j = 0; j < NH; ++j) g[j] = dup(0.f);
              if ((sflag[r0 + r] & kLast) && p.dht && on)
                ordered_load<NT>(p.dht + ((int64_t)sseq[r0 + r] * p.D + d) * p.N, n0, order, p.N, g);
            }
            float2 Bv[NH], Cv[NH], w1 = dup(0.f), w2 = dup(0.f), w3 = dup(0.f);
            pairs_load<NT>(&sb[r0 + r][m0], Bv);
            pairs_load<NT>(&sc[r0 + r][m0], Cv);
            const float2 q = su[r0 + r][cb];
            const float dyv = sdy[r0 + r][cb];
            float vb[NT], vc[NT];  // terms of dB and dC
#pragma unroll
            for (int j = 0; j < NH; ++j) {
              float2 ht = hp[r + 1][j];
              if (FLAG) ht = fma2(a[r][j], hp[r][j], mul2(dup(q.y), Bv[j]));  // the next row may have started anew
              g[j] = fma2(Cv[j], dup(dyv), g[j]);
              w1 = j ? fma2(g[j], Bv[j], w1) : mul2(g[j], Bv[j]);
              w3 = j ? fma2(Cv[j], ht, w3) : mul2(Cv[j], ht);
              const float2 tb = mul2(g[j], dup(q.y)), tc = mul2(ht, dup(dyv));
              vb[2 * j] = tb.x; vb[2 * j + 1] = tb.y;
              vc[2 * j] = tc.x; vc[2 * j + 1] = tc.y;
              g[j] = mul2(a[r][j], g[j]);
              const float2 w = mul2(g[j], hp[r][j]);
              w2 = j ? fma2(A[j], w, w2) : mul2(A[j], w);
              dA[j] = fma2(dup(q.x), w, dA[j]);
            }
            s1[rr] = w1.x + w1.y;
            s2[rr] = w2.x + w2.y;
            s3[rr] = w3.x + w3.y;
            // over the warp's channels: first the states are halved, then one of dB and dC is kept, then nothing is left to halve
            constexpr int KEEP = NT >> O::BITS;
            int m = LN;
#pragma unroll
            for (int i = 0; i < O::BITS; ++i, m <<= 1)
#pragma unroll
              for (int j = 0; j < (NT >> (i + 1)); ++j) {
                vb[j] += __shfl_xor_sync(0xffffffffu, vb[j + (NT >> (i + 1))], m);
                vc[j] += __shfl_xor_sync(0xffffffffu, vc[j + (NT >> (i + 1))], m);
              }
            float* out = &sr[warp][r0 + r][n0];
            if constexpr ((LN << O::BITS) < 32) {
              const bool up = lane & (LN << O::BITS);
              float keep = up ? vc[0] : vb[0];
              keep += __shfl_xor_sync(0xffffffffu, up ? vb[0] : vc[0], LN << O::BITS);
#pragma unroll
              for (int mm = LN << (O::BITS + 1); mm < 32; mm <<= 1) keep += __shfl_xor_sync(0xffffffffu, keep, mm);
              out[(up ? NP : 0) + order] = keep;
            } else {
#pragma unroll
              for (int j = 0; j < KEEP; ++j) {
                out[j ^ order] = vb[j];
                out[NP + (j ^ order)] = vc[j];
              }
            }
            if (FLAG && (sflag[r0 + r] & kFirst) && p.dh0 && on)
              ordered_store<NT>(p.dh0 + ((int64_t)sseq[r0 + r] * p.D + d) * p.N, n0, order, p.N, g);
          }
          const int o1 = fold<4, LN, 1>(s1, lane);  // over the lanes of a channel
          fold<4, LN, 1>(s2, lane);
          fold<4, LN, 1>(s3, lane);
          sq[0][r0 + r4 + o1][cb] = s1[0];
          sq[1][r0 + r4 + o1][cb] = s2[0];
          sq[2][r0 + r4 + o1][cb] = s3[0];
        }
      }
    };
    if (VAR && flagged) rows(std::true_type());
    else rows(std::false_type());
    __syncthreads();

    const int t = t0 + qr;
    if (qr < TS && t < t_end) {
      const bool none = VAR && (sflag[qr] & kNone);
      float odx[4], oddt[4], odz[4], sk[4];
      const float4 u0 = *reinterpret_cast<const float4*>(&su[qr][qc * 4]);
      const float4 u1 = *reinterpret_cast<const float4*>(&su[qr][qc * 4 + 2]);
      const float4 dy4 = *reinterpret_cast<const float4*>(&sdy[qr][qc * 4]);
      const float4 q0 = *reinterpret_cast<const float4*>(&sq[0][qr][qc * 4]);
      const float4 q1 = *reinterpret_cast<const float4*>(&sq[1][qr][qc * 4]);
      const float4 q2 = *reinterpret_cast<const float4*>(&sq[2][qr][qc * 4]);
      const float dl[4] = {u0.x, u0.z, u1.x, u1.z}, dy[4] = {dy4.x, dy4.y, dy4.z, dy4.w};
      const float gB[4] = {q0.x, q0.y, q0.z, q0.w}, aw[4] = {q1.x, q1.y, q1.z, q1.w}, ch[4] = {q2.x, q2.y, q2.z, q2.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) sk[i] = p.skip && i < valid ? p.skip[qd + i] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = xc.get(i);
        odx[i] = none ? 0.f : fmaf(dl[i], gB[i], sk[i] * dy[i]);
        float dv = fmaf(x, gB[i], aw[i] * kLn2);
        if (p.softplus) dv *= fast_sigmoid(dc.get(i) + bias[i]);
        oddt[i] = none ? 0.f : dv;
        dbias[i] += oddt[i];
        dskip[i] = none ? dskip[i] : fmaf(dy[i], x, dskip[i]);
        if (p.dz) {
          const float z = zc.get(i), zs = fast_sigmoid(z), y = fmaf(sk[i], x, ch[i]);
          odz[i] = none ? 0.f : gc.get(i) * y * zs * fmaf(z, 1.f - zs, 1.f);
        }
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
    ordered_store<NT>(p.pa + (sg * p.D + d) * p.N, n0, order, p.N, dA);
    if (!VAR && p.dh0 && k == 0) ordered_store<NT>(p.dh0 + ((int64_t)b * p.D + d) * p.N, n0, order, p.N, g);
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
// As the forward's: loads a tile ahead, the decays and inputs of eight rows before the rows themselves.
template <typename T, int LN, int NT, bool VAR>
__global__ void __launch_bounds__(128) k_scan_bwd_sum(const P p) {
  constexpr int TS = 32, DB = 128 / LN, NP = LN * NT, QC = DB / 4, RPP = 128 / QC, QN = RPP >= TS ? 1 : TS / RPP;
  constexpr int NH = NT / 2, BQ = TS * NP / 4, BN = (BQ + 127) / 128, RG = 8;
  __shared__ __align__(16) float2 su[TS][DB];  // delta, dy
  __shared__ __align__(16) float sc[TS][NP];
  __shared__ int sflag[TS], sseq[TS];
  __shared__ unsigned smark;
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
  Quad<T> dr[QN], gr[QN], zr[QN], cr[BN];
  int flag = 0, seq = 0;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int row = qr + j * RPP, t = t0 + row;
      const int v = (row < TS && t < t_end) ? valid : 0;
      quad_load<T>(static_cast<const T*>(p.dt) + b * p.ds[0] + t * p.ds[1] + qd, p.vd, v, dr[j]);
      quad_load<T>(static_cast<const T*>(p.dout) + b * p.os[0] + t * p.os[1] + qd, p.vo, v, gr[j]);
      quad_load<T>(static_cast<const T*>(p.z) + b * p.zs[0] + t * p.zs[1] + qd, p.vz, p.z ? v : 0, zr[j]);
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * 128, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      const int v = (q < BQ && t0 + row < t_end) ? min(max(p.N - n, 0), 4) : 0;
      quad_load<T>(static_cast<const T*>(p.cm) + b * p.cs[0] + (t0 + row) * p.cs[1] + grp * p.N + n, p.vc, v, cr[j]);
    }
    if (VAR && tid < TS) flag = t0 + tid < t_end ? row_flags(p, t0 + tid, seq) : 0;
  };
  unsigned broken = 0;
  const int last = t_end > t_first ? t_first + (t_end - t_first - 1) / TS * TS : t_first - TS;
  if (last >= t_first) fetch(last);
  for (int t0 = last; t0 >= t_first; t0 -= TS) {
    unsigned marks = 0;  // a bit for every row of the tile that begins or ends a sequence, or belongs to none
    if (VAR) {
      if (tid < TS) {
        sflag[tid] = flag;
        sseq[tid] = seq;
        marks = __ballot_sync(0xffffffffu, flag);
        if (tid == 0) smark = marks;
        broken |= __ballot_sync(0xffffffffu, flag & (kLast | kNone));
      }
      __syncthreads();
      marks = smark;
    }
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int row = qr + j * RPP;
      if (row >= TS) continue;
      const bool gone = t0 + row >= t_end || (VAR && (sflag[row] & kNone));
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = zr[j].get(i);
        const float dy = p.z ? gr[j].get(i) * z * fast_sigmoid(z) : gr[j].get(i);
        f[2 * i + 1] = gone ? 0.f : dy;
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float2 dl = make_float2(dr[j].get(i) + bias[i], dr[j].get(i + 1) + bias[i + 1]);
        if (p.softplus) dl = softplus2(dl);
        f[2 * i] = gone ? 0.f : dl.x;
        f[2 * i + 2] = gone ? 0.f : dl.y;
      }
      *reinterpret_cast<float4*>(&su[row][qc * 4]) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(&su[row][qc * 4 + 2]) = make_float4(f[4], f[5], f[6], f[7]);
    }
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int q = tid + j * 128, row = q / (NP / 4), n = (q - row * (NP / 4)) * 4;
      if (q >= BQ) continue;
      const bool none = VAR && (sflag[row] & kNone);
      float fc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) fc[i] = none ? 0.f : cr[j].get(i);
      *reinterpret_cast<float4*>(&sc[row][n]) = make_float4(fc[0], fc[1], fc[2], fc[3]);
    }
    __syncthreads();
    if (t0 > t_first) fetch(t0 - TS);
#pragma unroll 1
    for (int r0 = (min(TS, t_end - t0) - 1) / RG * RG; r0 >= 0; r0 -= RG) {  // rows at t_end and beyond: nothing moves
      if (VAR && (marks >> r0 & ((1u << RG) - 1))) {
#pragma unroll 1
        for (int r = min(r0 + RG, t_end - t0) - 1; r >= r0; --r) {
          const int f = sflag[r];
          if (f & (kLast | kNone)) {
#pragma unroll
            for (int j = 0; j < NH; ++j) g[j] = dup(0.f);
            if ((f & kLast) && p.dht && on) states_load<NT>(p.dht + ((int64_t)sseq[r] * p.D + d) * p.N, n0, p.N, g);
          }
          float2 Cv[NH];
          pairs_load<NT>(&sc[r][n0], Cv);
          const float2 q = su[r][cb];
#pragma unroll
          for (int j = 0; j < NH; ++j) g[j] = mul2(decay2(q.x, A[j]), fma2(Cv[j], dup(q.y), g[j]));
          dsum += q.x;
        }
        continue;
      }
      float2 a[RG][NH], in[RG][NH];
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        float2 Cv[NH];
        pairs_load<NT>(&sc[r0 + r][n0], Cv);
        const float2 q = su[r0 + r][cb];
        dsum += q.x;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          a[r][j] = decay2(q.x, A[j]);
          in[r][j] = mul2(Cv[j], dup(q.y));
        }
      }
#pragma unroll
      for (int r = RG - 1; r >= 0; --r)
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          const float2 s = make_float2(in[r][j].x + g[j].x, in[r][j].y + g[j].y);
          g[j] = mul2(a[r][j], s);
        }
    }
    __syncthreads();
  }
  if (on) {
    states_store<NT>(p.carry + (((int64_t)b * p.nseg + k) * p.D + d) * p.N, n0, p.N, g);
    if (nl == 0) p.sdelta[((int64_t)b * p.nseg + k) * p.D + d] = dsum;
  }
  if (VAR && blockIdx.x == 0 && tid == 0) p.broken[k] = broken != 0;
}

// The partial sums, each in a fixed order, in one launch: dB, dC [B, T, G, N] over the parts of a group (the first
// `bc_blocks` blocks), dA, dD and dbias over batch rows and segments (the rest).
template <typename T>
__global__ void __launch_bounds__(256) k_scan_fold(const P p, int64_t bc_blocks, T* __restrict__ dB, T* __restrict__ dC,
                                                   float* __restrict__ dA, float* __restrict__ dskip,
                                                   float* __restrict__ dbias) {
  if (blockIdx.x < bc_blocks) {
    const int64_t per = (int64_t)p.B * p.T * 2 * p.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= per * p.G) return;
    const int grp = (int)(i / per);
    const int64_t at = i - grp * per, row = at / (2 * p.N);
    const int c = (int)(at - row * 2 * p.N);
    const float* src = p.pbc + (int64_t)grp * p.parts * per + at;
    float s = 0.f;
    for (int k = 0; k < p.parts; ++k) s += src[k * per];
    T* o = c < p.N ? dB : dC;
    o[(row * p.G + grp) * p.N + (c < p.N ? c : c - p.N)] = from_f<T>(s);
    return;
  }
  const int64_t dn = (int64_t)p.D * p.N, i = (blockIdx.x - bc_blocks) * 256 + threadIdx.x;
  if (i >= dn + 2 * p.D) return;
  const int64_t j = i - dn;  // dD, then dbias
  float* o = i < dn ? dA + i : j < p.D ? dskip + j : dbias + (j - p.D);
  if ((i < dn ? dA : j < p.D ? dskip : dbias) == nullptr) return;
  const float* src = i < dn ? p.pa + i : p.pd + j;
  const int64_t stride = i < dn ? dn : 2 * (int64_t)p.D;
  float s = 0.f;
  for (int k = 0; k < p.B * p.nseg; ++k) s += src[k * stride];
  *o = s;
}

size_t plan_bwd(P& p, void* ws) {
  p.parts = blocks_of(p, kBwdThreads / lanes_of(p.N)) / p.G;
  split(p, p.parts * p.G, kBwdBlocks, 2);
  Carve c{static_cast<char*>(ws)};
  p.pbc = c.take((size_t)p.G * p.parts * p.B * p.T * 2 * p.N);
  p.pa = c.take((size_t)p.B * p.nseg * p.D * p.N);
  p.pd = c.take((size_t)p.B * p.nseg * 2 * p.D);
  return carve_segments(p, c);
}

}  // namespace ssm
}  // namespace tops

using namespace tops;
using namespace tops::ssm;

extern "C" {

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
  TOPS_CHECK_ARG(f.B == 0 || f.A, "ssm_scan_bwd: A is required");
  TOPS_CHECK_ARG(!rows || !f.z || a->dz, "ssm_scan_bwd: z needs dz");
  TOPS_CHECK_ARG(aligned_to(a->workspace, 16), "ssm_scan_bwd: workspace must be 16-byte aligned");
  P p = params(&f);
  const size_t need = plan_bwd(p, a->workspace);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "ssm_scan_bwd: workspace smaller than tops_gla_ssm_scan_bwd_workspace_size()");
  p.dout = a->dout; p.os[0] = a->dout_stride_b; p.os[1] = a->dout_stride_t;
  p.dht = a->dht; p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz; p.dh0 = a->dh0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = empty_states(p, p.dht, p.dh0, true, st)) return rc;
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
      if (bytes > 47 * 1024) {  // the rows' flags come on top
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return cuda_status(e, "ssm_scan_bwd");
      }
      kernel<<<dim3(p.parts * p.G, p.B, p.nseg), kBwdThreads, bytes, st>>>(p);
      return 0;
    });
    if (rc) return rc;
    TOPS_CUDA_LAUNCH_CHECK("ssm_scan_bwd");
  }
  LaunchTimer lt(st, "ssm_scan_fold");
  const int64_t bc = (int64_t)p.B * p.T * 2 * p.N * p.G, params_n = (int64_t)p.D * p.N + 2 * p.D;
  const int64_t bc_blocks = (bc + 255) / 256;
  by_type(f.dtype, [&](auto t) {
    using T = decltype(t);
    k_scan_fold<T><<<(unsigned)(bc_blocks + (params_n + 255) / 256), 256, 0, st>>>(
        p, bc_blocks, static_cast<T*>(a->dB), static_cast<T*>(a->dC), a->dA, a->dskip, a->ddt_bias);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("ssm_scan_fold");
  return TOPS_OK;
}

}  // extern "C"
