// Causal depthwise short convolution over time, channels last:
//   p_t = b + sum_{j < W} w[:, j] x_{t - W + 1 + j},   y = p  or  p sigmoid(p)
// Rows before a sequence's first are its carried state [N, D, W - 1] (last column = the
// newest input) or zeros.  Backward, with dp = dy y'(p):
//   dx_s = sum_k w[:, W - 1 - k] dp_{s + k},   dw[:, j] = sum_t dp_t x_{t - W + 1 + j},   db = sum_t dp_t
//
// Nothing is reused but the W - 1 rows before a row, so HBM bounds it: a thread owns V channels (16 bytes; 8 in the
// backward, whose sums need the registers) and walks down a strip of rows with the window in registers.  B8 T4096 D2048
// bf16, calls in a row: forward 57 us = 4.7 TB/s, backward 105 us = 3.8 TB/s and 115 with the parameters' sums.  The
// backward fills no unit (HBM 46 %, issue 59 %): 128 registers leave 14 warps an SM, too few to cover each other's waits.
#include <algorithm>

#include "rowtypes.cuh"

namespace tops {
namespace conv {

struct P {
  int B, T, D, N;  // N sequences
  int act, wdtype, wvec;  // wvec: the weights of V channels start on a vector
  const int32_t* cu;
  int64_t xb, xt;  // strides of x in elements (batch, row)
  const void* x;
  const void* w;
  const void* b;
  const void* state;
  void* y;
  void* fin;
  // backward
  int64_t gb, gt;  // strides of dy
  const void* dy;
  const void* dfin;
  void* dx;
  float* part;  // [strips][W + 1][D]: dw and db of one strip
  void* dstate;
  int strip, strips, dv;  // rows of a strip, strips of one batch row, column groups
};

__device__ __forceinline__ float act_fwd(float p, int act) { return act ? p * fast_sigmoid(p) : p; }
__device__ __forceinline__ float act_grad(float p, int act) {
  if (!act) return 1.f;
  const float s = fast_sigmoid(p);
  return s * fmaf(p, 1.f - s, 1.f);
}

// weights [V][W] and biases of V channels from d0: V W elements in a row
template <typename T, int V, int W>
__device__ __forceinline__ void load_params(const P& p, int d0, float (&w)[W][V], float (&bias)[V]) {
  float flat[W][V];  // W vectors of V elements
  if (p.wdtype == TOPS_F32 && sizeof(T) != 4) {
    const float* wp = static_cast<const float*>(p.w) + (int64_t)d0 * W;
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) flat[j][i] = wp[j * V + i];
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = p.b ? static_cast<const float*>(p.b)[d0 + i] : 0.f;
  } else {
    const T* wp = static_cast<const T*>(p.w) + (int64_t)d0 * W;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (p.wvec) Vx<T, V>::load(wp + j * V, flat[j]);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) flat[j][i] = to_f<T>(wp[j * V + i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = p.b ? to_f<T>(static_cast<const T*>(p.b)[d0 + i]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = flat[(i * W + j) / V][(i * W + j) % V];
}

// Rows on their way: every thread copies the vectors that it will use itself into its own column of shared memory, so
// that several batches of R rows are in flight without registers and no thread waits for another.
constexpr int R = 4;

// the sequence of row t of batch row b: [s, e) and its number (-1: none)
__device__ __forceinline__ SeqAt seq_of(const P& p, int b, int t) {
  if (p.cu == nullptr) return SeqAt{b, 0, p.T};
  return seq_at(p.cu, p.N, p.T, t);
}

// x at row t of a sequence that starts at s, channels d0.. (from the carried state before s)
template <typename T, int V, int W>
__device__ __forceinline__ void row_or_state(const P& p, int b, const SeqAt& q, int t, int d0, float (&r)[V]) {
  if (t >= q.s) {
    Vx<T, V>::load(static_cast<const T*>(p.x) + b * p.xb + t * p.xt + d0, r);
  } else if (p.state != nullptr && q.n >= 0) {
    const T* st = static_cast<const T*>(p.state) + ((int64_t)q.n * p.D + d0) * (W - 1) + (W - 1) + (t - q.s);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = to_f<T>(st[i * (W - 1)]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = 0.f;
  }
}

// p of a row from its window
template <int V, int W>
__device__ __forceinline__ void sum_of(const float (&w)[W][V], const float (&bias)[V], const float (&win)[W][V], float (&a)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = bias[i];
#pragma unroll
  for (int j = 0; j < W; ++j) fma_n<V>(a, w[j], win[j]);
}
template <int V, int W>
__device__ __forceinline__ void act_of(const P& p, const float (&w)[W][V], const float (&bias)[V],
                                       const float (&win)[W][V], float (&out)[V]) {
  sum_of<V, W>(w, bias, win, out);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = act_fwd(out[i], p.act);
}

// final state of sequence n, channels d0..: its last W - 1 inputs
template <typename T, int V, int W>
__device__ void final_state(const P& p, int n, int d0) {
  SeqAt q{n, 0, p.T};
  int b = n;
  if (p.cu != nullptr) {
    q.s = max(__ldg(p.cu + n), 0);
    q.e = max(q.s, min(__ldg(p.cu + n + 1), p.T));
    b = 0;
  }
  T* f = static_cast<T*>(p.fin) + ((int64_t)n * p.D + d0) * (W - 1);
#pragma unroll
  for (int c = 0; c < W - 1; ++c) {
    float r[V];
    row_or_state<T, V, W>(p, b, q, q.e - (W - 1) + c, d0, r);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i * (W - 1) + c] = from_f<T>(r[i]);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(128) k_conv_fwd(const P p) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int64_t unit = id / p.dv;
  const int d0 = (int)(id - unit * p.dv) * V;
  const int64_t nstrips = (int64_t)p.B * p.strips;
  if (unit >= nstrips) {
    const int64_t n = unit - nstrips;
    if (p.fin != nullptr && n < p.N) final_state<T, V, W>(p, (int)n, d0);
    return;
  }
  const int b = (int)(unit / p.strips);
  const int t0 = (int)(unit - (int64_t)b * p.strips) * p.strip;
  const int t1 = min(t0 + p.strip, p.T);
  const T* x = static_cast<const T*>(p.x) + b * p.xb + d0;
  constexpr int kAhead = 3, kSlots = R * (kAhead + 1);
  __shared__ Raw<T, V> ring[V == 1 ? 1 : kSlots][128];
  const int batches = (t1 - t0) / R;
  auto ask = [&](int g) {
    if (g < batches)
#pragma unroll
      for (int r = 0; r < R; ++r)
        copy_async<Raw<T, V>::B>(&ring[(g * R + r) % kSlots][threadIdx.x], x + (t0 + g * R + r) * p.xt);
    copies_commit();
  };
  if constexpr (V > 1)  // the first rows are on their way while the weights and the sequence are looked up
#pragma unroll
    for (int g = 0; g < kAhead; ++g) ask(g);
  float w[W][V], bias[V];
  load_params<T, V, W>(p, d0, w, bias);
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.T * p.D + d0;
  SeqAt q = seq_of(p, b, t0);
  float win[W][V];  // rows t - W + 1 .. t
#pragma unroll
  for (int j = 0; j < W - 1; ++j) row_or_state<T, V, W>(p, b, q, t0 - (W - 1) + j, d0, win[j + 1]);
  // one row, at any place of its sequence
  auto row = [&](int t) {
    if (t >= q.e || q.n < 0) {
      q = seq_of(p, b, t);
      if (q.n < 0) {
        float zero[V];
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        Vx<T, V>::store(y + (int64_t)t * p.D, zero);
        return;
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j) row_or_state<T, V, W>(p, b, q, t - (W - 1) + j, d0, win[j + 1]);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
    Vx<T, V>::load(x + t * p.xt, win[W - 1]);
    float out[V];
    act_of<V, W>(p, w, bias, win, out);
    Vx<T, V>::store(y + (int64_t)t * p.D, out);
  };
  if constexpr (V == 1) {
    for (int t = t0; t < t1; ++t) row(t);
    return;
  } else {
    for (int g = 0; g < batches; ++g) {
      ask(g + kAhead);
      copies_wait<kAhead>();
      const int t = t0 + g * R;
      if (t + R > q.e || q.n < 0) {  // a sequence ends here
        for (int r = 0; r < R; ++r) row(t + r);
        continue;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
        ring[(g * R + r) % kSlots][threadIdx.x].get(win[W - 1]);
        float out[V];
        act_of<V, W>(p, w, bias, win, out);
        Vx<T, V>::store(y + (int64_t)(t + r) * p.D, out);
      }
    }
    for (int t = t0 + batches * R; t < t1; ++t) row(t);
  }
}

// dp of a row from its window; dp holds the row's dy
template <int V, int W>
__device__ __forceinline__ void dp_of(const P& p, const float (&w)[W][V], const float (&bias)[V],
                                      const float (&win)[W][V], float (&dp)[V]) {
  float a[V];
  sum_of<V, W>(w, bias, win, a);
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = act_grad(a[i], p.act);
  mul_n<V>(dp, dp, a);
}

// Gradient of sequence n's carried state, channels d0..: its column c is read by the rows
// i <= c of the sequence (tap c - i) and, where the sequence is shorter than the state, by
// the final state's column c - len.
template <typename T, int V, int W>
__device__ void state_grad(const P& p, const float (&w)[W][V], const float (&bias)[V], int n, int d0) {
  SeqAt q{n, 0, p.T};
  int b = n;
  if (p.cu != nullptr) {
    q.s = max(__ldg(p.cu + n), 0);
    q.e = max(q.s, min(__ldg(p.cu + n + 1), p.T));
    b = 0;
  }
  const int len = q.e - q.s;
  float ds[W - 1][V];
#pragma unroll
  for (int c = 0; c < W - 1; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) ds[c][i] = 0.f;
#pragma unroll
  for (int r = 0; r < W - 1; ++r) {
    if (r < len) {
      float win[W][V], dp[V];
#pragma unroll
      for (int j = 0; j < W; ++j) row_or_state<T, V, W>(p, b, q, q.s + r - (W - 1) + j, d0, win[j]);
      Vx<T, V>::load(static_cast<const T*>(p.dy) + b * p.gb + (q.s + r) * p.gt + d0, dp);
      dp_of<V, W>(p, w, bias, win, dp);
#pragma unroll
      for (int c = r; c < W - 1; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) ds[c][i] = fmaf(w[c - r][i], dp[i], ds[c][i]);
    }
  }
  if (p.dfin != nullptr) {
    const T* f = static_cast<const T*>(p.dfin) + ((int64_t)n * p.D + d0) * (W - 1);
#pragma unroll
    for (int c = 0; c < W - 1; ++c)
      if (c >= len)
#pragma unroll
        for (int i = 0; i < V; ++i) ds[c][i] += to_f<T>(f[i * (W - 1) + c - len]);
  }
  T* o = static_cast<T*>(p.dstate) + ((int64_t)n * p.D + d0) * (W - 1);
#pragma unroll
  for (int c = 0; c < W - 1; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) o[i * (W - 1) + c] = from_f<T>(ds[c][i]);
}

// One strip: rows t0 .. t1 of dx need dp up to W - 1 rows further (computed again by the next
// strip, whose rows alone go into dw and db).
template <typename T, int V, int W>
__global__ void __launch_bounds__(128) k_conv_bwd(const P p) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int64_t unit = id / p.dv;
  const int d0 = (int)(id - unit * p.dv) * V;
  const int64_t nstrips = (int64_t)p.B * p.strips;
  if (unit >= nstrips) {
    if (p.dstate == nullptr || unit - nstrips >= p.N) return;
    float w[W][V], bias[V];
    load_params<T, V, W>(p, d0, w, bias);
    state_grad<T, V, W>(p, w, bias, (int)(unit - nstrips), d0);
    return;
  }
  const int b = (int)(unit / p.strips);
  const int t0 = (int)(unit - (int64_t)b * p.strips) * p.strip;
  const int t1 = min(t0 + p.strip, p.T);
  const T* x = static_cast<const T*>(p.x) + b * p.xb + d0;
  const T* dy = static_cast<const T*>(p.dy) + b * p.gb + d0;
  constexpr int kAhead = Raw<T, V>::B == 16 ? 1 : 3, kSlots = R * (kAhead + 1);  // 32 KB
  __shared__ Raw<T, V> ring[2][V == 1 ? 1 : kSlots][128];
  const int batches = (t1 - t0) / R;
  auto ask = [&](int g) {
    if (g < batches)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int t = t0 + g * R + r, at = (g * R + r) % kSlots;
        copy_async<Raw<T, V>::B>(&ring[0][at][threadIdx.x], x + t * p.xt);
        copy_async<Raw<T, V>::B>(&ring[1][at][threadIdx.x], dy + t * p.gt);
      }
    copies_commit();
  };
  if constexpr (V > 1)
#pragma unroll
    for (int g = 0; g < kAhead; ++g) ask(g);
  float w[W][V], bias[V];
  load_params<T, V, W>(p, d0, w, bias);
  T* dx = static_cast<T*>(p.dx) + (int64_t)b * p.T * p.D + d0;
  SeqAt q = seq_of(p, b, t0);
  float win[W][V], acc[W][V], dw[W][V], db[V];  // acc[k]: dx of row t - k so far
#pragma unroll
  for (int i = 0; i < V; ++i) db[i] = 0.f;
#pragma unroll
  for (int j = 0; j < W; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[j][i] = dw[j][i] = 0.f;
#pragma unroll
  for (int j = 0; j < W - 1; ++j) row_or_state<T, V, W>(p, b, q, t0 - (W - 1) + j, d0, win[j + 1]);
  // one row, at any place of its sequence (rows past T or the sequence add nothing)
  auto row = [&](int t) {
    if (t < p.T && (t >= q.e || q.n < 0)) {
      q = seq_of(p, b, t);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) row_or_state<T, V, W>(p, b, q, t - (W - 1) + j, d0, win[j + 1]);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
#pragma unroll
    for (int j = W - 1; j > 0; --j)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[j][i] = acc[j - 1][i];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[0][i] = 0.f;
    if (t < p.T && q.n >= 0) {
      float dp[V];
      Vx<T, V>::load(x + t * p.xt, win[W - 1]);
      Vx<T, V>::load(dy + t * p.gt, dp);
      dp_of<V, W>(p, w, bias, win, dp);
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (t - k >= q.s)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[k][i] = fmaf(w[W - 1 - k][i], dp[i], acc[k][i]);
      if (t < t1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          db[i] += dp[i];
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][i] = fmaf(dp[i], win[j][i], dw[j][i]);
        }
        if (p.dfin != nullptr && t >= q.e - (W - 1)) {  // the final state reads this row too
          const T* f = static_cast<const T*>(p.dfin) + ((int64_t)q.n * p.D + d0) * (W - 1) + t - q.e + (W - 1);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[0][i] += to_f<T>(f[i * (W - 1)]);
        }
      }
    }
    if (t - (W - 1) >= t0) Vx<T, V>::store(dx + (int64_t)(t - (W - 1)) * p.D, acc[W - 1]);
  };
  const int stop = t1 + W - 1;
  if constexpr (V == 1) {
    for (int t = t0; t < stop; ++t) row(t);
  } else {
    for (int g = 0; g < batches; ++g) {
      ask(g + kAhead);
      copies_wait<kAhead>();
      const int t = t0 + g * R;
      // fewer than W - 1 rows from the strip's begin or from an end of the sequence
      if (q.n < 0 || t < max(q.s, t0) + W - 1 || t + R > q.e - (W - 1)) {
        for (int r = 0; r < R; ++r) row(t + r);
        continue;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
#pragma unroll
        for (int j = W - 1; j > 0; --j)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[j][i] = acc[j - 1][i];
        float dp[V];
        ring[0][(g * R + r) % kSlots][threadIdx.x].get(win[W - 1]);
        ring[1][(g * R + r) % kSlots][threadIdx.x].get(dp);
        dp_of<V, W>(p, w, bias, win, dp);
        mul_n<V>(acc[0], w[W - 1], dp);
#pragma unroll
        for (int k = 1; k < W; ++k) fma_n<V>(acc[k], w[W - 1 - k], dp);
#pragma unroll
        for (int i = 0; i < V; ++i) db[i] += dp[i];
#pragma unroll
        for (int j = 0; j < W; ++j) fma_n<V>(dw[j], dp, win[j]);
        Vx<T, V>::store(dx + (int64_t)(t + r - (W - 1)) * p.D, acc[W - 1]);
      }
    }
    for (int t = t0 + batches * R; t < stop; ++t) row(t);
  }
  if (p.part != nullptr) {
    float* o = p.part + unit * (W + 1) * p.D + d0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j < W; ++j) o[(int64_t)j * p.D + i] = dw[j][i];
      o[(int64_t)W * p.D + i] = db[i];
    }
  }
}

// dw [D, W] and db [D] = the strips' sums, in a fixed order
__global__ void __launch_bounds__(1024) k_conv_dw(int64_t strips, int D, int W, int wdtype,
                                                  const float* __restrict__ part, void* dw, void* db) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int cols = (W + 1) * D;
  float s = 0.f;
  if (c < cols)
    for (int64_t i = threadIdx.y; i < strips; i += 32) s += part[i * cols + c];
  __shared__ float red[32][33];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    float t = 0.f;
    for (int y = 0; y < 32; ++y) t += red[y][threadIdx.x];
    const int j = c / D, d = c - j * D;
    if (j < W) {
      if (dw) store_param(dw, wdtype, (int64_t)d * W + j, t);
    } else if (db) {
      store_param(db, wdtype, d, t);
    }
  }
}

// One token of each of B rows: the window is the row's state and its input.
template <typename T, int V, int W>
__global__ void __launch_bounds__(128) k_conv_step(const P p) {
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int64_t b = id / p.dv;
  const int d0 = (int)(id - b * p.dv) * V;
  if (b >= p.B) return;
  float x[V], st[V * (W - 1)], out[V];
  Vx<T, V>::load(static_cast<const T*>(p.x) + b * p.xb + d0, x);
  const T* s = static_cast<const T*>(p.state) + (b * p.D + d0) * (W - 1);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {  // V (W - 1) elements in a row: W - 1 vectors
    float v[V];
    Vx<T, V>::load(s + j * V, v);
#pragma unroll
    for (int i = 0; i < V; ++i) st[j * V + i] = v[i];
  }
  float w[W][V], bias[V];
  load_params<T, V, W>(p, d0, w, bias);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float a = bias[i];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) a = fmaf(w[j][i], st[i * (W - 1) + j], a);
    a = fmaf(w[W - 1][i], x[i], a);
    out[i] = act_fwd(a, p.act);
  }
  Vx<T, V>::store(static_cast<T*>(p.y) + b * p.D + d0, out);
  T* f = static_cast<T*>(p.fin) + (b * p.D + d0) * (W - 1);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = j * V + i, ch = e / (W - 1), col = e % (W - 1);
      v[i] = col + 1 < W - 1 ? st[ch * (W - 1) + col + 1] : x[ch];
    }
    Vx<T, V>::store(f + j * V, v);
  }
}

template <typename F>
int by_width(int W, F f) {
  if (W == 2) return f(std::integral_constant<int, 2>());
  if (W == 3) return f(std::integral_constant<int, 3>());
  return f(std::integral_constant<int, 4>());
}

// calls f with (T, V, W); V is V16 channels (four in fp32) where every base and stride allows 16-byte accesses, else 1
template <int V16, typename F>
int by_type(int dtype, bool wide, int W, F f) {
  return by_width(W, [&](auto w) {
    constexpr int WW = decltype(w)::value;
    if (dtype == TOPS_F32)
      return wide ? f(float(), std::integral_constant<int, 4>(), std::integral_constant<int, WW>())
                  : f(float(), std::integral_constant<int, 1>(), std::integral_constant<int, WW>());
    if (dtype == TOPS_BF16)
      return wide ? f(__nv_bfloat16(), std::integral_constant<int, V16>(), std::integral_constant<int, WW>())
                  : f(__nv_bfloat16(), std::integral_constant<int, 1>(), std::integral_constant<int, WW>());
    return wide ? f(__half(), std::integral_constant<int, V16>(), std::integral_constant<int, WW>())
                : f(__half(), std::integral_constant<int, 1>(), std::integral_constant<int, WW>());
  });
}

int check(const tops_gla_conv_args* a) {
  TOPS_CHECK_ARG(a != nullptr, "causal_conv: args is NULL");
  TOPS_CHECK_ARG(a->B >= 0 && a->T >= 0 && a->D > 0 && a->N >= 0, "causal_conv: negative or zero dimension");
  if (a->B > kMaxRows || a->T > kMaxRows || a->D > kMaxChannels) return fail(TOPS_ERR_UNSUPPORTED, "causal_conv: too many rows or channels");
  if (a->W < 2 || a->W > 4) return fail(TOPS_ERR_UNSUPPORTED, "causal_conv: the kernel width must be 2, 3 or 4");
  TOPS_CHECK_ARG(dtype_known(a->dtype), "causal_conv: unknown dtype");
  TOPS_CHECK_ARG(a->w_dtype == a->dtype || a->w_dtype == TOPS_F32, "causal_conv: w_dtype must be dtype or TOPS_F32");
  TOPS_CHECK_ARG(a->activation == 0 || a->activation == 1, "causal_conv: activation must be 0 (none) or 1 (silu)");
  if (a->cu_seqlens) {
    TOPS_CHECK_ARG(a->B == 1, "causal_conv: cu_seqlens requires B == 1");
    TOPS_CHECK_ARG(a->N >= 1, "causal_conv: cu_seqlens requires N >= 1");
  } else {
    TOPS_CHECK_ARG(a->N == a->B, "causal_conv: N must equal B without cu_seqlens");
  }
  return TOPS_OK;
}

// elements are reachable by 16-byte accesses at every row
bool wide_ok(const tops_gla_conv_args* a) {
  const int es = dtype_bytes(a->dtype), v = 16 / es;
  return a->D % v == 0 && a->x_stride_b % v == 0 && a->x_stride_t % v == 0 && aligned_to(a->x, 16);
}

P params(const tops_gla_conv_args* a) {
  P p{};
  p.B = a->B; p.T = a->T; p.D = a->D; p.N = a->N;
  p.act = a->activation; p.wdtype = a->w_dtype;
  p.wvec = aligned_to(a->w, 16);
  p.cu = a->cu_seqlens;
  p.xb = a->x_stride_b; p.xt = a->x_stride_t;
  p.x = a->x; p.w = a->w; p.b = a->bias; p.state = a->initial_state;
  p.y = a->y; p.fin = a->final_state;
  return p;
}

// Rows of a strip: long strips read their W - 1 rows of halo (and write their partial sums)
// rarely, short ones give every SM threads to hide the loads with.
void split(P& p, int v, int64_t threads_wanted, int most) {
  p.dv = p.D / v;
  const int64_t rows = ((int64_t)p.B * p.T * p.dv + threads_wanted - 1) / threads_wanted;
  p.strip = (int)std::min<int64_t>(most, std::max<int64_t>(8, rows));
  p.strips = (p.T + p.strip - 1) / p.strip;
}

// Four blocks of 128 threads fill an SM's registers: strips that make one wave of them (forward) or two (backward), as
// far as the cap lets them (23 packed prompts of 9973 rows: 22 -> 18 us against strips of 8; backward B8 T4096 D2048: 1024
// threads an SM 108 us, 512: 114, 1536: 116, each between events of its own, which add some 3 us).
constexpr int64_t kFwdThreads = 148 * 512, kBwdThreads = 148 * 1024;

}  // namespace conv
}  // namespace tops

using namespace tops;
using namespace tops::conv;

extern "C" {

TOPS_API int tops_gla_causal_conv_fwd(const tops_gla_conv_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if ((int64_t)a->B * a->T == 0 && a->N == 0) return TOPS_OK;
  const bool rows = (int64_t)a->B * a->T > 0;
  TOPS_CHECK_ARG(!rows || (a->x && a->w && a->y), "causal_conv_fwd: x, w and y are required");
  if (!rows && !a->final_state) return TOPS_OK;
  const bool wide = wide_ok(a) && aligned_to(a->y, 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "causal_conv_fwd");
  by_type<8>(a->dtype, wide, a->W, [&](auto t, auto v, auto w) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = decltype(w)::value;
    P p = params(a);
    split(p, V, kFwdThreads, 32);
    const int64_t n = ((int64_t)p.B * p.strips + (p.fin ? p.N : 0)) * p.dv;
    k_conv_fwd<T, V, W><<<(unsigned)((n + 127) / 128), 128, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("causal_conv_fwd");
  return TOPS_OK;
}

TOPS_API size_t tops_gla_causal_conv_bwd_workspace_size(const tops_gla_conv_bwd_args* a) {
  if (a == nullptr || check(&a->f) != TOPS_OK || (!a->dw && !a->dbias)) return 0;
  size_t most = 0;  // of the two layouts (the alignment of the pointers decides between them)
  for (int v : {1, 4}) {
    if (a->f.D % v) continue;
    P p = params(&a->f);
    split(p, v, kBwdThreads, 256);
    most = std::max(most, (size_t)p.B * p.strips * (a->f.W + 1) * p.D * sizeof(float));
  }
  return most;
}

TOPS_API int tops_gla_causal_conv_bwd(const tops_gla_conv_bwd_args* a, void* stream) {
  TOPS_CHECK_ARG(a != nullptr, "causal_conv_bwd: args is NULL");
  if (int rc = check(&a->f)) return rc;
  const tops_gla_conv_args& f = a->f;
  const bool rows = (int64_t)f.B * f.T > 0;
  TOPS_CHECK_ARG(!rows || (f.x && f.w && a->dy && a->dx), "causal_conv_bwd: x, w, dy and dx are required");
  TOPS_CHECK_ARG(f.w, "causal_conv_bwd: w is required");
  const size_t need = tops_gla_causal_conv_bwd_workspace_size(a);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(TOPS_ERR_WORKSPACE, "causal_conv_bwd: workspace smaller than tops_gla_causal_conv_bwd_workspace_size()");
  const int v0 = 16 / dtype_bytes(f.dtype);
  const bool wide = wide_ok(&f) && aligned_to(a->dx, 16) && aligned_to(a->dy, 16) && a->dy_stride_b % v0 == 0 &&
                    a->dy_stride_t % v0 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int64_t strips = 0;
  if (rows || a->dstate) {
    LaunchTimer lt(st, "causal_conv_bwd");
    by_type<4>(f.dtype, wide, f.W, [&](auto t, auto v, auto w) {
      using T = decltype(t);
      constexpr int V = decltype(v)::value, W = decltype(w)::value;
      P p = params(&f);
      p.gb = a->dy_stride_b; p.gt = a->dy_stride_t;
      p.dy = a->dy; p.dfin = a->dfinal; p.dx = a->dx; p.dstate = a->dstate;
      p.part = (a->dw || a->dbias) ? static_cast<float*>(a->workspace) : nullptr;
      split(p, V, kBwdThreads, 256);
      strips = (int64_t)p.B * p.strips;
      const int64_t n = (strips + (p.dstate ? p.N : 0)) * p.dv;
      k_conv_bwd<T, V, W><<<(unsigned)((n + 127) / 128), 128, 0, st>>>(p);
      return 0;
    });
    TOPS_CUDA_LAUNCH_CHECK("causal_conv_bwd");
  }
  if (a->dw || a->dbias) {
    LaunchTimer lt(st, "causal_conv_dw");
    const int cols = (f.W + 1) * f.D;
    k_conv_dw<<<(cols + 31) / 32, dim3(32, 32), 0, st>>>(strips, f.D, f.W, f.w_dtype,
                                                         static_cast<const float*>(a->workspace), a->dw, a->dbias);
    TOPS_CUDA_LAUNCH_CHECK("causal_conv_dw");
  }
  return TOPS_OK;
}

TOPS_API int tops_gla_causal_conv_step(const tops_gla_conv_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  TOPS_CHECK_ARG(a->T == 1 && !a->cu_seqlens, "causal_conv_step: T must be 1, without cu_seqlens");
  if (a->B == 0) return TOPS_OK;
  TOPS_CHECK_ARG(a->x && a->w && a->initial_state && a->y && a->final_state,
                 "causal_conv_step: x, w, initial_state, y and final_state are required");
  const bool wide = wide_ok(a) && aligned_to(a->y, 16) && aligned_to(a->initial_state, 16) &&
                    aligned_to(a->final_state, 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LaunchTimer lt(st, "causal_conv_step");
  by_type<8>(a->dtype, wide, a->W, [&](auto t, auto v, auto w) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = decltype(w)::value;
    P p = params(a);
    p.dv = p.D / V;
    const int64_t n = (int64_t)p.B * p.dv;
    k_conv_step<T, V, W><<<(unsigned)((n + 127) / 128), 128, 0, st>>>(p);
    return 0;
  });
  TOPS_CUDA_LAUNCH_CHECK("causal_conv_step");
  return TOPS_OK;
}

}  // extern "C"
