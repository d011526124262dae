// Element access of the kernels that take every storage type with strides: vectors of V
// elements of T in as few aligned 16-byte accesses as V allows, fp32 arithmetic between.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace tops {

template <typename T, int V>
struct Vx {
  static constexpr int BYTES = V * (int)sizeof(T);
  static __device__ __forceinline__ void load(const T* p, float (&r)[V]) {
    alignas(16) T raw[V];
    load_raw(p, raw);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = to_f<T>(raw[i]);
  }
  static __device__ __forceinline__ void load_raw(const T* p, T (&raw)[V]) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i)
        reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) raw[i] = p[i];
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&r)[V]) {
    alignas(16) T raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = from_f<T>(r[i]);
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = raw[i];
    }
  }
};

// V elements as they lie in memory, taken apart only where they are used: a load's registers may not be touched before
template <typename T, int V>
struct Raw {
  static constexpr int B = V * (int)sizeof(T);
  alignas(B >= 16 ? 16 : B >= 4 ? B : 4) uint32_t w[B >= 4 ? B / 4 : 1];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (B % 16 == 0) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (B == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (B == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void get(float (&r)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) {
        r[i] = __uint_as_float(w[i]);
      } else {
        const uint16_t h = (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]);
        if constexpr (std::is_same<T, __half>::value) r[i] = __half2float(__ushort_as_half(h));
        else r[i] = __uint_as_float((uint32_t)h << 16);
      }
    }
  }
};

// copies of 8 or 16 bytes (or several of 16) from global to shared memory, in groups that are waited for by their order
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (BYTES > 16) {
    copy_async<16>(dst, src);
    copy_async<BYTES - 16>(static_cast<char*>(dst) + 16, static_cast<const char*>(src) + 16);
  } else if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(a), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int AHEAD>
__device__ __forceinline__ void copies_wait() {  // all but the last AHEAD groups have arrived
  asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
}

// element i of a small parameter tensor stored in `dtype` (enum tops_dtype)
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
  if (dtype == TOPS_F32) return static_cast<const float*>(p)[i];
  if (dtype == TOPS_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == TOPS_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == TOPS_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

constexpr float kLog2e = 1.44269504088896341f;

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
// d += a b, d = a b over V elements, two at a time
template <int V>
__device__ __forceinline__ void fma_n(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    d[0] = fmaf(a[0], b[0], d[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(d[i], d[i + 1]));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void mul_n(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    d[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = mul2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  }
}

// 1 / (1 + exp(-x)): both hardware approximations, off by at most 2^-22 each; 0 and 1 at the infinities
__device__ __forceinline__ float fast_sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(-kLog2e * x)));
  return r;
}

// ---------------------------------------------------------------------------
// packed sequences: rows [cu[n], cu[n+1]) of one axis of T rows.  The offsets lie on the
// device and are not read by the host, so every value is clamped to the axis here: wrong
// offsets give wrong rows, never an access out of range.  A row that no sequence covers
// belongs to none (n = -1).
// ---------------------------------------------------------------------------
struct SeqAt {
  int n, s, e;
};

__device__ __forceinline__ SeqAt seq_at(const int32_t* __restrict__ cu, int N, int T, int t) {
  int lo = 0, hi = N - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid; else hi = mid - 1;
  }
  SeqAt q{lo, max(__ldg(cu + lo), 0), min(__ldg(cu + lo + 1), T)};
  if (t < q.s || t >= q.e) q.n = -1;
  return q;
}

// rows and channels are counted in 32 bits; a tile may step past the last row
constexpr int kMaxRows = INT32_MAX - 65535, kMaxChannels = 1 << 28;
inline bool dtype_known(int d) { return d == TOPS_F32 || d == TOPS_BF16 || d == TOPS_F16; }
inline int dtype_bytes(int d) { return d == TOPS_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace tops
