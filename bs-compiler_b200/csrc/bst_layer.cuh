// bst_layer.cuh — device and host helpers shared by the layer kernels (norm, convolution, scan).
//
// Elements are float, bf16 or fp16; all arithmetic is fp32, rounded once when a result is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "bst_internal.h"

namespace bst {

int sm_count();  // bst_core.cu

using bf16 = __nv_bfloat16;
using fp16 = __half;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(fp16 v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ fp16 from_f<fp16>(float v) { return __float2half_rn(v); }

// V elements that move as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Chunk {
  T v[V];
};

// Elements [0, n) of a chunk, as one access where `vec` (the caller has checked alignment) and all are meant.
template <typename T, int V>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T, V>& c, int n, bool vec) {
  if (vec && n >= V) {
    *reinterpret_cast<Chunk<T, V>*>(p) = c;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = c.v[i];
  }
}

// All V elements or none (zeros): one predicated access, so that the loads of a loop's next turn can stay in flight
// (a choice between two ways to load makes the thread wait for the values where the ways meet).
template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> load_whole(const T* p, bool on) {
  Chunk<T, V> c{};
  if (on) c = *reinterpret_cast<const Chunk<T, V>*>(p);
  return c;
}
template <typename T, int V>
__device__ __forceinline__ void store_whole(T* p, const Chunk<T, V>& c, bool on) {
  if (on) *reinterpret_cast<Chunk<T, V>*>(p) = c;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x and 1/x by the special-function unit (relative error about 2^-22 and 2^-23).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + e^-x); 0 and 1 at the far ends, where e^-x overflows or vanishes.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-x * kLog2e)); }

// softplus(x) = max(x, 0) + log1p(t) with t = e^-|x| in (0, 1].  log1p(t) = 2 atanh(s), s = t / (2 + t)
// <= 1/3, and atanh(s) = s (1 + q P(q)), q = s^2 <= 1/9: no cancellation at any x, so a step size of 1e-4
// keeps its relative accuracy.  P is a weighted least-squares fit on Chebyshev nodes; with four
// coefficients the result is good to 5e-9 before rounding.
constexpr float kAtanh1 = 0.33333208f, kAtanh2 = 0.20010764f, kAtanh3 = 0.14000901f, kAtanh4 = 0.14005998f;
__device__ __forceinline__ float softplus(float x) {
  const float t = ex2(-fabsf(x) * kLog2e);
  const float s = t * rcp(2.f + t);
  const float q = s * s;
  float p = fmaf(kAtanh4, q, kAtanh3);
  p = fmaf(p, q, kAtanh2);
  p = fmaf(p, q, kAtanh1);
  p = fmaf(p, q, 1.f);
  return fmaf(2.f * s, p, x < 0.f ? 0.f : x);  // a NaN is kept: x < 0 is false for it
}

// Two fp32 lanes per instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// sigmoid and softplus of two values, their fused operations paired.
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  const float2 e = ex2_2(mul2(x, both(-kLog2e)));
  const float2 d = add2(e, both(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
__device__ __forceinline__ float2 softplus2(float2 x) {
  const float2 t = ex2_2(make_float2(-fabsf(x.x) * kLog2e, -fabsf(x.y) * kLog2e));
  const float2 w = add2(t, both(2.f));
  const float2 s = mul2(t, make_float2(rcp(w.x), rcp(w.y)));
  const float2 q = mul2(s, s);
  float2 p = fma2(both(kAtanh4), q, both(kAtanh3));
  p = fma2(p, q, both(kAtanh2));
  p = fma2(p, q, both(kAtanh1));
  p = fma2(p, q, both(1.f));
  // max(x, 0) that keeps a NaN: x < 0 is false for it.
  const float2 m = make_float2(x.x < 0.f ? 0.f : x.x, x.y < 0.f ? 0.f : x.y);
  return fma2(add2(s, s), p, m);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Sums v[0..NV) over LANES lanes that are BASE apart (LANES, BASE powers of two), and leaves each of
// them NV / LANES of the totals in v[0..): lane l of the group has those of values [l NV/LANES, ...).
// Each step halves the values that a lane still carries, so NV - NV/LANES shuffles do what
// NV log2(LANES) would in a plain butterfly.
template <int NV, int LANES, int BASE>
__device__ __forceinline__ void reduce_scatter(float (&v)[NV], int lane) {
  static_assert(NV % LANES == 0, "each lane ends with a whole number of values");
  int n = NV;
#pragma unroll
  for (int m = LANES / 2; m >= 1; m >>= 1) {
    const bool up = (lane & (m * BASE)) != 0;
    n >>= 1;
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) {
      if (i < n) {
        const float send = up ? v[i] : v[i + n];
        const float keep = up ? v[i + n] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m * BASE);
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------
inline int layer_elem_size(int dtype) { return dtype == BST_F32 ? 4 : 2; }
inline bool layer_dtype(int dtype) { return dtype == BST_F32 || dtype == BST_BF16 || dtype == BST_F16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int launched(const char* kernel) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, kernel);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return BST_OK;
}

// f(T{}) with the element type of a checked dtype.
template <class F>
int with_type(int dtype, F&& f) {
  if (dtype == BST_F32) return f(float{});
  if (dtype == BST_BF16) return f(bf16{});
  return f(fp16{});
}

}  // namespace bst
