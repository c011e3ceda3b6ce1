// Helpers shared by the layer operators around the scan (add_rms_norm.cu, short_conv.cu, token_scan.cu,
// token_scan_bwd.cu, token_step.cu): vectors of elements widened to fp32, block sums, the activation
// functions, and the slot of a row of a single-token call.
#pragma once

#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "ssd_common.cuh"
#include "ssd_launch.h"

namespace ssd {

// SMs of a B200, what the plans below count blocks against (a workspace query and its launch have to agree).
constexpr int kSMs = 148;

// ---- V consecutive elements of type T, widened to fp32 ---------------------------------------------
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T e[V];
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// ---- two fp32 numbers in one 64-bit register: the packed multiply-adds issue once for both -----------
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }
// the two 16-bit elements of a word as fp32
template <typename T> __device__ __forceinline__ f32x2 widen_pair(uint32_t w);
template <> __device__ __forceinline__ f32x2 widen_pair<__nv_bfloat16>(uint32_t w) {
  return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ f32x2 widen_pair<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pack2(f.x, f.y);
}

// elements 2 i and 2 i + 1 of a vector as fp32
template <int V>
__device__ __forceinline__ f32x2 pair_of(const Pack<float, V>& p, int i) { return pack2(p.e[2 * i], p.e[2 * i + 1]); }
template <int V, typename T>
__device__ __forceinline__ f32x2 pair_of(const Pack<T, V>& p, int i) {
  uint32_t w;
  memcpy(&w, &p.e[2 * i], 4);
  return widen_pair<T>(w);
}

template <typename T> struct Pairs;
template <> struct Pairs<float> {
  static __device__ __forceinline__ void put(float* e, float a, float b) { e[0] = a, e[1] = b; }
};
template <> struct Pairs<__nv_bfloat16> {
  static __device__ __forceinline__ void put(__nv_bfloat16* e, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    memcpy(e, &v, 4);
  }
};
template <> struct Pairs<__half> {
  static __device__ __forceinline__ void put(__half* e, float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    memcpy(e, &v, 4);
  }
};

template <typename T, int V>
__device__ __forceinline__ void widen_all(const Pack<T, V>& p, float (&v)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) unpack2(pair_of(p, i / 2), v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = widen(p.e[i]);
  }
}
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  widen_all(*reinterpret_cast<const Pack<T, V>*>(p), v);
}
template <int V, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  Pack<T, V> t;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) Pairs<T>::put(&t.e[i], v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t.e[i] = narrow<T>(v[i]);
  }
  *reinterpret_cast<Pack<T, V>*>(p) = t;
}

// v = f(v, w) element by element; pairs go through one packed operation
template <int V>
__device__ __forceinline__ void vec_add(float (&v)[V], const float (&w)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) unpack2(add2(pack2(v[i], v[i + 1]), pack2(w[i], w[i + 1])), v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += w[i];
  }
}
template <int V>
__device__ __forceinline__ void vec_mul(float (&v)[V], const float (&w)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) unpack2(mul2(pack2(v[i], v[i + 1]), pack2(w[i], w[i + 1])), v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= w[i];
  }
}
// c = a * b + c
template <int V>
__device__ __forceinline__ void vec_fma(const float (&a)[V], const float (&b)[V], float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) unpack2(fma2(pack2(a[i], a[i + 1]), pack2(b[i], b[i + 1]), pack2(c[i], c[i + 1])), c[i], c[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = fmaf(a[i], b[i], c[i]);
  }
}
// V parameters (weights, biases) of any of the three types, always read as V separate elements or, in
// fp32 and aligned, as 16-byte vectors; read once per thread, so the branch costs nothing.
template <int V>
__device__ __forceinline__ void load_param(const void* base, int dtype, int64_t idx, float (&v)[V]) {
  if (V % 4 == 0 && dtype == SSD_F32 && (reinterpret_cast<uintptr_t>(static_cast<const float*>(base) + idx) & 15) == 0) {
#pragma unroll
    for (int i = 0; i + 3 < V; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + idx + i);
      v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = load_f(base, dtype, idx + i);
}

// One parameter of any of the three types in two steps: `load` issues it -- into one register or the other,
// with no branch that would wait for it -- and `value` converts it where it is used.
struct AnyParam {
  uint32_t w = 0;
  uint16_t h = 0;
  __device__ __forceinline__ void load(const void* base, int dtype, int64_t idx) {
    if (dtype == SSD_F32) w = static_cast<const uint32_t*>(base)[idx];
    if (dtype != SSD_F32) h = static_cast<const uint16_t*>(base)[idx];
  }
  __device__ __forceinline__ float value(int dtype) const {
    const float b = __uint_as_float((uint32_t)h << 16), f = __half2float(__ushort_as_half(h));
    return dtype == SSD_F32 ? __uint_as_float(w) : dtype == SSD_BF16 ? b : f;
  }
};

// ---- activations -----------------------------------------------------------------------------------
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + exp(-v)): zero where the exponential overflows
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_approx(1.0f + ex2_approx(v * -1.4426950408889634f)); }
__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f(v); }
// d/dv of v * sigmoid(v)
__device__ __forceinline__ float dsilu_f(float v) {
  const float g = sigmoid_f(v);
  return g * (1.0f + v * (1.0f - g));
}
template <int V>
__device__ __forceinline__ void vec_silu(float (&v)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      float a, b;
      const f32x2 w = pack2(v[i], v[i + 1]);
      unpack2(mul2(w, both(-1.4426950408889634f)), a, b);
      unpack2(add2(both(1.0f), pack2(ex2_approx(a), ex2_approx(b))), a, b);
      unpack2(mul2(w, pack2(rcp_approx(a), rcp_approx(b))), v[i], v[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = silu_f(v[i]);
  }
}
// log(1 + exp(v)), exact to a few units in the last place also where it is small: the layer's steps lie
// between 1e-4 and 1e-1, where log(exp(v) + 1) would keep three digits.  With e = exp(-|v|) <= 1,
// log(1 + e) = 2 atanh(e / (2 + e)), whose argument is at most 1/3: seven terms of the series leave 2e-8.
__device__ __forceinline__ float softplus_f(float v) {
  const float e = ex2_approx(fabsf(v) * -1.4426950408889634f);
  const float s = e * rcp_approx(2.0f + e), s2 = s * s;
  float r = fmaf(s2, 1.0f / 13.0f, 1.0f / 11.0f);
  r = fmaf(s2, r, 1.0f / 9.0f);
  r = fmaf(s2, r, 1.0f / 7.0f);
  r = fmaf(s2, r, 1.0f / 5.0f);
  r = fmaf(s2, r, 1.0f / 3.0f);
  r = fmaf(s * s2, r, s);
  return fmaf(2.0f, r, fmaxf(v, 0.0f));          // r is a NaN where v is
}
// v held between lo and hi; a NaN stays one
__device__ __forceinline__ float clamp_f(float v, float lo, float hi) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(lo));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(hi));
  return r;
}
// dt' of one position and channel
__device__ __forceinline__ float scan_dt(float raw, bool softplus, float lo, float hi) {
  return clamp_f(softplus ? softplus_f(raw) : raw, lo, hi);
}

// ---- block-wide sum and maximum --------------------------------------------------------------------
// `slots` is shared memory for 32 floats that no other reduction in flight uses.  Every thread gets the
// result; the order of the additions depends on the block's size alone.
template <bool MAX>
__device__ __forceinline__ float combine(float a, float b) {
  if (!MAX) return a + b;
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));   // a NaN stays
  return r;
}
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* slots) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = combine<MAX>(v, __shfl_xor_sync(0xffffffffu, v, off));
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  v = slots[(threadIdx.x & 31) < warps ? (threadIdx.x & 31) : 0];
  if (!MAX && (threadIdx.x & 31) >= warps) v = 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = combine<MAX>(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// two sums with one barrier; slots[0] and slots[1] as above
__device__ __forceinline__ void block_reduce2(float& u, float& v, float (*slots)[32]) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, off);
    v += __shfl_xor_sync(0xffffffffu, v, off);
  }
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  if (lane == 0) slots[0][threadIdx.x >> 5] = u, slots[1][threadIdx.x >> 5] = v;
  __syncthreads();
  u = lane < warps ? slots[0][lane] : 0.0f;
  v = lane < warps ? slots[1][lane] : 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, off);
    v += __shfl_xor_sync(0xffffffffu, v, off);
  }
}

// ---- the state slot of a row of a single-token call --------------------------------------------------
// A row is padding (it gets zeros and touches no state) if its index lies outside the slots, or if an
// earlier row names the same slot: two rows would race on it.  step_slot gives the slot or -1;
// step_taken, called by every thread of the block behind its loads and before its stores, says whether an
// earlier row has it: the search runs while the loads are in flight.
__device__ __forceinline__ int step_slot(const int32_t* indices, int row, int slots) {
  const int slot = indices == nullptr ? row : indices[row];
  return slot < slots ? slot : -1;
}
__device__ __forceinline__ bool step_taken(const int32_t* indices, int row, int slot) {
  if (indices == nullptr) return false;
  bool taken = false;
  for (int j = threadIdx.x; j < row; j += blockDim.x) taken |= indices[j] == slot;
  return __syncthreads_or(taken) != 0;
}

// ---- alignment of what a vector access of `bytes` needs --------------------------------------------
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline bool rows_aligned(const void* p, const int64_t* stride, int n, int elem, size_t bytes) {
  if (!aligned_to(p, bytes)) return false;
  for (int i = 0; i < n; ++i)
    if ((stride[i] * elem) % (int64_t)bytes != 0) return false;
  return true;
}

// calls f with a value of the type that `dtype` names
template <typename F>
int with_type(int dtype, F f) {
  switch (dtype) {
    case SSD_BF16: return f(__nv_bfloat16());
    case SSD_F16: return f(__half());
    default: return f(float());
  }
}

}  // namespace ssd
