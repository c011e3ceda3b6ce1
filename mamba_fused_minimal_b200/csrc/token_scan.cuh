// What the forward scan (token_scan.cu) and its gradients (token_scan_bwd.cu) share.
#pragma once

#include "layer_common.cuh"

namespace ssd {

struct ScanArgs {
  const void* x;
  const void* dt;
  const void* A;
  const void* B;
  const void* C;
  const void* D;
  const void* z;
  const void* bias;
  const void* init;
  const int32_t* seq;
  void* out;
  void* out_x;
  float* final_states;
  float* ckpt;
  float* seg_state;      // (b, segments, d, n): the state a segment leaves from a zero start
  float2* seg_decay;     // (b, segments, d): (sum of dt', 0 where the segment drops what it was given, else 1)
  int dt_f32, A_dtype, D_dtype, bias_dtype, init_dtype;
  int seqlen, channels, ngroups, dstate, per_group, tiles_per_group;
  int softplus;
  float dt_min, dt_max;
  int64_t x_sb, x_sl, dt_sb, dt_sl, z_sb, z_sl;
  int64_t B_sb, B_sl, B_sg, C_sb, C_sl, C_sg;
  int64_t s_sb, s_sl;
  int seg_len, segments; // positions of a segment (a multiple of the tile's), segments of a sequence
};

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
constexpr float kLog2e = 1.4426950408889634f;

// V consecutive elements.  VEC: the vector is aligned and read as a whole, `count` or not -- the caller
// points at elements that exist and masks what it makes of them.  A load under a condition would be
// waited for where the branches meet; this one is not waited for before its words are used (measured on
// 2 x 4096 x 5120 channels of 16 components: 712 us with conditional loads, 576 us without).  Else the
// first `count` elements exist and the others read as zero.
template <int V, bool VEC, typename T>
__device__ __forceinline__ Pack<T, V> load_some(const T* p, int count) {
  Pack<T, V> t;
  if constexpr (VEC) {
    t = *reinterpret_cast<const Pack<T, V>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t.e[i] = i < count ? p[i] : narrow<T>(0.0f);
  }
  return t;
}
template <int V, bool VEC, typename T>
__device__ __forceinline__ void store_some(T* p, const float (&v)[V], int count) {
  if constexpr (VEC) {
    if (count > 0) store_vec<V>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < count) p[i] = narrow<T>(v[i]);
  }
}

// bit t: position t0 + t belongs to another sequence than the one before it (positions before the first
// belong to sequence 0).  One warp-wide vote over 32 positions.
__device__ __forceinline__ uint32_t reset_mask(const ScanArgs& a, int b, int t0, int lane) {
  bool reset = false;
  const int t = t0 + lane;
  if (t < a.seqlen) {
    const int64_t at = b * a.s_sb + (int64_t)t * a.s_sl;
    reset = a.seq[at] != (t > 0 ? a.seq[at - a.s_sl] : 0);
  }
  return __ballot_sync(0xffffffffu, reset);
}

ScanArgs scan_args(const ssd_token_scan_params_t& p);

}  // namespace ssd
