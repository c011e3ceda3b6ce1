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
  float* out_x;          // y before the gate, which dz is made of: in 32 bits, so that dz is rounded once
  float* final_states;
  float* ckpt;
  float* seg_state;      // (b, segments, d, n): the state a segment leaves from a zero start
  float2* seg_decay;     // (b, segments, d): (sum of dt', 0 where the segment drops what it was given, else 1)
  int dt_f32, A_dtype, D_dtype, bias_dtype, init_dtype;
  int seqlen, channels, ngroups, dstate, per_group, tiles_per_group;
  int softplus, limits;
  float dt_min, dt_max;
  int64_t x_sb, x_sl, dt_sb, dt_sl, z_sb, z_sl;
  int64_t B_sb, B_sl, B_sg, C_sb, C_sl, C_sg;
  int64_t s_sb, s_sl;
  int seg_len, segments; // positions of a segment (a multiple of the tile's), segments of a sequence
};

// softplus_f and silu_f of a pair: the same operations in the same order
__device__ __forceinline__ f32x2 softplus2(f32x2 v) {
  float a, b, c, d;
  unpack2(v, a, b);
  const f32x2 e = pack2(ex2_approx(fabsf(a) * -1.4426950408889634f), ex2_approx(fabsf(b) * -1.4426950408889634f));
  unpack2(add2(e, both(2.0f)), c, d);
  const f32x2 s = mul2(e, pack2(rcp_approx(c), rcp_approx(d))), s2 = mul2(s, s);
  f32x2 r = fma2(s2, both(1.0f / 13.0f), both(1.0f / 11.0f));
  r = fma2(s2, r, both(1.0f / 9.0f));
  r = fma2(s2, r, both(1.0f / 7.0f));
  r = fma2(s2, r, both(1.0f / 5.0f));
  r = fma2(s2, r, both(1.0f / 3.0f));
  r = fma2(mul2(s, s2), r, s);
  return fma2(both(2.0f), r, pack2(fmaxf(a, 0.0f), fmaxf(b, 0.0f)));
}
__device__ __forceinline__ f32x2 silu2(f32x2 v) {
  float a, b;
  unpack2(mul2(v, both(-1.4426950408889634f)), a, b);
  unpack2(add2(both(1.0f), pack2(ex2_approx(a), ex2_approx(b))), a, b);
  return mul2(v, pack2(rcp_approx(a), rcp_approx(b)));
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
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; i += 2) Pairs<T>::put(&t.e[i], v[i], v[i + 1]);
    if (count > 0) *reinterpret_cast<Pack<T, V>*>(p) = t;
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

// What of a state is left behind a segment whose dt' add up to `sum`; A2 is A log2(e).  Zero stays zero where A > 0
// and the decay passes the largest number.
__device__ __forceinline__ float through_segment(float A2, float sum, float state) { return state == 0.0f ? 0.0f : ex2_approx(A2 * sum) * state; }

ScanArgs scan_args(const ssd_token_scan_params_t& p);

}  // namespace ssd
