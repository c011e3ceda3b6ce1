// Short causal convolution over the sequence, one filter of 2 to 4 taps for each channel: prompts,
// gradients, single tokens.
//
//   pre[t] = bias + sum_j wr[j] x[t - j],  wr[j] = weight[width - 1 - j];   out = pre or silu(pre)
//   dpre = dout * silu'(pre);  dx[s] = sum_j wr[j] dpre[s + j];  dwr[j] = sum_t dpre[t] x[t - j]
//
// Every element is read and written once: the bound is memory bandwidth.  Channels are contiguous, so a
// thread owns a vector of channels and walks a strip of positions with the last width - 1 inputs in
// registers; only a strip's first width - 1 positions are read twice.  Measured: 8 x 4096 x 5376 bf16 out of a
// wider buffer 144 to 152 us (4.6 to 4.9 TB/s of 6.5 for a copy): the loads in flight are held in registers, 96 a
// thread, which leaves 20 warps an SM; packed 3 x 2049 x 1792 gradients 41 us, bound by issue (66 %).
#include "layer_common.cuh"

namespace ssd {
namespace {

constexpr int kConvThreads = 128;
constexpr int kGroup = 8;         // positions whose loads are issued together, one group ahead of their use
constexpr int kStrip = 64;        // most positions of a strip

// Positions of a strip: 64, or fewer where the strips would leave most of the GPU idle (993 x 984 channels, 32
// blocks of 64 positions: 20 us).  With the `halo` positions behind it that a gradient strip walks, too, it is a
// whole number of groups.
int strip_of(int batch, int seqlen, int channels, int halo) {
  int n = kStrip;
  const int64_t rows = (int64_t)batch * ((channels + 511) / 512);
  while (n > kGroup && rows * ((seqlen + n - halo - 1) / (n - halo)) < 2 * kSMs) n /= 2;
  return n - halo;
}

struct ConvArgs {
  const void* x;
  const void* weight;
  const void* bias;
  const void* init;
  const int32_t* seq;
  void* out;
  void* final_states;
  int weight_dtype, bias_dtype;
  int seqlen, channels, strip;
  int silu;
  int64_t x_sb, x_sl, s_sb, s_sl;
};

// The sequence number of position t; positions before the first belong to sequence 0.
__device__ __forceinline__ int seq_at(const ConvArgs& a, int64_t base, int t) { return t < 0 ? 0 : a.seq[base + (int64_t)t * a.s_sl]; }

// Weights of V channels as wr[j][v], and the bias.
template <int W, int V>
__device__ __forceinline__ void load_filter(const void* weight, int wdt, const void* bias, int bdt, int c, float (&wr)[W][V], float (&bs)[V]) {
  float flat[V * W];
  load_param<V * W>(weight, wdt, (int64_t)c * W, flat);
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < W; ++j) wr[j][v] = flat[v * W + (W - 1 - j)];
    bs[v] = 0.0f;
  }
  if (bias) load_param<V>(bias, bdt, c, bs);
}

// Input of position t (t may lie before the first: initial states or zero).
template <typename T, int W, int V>
__device__ __forceinline__ void load_input(const ConvArgs& a, const T* x, int b, int c, int t, float (&v)[V]) {
  if (t >= 0) {
    load_vec<V>(x + (int64_t)t * a.x_sl, v);
  } else if (a.init != nullptr && t >= -(W - 1)) {
    load_vec<V>(static_cast<const T*>(a.init) + ((int64_t)b * (W - 1) + (t + W - 1)) * a.channels + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

// The value j positions before position `at` of the window, masked where it belongs to another sequence (a
// select: what is masked may be an infinity or a NaN).
template <int V, bool SEQ, int N>
__device__ __forceinline__ void masked(const float (&v)[N][V], const int (&id)[N], int at, int j, float (&past)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) past[i] = !SEQ || id[at - j] == id[at] ? v[at - j][i] : 0.0f;
}
// the pre-activation of position `at` of the window
template <int W, int V, bool SEQ, int N>
__device__ __forceinline__ void tap(const float (&wr)[W][V], const float (&bs)[V], const float (&v)[N][V], const int (&id)[N], int at, float (&y)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) y[i] = bs[i];
  vec_fma(wr[0], v[at], y);
#pragma unroll
  for (int j = 1; j < W; ++j) {
    float past[V];
    masked<V, SEQ>(v, id, at, j, past);
    vec_fma(wr[j], past, y);
  }
}

// Channels are contiguous, so a thread takes V of them; 8 bytes a load leave the registers for eight loads in
// flight and the next eight behind them.  Every load is unconditional (the position is clamped to the strip):
// one under a condition would be waited for at once.
// FULL: the strip is the longest, a constant (with its length read at run time the packed gradients took 72 us
// instead of 66).
template <typename T, int W, int V, bool SEQ, bool FULL>
__global__ void __launch_bounds__(kConvThreads) short_conv_fwd_kernel(ConvArgs a) {
  const int c = (blockIdx.x * kConvThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int b = blockIdx.z;
  const int strip = FULL ? kStrip : a.strip;
  const int t0 = blockIdx.y * strip, t1 = min(t0 + strip, a.seqlen);
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + c;
  T* out = static_cast<T*>(a.out) + ((int64_t)b * a.seqlen) * a.channels + c;
  const int64_t sbase = SEQ ? b * a.s_sb : 0;
  Pack<T, V> next[kGroup];
  int next_id[kGroup];
  const auto fetch = [&](int t) {
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int at = min(t + u, t1 - 1);
      next[u] = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)at * a.x_sl);
      next_id[u] = SEQ ? seq_at(a, sbase, at) : 0;
    }
  };
  fetch(t0);
  float wr[W][V], bs[V];
  load_filter<W, V>(a.weight, a.weight_dtype, a.bias, a.bias_dtype, c, wr, bs);
  float v[W - 1 + kGroup][V];          // v[W - 1 + u] = x[t + u], before it the last width - 1 inputs
  int id[W - 1 + kGroup];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    load_input<T, W, V>(a, x, b, c, t0 - (W - 1) + j, v[j]);
    id[j] = SEQ ? seq_at(a, sbase, t0 - (W - 1) + j) : 0;
  }
  for (int t = t0; t < t1; t += kGroup) {
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      widen_all(next[u], v[W - 1 + u]);
      id[W - 1 + u] = next_id[u];
    }
    if (t + kGroup < t1) fetch(t + kGroup);
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      float y[V];
      tap<W, V, SEQ>(wr, bs, v, id, W - 1 + u, y);
      if (a.silu) vec_silu(y);
      if (t + u < t1) store_vec<V>(out + (int64_t)(t + u) * a.channels, y);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[kGroup + j][i];
      id[j] = id[kGroup + j];
    }
  }
  if (a.final_states != nullptr && t1 == a.seqlen) {
    T* fin = static_cast<T*>(a.final_states) + (int64_t)b * (W - 1) * a.channels + c;
    const int last = SEQ ? seq_at(a, sbase, a.seqlen - 1) : 0;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const int t = a.seqlen - (W - 1) + j;
      float y[V];
      load_input<T, W, V>(a, x, b, c, t, y);
      if (SEQ && seq_at(a, sbase, t) != last) {
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = 0.0f;
      }
      store_vec<V>(fin + (int64_t)j * a.channels, y);
    }
  }
}

// ---- gradients --------------------------------------------------------------------------------------
struct ConvBwdArgs {
  ConvArgs f;
  const void* dout;
  const void* dfinal;
  void* dx;
  void* dinit;
  float* partial;      // (strips, width + 1, channels): the strip's share of dwr[0..width-1] and dbias
  int64_t d_sb, d_sl;
};

// A strip walks its positions and the width - 1 behind it (whose dpre its last dx need), in groups whose
// loads are issued one group ahead; dx of a position is complete once dpre of the width - 1 positions after it
// is known.
template <typename T, int W, int V, bool SEQ, bool FULL>
__global__ void __launch_bounds__(kConvThreads, 5) short_conv_bwd_kernel(ConvBwdArgs g) {
  const ConvArgs& a = g.f;
  const int c = (blockIdx.x * kConvThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int b = blockIdx.z;
  const int strip = FULL ? kStrip - (W - 1) : a.strip;
  const int t0 = blockIdx.y * strip, t1 = min(t0 + strip, a.seqlen);
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + c;
  const T* dout = static_cast<const T*>(g.dout) + b * g.d_sb + c;
  T* dx = static_cast<T*>(g.dx) + ((int64_t)b * a.seqlen) * a.channels + c;
  const int64_t sbase = SEQ ? b * a.s_sb : 0;
  const int last_id = SEQ ? seq_at(a, sbase, a.seqlen - 1) : 0;
  Pack<T, V> next[kGroup], next_d[kGroup];
  int next_id[kGroup];
  const auto fetch = [&](int t) {
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int at = min(t + u, a.seqlen - 1);
      next[u] = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)at * a.x_sl);
      next_d[u] = *reinterpret_cast<const Pack<T, V>*>(dout + (int64_t)at * g.d_sl);
      next_id[u] = SEQ ? seq_at(a, sbase, at) : 0;
    }
  };
  fetch(t0);
  float wr[W][V], bs[V], dw[W][V], db[V];
  load_filter<W, V>(a.weight, a.weight_dtype, a.bias, a.bias_dtype, c, wr, bs);
  float v[W - 1 + kGroup][V], dp[W - 1 + kGroup][V];       // x and dpre; [W - 1 + u] is position t + u
  int id[W - 1 + kGroup];
  const bool first = t0 == 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][i] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    load_input<T, W, V>(a, x, b, c, t0 - (W - 1) + j, v[j]);
    id[j] = SEQ ? seq_at(a, sbase, t0 - (W - 1) + j) : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) dp[j][i] = 0.0f;           // not of this strip, and zero before the first position
  }
  for (int t = t0; t < t1 + W - 1; t += kGroup) {
    Pack<T, V> d[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      widen_all(next[u], v[W - 1 + u]);
      d[u] = next_d[u];
      id[W - 1 + u] = next_id[u];
    }
    if (t + kGroup < t1 + W - 1) fetch(t + kGroup);
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int at = W - 1 + u, now = t + u;
      float pre[V];
      tap<W, V, SEQ>(wr, bs, v, id, at, pre);
      widen_all(d[u], dp[at]);
      if (a.silu) {
#pragma unroll
        for (int i = 0; i < V; ++i) pre[i] = dsilu_f(pre[i]);
        vec_mul(dp[at], pre);
      }
      if (now >= a.seqlen) {                               // behind the last position there is no dpre
#pragma unroll
        for (int i = 0; i < V; ++i) dp[at][i] = 0.0f;
      }
      if (now < t1) {
        vec_add(db, dp[at]);
        vec_fma(dp[at], v[at], dw[0]);
#pragma unroll
        for (int j = 1; j < W; ++j) {
          float past[V];
          masked<V, SEQ>(v, id, at, j, past);
          vec_fma(dp[at], past, dw[j]);
        }
      }
      // the position width - 1 back, s, at u in the window: dx[s] = sum_j wr[j] dpre[s + j]
      const int s = now - (W - 1);
      if ((s >= t0 || (first && g.dinit != nullptr)) && s < t1) {
        float r[V];
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
          float after[V];
#pragma unroll
          for (int i = 0; i < V; ++i) after[i] = !SEQ || id[u] == id[u + j] ? dp[u + j][i] : 0.0f;
          vec_fma(wr[j], after, r);
        }
        const int k = s - (a.seqlen - (W - 1));
        if (g.dfinal != nullptr && k >= 0 && (!SEQ || id[u] == last_id)) {
          float f[V];
          load_vec<V>(static_cast<const T*>(g.dfinal) + ((int64_t)b * (W - 1) + k) * a.channels + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) r[i] += f[i];
        }
        if (s >= 0)
          store_vec<V>(dx + (int64_t)s * a.channels, r);
        else
          store_vec<V>(static_cast<T*>(g.dinit) + ((int64_t)b * (W - 1) + (s + W - 1)) * a.channels + c, r);
      }
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[kGroup + j][i], dp[j][i] = dp[kGroup + j][i];
      id[j] = id[kGroup + j];
    }
  }
  float* part = g.partial + ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * (W + 1)) * a.channels + c;
#pragma unroll
  for (int j = 0; j < W; ++j) store_vec<V>(part + (int64_t)j * a.channels, dw[j]);
  store_vec<V>(part + (int64_t)W * a.channels, db);
}

// dweight[c][k] and dbias[c] from the strips' shares, added in a fixed order.
template <int W>
__global__ void __launch_bounds__(1024) short_conv_sum_kernel(const float* partial, float* dweight, float* dbias, int strips, int channels) {
  __shared__ float s[32][33];
  const int j = blockIdx.y;
  const int col = blockIdx.x * 32 + threadIdx.x;
  float acc = 0.0f;
  if (col < channels) {
#pragma unroll 4
    for (int p = threadIdx.y; p < strips; p += 32) acc += partial[((int64_t)p * (W + 1) + j) * channels + col];
  }
  s[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  float v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < channels) {
    if (j < W)
      dweight[(int64_t)c * W + (W - 1 - j)] = v;
    else if (dbias != nullptr)
      dbias[c] = v;
  }
}

// ---- single tokens ----------------------------------------------------------------------------------
struct ConvStepArgs {
  const void* x;
  void* state;
  const void* weight;
  const void* bias;
  const int32_t* indices;
  void* out;
  int weight_dtype, bias_dtype;
  int slots, channels;
  int silu;
  int64_t x_sb, st_ss, st_sp;
};

template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) short_conv_step_kernel(ConvStepArgs a) {
  const int row = blockIdx.y;
  const int slot = step_slot(a.indices, row, a.slots);
  const int c = (blockIdx.x * kConvThreads + threadIdx.x) * V;
  // every load is issued before anything is used, clamped instead of under a condition
  const bool inside = c < a.channels;
  const int cc = inside ? c : 0;
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.channels + cc;
  T* st = static_cast<T*>(a.state) + (int64_t)max(slot, 0) * a.st_ss + cc;
  const Pack<T, V> xr = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.x) + row * a.x_sb + cc);
  Pack<T, V> old[W - 1];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) old[j] = *reinterpret_cast<const Pack<T, V>*>(st + (int64_t)j * a.st_sp);    // oldest first
  float y[V], in[V], past[W - 1][V], wr[W][V], bs[V];
  load_filter<W, V>(a.weight, a.weight_dtype, a.bias, a.bias_dtype, cc, wr, bs);
  const bool taken = step_taken(a.indices, row, slot);
  if (!inside) return;
  if (slot < 0 || taken) {
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = 0.0f;
    store_vec<V>(out, y);
    return;
  }
  widen_all(xr, in);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) widen_all(old[j], past[j]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float acc = fmaf(wr[0][i], in[i], bs[i]);
#pragma unroll
    for (int j = 1; j < W; ++j) acc = fmaf(wr[j][i], past[W - 1 - j][i], acc);
    y[i] = a.silu ? silu_f(acc) : acc;
  }
  store_vec<V>(out, y);
#pragma unroll
  for (int j = 0; j < W - 2; ++j) *reinterpret_cast<Pack<T, V>*>(st + (int64_t)j * a.st_sp) = old[j + 1];
  *reinterpret_cast<Pack<T, V>*>(st + (int64_t)(W - 2) * a.st_sp) = xr;
}

ConvArgs conv_args(const ssd_short_conv_params_t& p) {
  ConvArgs a;
  a.x = p.x;
  a.weight = p.weight;
  a.bias = p.bias;
  a.init = p.initial_states;
  a.seq = p.seq_idx;
  a.out = p.out;
  a.final_states = p.final_states;
  a.weight_dtype = p.weight_dtype;
  a.bias_dtype = p.bias_dtype;
  a.seqlen = p.seqlen;
  a.channels = p.channels;
  a.silu = p.silu;
  a.x_sb = p.x_stride[0], a.x_sl = p.x_stride[1];
  a.s_sb = p.seq_idx_stride[0], a.s_sl = p.seq_idx_stride[1];
  return a;
}

// calls f with the filter's width as a constant
template <typename F>
int with_width(int width, F f) {
  switch (width) {
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    default: return f(std::integral_constant<int, 4>());
  }
}

int strips_of(int seqlen, int strip) { return (seqlen + strip - 1) / strip; }

}  // namespace

int launch_short_conv_fwd(const ssd_short_conv_params_t& p, cudaStream_t stream) {
  ConvArgs a = conv_args(p);
  a.strip = strip_of(p.batch, p.seqlen, p.channels, 0);
  const int strips = strips_of(p.seqlen, a.strip);
  SSD_REQUIRE(strips <= 65535 && p.batch <= 65535, SSD_ERR_UNSUPPORTED, "short conv: seqlen %d or batch %d too large", p.seqlen, p.batch);
  return with_type(p.x_dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 4;
    constexpr size_t kBytes = V * sizeof(T);
    const bool vec = p.channels % V == 0 && rows_aligned(p.x, p.x_stride, 2, sizeof(T), kBytes) && aligned_to(p.out, kBytes) &&
                     aligned_to(p.initial_states, kBytes) && aligned_to(p.final_states, kBytes);
    return with_width(p.width, [&](auto w) {
      constexpr int W = decltype(w)::value;
      const auto go = [&](auto v, auto s) -> int {
        constexpr int N = decltype(v)::value;
        const dim3 grid((p.channels + kConvThreads * N - 1) / (kConvThreads * N), strips, p.batch);
        if (a.strip == kStrip)
          short_conv_fwd_kernel<T, W, N, decltype(s)::value, true><<<grid, kConvThreads, 0, stream>>>(a);
        else
          short_conv_fwd_kernel<T, W, N, decltype(s)::value, false><<<grid, kConvThreads, 0, stream>>>(a);
        SSD_CUDA_OK(cudaGetLastError());
        return SSD_OK;
      };
      const std::integral_constant<int, V> wide;
      const std::integral_constant<int, 1> one;
      if (p.seq_idx) return vec ? go(wide, std::true_type()) : go(one, std::true_type());
      return vec ? go(wide, std::false_type()) : go(one, std::false_type());
    });
  });
}

size_t short_conv_bwd_workspace(const ssd_short_conv_bwd_params_t& p) {
  const ssd_short_conv_params_t& c = p.conv;
  const int strips = strips_of(c.seqlen, strip_of(c.batch, c.seqlen, c.channels, c.width - 1));
  return (size_t)c.batch * strips * (c.width + 1) * c.channels * sizeof(float);
}

int launch_short_conv_bwd(const ssd_short_conv_bwd_params_t& q, cudaStream_t stream) {
  const ssd_short_conv_params_t& p = q.conv;
  ConvBwdArgs g;
  g.f = conv_args(p);
  g.dout = q.dout;
  g.dfinal = q.dfinal_states;
  g.dx = q.dx;
  g.dinit = q.dinitial_states;
  g.partial = static_cast<float*>(q.workspace);
  g.d_sb = q.dout_stride[0], g.d_sl = q.dout_stride[1];
  g.f.strip = strip_of(p.batch, p.seqlen, p.channels, p.width - 1);
  const int strips = strips_of(p.seqlen, g.f.strip);
  SSD_REQUIRE(strips <= 65535 && p.batch <= 65535, SSD_ERR_UNSUPPORTED, "short conv: seqlen %d or batch %d too large", p.seqlen, p.batch);
  return with_type(p.x_dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 2;
    constexpr size_t kBytes = V * sizeof(T);
    const bool vec = p.channels % V == 0 && rows_aligned(p.x, p.x_stride, 2, sizeof(T), kBytes) &&
                     rows_aligned(q.dout, q.dout_stride, 2, sizeof(T), kBytes) && aligned_to(q.dx, kBytes) &&
                     aligned_to(p.initial_states, kBytes) && aligned_to(q.dfinal_states, kBytes) && aligned_to(q.dinitial_states, kBytes);
    return with_width(p.width, [&](auto w) {
      constexpr int W = decltype(w)::value;
      const auto go = [&](auto v, auto s) -> int {
        constexpr int N = decltype(v)::value;
        const dim3 grid((p.channels + kConvThreads * N - 1) / (kConvThreads * N), strips, p.batch);
        if (g.f.strip == kStrip - (W - 1))
          short_conv_bwd_kernel<T, W, N, decltype(s)::value, true><<<grid, kConvThreads, 0, stream>>>(g);
        else
          short_conv_bwd_kernel<T, W, N, decltype(s)::value, false><<<grid, kConvThreads, 0, stream>>>(g);
        SSD_CUDA_OK(cudaGetLastError());
        short_conv_sum_kernel<W><<<dim3((p.channels + 31) / 32, W + 1), dim3(32, 32), 0, stream>>>(g.partial, q.dweight, q.dbias,
                                                                                                    strips * p.batch, p.channels);
        SSD_CUDA_OK(cudaGetLastError());
        return SSD_OK;
      };
      const std::integral_constant<int, V> wide;
      const std::integral_constant<int, 1> one;
      if (p.seq_idx) return vec ? go(wide, std::true_type()) : go(one, std::true_type());
      return vec ? go(wide, std::false_type()) : go(one, std::false_type());
    });
  });
}

int launch_short_conv_step(const ssd_short_conv_step_params_t& p, cudaStream_t stream) {
  ConvStepArgs a;
  a.x = p.x;
  a.state = p.conv_state;
  a.weight = p.weight;
  a.bias = p.bias;
  a.indices = p.state_indices;
  a.out = p.out;
  a.weight_dtype = p.weight_dtype;
  a.bias_dtype = p.bias_dtype;
  a.slots = p.slots;
  a.channels = p.channels;
  a.silu = p.silu;
  a.x_sb = p.x_stride;
  a.st_ss = p.state_stride[0], a.st_sp = p.state_stride[1];
  SSD_REQUIRE(p.batch <= 65535, SSD_ERR_UNSUPPORTED, "short conv step: batch %d too large", p.batch);
  return with_type(p.x_dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 4;
    constexpr size_t kBytes = V * sizeof(T);
    const bool vec = p.channels % V == 0 && rows_aligned(p.x, &p.x_stride, 1, sizeof(T), kBytes) &&
                     rows_aligned(p.conv_state, p.state_stride, 2, sizeof(T), kBytes) && aligned_to(p.out, kBytes);
    return with_width(p.width, [&](auto w) {
      constexpr int W = decltype(w)::value;
      const auto go = [&](auto v) -> int {
        constexpr int N = decltype(v)::value;
        const dim3 grid((p.channels + kConvThreads * N - 1) / (kConvThreads * N), p.batch);
        short_conv_step_kernel<T, W, N><<<grid, kConvThreads, 0, stream>>>(a);
        SSD_CUDA_OK(cudaGetLastError());
        return SSD_OK;
      };
      return vec ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>());
    });
  });
}

}  // namespace ssd
