// Residual addition + root-mean-square norm (forward with an output in x's type or in 8 bits, gradients).
//
//   t = x + residual;  r = (mean t^2 + eps)^(-1/2);  y = t r w
//   8 bits: scale = max|y| / M, q = round(y / scale), M = 127 or 448
//
// Both directions move every element once and compute little: the bound is memory bandwidth.  A block
// holds a row in registers between the sum over it and the writing, so nothing is read twice.  Measured:
// 32768 x 2560 bf16 with residual to e4m3 104 to 109 us (5.4 to 5.6 TB/s of 6.5 for a copy; 115 with a weight in bf16,
// which is read element by element), 8188 x 4096 with an fp32 residual forward and gradients 164 to 166 us (5.7 TB/s).
// Gradients of longer rows do not fit the registers of a block that size and spill: 4092 x 8192 205 us, floor 143.
#include "layer_common.cuh"

namespace ssd {
namespace {

constexpr int kMaxThreads = 1024;

struct NormArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* out;
  void* residual_out;
  float* rstd;
  float* scales;
  int weight_dtype, seqlen, dim;
  int64_t x_sb, x_sl, r_sb, r_sl;
  float eps;
};

// Rows whose largest |y| lies below kTiny are multiplied by kLift, and their scale too, before codes are made of
// them: both are powers of two, so nothing is rounded by it.  Lifted values lie between 2^-49 and 2^40.
constexpr float kTiny = 0x1p-60f;
constexpr float kLift = 0x1p100f;

// What an output element is made of: y for the input's types, y / scale for the 8-bit types.
struct I8 {};
struct E4M3 {};
template <typename O> struct OutKind { static constexpr float kMost = 0.0f; };
template <> struct OutKind<I8> { static constexpr float kMost = 127.0f; };
template <> struct OutKind<E4M3> { static constexpr float kMost = 448.0f; };

// y / scale, rounded as a division rounds: the product with the reciprocal, corrected by what it left over, which a
// fused multiply-add finds exactly (Markstein, IBM Journal of Research and Development 34, 1990).  That holds while
// neither the reciprocal nor what is left over leaves fp32's range: smaller rows are lifted first, see kTiny.
template <int V>
__device__ __forceinline__ void quotients(const float (&y)[V], float scale, float inv, float (&q)[V]) {
  float left[V], iv[V], sc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) q[i] = iv[i] = inv, sc[i] = -scale, left[i] = y[i];
  vec_mul(q, y);
  vec_fma(q, sc, left);
  vec_fma(left, iv, q);
}

template <typename O, int V>
__device__ __forceinline__ void store_out(void* base, int64_t idx, const float (&y)[V], float scale, float inv) {
  if constexpr (std::is_same<O, I8>::value) {
    Pack<int8_t, V> t;
    float q[V];
    quotients(y, scale, inv, q);
#pragma unroll
    for (int i = 0; i < V; ++i) t.e[i] = (int8_t)max(-127, min(127, __float2int_rn(q[i])));
    *reinterpret_cast<Pack<int8_t, V>*>(static_cast<int8_t*>(base) + idx) = t;
  } else if constexpr (std::is_same<O, E4M3>::value) {
    float q[V];
    quotients(y, scale, inv, q);
    if constexpr (V % 2 == 0) {
      Pack<uint16_t, V / 2> t;
#pragma unroll
      for (int i = 0; i < V; i += 2) t.e[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(q[i], q[i + 1]), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<Pack<uint16_t, V / 2>*>(static_cast<uint8_t*>(base) + idx) = t;
    } else {
      static_cast<uint8_t*>(base)[idx] = __nv_cvt_float_to_fp8(q[0], __NV_SATFINITE, __NV_E4M3);
    }
  } else {
    store_vec<V>(static_cast<O*>(base) + idx, y);
  }
}

// w = v rounded to R
template <typename R, int V>
__device__ __forceinline__ void round_all(const float (&v)[V], float (&w)[V]) {
  Pack<R, V> t;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      Pairs<R>::put(&t.e[i], v[i], v[i + 1]);
      unpack2(pair_of(t, i / 2), w[i], w[i + 1]);
    }
  } else {
    w[0] = widen(narrow<R>(v[0]));
  }
}

// One row per block.  VPT > 0: the row is held in registers, VPT vectors of V elements per thread;
// VPT == 0: rows longer than the registers hold are read again (from L2) for each pass.
template <typename T, typename R, typename O, int V, int VPT>
__global__ void __launch_bounds__(kMaxThreads) add_rms_norm_kernel(NormArgs a) {
  __shared__ float slots[3][32];
  constexpr bool kHold = VPT > 0;
  constexpr bool kScaled = OutKind<O>::kMost > 0.0f;
  const int64_t row = blockIdx.x;
  const int b = (int)(row / a.seqlen), l = (int)(row - (int64_t)b * a.seqlen);
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + l * a.x_sl;
  const R* res = a.residual ? static_cast<const R*>(a.residual) + b * a.r_sb + l * a.r_sl : nullptr;
  const int64_t obase = row * a.dim;
  float t[kHold ? VPT : 1][V];

  const auto fetch = [&](int col, float (&v)[V]) {
    load_vec<V>(x + col, v);
    if (res) {
      float u[V];
      load_vec<V>(res + col, u);
      vec_add(v, u);
    }
  };
  // two sums of squares: of t, which y is made of, and of t as it is kept, whose rstd the gradients use
  // (they see nothing but what was kept)
  float sums[V], kepts[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sums[i] = kepts[i] = 0.0f;
  // an 8-bit output has no gradients
  constexpr bool kRounds = sizeof(R) < 4 && !kScaled;
  const auto square = [&](const float (&v)[V]) {
    vec_fma(v, v, sums);
    if constexpr (kRounds) {
      float w[V];
      round_all<R>(v, w);
      vec_fma(w, w, kepts);
    }
  };
  if constexpr (kHold) {
    // all of the row's loads first, none of them under a condition that would be waited for: columns past
    // the end read the last ones and become zero
    Pack<T, V> xr[VPT];
    Pack<R, V> rr[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) xr[k] = *reinterpret_cast<const Pack<T, V>*>(x + min((int)(k * blockDim.x + threadIdx.x) * V, a.dim - V));
    if (res) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) rr[k] = *reinterpret_cast<const Pack<R, V>*>(res + min((int)(k * blockDim.x + threadIdx.x) * V, a.dim - V));
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      widen_all(xr[k], t[k]);
      if (res) {
        float u[V];
        widen_all(rr[k], u);
        vec_add(t[k], u);
      }
      if ((int)(k * blockDim.x + threadIdx.x) * V >= a.dim) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] = 0.0f;
      }
      square(t[k]);
    }
  } else {
    for (int col = threadIdx.x * V; col < a.dim; col += blockDim.x * V) {
      fetch(col, t[0]);
      square(t[0]);
    }
  }
  float sum = sums[0], kept = kepts[0];
#pragma unroll
  for (int i = 1; i < V; ++i) sum += sums[i], kept += kepts[i];
  if (kRounds) {
    block_reduce2(sum, kept, slots);
  } else {
    kept = sum = block_reduce<false>(sum, slots[0]);
  }
  const float r = rsqrtf(sum / (float)a.dim + a.eps);
  if (!kScaled && threadIdx.x == 0) a.rstd[row] = rsqrtf(kept / (float)a.dim + a.eps);

  // y of one vector; `keep` writes the sum beside it
  const auto finish = [&](int col, float (&v)[V], bool keep) {
    if (keep && a.residual_out) store_vec<V>(static_cast<R*>(a.residual_out) + obase + col, v);
    float w[V];
    load_param<V>(a.weight, a.weight_dtype, col, w);
    float rr[V];
#pragma unroll
    for (int i = 0; i < V; ++i) rr[i] = r;
    vec_mul(v, rr);
    vec_mul(v, w);
  };
  if constexpr (!kScaled) {
    if (kHold) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int col = (k * blockDim.x + threadIdx.x) * V;
        if (col < a.dim) {
          finish(col, t[k], true);
          store_out<O, V>(a.out, obase + col, t[k], 0.0f, 0.0f);
        }
      }
    } else {
      for (int col = threadIdx.x * V; col < a.dim; col += blockDim.x * V) {
        fetch(col, t[0]);
        finish(col, t[0], true);
        store_out<O, V>(a.out, obase + col, t[0], 0.0f, 0.0f);
      }
    }
  } else {
    float most = 0.0f;
    if (kHold) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int col = (k * blockDim.x + threadIdx.x) * V;
        if (col < a.dim) {
          finish(col, t[k], true);
#pragma unroll
          for (int i = 0; i < V; ++i) most = combine<true>(most, fabsf(t[k][i]));
        }
      }
    } else {
      for (int col = threadIdx.x * V; col < a.dim; col += blockDim.x * V) {
        fetch(col, t[0]);
        finish(col, t[0], true);
#pragma unroll
        for (int i = 0; i < V; ++i) most = combine<true>(most, fabsf(t[0][i]));
      }
    }
    most = block_reduce<true>(most, slots[2]);
    // an infinite y has no scale either: infinity becomes the NaN that marks such a row
    const float scale = most <= 3.4028235e38f ? most / OutKind<O>::kMost : __int_as_float(0x7fc00000);
    if (threadIdx.x == 0) a.scales[row] = scale;
    // the same for every thread of the block
    const bool tiny = most < kTiny;
    const float scale_up = tiny ? scale * kLift : scale;
    // zero for a row of zeros (and one so small that its scale is zero)
    const float inv = tiny ? (scale > 0.0f ? 1.0f / scale_up : 0.0f) : OutKind<O>::kMost / most;
    const auto lift = [&](float (&v)[V]) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= kLift;
    };
    if (kHold) {
      if (tiny) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) lift(t[k]);
      }
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int col = (k * blockDim.x + threadIdx.x) * V;
        if (col < a.dim) store_out<O, V>(a.out, obase + col, t[k], scale_up, inv);
      }
    } else {
      for (int col = threadIdx.x * V; col < a.dim; col += blockDim.x * V) {
        fetch(col, t[0]);
        finish(col, t[0], false);
        if (tiny) lift(t[0]);
        store_out<O, V>(a.out, obase + col, t[0], scale_up, inv);
      }
    }
  }
}

int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Threads and vectors per thread of a row of `nvec` vectors: `most` vectors per thread at most (the
// registers they take); 0 vectors per thread where the row does not fit a block's registers.
void row_shape(int nvec, int64_t rows, int want, int most, int* threads, int* vpt) {
  int v = 1;
  // few rows: one vector per thread, the shortest way through a row.  Many rows: blocks of about `want`
  // threads, so that several rows are in flight on an SM and one row's sums hide behind another's loads.
  if (rows < 2 * kSMs) want = kMaxThreads;
  while (v < most && (nvec + v - 1) / v > want) v *= 2;
  *vpt = v;
  *threads = round_up((nvec + v - 1) / v, 32);
  if (*threads > kMaxThreads) {
    *vpt = 0;
    *threads = 512;
  }
}

template <typename T, typename R, typename O, int V>
int launch_norm_v(const NormArgs& a, int64_t rows, cudaStream_t stream) {
  int threads, vpt;
  row_shape((a.dim + V - 1) / V, rows, 256, V == 8 ? 4 : 8, &threads, &vpt);
  const unsigned grid = (unsigned)rows;
  switch (vpt) {
    case 1: add_rms_norm_kernel<T, R, O, V, 1><<<grid, threads, 0, stream>>>(a); break;
    case 2: add_rms_norm_kernel<T, R, O, V, 2><<<grid, threads, 0, stream>>>(a); break;
    case 4: add_rms_norm_kernel<T, R, O, V, 4><<<grid, threads, 0, stream>>>(a); break;
    case 8:
      if constexpr (V < 8) add_rms_norm_kernel<T, R, O, V, 8><<<grid, threads, 0, stream>>>(a);
      break;
    default: add_rms_norm_kernel<T, R, O, V, 0><<<grid, threads, 0, stream>>>(a); break;
  }
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

template <typename T, typename R, typename O>
int launch_norm(const NormArgs& a, const ssd_add_rms_norm_params_t& p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int64_t rows = (int64_t)p.batch * p.seqlen;
  const bool vec = p.dim % V == 0 && rows_aligned(p.x, p.x_stride, 2, sizeof(T), 16) && aligned_to(p.out, V) &&
                   (sizeof(O) == 1 || aligned_to(p.out, 16)) &&
                   (p.residual == nullptr || rows_aligned(p.residual, p.residual_stride, 2, sizeof(R), 16)) &&
                   (p.residual_out == nullptr || aligned_to(p.residual_out, 16));
  return vec ? launch_norm_v<T, R, O, V>(a, rows, stream) : launch_norm_v<T, R, O, 1>(a, rows, stream);
}

// =====================================================================================================
// gradients
// =====================================================================================================
struct NormBwdArgs {
  const void* dout;
  const void* total;
  const void* weight;
  const float* rstd;
  const void* dresidual;
  void* dx;
  void* dresidual_in;
  float* partial;      // (grid, dim)
  int weight_dtype, seqlen, dim;
  int64_t rows;
  int64_t d_sb, d_sl, t_sb, t_sl, r_sb, r_sl;
};

// A block walks rows blockIdx.x, + gridDim.x, ...; each thread keeps its columns' share of the weight
// gradient in registers and writes it once, as the block's row of `partial`.  The second kernel adds the
// rows of `partial` in a fixed order, so the result does not depend on which block ran first.
// Where the registers allow it (one vector per thread, up to 512 threads) the next row's loads are issued
// before this row's sum is joined, so the barrier's wait is theirs too.
template <typename T, typename S, int V, int VPT, int THREADS>
__global__ void __launch_bounds__(THREADS) add_rms_norm_bwd_kernel(NormBwdArgs a) {
  constexpr bool kNext = VPT == 1 && THREADS <= 512;
  __shared__ float slots[2][32];
  float w[VPT][V], dw[VPT][V];
  int col[VPT];
  bool in[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    col[k] = (int)(k * blockDim.x + threadIdx.x) * V;
    in[k] = col[k] < a.dim;
    col[k] = min(col[k], a.dim - V);       // past the end: the last columns, masked by w = 0 and not stored
    load_param<V>(a.weight, a.weight_dtype, col[k], w[k]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[k][i] = 0.0f;
      if (!in[k]) w[k][i] = 0.0f;
    }
  }
  Pack<T, V> gr[VPT];
  Pack<S, V> tr[VPT], rr[VPT];
  float r_next;
  const auto fetch = [&](int64_t row) {
    const int b = (int)(row / a.seqlen), l = (int)(row - (int64_t)b * a.seqlen);
    const T* dout = static_cast<const T*>(a.dout) + b * a.d_sb + l * a.d_sl;
    const S* total = static_cast<const S*>(a.total) + b * a.t_sb + l * a.t_sl;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      gr[k] = *reinterpret_cast<const Pack<T, V>*>(dout + col[k]);
      tr[k] = *reinterpret_cast<const Pack<S, V>*>(total + col[k]);
    }
    if (a.dresidual) {
      const S* dres = static_cast<const S*>(a.dresidual) + b * a.r_sb + l * a.r_sl;
#pragma unroll
      for (int k = 0; k < VPT; ++k) rr[k] = *reinterpret_cast<const Pack<S, V>*>(dres + col[k]);
    }
    r_next = a.rstd[row];
  };
  if (kNext) fetch(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    if (!kNext) fetch(row);
    const float r = r_next;
    float g[VPT][V], hat[VPT][V], u[VPT][V], sums[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sums[i] = 0.0f, s[i] = r;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      widen_all(gr[k], g[k]);
      widen_all(tr[k], hat[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) u[k][i] = 0.0f;
      if (a.dresidual) widen_all(rr[k], u[k]);
      vec_mul(hat[k], s);
      vec_fma(g[k], hat[k], dw[k]);
      vec_mul(g[k], w[k]);
      vec_fma(g[k], hat[k], sums);
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += sums[i];
    if (kNext && row + gridDim.x < a.rows) fetch(row + gridDim.x);
    const float mean = block_reduce<false>(sum, slots[turn]) / (float)a.dim;
    float m[V];
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = -mean;
    const int64_t obase = row * a.dim;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!in[k]) continue;
      vec_fma(hat[k], m, g[k]);
      vec_fma(g[k], s, u[k]);
      store_vec<V>(static_cast<T*>(a.dx) + obase + col[k], u[k]);
      if (a.dresidual_in) store_vec<V>(static_cast<S*>(a.dresidual_in) + obase + col[k], u[k]);
    }
  }
  float* part = a.partial + (int64_t)blockIdx.x * a.dim;
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (in[k]) store_vec<V>(part + col[k], dw[k]);
}

// The same for rows longer than a block's registers hold: every row is read twice and the weight
// gradient comes from a kernel of its own that walks columns.
template <typename T, typename S>
__global__ void __launch_bounds__(kMaxThreads) add_rms_norm_bwd_long_kernel(NormBwdArgs a) {
  __shared__ float slots[2][32];
  const int64_t row = blockIdx.x;
  const int b = (int)(row / a.seqlen), l = (int)(row - (int64_t)b * a.seqlen);
  const T* dout = static_cast<const T*>(a.dout) + b * a.d_sb + l * a.d_sl;
  const S* total = static_cast<const S*>(a.total) + b * a.t_sb + l * a.t_sl;
  const S* dres = a.dresidual ? static_cast<const S*>(a.dresidual) + b * a.r_sb + l * a.r_sl : nullptr;
  const float r = a.rstd[row];
  float sum = 0.0f;
  for (int col = threadIdx.x; col < a.dim; col += blockDim.x)
    sum += widen(dout[col]) * load_f(a.weight, a.weight_dtype, col) * (widen(total[col]) * r);
  const float mean = block_reduce<false>(sum, slots[0]) / (float)a.dim;
  for (int col = threadIdx.x; col < a.dim; col += blockDim.x) {
    const float g = widen(dout[col]) * load_f(a.weight, a.weight_dtype, col);
    float u = r * (g - widen(total[col]) * r * mean);
    if (dres) u += widen(dres[col]);
    static_cast<T*>(a.dx)[row * a.dim + col] = narrow<T>(u);
    if (a.dresidual_in) static_cast<S*>(a.dresidual_in)[row * a.dim + col] = narrow<S>(u);
  }
}
template <typename T, typename S>
__global__ void __launch_bounds__(256) add_rms_norm_bwd_long_weight_kernel(NormBwdArgs a) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= a.dim) return;
  float acc = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const int b = (int)(row / a.seqlen), l = (int)(row - (int64_t)b * a.seqlen);
    acc += widen(static_cast<const T*>(a.dout)[b * a.d_sb + l * a.d_sl + col]) *
           (widen(static_cast<const S*>(a.total)[b * a.t_sb + l * a.t_sl + col]) * a.rstd[row]);
  }
  a.partial[(int64_t)blockIdx.y * a.dim + col] = acc;
}

// out[c] = sum over p of partial[p][c]: 32 columns and 32 strides of rows per block, joined in a fixed order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* partial, float* out, int parts, int dim) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float acc = 0.0f;
  if (col < dim) {
#pragma unroll 4
    for (int p = threadIdx.y; p < parts; p += 32) acc += partial[(int64_t)p * dim + col];
  }
  s[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  float v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < dim) out[c] = v;
}

// Rows of `partial`: as many blocks as are resident at once -- two an SM, up to eight of short rows, whose
// blocks are small -- and no more than there are rows.
int bwd_parts(int64_t rows, int dim) {
  const int per_sm = dim >= 4096 ? 2 : dim <= 1024 ? 8 : 8192 / dim;
  const int64_t most = per_sm * kSMs;
  return (int)(rows < most ? rows : most);
}

template <typename T, typename S, int V>
int launch_norm_bwd_v(const NormBwdArgs& a, cudaStream_t stream) {
  int threads, vpt;
  row_shape((a.dim + V - 1) / V, a.rows, V == 1 ? 128 : 512, V == 8 ? 2 : V == 1 ? 8 : 4, &threads, &vpt);
  const int parts = bwd_parts(a.rows, a.dim);
  switch (vpt) {
    case 1:
      if (threads <= 512)
        add_rms_norm_bwd_kernel<T, S, V, 1, 512><<<parts, threads, 0, stream>>>(a);
      else
        add_rms_norm_bwd_kernel<T, S, V, 1, kMaxThreads><<<parts, threads, 0, stream>>>(a);
      break;
    case 2:
      if (threads <= 640)
        add_rms_norm_bwd_kernel<T, S, V, 2, 640><<<parts, threads, 0, stream>>>(a);
      else
        add_rms_norm_bwd_kernel<T, S, V, 2, kMaxThreads><<<parts, threads, 0, stream>>>(a);
      break;
    case 4:
      if constexpr (V < 8) add_rms_norm_bwd_kernel<T, S, V, 4, kMaxThreads><<<parts, threads, 0, stream>>>(a);
      break;
    case 8:
      if constexpr (V == 1) {
        if (threads <= 640)
          add_rms_norm_bwd_kernel<T, S, V, 8, 640><<<parts, threads, 0, stream>>>(a);
        else
          add_rms_norm_bwd_kernel<T, S, V, 8, kMaxThreads><<<parts, threads, 0, stream>>>(a);
      }
      break;
    default:
      add_rms_norm_bwd_long_kernel<T, S><<<(unsigned)a.rows, 1024, 0, stream>>>(a);
      SSD_CUDA_OK(cudaGetLastError());
      add_rms_norm_bwd_long_weight_kernel<T, S><<<dim3((a.dim + 255) / 256, parts), 256, 0, stream>>>(a);
      break;
  }
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

template <typename T, typename S>
int launch_norm_bwd(const NormBwdArgs& a, const ssd_add_rms_norm_bwd_params_t& p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.dim % V == 0 && rows_aligned(p.dout, p.dout_stride, 2, sizeof(T), 16) &&
                   rows_aligned(p.total, p.total_stride, 2, sizeof(S), 16) && aligned_to(p.dx, 16) &&
                   (p.dresidual == nullptr || rows_aligned(p.dresidual, p.dresidual_stride, 2, sizeof(S), 16)) &&
                   (p.dresidual_in == nullptr || aligned_to(p.dresidual_in, 16));
  return vec ? launch_norm_bwd_v<T, S, V>(a, stream) : launch_norm_bwd_v<T, S, 1>(a, stream);
}

}  // namespace

int launch_add_rms_norm(const ssd_add_rms_norm_params_t& p, cudaStream_t stream) {
  NormArgs a;
  a.x = p.x;
  a.residual = p.residual;
  a.weight = p.weight;
  a.out = p.out;
  a.residual_out = p.residual_out;
  a.rstd = p.rstd;
  a.scales = p.scales;
  a.weight_dtype = p.weight_dtype;
  a.seqlen = p.seqlen;
  a.dim = p.dim;
  a.x_sb = p.x_stride[0], a.x_sl = p.x_stride[1];
  a.r_sb = p.residual_stride[0], a.r_sl = p.residual_stride[1];
  a.eps = p.eps;
  return with_type(p.x_dtype, [&](auto t) {
    using T = decltype(t);
    const auto go = [&](auto r) {
      using R = decltype(r);
      if (p.out_dtype == SSD_I8) return launch_norm<T, R, I8>(a, p, stream);
      if (p.out_dtype == SSD_E4M3) return launch_norm<T, R, E4M3>(a, p, stream);
      return launch_norm<T, R, T>(a, p, stream);
    };
    return p.residual_dtype == SSD_F32 ? go(float()) : go(T());
  });
}

size_t add_rms_norm_bwd_workspace(const ssd_add_rms_norm_bwd_params_t& p) {
  return (size_t)bwd_parts((int64_t)p.batch * p.seqlen, p.dim) * p.dim * sizeof(float);
}

int launch_add_rms_norm_bwd(const ssd_add_rms_norm_bwd_params_t& p, cudaStream_t stream) {
  NormBwdArgs a;
  a.dout = p.dout;
  a.total = p.total;
  a.weight = p.weight;
  a.rstd = p.rstd;
  a.dresidual = p.dresidual;
  a.dx = p.dx;
  a.dresidual_in = p.dresidual_in;
  a.partial = static_cast<float*>(p.workspace);
  a.weight_dtype = p.weight_dtype;
  a.seqlen = p.seqlen;
  a.dim = p.dim;
  a.rows = (int64_t)p.batch * p.seqlen;
  a.d_sb = p.dout_stride[0], a.d_sl = p.dout_stride[1];
  a.t_sb = p.total_stride[0], a.t_sl = p.total_stride[1];
  a.r_sb = p.dresidual_stride[0], a.r_sl = p.dresidual_stride[1];
  const int rc = with_type(p.x_dtype, [&](auto t) {
    using T = decltype(t);
    return p.total_dtype == SSD_F32 ? launch_norm_bwd<T, float>(a, p, stream) : launch_norm_bwd<T, T>(a, p, stream);
  });
  if (rc != SSD_OK) return rc;
  sum_partials_kernel<<<(p.dim + 31) / 32, dim3(32, 32), 0, stream>>>(a.partial, p.dweight, bwd_parts(a.rows, p.dim), p.dim);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

}  // namespace ssd
