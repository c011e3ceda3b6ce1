// One position of the selective scan for each running sequence, the state updated in place:
//
//   h[n] = exp(dt' A[n]) h[n] + dt' x B[n];   y = C . h + D x;   out = y or y silu(z)
//
// The state is read and written once and everything else is small: memory bandwidth bounds a full batch,
// latency a single sequence.  A row is the dstate components of one (head, p); LPR adjacent lanes hold it
// as 16-byte vectors, and all loads of a thread's U rows are issued before the first is used, none of them
// under a condition that would be waited for.  With one decay a head (the Mamba2 form) a block stays
// inside a head and forms dt' and the decay once; with a decay for each component every row has its own.
// Measured: 128 sequences of 80 heads of 64 x 128 in fp32 125 to 129 us (5.2 to 5.4 TB/s of 6.5 for a copy), one sequence of
// 1536 channels of 16 6.3 us replayed.
#include "layer_common.cuh"

namespace ssd {
namespace {

constexpr int kStepThreads = 128;

struct StepArgs {
  ssd_token_scan_step_params_t p;
  int row_blocks;       // PER_HEAD: blocks of a head's rows
  int vec_bc;           // B and C: vectors of a thread's components are aligned
  int vec_A;            // A: fp32 and such vectors are aligned
};

// V values of each lane's U rows summed over LPR lanes: the lanes trade halves while they hold several rows.
// Afterwards v[0 .. R - 1], R = max(1, U / LPR), are the sums of rows first_row(lane) on.
template <int LPR, int U>
__device__ __forceinline__ void sum_rows(float (&v)[U], int lane) {
  int count = U;
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) {
    if (count > 1) {
      const int half = count / 2;
      const bool up = lane & off;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
      }
      count = half;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
}
template <int LPR, int U>
__device__ __forceinline__ int first_row(int lane) {
  int count = U, row = 0;
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) {
    if (count > 1) {
      count /= 2;
      if (lane & off) row += count;
    }
  }
  return row;
}

template <typename T, typename S, int VS, int LPR, int U, bool PER_HEAD>
__global__ void __launch_bounds__(kStepThreads, 5) token_step_kernel(StepArgs args) {
  const ssd_token_scan_step_params_t& p = args.p;
  constexpr int kGroups = kStepThreads / LPR;        // rows side by side
  constexpr int R = U / LPR > 1 ? U / LPR : 1;       // rows a lane finishes
  const int b = blockIdx.y;
  const int slot = step_slot(p.state_indices, b, p.slots);
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int P = p.headdim, n = p.dstate;
  const int heads_per_group = p.nheads / p.ngroups;

  // row u of the thread's, clamped to one that exists
  const int rows = PER_HEAD ? P : p.nheads * P;
  const int r0 = (PER_HEAD ? blockIdx.x % args.row_blocks : blockIdx.x) * (kGroups * U) + grp;
  const int block_head = PER_HEAD ? blockIdx.x / args.row_blocks : 0;
  const auto head_of = [&](int r) { return PER_HEAD ? block_head : P == 1 ? r : r / P; };
  const auto p_of = [&](int r) { return PER_HEAD ? r : P == 1 ? 0 : r % P; };
  const auto row_of = [&](int u) { return min(r0 + u * kGroups, rows - 1); };
  const bool live = slot >= 0;
  S* const state = static_cast<S*>(p.state) + (int64_t)max(slot, 0) * p.state_stride[0];
  const T* const xb = static_cast<const T*>(p.x) + b * p.x_stride[0];
  const T* const zb = static_cast<const T*>(p.z) + b * p.z_stride[0];
  constexpr int H = PER_HEAD ? 1 : U;                // rows with a dt' of their own
  T x[U], xf[R], zf[R];
  AnyParam dtr[H], br[H], ar[H], Df[R];
  Pack<S, VS> st[U];
  int64_t at[U];
  float acc[U];
  const int mine0 = lane * VS < n ? lane * VS : 0;   // this lane's first components, clamped
  // rows of one head, or heads of one row: kGroups rows further lies the same distance further, and one 64-bit
  // product serves all; a row past the end reads the first one's values
  const bool even = PER_HEAD || P == 1;
  const int64_t s_step = kGroups * (PER_HEAD ? p.state_stride[2] : p.state_stride[1]), x_step = kGroups * (PER_HEAD ? p.x_stride[2] : p.x_stride[1]);
  const int first = row_of(0), h0 = head_of(first), p0 = p_of(first);
  const int64_t at0 = h0 * p.state_stride[1] + p0 * p.state_stride[2], x0 = h0 * p.x_stride[1] + p0 * p.x_stride[2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = row_of(u), h = head_of(r), pp = p_of(r);
    const bool there = r0 + u * kGroups < rows;
    at[u] = even ? at0 + (there ? u * s_step : 0) : h * p.state_stride[1] + pp * p.state_stride[2];
    st[u] = *reinterpret_cast<const Pack<S, VS>*>(state + at[u] + mine0);
    x[u] = xb[even ? x0 + (there ? u * x_step : 0) : h * p.x_stride[1] + pp * p.x_stride[2]];
    if (u < H) {
      dtr[u].load(p.dt, p.dt_dtype, b * p.dt_stride[0] + h * p.dt_stride[1]);
      if (p.dt_bias) br[u].load(p.dt_bias, p.bias_dtype, h * p.bias_stride);
      if (PER_HEAD) ar[u].load(p.A, p.A_dtype, h * p.A_stride[0]);
    }
    acc[u] = 0.0f;
  }
  // the rows this lane finishes
  const int uf = first_row<LPR, U>(lane);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = row_of(uf + i), h = head_of(r), pp = p_of(r);
    xf[i] = xb[h * p.x_stride[1] + pp * p.x_stride[2]];
    if (p.z) zf[i] = zb[h * p.z_stride[1] + pp * p.z_stride[2]];
    if (p.D) Df[i].load(p.D, p.D_dtype, h * p.D_stride[0] + pp * p.D_stride[1]);
  }
  const bool idle = step_taken(p.state_indices, b, slot) || !live;
  float dt[H], decay[H];
#pragma unroll
  for (int u = 0; u < H; ++u) {
    float raw = dtr[u].value(p.dt_dtype);
    if (p.dt_bias) raw += br[u].value(p.bias_dtype);
    dt[u] = scan_dt(raw, p.dt_softplus, p.dt_min, p.dt_max);
    decay[u] = PER_HEAD ? ex2_approx(dt[u] * (ar[u].value(p.A_dtype) * 1.4426950408889634f)) : 0.0f;
  }

  for (int n0 = 0; n0 < n; n0 += LPR * VS) {
    const int nn = n0 + lane * VS;
    const bool in = nn < n;
    float Bv[VS], Cv[VS];
    const auto load_bc = [&](int h) {
      const int g = p.ngroups == 1 ? 0 : h / heads_per_group, at = in ? nn : 0;
      const T* Bp = static_cast<const T*>(p.B) + b * p.B_stride[0] + g * p.B_stride[1] + at;
      const T* Cp = static_cast<const T*>(p.C) + b * p.C_stride[0] + g * p.C_stride[1] + at;
      if (args.vec_bc) {
        load_vec<VS>(Bp, Bv);
        load_vec<VS>(Cp, Cv);
      } else {
#pragma unroll
        for (int i = 0; i < VS; ++i) Bv[i] = widen(Bp[i]), Cv[i] = widen(Cp[i]);
      }
    };
    if (PER_HEAD) load_bc(head_of(0));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[VS], Av[VS], w[VS];
      if (n0 > 0 && in) st[u] = *reinterpret_cast<const Pack<S, VS>*>(state + at[u] + nn);
      if (!PER_HEAD) {
        const int h = head_of(row_of(u));
        load_bc(h);
        const int64_t a0 = h * p.A_stride[0] + (in ? nn : 0) * p.A_stride[1];
        if (args.vec_A) {
          load_vec<VS>(static_cast<const float*>(p.A) + a0, Av);
        } else {
#pragma unroll
          for (int i = 0; i < VS; ++i) Av[i] = load_f(p.A, p.A_dtype, a0 + i * p.A_stride[1]);
        }
      }
      const float d = dt[PER_HEAD ? 0 : u], ux = d * widen(x[u]);
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        Av[i] = PER_HEAD ? decay[0] : ex2_approx(d * (Av[i] * 1.4426950408889634f));
        v[i] = ux;
        w[i] = widen(st[u].e[i]);
      }
      vec_mul(v, Bv);
      vec_fma(Av, w, v);
      if (in) {
#pragma unroll
        for (int i = 0; i < VS; ++i) acc[u] = fmaf(v[i], Cv[i], acc[u]);      // y sees the state before it is rounded to its type
        if (!idle && r0 + u * kGroups < rows) store_vec<VS>(state + at[u] + nn, v);
      }
    }
  }
  sum_rows<LPR, U>(acc, lane);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + (uf + i) * kGroups;
    // with more lanes than rows several lanes hold a row's sum: the first of them writes
    if (r >= rows || (LPR > U && (lane & (LPR / U - 1)) != 0)) continue;
    const int h = head_of(r), pp = p_of(r);
    float y = acc[i];
    if (p.D) y = fmaf(Df[i].value(p.D_dtype), widen(xf[i]), y);
    if (p.z) y *= silu_f(widen(zf[i]));
    static_cast<T*>(p.out)[((int64_t)b * p.nheads + h) * P + pp] = narrow<T>(idle ? 0.0f : y);
  }
}

template <typename T, typename S, int VS, int LPR, bool PER_HEAD>
int launch_step(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  constexpr int U = PER_HEAD ? 8 : 4;
  constexpr int kRows = kStepThreads / LPR * U;
  StepArgs a;
  a.p = p;
  a.row_blocks = (p.headdim + kRows - 1) / kRows;
  constexpr size_t kBytes = VS * sizeof(T) < 16 ? VS * sizeof(T) : 16;
  a.vec_bc = rows_aligned(p.B, p.B_stride, 2, sizeof(T), kBytes) && rows_aligned(p.C, p.C_stride, 2, sizeof(T), kBytes) && p.dstate % VS == 0;
  a.vec_A = p.A_dtype == SSD_F32 && p.A_stride[1] == 1 && rows_aligned(p.A, p.A_stride, 1, 4, VS * 4 < 16 ? VS * 4 : 16) && p.dstate % VS == 0;
  const int64_t blocks = PER_HEAD ? (int64_t)a.row_blocks * p.nheads : ((int64_t)p.nheads * p.headdim + kRows - 1) / kRows;
  SSD_REQUIRE((int64_t)p.nheads * p.headdim <= 0x7fffffff - kRows && blocks <= 0x7fffffff && p.batch <= 65535, SSD_ERR_UNSUPPORTED, "token scan step: too many rows or batch %d too large", p.batch);
  token_step_kernel<T, S, VS, LPR, U, PER_HEAD><<<dim3((unsigned)blocks, p.batch), kStepThreads, 0, stream>>>(a);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

template <typename T, typename S, bool PER_HEAD>
int launch_step_lanes(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  constexpr int VS = 16 / sizeof(S);
  const bool vec = p.dstate % VS == 0 && rows_aligned(p.state, p.state_stride, 3, sizeof(S), 16);
  if (!vec) return launch_step<T, S, 1, 32, PER_HEAD>(p, stream);
  const int need = p.dstate / VS;
  if (need <= 2) return launch_step<T, S, VS, 2, PER_HEAD>(p, stream);
  if (need <= 4) return launch_step<T, S, VS, 4, PER_HEAD>(p, stream);
  if (need <= 8) return launch_step<T, S, VS, 8, PER_HEAD>(p, stream);
  if (need <= 16) return launch_step<T, S, VS, 16, PER_HEAD>(p, stream);
  return launch_step<T, S, VS, 32, PER_HEAD>(p, stream);
}

}  // namespace

int launch_token_step(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  return with_type(p.x_dtype, [&](auto t) -> int {
    using T = decltype(t);
    const auto go = [&](auto s) -> int {
      using S = decltype(s);
      // one decay a head, and enough rows in a head to fill a block's rows
      return p.A_stride[1] == 0 && p.headdim >= 16 ? launch_step_lanes<T, S, true>(p, stream) : launch_step_lanes<T, S, false>(p, stream);
    };
    return p.state_dtype == SSD_F32 ? go(float()) : go(T());
  });
}

}  // namespace ssd
