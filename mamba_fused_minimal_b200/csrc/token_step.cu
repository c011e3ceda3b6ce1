// One position of the selective scan for each running sequence, the state updated in place:
//
//   h[n] = exp(dt' A[n]) h[n] + dt' x B[n];   y = C . h + D x;   out = y or y silu(z)
//
// The state is read and written once and everything else is small: memory bandwidth bounds a full batch,
// latency a single sequence.  A row is the dstate components of one (head, p); LPR adjacent lanes hold it
// as 16-byte vectors, and a thread's U rows are all loaded before the first is used.  With one decay a
// head (the Mamba2 form) a block stays inside a head and forms dt' and the decay once; with a decay for
// each component every row has its own.
#include "layer_common.cuh"

namespace ssd {
namespace {

constexpr int kStepThreads = 128;

struct StepArgs {
  ssd_token_scan_step_params_t p;
  int row_blocks;       // PER_HEAD: blocks of a head's rows
};

template <typename S, int VS, int LPR, int U, bool PER_HEAD>
__global__ void __launch_bounds__(kStepThreads) token_step_kernel(StepArgs args) {
  const ssd_token_scan_step_params_t& p = args.p;
  constexpr int kGroups = kStepThreads / LPR;        // rows side by side
  const int b = blockIdx.y;
  const int slot = step_slot(p.state_indices, b, p.slots);
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int P = p.headdim, n = p.dstate;
  const int heads_per_group = p.nheads / p.ngroups;

  int hh[U], pp[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (PER_HEAD) {
      hh[u] = blockIdx.x / args.row_blocks;
      pp[u] = (blockIdx.x % args.row_blocks) * (kGroups * U) + u * kGroups + grp;
      in[u] = pp[u] < P;
    } else {
      const int64_t r = (int64_t)blockIdx.x * (kGroups * U) + u * kGroups + grp;
      in[u] = r < (int64_t)p.nheads * P;
      hh[u] = in[u] ? (int)(r / P) : 0;
      pp[u] = in[u] ? (int)(r % P) : 0;
    }
  }
  const bool live = slot >= 0;
  S* const state = static_cast<S*>(p.state) + (int64_t)max(slot, 0) * p.state_stride[0];
  float acc[U], x[U], dt[U], decay[U];
#pragma unroll
  for (int u = 0; u < U; ++u) acc[u] = x[u] = dt[u] = decay[u] = 0.0f;
  bool taken = false;

  for (int n0 = 0; n0 < n; n0 += LPR * VS) {
    const int nn = n0 + lane * VS;
    const bool mine = nn < n;
    float st[U][VS];
    if (live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (in[u] && mine) {
          load_vec<VS>(state + hh[u] * p.state_stride[1] + pp[u] * p.state_stride[2] + nn, st[u]);
        } else {
#pragma unroll
          for (int i = 0; i < VS; ++i) st[u][i] = 0.0f;
        }
      }
    }
    if (n0 == 0) {
      if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!in[u]) continue;
          x[u] = load_f(p.x, p.x_dtype, b * p.x_stride[0] + hh[u] * p.x_stride[1] + pp[u] * p.x_stride[2]);
          if (PER_HEAD && u > 0 && in[0]) {
            dt[u] = dt[0];
            decay[u] = decay[0];
            continue;
          }
          float raw = load_f(p.dt, p.dt_dtype, b * p.dt_stride[0] + hh[u] * p.dt_stride[1]);
          if (p.dt_bias) raw += load_f(p.dt_bias, p.bias_dtype, hh[u] * p.bias_stride);
          dt[u] = scan_dt(raw, p.dt_softplus, p.dt_min, p.dt_max);
          if (PER_HEAD) decay[u] = __expf(dt[u] * load_f(p.A, p.A_dtype, hh[u] * p.A_stride[0]));
        }
      }
      taken = step_taken(p.state_indices, b, slot);
    }
    if (!live || taken) break;
    if (!mine) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in[u]) continue;
      const int g = hh[u] / heads_per_group;
      float Bv[VS], Cv[VS], Av[VS];
      load_param<VS>(p.B, p.x_dtype, b * p.B_stride[0] + g * p.B_stride[1] + nn, Bv);
      load_param<VS>(p.C, p.x_dtype, b * p.C_stride[0] + g * p.C_stride[1] + nn, Cv);
      if (!PER_HEAD) {
#pragma unroll
        for (int i = 0; i < VS; ++i) Av[i] = load_f(p.A, p.A_dtype, hh[u] * p.A_stride[0] + (nn + i) * p.A_stride[1]);
      }
      const float ux = dt[u] * x[u];
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const float a = PER_HEAD ? decay[u] : __expf(dt[u] * Av[i]);
        st[u][i] = fmaf(a, st[u][i], ux * Bv[i]);
        acc[u] = fmaf(st[u][i], Cv[i], acc[u]);      // y sees the state before it is rounded to its type
      }
      store_vec<VS>(state + hh[u] * p.state_stride[1] + pp[u] * p.state_stride[2] + nn, st[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float y = acc[u];
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) y += __shfl_xor_sync(0xffffffffu, y, off);
    if (lane == 0 && in[u]) {
      if (live && !taken) {
        if (p.D) y += load_f(p.D, p.D_dtype, hh[u] * p.D_stride[0] + pp[u] * p.D_stride[1]) * x[u];
        if (p.z) y *= silu_f(load_f(p.z, p.x_dtype, b * p.z_stride[0] + hh[u] * p.z_stride[1] + pp[u] * p.z_stride[2]));
      } else {
        y = 0.0f;
      }
      store_f(p.out, p.x_dtype, ((int64_t)b * p.nheads + hh[u]) * P + pp[u], y);
    }
  }
}

template <typename S, int VS, int LPR, bool PER_HEAD>
int launch_step(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  constexpr int U = PER_HEAD ? 8 : 4;
  constexpr int kRows = kStepThreads / LPR * U;
  StepArgs a;
  a.p = p;
  a.row_blocks = (p.headdim + kRows - 1) / kRows;
  const int64_t blocks = PER_HEAD ? (int64_t)a.row_blocks * p.nheads : ((int64_t)p.nheads * p.headdim + kRows - 1) / kRows;
  SSD_REQUIRE(blocks <= 0x7fffffff && p.batch <= 65535, SSD_ERR_UNSUPPORTED, "token scan step: too many rows or batch %d too large", p.batch);
  token_step_kernel<S, VS, LPR, U, PER_HEAD><<<dim3((unsigned)blocks, p.batch), kStepThreads, 0, stream>>>(a);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

template <typename S, bool PER_HEAD>
int launch_step_lanes(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  constexpr int VS = 16 / sizeof(S);
  const bool vec = p.dstate % VS == 0 && rows_aligned(p.state, p.state_stride, 3, sizeof(S), 16);
  if (!vec) return launch_step<S, 1, 32, PER_HEAD>(p, stream);
  const int need = p.dstate / VS;
  if (need <= 2) return launch_step<S, VS, 2, PER_HEAD>(p, stream);
  if (need <= 4) return launch_step<S, VS, 4, PER_HEAD>(p, stream);
  if (need <= 8) return launch_step<S, VS, 8, PER_HEAD>(p, stream);
  if (need <= 16) return launch_step<S, VS, 16, PER_HEAD>(p, stream);
  return launch_step<S, VS, 32, PER_HEAD>(p, stream);
}

}  // namespace

int launch_token_step(const ssd_token_scan_step_params_t& p, cudaStream_t stream) {
  return with_type(p.state_dtype, [&](auto s) -> int {
    using S = decltype(s);
    // one decay a head, and enough rows in a head to fill a block's rows
    return p.A_stride[1] == 0 && p.headdim >= 16 ? launch_step_lanes<S, true>(p, stream) : launch_step_lanes<S, false>(p, stream);
  });
}

}  // namespace ssd
