// Gradients of the selective scan.  With a_t = exp(dt' A), u_t = dt' x, g = dL/dh:
//
//   g_t = C_t dy_t + a_{t+1} g_{t+1}                 (from the last position to the first)
//   dC_t = sum over channels of dy_t h_t             dB_t = sum over channels of g_t u_t
//   dx = dt' (g . B) + D dy                          ddt' = x (g . B) + sum_n A a h_before g
//   dA = sum over positions of dt' a h_before g      dz = dout y silu'(z),  dy = dout silu(z)
//
// A thread owns one component of one channel's state.  The forward pass left the states before every 16th
// position, so a tile of 16 positions is recomputed from its checkpoint into registers (a and a h_before:
// one exponential per position and component, as in the forward pass) and then walked backwards.  What
// is summed over components (g . B and the A term) is exchanged between the lanes of a channel; what is
// summed over channels (dB, dC) is added up over the block's channels in shared memory and leaves as the
// block's share, which a second kernel adds over the blocks in a fixed order.
#include "token_scan.cuh"

namespace ssd {
namespace {

constexpr int kBwdThreads = 512;
constexpr int kBwdWarps = kBwdThreads / 32;
constexpr int kT = SSD_TOKEN_SCAN_CHECKPOINT;     // positions of a tile
constexpr int kPitch = kT + 4;                    // row pitch in shared memory

struct ScanBwdArgs {
  ScanArgs f;
  const void* dout;
  const float* dfinal;
  void* dx;
  void* ddt;
  void* dz;
  float* dinit;
  float* part_bc;      // (b, l, g, tiles_per_group, 2, n): the blocks' shares of dB and dC
  float* part_A;       // (b, d, n)
  float* part_D;       // (b, d)
  float* part_bias;    // (b, d)
  int64_t d_sb, d_sl;
};

template <int NP>
struct BwdShape {
  static constexpr int kChannels = kBwdThreads / NP;              // channels of a block
  static constexpr int kSlabs = NP > 32 ? NP / 32 : 1;            // warps that share a channel
  static constexpr int kRow = NP == 8 ? 16 : NP == 16 ? 32 : 64;  // a warp's dB and dC of one position
  static constexpr int kItems = kT * kChannels;                   // (position, channel) pairs of a tile
  static constexpr int kPer = kItems > kBwdThreads ? kItems / kBwdThreads : 1;
  static constexpr int kBc = 2 * kT * NP;
  static constexpr int kPerBc = kBc > kBwdThreads ? kBc / kBwdThreads : 1;
  static constexpr size_t kSmem = sizeof(float) * ((3 * kChannels + 2 * NP) * kPitch + 2 * kChannels * kSlabs * kPitch + kBwdWarps * kT * kRow);
};

template <typename T, int NP>
__global__ void __launch_bounds__(kBwdThreads) token_scan_bwd_kernel(ScanBwdArgs q) {
  using Sh = BwdShape<NP>;
  constexpr int CH = Sh::kChannels, SL = Sh::kSlabs, ROW = Sh::kRow, PER = Sh::kPer;
  constexpr bool kAhead = NP <= 64;      // the tile before waits in registers while this one is computed
  const ScanArgs& a = q.f;
  extern __shared__ float4 smem4[];
  float* s_d = reinterpret_cast<float*>(smem4);      // [CH][kPitch] dt'
  float* s_u = s_d + CH * kPitch;                    // dt' x
  float* s_g = s_u + CH * kPitch;                    // dy
  float* s_B = s_g + CH * kPitch;                    // [NP][kPitch]
  float* s_C = s_B + NP * kPitch;
  float* s_p = s_C + NP * kPitch;                    // [2][CH][SL][kPitch]: g . B and the A term
  float* s_bc = s_p + 2 * CH * SL * kPitch;          // [warps][kT][ROW]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int grp = blockIdx.x / a.tiles_per_group, tile_c = blockIdx.x % a.tiles_per_group;
  const int b = blockIdx.y;
  const int c0 = grp * a.per_group + tile_c * CH;
  const int nch = min(CH, a.per_group - tile_c * CH);

  // what this thread loads and stores: item i is position i / CH, channel i % CH
  const int lc = tid % CH;
  const float Dv = a.D && lc < nch ? load_f(a.D, a.D_dtype, c0 + lc) : 0.0f;
  const float bias = a.bias && lc < nch ? load_f(a.bias, a.bias_dtype, c0 + lc) : 0.0f;
  float sum_D = 0.0f, sum_bias = 0.0f;

  // what this thread computes
  const int n = tid % NP, ch = tid / NP;
  const bool has = ch < nch && n < a.dstate;
  const float A = has ? load_f(a.A, a.A_dtype, (int64_t)(c0 + ch) * a.dstate + n) : 0.0f;
  const float A2 = A * kLog2e;
  const int64_t state_at = ((int64_t)b * a.channels + c0 + ch) * a.dstate + n;
  float carry = has && q.dfinal ? q.dfinal[state_at] : 0.0f;      // a_{t+1} g_{t+1}
  float sum_A = 0.0f;

  const int tiles = (a.seqlen + kT - 1) / kT;
  // as they were loaded: nothing waits for them before they are used
  T xr[PER], dr[PER], gr[PER], zr[PER], yr[PER], bcr[kAhead ? Sh::kPerBc : 1];
  float dr32[PER], h_next = 0.0f;
  const T zero = narrow<T>(0.0f);
  const auto read = [&](const void* base, int64_t at) { return static_cast<const T*>(base)[at]; };
  const auto load_bc = [&](int k, int t0) {
    const int item = k * kBwdThreads + tid;
    if (Sh::kBc < kBwdThreads && item >= Sh::kBc) return zero;
    const int nn = item % NP, t = t0 + (item / NP) % kT;
    const bool is_c = item >= kT * NP;
    if (nn >= a.dstate || t >= a.seqlen) return zero;
    return is_c ? read(a.C, b * a.C_sb + (int64_t)t * a.C_sl + grp * a.C_sg + nn) : read(a.B, b * a.B_sb + (int64_t)t * a.B_sl + grp * a.B_sg + nn);
  };
  const auto store_bc = [&](int k, T v) {
    const int item = k * kBwdThreads + tid;
    if (Sh::kBc < kBwdThreads && item >= Sh::kBc) return;
    (item >= kT * NP ? s_C : s_B)[(item % NP) * kPitch + (item / NP) % kT] = widen(v);
  };
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int item = e * kBwdThreads + tid, t = t0 + item / CH;
      xr[e] = dr[e] = gr[e] = zr[e] = yr[e] = zero;
      dr32[e] = 0.0f;
      if (item >= Sh::kItems || t >= a.seqlen || lc >= nch) continue;
      const int64_t c = c0 + lc;
      xr[e] = read(a.x, b * a.x_sb + (int64_t)t * a.x_sl + c);
      const int64_t dat = b * a.dt_sb + (int64_t)t * a.dt_sl + c;
      if (a.dt_f32)
        dr32[e] = static_cast<const float*>(a.dt)[dat];
      else
        dr[e] = read(a.dt, dat);
      gr[e] = read(q.dout, b * q.d_sb + (int64_t)t * q.d_sl + c);
      if (a.z) {
        zr[e] = read(a.z, b * a.z_sb + (int64_t)t * a.z_sl + c);
        yr[e] = read(a.out_x, ((int64_t)b * a.seqlen + t) * a.channels + c);
      }
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < Sh::kPerBc; ++k) bcr[k] = load_bc(k, t0);
    }
    if (has) h_next = a.ckpt[(((int64_t)b * tiles + t0 / kT) * a.channels + c0 + ch) * a.dstate + n];
  };

  fetch((tiles - 1) * kT);
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const int t0 = tile * kT;
    float d[PER], x[PER], dy[PER], raw[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int item = e * kBwdThreads + tid, lt = item / CH, t = t0 + lt;
      if (item >= Sh::kItems) continue;
      const bool in = t < a.seqlen && lc < nch;
      x[e] = widen(xr[e]);
      raw[e] = (a.dt_f32 ? dr32[e] : widen(dr[e])) + bias;
      d[e] = in ? scan_dt(raw[e], a.softplus, a.dt_min, a.dt_max) : 0.0f;
      dy[e] = widen(gr[e]);
      if (a.z) {
        const float zv = widen(zr[e]);
        if (in) static_cast<T*>(q.dz)[((int64_t)b * a.seqlen + t) * a.channels + c0 + lc] = narrow<T>(dy[e] * widen(yr[e]) * dsilu_f(zv));
        dy[e] *= silu_f(zv);
      }
      s_d[lc * kPitch + lt] = d[e];
      s_u[lc * kPitch + lt] = d[e] * x[e];
      s_g[lc * kPitch + lt] = dy[e];
      sum_D += dy[e] * x[e];
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < Sh::kPerBc; ++k) store_bc(k, bcr[k]);
    } else {
#pragma unroll 4
      for (int k = 0; k < Sh::kPerBc; ++k) store_bc(k, load_bc(k, t0));
    }
    float h = h_next;
    const uint32_t resets = a.seq ? reset_mask(a, b, t0, lane) : 0u;
    __syncthreads();
    if (tile > 0) fetch(t0 - kT);

    // forwards through the tile: the decays, and what of the state before reaches each position
    float dec[kT], kept[kT];
#pragma unroll
    for (int t = 0; t < kT; t += 4) {
      const float4 d4 = *reinterpret_cast<const float4*>(&s_d[ch * kPitch + t]);
      const float4 u4 = *reinterpret_cast<const float4*>(&s_u[ch * kPitch + t]);
      const float4 B4 = *reinterpret_cast<const float4*>(&s_B[n * kPitch + t]);
      const float dd[4] = {d4.x, d4.y, d4.z, d4.w}, uu[4] = {u4.x, u4.y, u4.z, u4.w}, BB[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dec[t + i] = resets >> (t + i) & 1u ? 0.0f : ex2_approx(dd[i] * A2);
        kept[t + i] = resets >> (t + i) & 1u ? 0.0f : dec[t + i] * h;
        h = fmaf(uu[i], BB[i], kept[t + i]);
      }
    }
    // and backwards
#pragma unroll
    for (int t = kT - 4; t >= 0; t -= 4) {
      const float4 d4 = *reinterpret_cast<const float4*>(&s_d[ch * kPitch + t]);
      const float4 u4 = *reinterpret_cast<const float4*>(&s_u[ch * kPitch + t]);
      const float4 g4 = *reinterpret_cast<const float4*>(&s_g[ch * kPitch + t]);
      const float4 B4 = *reinterpret_cast<const float4*>(&s_B[n * kPitch + t]);
      const float4 C4 = *reinterpret_cast<const float4*>(&s_C[n * kPitch + t]);
      const float dd[4] = {d4.x, d4.y, d4.z, d4.w}, uu[4] = {u4.x, u4.y, u4.z, u4.w}, yy[4] = {g4.x, g4.y, g4.z, g4.w};
      const float BB[4] = {B4.x, B4.y, B4.z, B4.w}, CC[4] = {C4.x, C4.y, C4.z, C4.w};
      float p1[4], p2[4];
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        const float g = fmaf(CC[i], yy[i], carry);
        const float vC = yy[i] * fmaf(uu[i], BB[i], kept[t + i]);
        const float vB = g * uu[i];
        const float m = g * kept[t + i];
        p1[i] = g * BB[i];
        p2[i] = m * A;
        sum_A = fmaf(m, dd[i], sum_A);
        carry = g * dec[t + i];
        float* row = s_bc + (warp * kT + t + i) * ROW;
        if constexpr (NP >= 32) {
          row[lane] = vB;
          row[32 + lane] = vC;
        } else {
          // lanes 0..15 keep dB, lanes 16..31 dC, of the channels 16 lanes apart
          float v = (lane < 16 ? vB : vC) + __shfl_xor_sync(0xffffffffu, lane < 16 ? vC : vB, 16);
          if constexpr (NP == 8) {
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            if ((lane & 8) == 0) row[(lane >> 4) * 8 + (lane & 7)] = v;
          } else {
            row[lane] = v;
          }
        }
      }
      // eight sums (two kinds, four positions) over the channel's lanes: the lanes trade halves until each
      // of eight holds one sum
      const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (b0 ? p2[i] : p1[i]) + __shfl_xor_sync(0xffffffffu, b0 ? p1[i] : p2[i], 1);
      float v0 = (b1 ? w[1] : w[0]) + __shfl_xor_sync(0xffffffffu, b1 ? w[0] : w[1], 2);
      float v1 = (b1 ? w[3] : w[2]) + __shfl_xor_sync(0xffffffffu, b1 ? w[2] : w[3], 2);
      float r = (b2 ? v1 : v0) + __shfl_xor_sync(0xffffffffu, b2 ? v0 : v1, 4);
#pragma unroll
      for (int off = 8; off < (NP < 32 ? NP : 32); off <<= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
      if ((n & 31) < 8) s_p[(((lane & 1) * CH + ch) * SL + n / 32) * kPitch + t + ((lane >> 1) & 3)] = r;
    }
    __syncthreads();

#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int item = e * kBwdThreads + tid, lt = item / CH, t = t0 + lt;
      if (item >= Sh::kItems || t >= a.seqlen || lc >= nch) continue;
      float gB = 0.0f, gA = 0.0f;
#pragma unroll
      for (int s = 0; s < SL; ++s) {
        gB += s_p[(lc * SL + s) * kPitch + lt];
        gA += s_p[((CH + lc) * SL + s) * kPitch + lt];
      }
      float dd = x[e] * gB + gA;
      if (a.softplus || a.dt_min > -INFINITY || a.dt_max < INFINITY) {
        const float v = a.softplus ? softplus_f(raw[e]) : raw[e];
        if (v < a.dt_min || v > a.dt_max) dd = 0.0f;
        if (a.softplus) dd *= sigmoid_f(raw[e]);
      }
      sum_bias += dd;
      const int64_t at = ((int64_t)b * a.seqlen + t) * a.channels + c0 + lc;
      static_cast<T*>(q.dx)[at] = narrow<T>(fmaf(d[e], gB, Dv * dy[e]));
      if (a.dt_f32)
        static_cast<float*>(q.ddt)[at] = dd;
      else
        static_cast<T*>(q.ddt)[at] = narrow<T>(dd);
    }
    // the block's share of dB and dC: over the warps (their channels) in order
    constexpr int kOuts = kT * SL * ROW, kSum = kBwdWarps / SL;
#pragma unroll 1
    for (int o = tid; o < kOuts; o += kBwdThreads) {
      const int j = o % ROW, slab = (o / ROW) % SL, t = o / (ROW * SL);
      const int nn = slab * 32 + j % (ROW / 2);
      if (nn >= a.dstate || t0 + t >= a.seqlen) continue;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < kSum; ++s) v += s_bc[((s * SL + slab) * kT + t) * ROW + j];
      q.part_bc[((((int64_t)b * a.seqlen + t0 + t) * a.ngroups + grp) * a.tiles_per_group + tile_c) * (2 * a.dstate) +
                (j / (ROW / 2)) * a.dstate + nn] = v;
    }
  }

  if (has) {
    q.part_A[state_at] = sum_A;
    if (q.dinit) q.dinit[state_at] = carry;
  }
  // dD and the bias's gradient: over the threads of a channel in order
  __syncthreads();
  s_bc[tid] = sum_D;
  s_bc[kBwdThreads + tid] = sum_bias;
  __syncthreads();
  if (tid < nch) {
    float u = 0.0f, v = 0.0f;
    for (int s = tid; s < min(kBwdThreads, Sh::kItems); s += CH) u += s_bc[s], v += s_bc[kBwdThreads + s];
    q.part_D[(int64_t)b * a.channels + c0 + tid] = u;
    q.part_bias[(int64_t)b * a.channels + c0 + tid] = v;
  }
}

// dB and dC: over the blocks' shares in order.  One thread per (position, group, kind, component).
template <typename T>
__global__ void __launch_bounds__(256) sum_bc_kernel(const float* part, T* dB, T* dC, int64_t rows, int tiles, int dstate) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * 2 * dstate) return;
  const int64_t row = i / (2 * dstate);
  const int j = (int)(i - row * 2 * dstate);
  const float* p = part + row * tiles * (2 * dstate) + j;
  float v = 0.0f;
#pragma unroll 8
  for (int k = 0; k < tiles; ++k) v += p[(int64_t)k * 2 * dstate];
  if (j < dstate)
    dB[row * dstate + j] = narrow<T>(v);
  else
    dC[row * dstate + j - dstate] = narrow<T>(v);
}

// dA, dD and the bias's gradient: over the batch in order.
__global__ void __launch_bounds__(256) sum_batch_kernel(ScanBwdArgs q, int batch, float* dA, float* dD, float* dbias) {
  const int64_t dn = (int64_t)q.f.channels * q.f.dstate, d = q.f.channels;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const float* p;
  float* out;
  int64_t at, pitch;
  if (i < dn) {
    p = q.part_A, out = dA, at = i, pitch = dn;
  } else if (i < dn + d) {
    p = q.part_D, out = dD, at = i - dn, pitch = d;
  } else if (i < dn + 2 * d) {
    p = q.part_bias, out = dbias, at = i - dn - d, pitch = d;
  } else {
    return;
  }
  if (out == nullptr) return;
  float v = 0.0f;
#pragma unroll 4
  for (int b = 0; b < batch; ++b) v += p[b * pitch + at];
  out[at] = v;
}

int padded_state(int n) { return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256; }

int bwd_tiles(const ssd_token_scan_params_t& p) {
  const int ch = kBwdThreads / padded_state(p.dstate);
  return (p.channels / p.ngroups + ch - 1) / ch;
}

struct BwdWorkspace {
  size_t bc, A, D, total;      // offsets in floats: shares of dB and dC, dA, dD; the bias's follow dD's
};
BwdWorkspace bwd_workspace(const ssd_token_scan_params_t& p) {
  BwdWorkspace w;
  w.bc = 0;
  w.A = (size_t)p.batch * p.seqlen * p.ngroups * bwd_tiles(p) * 2 * p.dstate;
  w.D = w.A + (size_t)p.batch * p.channels * p.dstate;
  w.total = w.D + 2 * (size_t)p.batch * p.channels;
  return w;
}

template <typename T, int NP>
int launch_bwd(const ScanBwdArgs& q, int batch, cudaStream_t stream) {
  constexpr size_t smem = BwdShape<NP>::kSmem;
  if (smem > 48 * 1024)
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_bwd_kernel<T, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  token_scan_bwd_kernel<T, NP><<<dim3(q.f.ngroups * q.f.tiles_per_group, batch), kBwdThreads, smem, stream>>>(q);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

}  // namespace

size_t token_scan_bwd_workspace(const ssd_token_scan_bwd_params_t& p) { return bwd_workspace(p.scan).total * sizeof(float); }

int launch_token_scan_bwd(const ssd_token_scan_bwd_params_t& r, cudaStream_t stream) {
  const ssd_token_scan_params_t& p = r.scan;
  const BwdWorkspace w = bwd_workspace(p);
  ScanBwdArgs q;
  q.f = scan_args(p);
  q.f.tiles_per_group = bwd_tiles(p);
  q.dout = r.dout;
  q.dfinal = r.dfinal_states;
  q.dx = r.dx, q.ddt = r.ddt, q.dz = r.dz, q.dinit = r.dinitial_states;
  float* ws = static_cast<float*>(r.workspace);
  q.part_bc = ws + w.bc;
  q.part_A = ws + w.A;
  q.part_D = ws + w.D;
  q.part_bias = q.part_D + (size_t)p.batch * p.channels;
  q.d_sb = r.dout_stride[0], q.d_sl = r.dout_stride[1];
  SSD_REQUIRE(p.batch <= 65535, SSD_ERR_UNSUPPORTED, "token scan: batch %d too large", p.batch);
  return with_type(p.x_dtype, [&](auto t) -> int {
    using T = decltype(t);
    int rc;
    switch (padded_state(p.dstate)) {
      case 8: rc = launch_bwd<T, 8>(q, p.batch, stream); break;
      case 16: rc = launch_bwd<T, 16>(q, p.batch, stream); break;
      case 32: rc = launch_bwd<T, 32>(q, p.batch, stream); break;
      case 64: rc = launch_bwd<T, 64>(q, p.batch, stream); break;
      case 128: rc = launch_bwd<T, 128>(q, p.batch, stream); break;
      default: rc = launch_bwd<T, 256>(q, p.batch, stream); break;
    }
    if (rc != SSD_OK) return rc;
    const int64_t rows = (int64_t)p.batch * p.seqlen * p.ngroups, outs = rows * 2 * p.dstate;
    sum_bc_kernel<T><<<(unsigned)((outs + 255) / 256), 256, 0, stream>>>(q.part_bc, static_cast<T*>(r.dB), static_cast<T*>(r.dC), rows,
                                                                       q.f.tiles_per_group, p.dstate);
    SSD_CUDA_OK(cudaGetLastError());
    const int64_t par = (int64_t)p.channels * (p.dstate + 2);
    sum_batch_kernel<<<(unsigned)((par + 255) / 256), 256, 0, stream>>>(q, p.batch, r.dA, r.dD, r.ddt_bias);
    SSD_CUDA_OK(cudaGetLastError());
    return SSD_OK;
  });
}

}  // namespace ssd
