// Selective scan, position by position: h[n] = a h[n] + dt' x B[n], a = exp(dt' A[n]), y = C . h + D x.
//
// Each (position, channel, component) needs one exponential and four multiply-adds, and nothing of it can
// be shared between channels, so at dstate 16 the special function units (16 exponentials per clock and
// SM) bound the kernel, ahead of memory (x, dt, z and out once).  A thread holds NS components of one
// channel's state in registers and LPC adjacent lanes share a channel: the recurrence along the positions
// never leaves a thread, and only y is summed over the LPC lanes, four positions at a time (the lanes trade
// halves, so that four sums over four lanes take three exchanges).
//
// A block takes 16 channels and walks the positions in tiles of 32.  The tile's x, dt, B and C are turned
// into fp32 with positions contiguous in shared memory, so that one 16-byte read gives a thread four
// positions; dt' is formed once per position and channel there.  The next tile's loads are in flight while
// this one is computed.
//
// Few channels and a long sequence: the sequence is cut into segments that run side by side.  A first pass
// leaves each segment's state from a zero start and the sum of its dt'; since the decay over a segment is
// exp(A * sum dt'), the second pass's blocks form the state they start from by themselves.  The
// exponentials are computed twice, so this is done only where the GPU would otherwise stand idle.
#include "token_scan.cuh"

namespace ssd {
namespace {

constexpr int kCh = 16;            // channels of a block
constexpr int kTile = 32;          // positions of a tile
constexpr int kLd = kTile + 4;     // row pitch in shared memory: 16-byte aligned, rows in different banks

template <typename T, int LPC, int NS, bool STATE>
__global__ void __launch_bounds__(kCh* LPC) token_scan_kernel(ScanArgs a) {
  constexpr int NT = kCh * LPC;          // threads
  constexpr int EV = kTile / LPC;        // elements of x a thread loads per tile
  constexpr int VPR = kCh / EV;          // such vectors per position
  constexpr int NP = LPC * NS;           // components, padded
  constexpr bool kAhead = NS <= 4;       // B and C of the next tile wait in registers too
  extern __shared__ float4 smem4[];
  float* s_d = reinterpret_cast<float*>(smem4);       // [kCh][kLd] dt'
  float* s_u = s_d + kCh * kLd;                       // dt' * x
  float* s_y = s_u + kCh * kLd;
  float* s_B = s_y + kCh * kLd;                       // [NP][kLd]
  float* s_C = s_B + NP * kLd;
  const int tid = threadIdx.x;
  const int g = blockIdx.x / a.tiles_per_group, tile_c = blockIdx.x % a.tiles_per_group;
  const int b = blockIdx.z, seg = blockIdx.y;
  const int c0 = g * a.per_group + tile_c * kCh;                     // first channel of the block
  const int nch = min(kCh, a.per_group - tile_c * kCh);
  const int t_begin = seg * a.seg_len, t_end = min(a.seqlen, t_begin + a.seg_len);

  // what this thread loads and stores: EV channels of one position
  const int lt = tid / VPR, lc = (tid % VPR) * EV;
  const int lcount = max(0, min(EV, nch - lc));
  const T* xp = static_cast<const T*>(a.x) + b * a.x_sb + c0 + lc;
  const T* zp = static_cast<const T*>(a.z) + b * a.z_sb + c0 + lc;
  const int64_t dt_off = b * a.dt_sb + c0 + lc;
  const T* Bp = static_cast<const T*>(a.B) + b * a.B_sb + g * a.B_sg;
  const T* Cp = static_cast<const T*>(a.C) + b * a.C_sb + g * a.C_sg;
  float dv[EV], bv[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) {
    dv[e] = a.D && e < lcount ? load_f(a.D, a.D_dtype, c0 + lc + e) : 0.0f;
    bv[e] = a.bias && e < lcount ? load_f(a.bias, a.bias_dtype, c0 + lc + e) : 0.0f;
  }

  // what this thread computes: components q, q + LPC, ... of channel ch
  const int q = tid % LPC, ch = tid / LPC;
  const bool has = ch < nch;
  float A2[NS], h[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int n = s * LPC + q;
    const bool in = has && n < a.dstate;
    A2[s] = in ? load_f(a.A, a.A_dtype, (int64_t)(c0 + ch) * a.dstate + n) * kLog2e : 0.0f;
    h[s] = in && a.init ? load_f(a.init, a.init_dtype, ((int64_t)b * a.channels + c0 + ch) * a.dstate + n) : 0.0f;
    if (STATE && seg > 0) h[s] = 0.0f;
  }
  if (!STATE && seg > 0) {
    // the state this segment starts from: what the earlier ones leave, in order (the first of them
    // started from the initial state)
#pragma unroll
    for (int s = 0; s < NS; ++s) h[s] = 0.0f;
    if (has) {
      for (int j = 0; j < seg; ++j) {
        const int64_t at = ((int64_t)b * a.segments + j) * a.channels + c0 + ch;
        const float2 dec = a.seg_decay[at];
        const bool keeps = j > 0 && dec.y != 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const int n = s * LPC + q;
          if (n < a.dstate) h[s] = (keeps ? ex2_approx(A2[s] * dec.x) * h[s] : 0.0f) + a.seg_state[at * a.dstate + n];
        }
      }
    }
  }
  float sum_dt = 0.0f;
  bool dropped = false;

  Pack<T, EV> xr, zr;
  float dr[EV];
  Pack<T, 4> bc[kAhead ? NS : 1];
  const auto load_bc = [&](int k, int t0) {
    const int item = k * NT + tid;
    const bool is_c = item >= kTile * NP / 4;
    const int r = is_c ? item - kTile * NP / 4 : item;
    const int t = t0 + r / (NP / 4), n = (r % (NP / 4)) * 4;
    const T* p = is_c ? Cp + (int64_t)t * a.C_sl : Bp + (int64_t)t * a.B_sl;
    const bool want = t < t_end && !(STATE && is_c);
    return load_some<4>(p + n, want ? a.dstate - n : 0, a.vec_bc);
  };
  const auto store_bc = [&](int k, const Pack<T, 4>& v) {
    const int item = k * NT + tid;
    const bool is_c = item >= kTile * NP / 4;
    const int r = is_c ? item - kTile * NP / 4 : item;
    const int t = r / (NP / 4), n = (r % (NP / 4)) * 4;
    float* s = is_c ? s_C : s_B;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[(n + i) * kLd + t] = widen(v.e[i]);
  };
  const auto fetch = [&](int t0) {
    const int t = t0 + lt;
    const int count = t < t_end ? lcount : 0;
    xr = load_some<EV>(xp + (int64_t)t * a.x_sl, count, a.vec);
    if (a.dt_f32) {
      const Pack<float, EV> r = load_some<EV>(static_cast<const float*>(a.dt) + dt_off + (int64_t)t * a.dt_sl, count, a.vec);
#pragma unroll
      for (int e = 0; e < EV; ++e) dr[e] = r.e[e];
    } else {
      const Pack<T, EV> r = load_some<EV>(static_cast<const T*>(a.dt) + dt_off + (int64_t)t * a.dt_sl, count, a.vec);
#pragma unroll
      for (int e = 0; e < EV; ++e) dr[e] = widen(r.e[e]);
    }
    if (!STATE && a.z) zr = load_some<EV>(zp + (int64_t)t * a.z_sl, count, a.vec);
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < NS; ++k) bc[k] = load_bc(k, t0);
    }
  };

  fetch(t_begin);
  for (int t0 = t_begin; t0 < t_end; t0 += kTile) {
    // positions past the end get dt' = 0 and x = B = C = 0: they leave the state as it is
    const int count = t0 + lt < t_end ? lcount : 0;
    float xv[EV];
    Pack<T, EV> zv = zr;
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      xv[e] = widen(xr.e[e]);
      const float d = e < count ? scan_dt(dr[e] + bv[e], a.softplus, a.dt_min, a.dt_max) : 0.0f;
      s_d[(lc + e) * kLd + lt] = d;
      s_u[(lc + e) * kLd + lt] = d * xv[e];
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < NS; ++k) store_bc(k, bc[k]);
    } else {
#pragma unroll 4
      for (int k = 0; k < NS; ++k) store_bc(k, load_bc(k, t0));
    }
    const uint32_t resets = a.seq ? reset_mask(a, b, t0, tid & 31) : 0u;
    __syncthreads();
    if (t0 + kTile < t_end) fetch(t0 + kTile);

    const int stop = min(kTile, t_end - t0);
    for (int t = 0; t < stop; t += 4) {
      if (!STATE && a.ckpt && (t & (SSD_TOKEN_SCAN_CHECKPOINT - 1)) == 0 && has) {
        const int64_t nck = (a.seqlen + SSD_TOKEN_SCAN_CHECKPOINT - 1) / SSD_TOKEN_SCAN_CHECKPOINT;
        float* dst = a.ckpt + (((int64_t)b * nck + (t0 + t) / SSD_TOKEN_SCAN_CHECKPOINT) * a.channels + c0 + ch) * a.dstate;
#pragma unroll
        for (int s = 0; s < NS; ++s)
          if (s * LPC + q < a.dstate) dst[s * LPC + q] = h[s];
      }
      const float4 d4 = *reinterpret_cast<const float4*>(&s_d[ch * kLd + t]);
      const float4 u4 = *reinterpret_cast<const float4*>(&s_u[ch * kLd + t]);
      const float d[4] = {d4.x, d4.y, d4.z, d4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const uint32_t r4 = (resets >> t) & 15u;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const float4 B4 = *reinterpret_cast<const float4*>(&s_B[(s * LPC + q) * kLd + t]);
        const float Bv[4] = {B4.x, B4.y, B4.z, B4.w};
        float Cv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!STATE) {
          const float4 C4 = *reinterpret_cast<const float4*>(&s_C[(s * LPC + q) * kLd + t]);
          Cv[0] = C4.x, Cv[1] = C4.y, Cv[2] = C4.z, Cv[3] = C4.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (r4 >> i & 1u) h[s] = 0.0f;
          h[s] = fmaf(ex2_approx(d[i] * A2[s]), h[s], u[i] * Bv[i]);
          if (!STATE) y[i] = fmaf(h[s], Cv[i], y[i]);
        }
      }
      if (STATE) {
        sum_dt += (d[0] + d[1]) + (d[2] + d[3]);
        dropped |= r4 != 0u;
      } else {
        // four sums over the channel's lanes: lanes trade halves until each of four holds one position
        const bool odd = q & 1, high = q & 2;
        float y01 = odd ? y[1] : y[0], y23 = odd ? y[3] : y[2];
        y01 += __shfl_xor_sync(0xffffffffu, odd ? y[0] : y[1], 1);
        y23 += __shfl_xor_sync(0xffffffffu, odd ? y[2] : y[3], 1);
        float r = high ? y23 : y01;
        r += __shfl_xor_sync(0xffffffffu, high ? y01 : y23, 2);
#pragma unroll
        for (int off = 4; off < LPC; off <<= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
        if (q < 4) s_y[ch * kLd + t + q] = r;
      }
    }
    __syncthreads();
    if (!STATE && count > 0) {
      const int64_t at = ((int64_t)b * a.seqlen + t0 + lt) * a.channels + c0 + lc;
      float o[EV];
#pragma unroll
      for (int e = 0; e < EV; ++e) o[e] = s_y[(lc + e) * kLd + lt] + dv[e] * xv[e];
      if (a.z) {
        if (a.out_x) store_some<EV>(static_cast<T*>(a.out_x) + at, o, count, a.vec);
#pragma unroll
        for (int e = 0; e < EV; ++e) o[e] *= silu_f(widen(zv.e[e]));
      }
      store_some<EV>(static_cast<T*>(a.out) + at, o, count, a.vec);
    }
  }

  if (!has) return;
  float* dst = STATE ? a.seg_state + (((int64_t)b * a.segments + seg) * a.channels + c0 + ch) * a.dstate
                     : a.final_states + ((int64_t)b * a.channels + c0 + ch) * a.dstate;
  if (STATE || t_end == a.seqlen) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
      if (s * LPC + q < a.dstate) dst[s * LPC + q] = h[s];
  }
  if (STATE && q == 0) a.seg_decay[((int64_t)b * a.segments + seg) * a.channels + c0 + ch] = make_float2(sum_dt, dropped ? 0.0f : 1.0f);
}

// How a problem is laid out over the GPU.
struct ScanPlan {
  int lpc, ns, tiles_per_group, segments, seg_len;
};

ScanPlan plan_scan(const ssd_token_scan_params_t& p) {
  ScanPlan s;
  const int per_group = p.channels / p.ngroups;
  s.tiles_per_group = (per_group + kCh - 1) / kCh;
  const int64_t blocks = (int64_t)p.batch * p.ngroups * s.tiles_per_group;
  // lanes per channel: more lanes give more threads, fewer lanes fewer exchanges and a smaller share of
  // per-tile work; the fewest that leave each scheduler two warps
  const int n = p.dstate <= 8 ? 8 : p.dstate <= 16 ? 16 : p.dstate <= 32 ? 32 : p.dstate <= 64 ? 64 : p.dstate <= 128 ? 128 : 256;
  s.lpc = n <= 16 ? 4 : n <= 32 ? 8 : 16;
  const int most = n < 16 ? n : 16;
  while (s.lpc < most && blocks * s.lpc / 2 < 148 * 8) s.lpc *= 2;
  s.ns = n / s.lpc;
  // segments: only where the blocks leave most of the GPU idle, and none shorter than 256 positions
  s.segments = 1;
  const int64_t warps = blocks * s.lpc / 2;
  if (warps < 148 * 4) {
    const int64_t want = (148 * 12 + warps - 1) / warps, room = p.seqlen / 256;
    s.segments = (int)(want < room ? want : room);
    if (s.segments > 128) s.segments = 128;
    if (s.segments < 3) s.segments = 1;          // the state pass doubles the work
  }
  s.seg_len = ((p.seqlen + s.segments - 1) / s.segments + kTile - 1) / kTile * kTile;
  s.segments = (p.seqlen + s.seg_len - 1) / s.seg_len;
  return s;
}

template <typename T, int LPC, int NS>
int launch_plan(const ScanArgs& a, int batch, cudaStream_t stream) {
  const size_t smem = (3 * kCh + 2 * LPC * NS) * kLd * sizeof(float);
  dim3 grid(a.ngroups * a.tiles_per_group, a.segments, batch);
  if (smem > 48 * 1024) {
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_kernel<T, LPC, NS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_kernel<T, LPC, NS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  }
  if (a.segments > 1) {
    grid.y = a.segments - 1;                     // nothing starts from the last segment's state
    token_scan_kernel<T, LPC, NS, true><<<grid, kCh * LPC, smem, stream>>>(a);
    SSD_CUDA_OK(cudaGetLastError());
    grid.y = a.segments;
  }
  token_scan_kernel<T, LPC, NS, false><<<grid, kCh * LPC, smem, stream>>>(a);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

size_t seg_state_bytes(const ssd_token_scan_params_t& p, const ScanPlan& s) {
  return s.segments > 1 ? (size_t)p.batch * s.segments * p.channels * p.dstate * sizeof(float) : 0;
}

}  // namespace

ScanArgs scan_args(const ssd_token_scan_params_t& p) {
  ScanArgs a;
  a.x = p.x, a.dt = p.dt, a.A = p.A, a.B = p.B, a.C = p.C, a.D = p.D, a.z = p.z;
  a.bias = p.dt_bias, a.init = p.initial_states, a.seq = p.seq_idx;
  a.out = p.out, a.out_x = p.out_x, a.final_states = p.final_states, a.ckpt = p.checkpoints;
  a.seg_state = nullptr, a.seg_decay = nullptr;
  a.dt_f32 = p.dt_dtype == SSD_F32;
  a.A_dtype = p.A_dtype, a.D_dtype = p.D_dtype, a.bias_dtype = p.bias_dtype, a.init_dtype = p.init_dtype;
  a.seqlen = p.seqlen, a.channels = p.channels, a.ngroups = p.ngroups, a.dstate = p.dstate;
  a.per_group = p.channels / p.ngroups, a.tiles_per_group = 0;
  a.softplus = p.dt_softplus, a.dt_min = p.dt_min, a.dt_max = p.dt_max;
  a.x_sb = p.x_stride[0], a.x_sl = p.x_stride[1];
  a.dt_sb = p.dt_stride[0], a.dt_sl = p.dt_stride[1];
  a.z_sb = p.z_stride[0], a.z_sl = p.z_stride[1];
  a.B_sb = p.B_stride[0], a.B_sl = p.B_stride[1], a.B_sg = p.B_stride[2];
  a.C_sb = p.C_stride[0], a.C_sl = p.C_stride[1], a.C_sg = p.C_stride[2];
  a.s_sb = p.seq_idx_stride[0], a.s_sl = p.seq_idx_stride[1];
  const int es = dtype_size(p.x_dtype), ds = dtype_size(p.dt_dtype);
  // a thread's vector of channels begins at a multiple of its own length within the group: aligned if
  // groups and rows are aligned to 16 bytes of the type
  a.vec = a.per_group % (16 / es) == 0 && p.channels % (16 / es) == 0 && rows_aligned(p.x, p.x_stride, 2, es, 16) &&
          rows_aligned(p.dt, p.dt_stride, 2, ds, 16) && (p.z == nullptr || rows_aligned(p.z, p.z_stride, 2, es, 16)) &&
          aligned_to(p.out, 16) && aligned_to(p.out_x, 16);
  a.vec_bc = p.dstate % 4 == 0 && rows_aligned(p.B, p.B_stride, 3, es, 4 * es) && rows_aligned(p.C, p.C_stride, 3, es, 4 * es);
  a.seg_len = p.seqlen, a.segments = 1;
  return a;
}

size_t token_scan_workspace(const ssd_token_scan_params_t& p) {
  const ScanPlan s = plan_scan(p);
  return s.segments > 1 ? seg_state_bytes(p, s) + (size_t)p.batch * s.segments * p.channels * sizeof(float2) + 16 : 0;
}

int launch_token_scan(const ssd_token_scan_params_t& p, cudaStream_t stream) {
  const ScanPlan s = plan_scan(p);
  ScanArgs a = scan_args(p);
  a.tiles_per_group = s.tiles_per_group;
  a.segments = s.segments;
  a.seg_len = s.seg_len;
  if (s.segments > 1) {
    a.seg_state = static_cast<float*>(p.workspace);
    a.seg_decay = reinterpret_cast<float2*>(static_cast<char*>(p.workspace) + (seg_state_bytes(p, s) + 15) / 16 * 16);
  }
  SSD_REQUIRE(p.batch <= 65535, SSD_ERR_UNSUPPORTED, "token scan: batch %d too large", p.batch);
  return with_type(p.x_dtype, [&](auto t) -> int {
    using T = decltype(t);
    switch (s.lpc * 1000 + s.ns) {
      case 4002: return launch_plan<T, 4, 2>(a, p.batch, stream);
      case 8001: return launch_plan<T, 8, 1>(a, p.batch, stream);
      case 4004: return launch_plan<T, 4, 4>(a, p.batch, stream);
      case 8002: return launch_plan<T, 8, 2>(a, p.batch, stream);
      case 16001: return launch_plan<T, 16, 1>(a, p.batch, stream);
      case 8004: return launch_plan<T, 8, 4>(a, p.batch, stream);
      case 16002: return launch_plan<T, 16, 2>(a, p.batch, stream);
      case 16004: return launch_plan<T, 16, 4>(a, p.batch, stream);
      case 16008: return launch_plan<T, 16, 8>(a, p.batch, stream);
      default: return launch_plan<T, 16, 16>(a, p.batch, stream);
    }
  });
}

}  // namespace ssd
