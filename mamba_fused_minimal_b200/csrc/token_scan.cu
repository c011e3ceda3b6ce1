// Selective scan, position by position: h[n] = a h[n] + dt' x B[n], a = exp(dt' A[n]), y = C . h + D x.
//
// Each (position, channel, component) needs one exponential and four multiply-adds, and nothing of it can
// be shared between channels, so at dstate 16 the special function units (16 exponentials per clock and
// SM) bound the kernel, ahead of memory (x, dt, z and out once).  A thread holds NS components of K
// channels' states in registers and LPC adjacent lanes share a channel: the recurrence along the positions
// never leaves a thread, and only y is summed over the LPC lanes.
//
// A block takes 16 channels and walks the positions in tiles of 32.  dt' is formed once per position and
// channel and put beside dt' x in shared memory, B and C are widened there.  What a lane reads back per
// component and position has to pass the shared memory's 128 bytes a clock whether it is broadcast or not;
// K = 2 channels per thread share each B and C.  The multiply-adds work on pairs of components (packed
// fp32), which halves their issue slots.
//
// Few channels and a long sequence: the sequence is cut into segments that run side by side.  A first pass
// leaves each segment's state from a zero start and the sum of its dt'; since the decay over a segment is
// exp(A * sum dt'), the second pass's blocks form the state they start from by themselves.  The
// exponentials are computed twice, so this is done only where the GPU would otherwise stand idle.
#include "token_scan.cuh"

#ifndef SSD_SCAN_K
#define SSD_SCAN_K 1
#endif
#ifndef SSD_SCAN_UNROLL
#define SSD_SCAN_UNROLL 1
#endif

namespace ssd {
namespace {

constexpr int kUnroll = SSD_SCAN_UNROLL;
constexpr int kCh = 16;            // channels of a block
constexpr int kTile = 32;          // positions of a tile
constexpr int kLdu = 2 * kTile + 4;   // row pitches in shared memory: a channel's rows start in different banks
constexpr int kLdy = 4 * kTile + 4;

constexpr int kHelpers = 64;       // threads that load, prepare and store
constexpr int kVec = kTile * kCh / kHelpers;   // elements of x such a thread loads per tile
constexpr int kPerRow = kCh / kVec;            // such vectors per position

// LPC lanes share a channel, a thread holds NS components of K channels.
template <int LPC, int NS, int K>
struct ScanShape {
  static constexpr int kCompute = kCh * LPC / K;      // threads that hold states
  static constexpr int kThreads = kCompute + kHelpers;
  static constexpr int kState = LPC * NS;             // components, padded
  static constexpr int kChunk = NS < 4 ? NS : 4;      // components that are read together
  static constexpr int kGroups = NS / kChunk;
  static constexpr int kRow = 2 * kState;             // a position's B and C
  static constexpr int kItems = 2 * kTile * kState / kChunk;   // chunks of a tile's B and C
  static constexpr int kPer = kItems / kHelpers;
  static constexpr bool kAhead = kPer <= 16;          // B and C of the next tile wait in registers, too
  static constexpr int kStage = kCh * (kLdu + kLdy) + kTile * kRow;   // floats of a tile in shared memory
  static constexpr size_t kSmem = 2 * sizeof(float) * kStage;
  // blocks an SM should hold: what leaves each thread about 100 registers
  static constexpr int kResident = kThreads <= 128 ? 5 : kThreads <= 192 ? 3 : 1;
};

// Named barriers FIRST and FIRST + 1, one for each stage: COUNT threads meet, of which some only leave word
// (arrive) and go on.  The numbers are constants: with computed ones the block would claim all sixteen
// barriers, and an SM has enough for four such blocks.
template <int FIRST, int COUNT>
__device__ __forceinline__ void bar_sync(int stage) {
  if (stage == 0)
    asm volatile("bar.sync %0, %1;" ::"n"(FIRST), "n"(COUNT) : "memory");
  else
    asm volatile("bar.sync %0, %1;" ::"n"(FIRST + 1), "n"(COUNT) : "memory");
}
template <int FIRST, int COUNT>
__device__ __forceinline__ void bar_arrive(int stage) {
  if (stage == 0)
    asm volatile("bar.arrive %0, %1;" ::"n"(FIRST), "n"(COUNT) : "memory");
  else
    asm volatile("bar.arrive %0, %1;" ::"n"(FIRST + 1), "n"(COUNT) : "memory");
}

template <typename T, int LPC, int NS, int K, bool STATE, bool VEC>
__global__ void __launch_bounds__(ScanShape<LPC, NS, K>::kThreads, ScanShape<LPC, NS, K>::kResident) token_scan_kernel(ScanArgs a) {
  using Sh = ScanShape<LPC, NS, K>;
  constexpr int NT = Sh::kThreads, EV = kVec, CB = Sh::kChunk, GR = Sh::kGroups, CK = kCh / K;
  extern __shared__ float4 smem4[];
  // a stage: du [kCh][kLdu], (dt', dt' x) of each position; y [kCh][kLdy], four shares of y of each
  // position; bc [kTile][GR][LPC][B: CB, C: CB]
  float* const s_stage = reinterpret_cast<float*>(smem4);
  const int g = blockIdx.x / a.tiles_per_group, tile_c = blockIdx.x % a.tiles_per_group;
  const int b = blockIdx.z, seg = blockIdx.y;
  const int c0 = g * a.per_group + tile_c * kCh;                     // first channel of the block
  const int nch = min(kCh, a.per_group - tile_c * kCh);
  const int t_begin = seg * a.seg_len, t_end = min(a.seqlen, t_begin + a.seg_len);

  const int tiles = (t_end - t_begin + kTile - 1) / kTile;
  // The two kinds of threads meet twice a tile: barrier 1 + stage when the tile is prepared, barrier 3 + stage
  // when it is computed.  The helpers prepare tile i + 2 only after they have stored tile i, so a stage is
  // never written while it is read.
  if (threadIdx.x >= Sh::kCompute) {
    const int tid = threadIdx.x - Sh::kCompute;
    // what this thread loads and stores: EV channels of one position
    const int lt = tid / kPerRow, lc = (tid % kPerRow) * EV;
    const int lcount = max(0, min(EV, nch - lc));
    const int lfrom = c0 + (lcount > 0 ? lc : 0);
    const T* xp = static_cast<const T*>(a.x) + b * a.x_sb + lfrom;
    const T* zp = static_cast<const T*>(a.z) + b * a.z_sb + lfrom;
    const int64_t dt_off = b * a.dt_sb + lfrom;
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_sb + g * a.B_sg;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_sb + g * a.C_sg;
    float dv[EV], bv[EV];
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      dv[e] = a.D && e < lcount ? load_f(a.D, a.D_dtype, c0 + lc + e) : 0.0f;
      bv[e] = a.bias && e < lcount ? load_f(a.bias, a.bias_dtype, c0 + lc + e) : 0.0f;
    }

    Pack<T, EV> xr, dr16;
    Pack<float, EV> dr32;
    Pack<T, CB> bcr[Sh::kAhead ? Sh::kPer : 1];
    // chunk k of this thread of the tile's B and C: CB components of one position
    const auto load_bc = [&](int k, int t0) {
      const int item = k * kHelpers + tid;
      const int n = item % (GR * LPC) * CB, tb = min(t0 + item / (GR * LPC) % kTile, t_end - 1);
      const T* src = item >= Sh::kItems / 2 ? Cp + (int64_t)tb * a.C_sl : Bp + (int64_t)tb * a.B_sl;
      if constexpr (VEC)
        return load_some<CB, true>(src + (n < a.dstate ? n : 0), CB);
      else
        return load_some<CB, false>(src + n, a.dstate - n);
    };
    const auto place_bc = [&](float* s_bc, int k, const Pack<T, CB>& r) {
      const int item = k * kHelpers + tid;
      const int gl = item % (GR * LPC), t = item / (GR * LPC) % kTile;
      const int lane = gl / GR, grp = gl % GR;                       // component gl * CB = lane * NS + grp * CB
      float v[CB];
#pragma unroll
      for (int i = 0; i < CB; ++i) v[i] = gl * CB + i < a.dstate ? widen(r.e[i]) : 0.0f;
      store_vec<CB>(s_bc + t * Sh::kRow + (grp * LPC + lane) * 2 * CB + (item >= Sh::kItems / 2 ? CB : 0), v);
    };
    // The next tile's values, left as they are loaded.  Positions past the end read the last one's, channels
    // past the group's the first one's; what is made of them is masked.
    const auto fetch = [&](int t0) {
      const int t = min(t0 + lt, t_end - 1), count = lcount;
      xr = load_some<EV, VEC>(xp + (int64_t)t * a.x_sl, count);
      if (a.dt_f32)
        dr32 = load_some<EV, VEC>(static_cast<const float*>(a.dt) + dt_off + (int64_t)t * a.dt_sl, count);
      else
        dr16 = load_some<EV, VEC>(static_cast<const T*>(a.dt) + dt_off + (int64_t)t * a.dt_sl, count);
      if constexpr (Sh::kAhead) {
#pragma unroll
        for (int k = 0; k < Sh::kPer; ++k)
          if (!STATE || k * kHelpers < Sh::kItems / 2) bcr[k] = load_bc(k, t0);
      }
    };
    const auto prepare = [&](int i) {
      float* const s_du = s_stage + (i & 1) * Sh::kStage;
      // positions past the end get dt' = dt' x = 0: they leave the state as it is
      const int count = t_begin + i * kTile + lt < t_end ? lcount : 0;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float raw = (a.dt_f32 ? dr32.e[e] : widen(dr16.e[e])) + bv[e];
        const float d = e < count ? scan_dt(raw, a.softplus, a.dt_min, a.dt_max) : 0.0f;
        const float u = e < count ? d * widen(xr.e[e]) : 0.0f;
        *reinterpret_cast<float2*>(&s_du[(lc + e) * kLdu + 2 * lt]) = make_float2(d, u);
      }
      float* const s_bc = s_du + kCh * (kLdu + kLdy);
      constexpr int kMine = STATE ? Sh::kPer / 2 : Sh::kPer;         // the second half is C
      if constexpr (Sh::kAhead) {
#pragma unroll
        for (int k = 0; k < kMine; ++k) place_bc(s_bc, k, bcr[k]);
      } else {
#pragma unroll 8
        for (int k = 0; k < kMine; ++k) place_bc(s_bc, k, load_bc(k, t_begin + i * kTile));
      }
      bar_arrive<1, NT>(i & 1);
    };
    fetch(t_begin);
    prepare(0);
    if (tiles > 1) fetch(t_begin + kTile);
    for (int i = 0; i < tiles; ++i) {
      const int t0 = t_begin + i * kTile;
      if (i + 1 < tiles) prepare(i + 1);
      if (i + 2 < tiles) fetch(t0 + 2 * kTile);
      // x and z of the tile whose y is awaited, read (again) while it is computed
      Pack<T, EV> xk, zk;
      if (!STATE) {
        const int t = min(t0 + lt, t_end - 1);
        xk = load_some<EV, VEC>(xp + (int64_t)t * a.x_sl, lcount);
        if (a.z) zk = load_some<EV, VEC>(zp + (int64_t)t * a.z_sl, lcount);
      }
      bar_sync<3, NT>(i & 1);
      const int count = t0 + lt < t_end ? lcount : 0;
      if (!STATE && count > 0) {
        const float* s_y = s_stage + (i & 1) * Sh::kStage + kCh * kLdu;
        const int64_t at = ((int64_t)b * a.seqlen + t0 + lt) * a.channels + c0 + lc;
        float o[EV];
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const float4 y4 = *reinterpret_cast<const float4*>(&s_y[(lc + e) * kLdy + 4 * lt]);
          o[e] = fmaf(dv[e], widen(xk.e[e]), (y4.x + y4.y) + (y4.z + y4.w));
        }
        if (a.z) {
          if (a.out_x) store_some<EV, VEC>(static_cast<T*>(a.out_x) + at, o, count);
#pragma unroll
          for (int e = 0; e < EV; ++e) o[e] *= silu_f(widen(zk.e[e]));
        }
        store_some<EV, VEC>(static_cast<T*>(a.out) + at, o, count);
      }
    }
    return;
  }

  const int tid = threadIdx.x;
  // what this thread computes: components n0 .. n0 + NS - 1, in pairs, of channels ch, ch + CK, ...
  const int q = tid % LPC, ch = tid / LPC;
  const int n0 = q * NS;
  const int64_t state_at = ((int64_t)b * a.channels + c0 + ch) * a.dstate + n0;
  f32x2 A2[K][NS / 2], h[K][NS / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int s = 0; s < NS; s += 2) {
      float A[2], v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = ch + k * CK < nch && n0 + s + i < a.dstate;
        const int64_t at = (int64_t)k * CK * a.dstate + s + i;
        A[i] = in ? load_f(a.A, a.A_dtype, (int64_t)(c0 + ch) * a.dstate + n0 + at) * kLog2e : 0.0f;
        v[i] = in && a.init && seg == 0 ? load_f(a.init, a.init_dtype, state_at + at) : 0.0f;
      }
      A2[k][s / 2] = pack2(A[0], A[1]);
      h[k][s / 2] = pack2(v[0], v[1]);
    }
  }
  // the states of the thread's channels into an array (..., channels, dstate) whose element of the block's
  // first channel is at `base`
  const auto store_state = [&](float* base) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ch + k * CK >= nch) continue;
      float* dst = base + (int64_t)(ch + k * CK) * a.dstate + n0;
#pragma unroll
      for (int s = 0; s < NS; s += 2) {
        float v[2];
        unpack2(h[k][s / 2], v[0], v[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (n0 + s + i < a.dstate) dst[s + i] = v[i];
      }
    }
  };
  if (!STATE && seg > 0) {
    // the state this segment starts from: what the earlier ones leave, in order (the first of them
    // started from the initial state)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ch + k * CK >= nch) continue;
      for (int j = 0; j < seg; ++j) {
        const int64_t at = ((int64_t)b * a.segments + j) * a.channels + c0 + ch + k * CK;
        const float2 dec = a.seg_decay[at];
        const bool keeps = j > 0 && dec.y != 0.0f;
#pragma unroll
        for (int s = 0; s < NS; s += 2) {
          float A[2], v[2];
          unpack2(A2[k][s / 2], A[0], A[1]);
          unpack2(h[k][s / 2], v[0], v[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (n0 + s + i < a.dstate) v[i] = (keeps ? ex2_approx(A[i] * dec.x) * v[i] : 0.0f) + a.seg_state[at * a.dstate + n0 + s + i];
          }
          h[k][s / 2] = pack2(v[0], v[1]);
        }
      }
    }
  }
  float sum_dt[K];
#pragma unroll
  for (int k = 0; k < K; ++k) sum_dt[k] = 0.0f;
  bool dropped = false;

  // four positions of the tile; RESET: `r4` says which of them drop the state before
  const auto four = [&](int t, const float* s_du, const float* s_bc, float* s_y, auto reset, uint32_t r4) {
    constexpr bool RESET = decltype(reset)::value;
    float d[K][4], u[K][4], y[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* du = &s_du[(ch + k * CK) * kLdu + 2 * t];
      const float4 lo = *reinterpret_cast<const float4*>(du), hi = *reinterpret_cast<const float4*>(du + 4);
      d[k][0] = lo.x, u[k][0] = lo.y, d[k][1] = lo.z, u[k][1] = lo.w;
      d[k][2] = hi.x, u[k][2] = hi.y, d[k][3] = hi.z, u[k][3] = hi.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 y2[K];
#pragma unroll
      for (int m = 0; m < GR; ++m) {
        const float* row = s_bc + (t + i) * Sh::kRow + (m * LPC + q) * 2 * CB;
        f32x2 Bv[CB / 2], Cv[CB / 2];
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(row);
        Bv[0] = v.x;
        if constexpr (CB == 2) {
          Cv[0] = v.y;
        } else {
          Bv[1] = v.y;
          if (!STATE) {
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(row + CB);
            Cv[0] = w.x, Cv[1] = w.y;
          }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const f32x2 dd = pack2(d[k][i], d[k][i]), uu = pack2(u[k][i], u[k][i]);
#pragma unroll
          for (int s = 0; s < CB / 2; ++s) {
            const int at = m * (CB / 2) + s;
            f32x2& hh = h[k][at];
            if (RESET && (r4 >> i & 1u)) hh = 0;
            float e0, e1;
            unpack2(mul2(dd, A2[k][at]), e0, e1);
            hh = fma2(pack2(ex2_approx(e0), ex2_approx(e1)), hh, mul2(uu, Bv[s]));
            if (!STATE) y2[k] = at == 0 ? mul2(hh, Cv[s]) : fma2(hh, Cv[s], y2[k]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (STATE) {
          sum_dt[k] += d[k][i];
        } else {
          float lo, hi;
          unpack2(y2[k], lo, hi);
          y[k][i] = lo + hi;
        }
      }
    }
    if (STATE) return;
    // y is summed over the channel's lanes: lanes beyond four trade halves until four shares are left, which
    // go to shared memory and are added where y is used
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float* dst = &s_y[(ch + k * CK) * kLdy + 4 * t + (q & 3)];
      if constexpr (LPC == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[4 * i] = y[k][i];
      } else {
        const bool b2 = q & 4;
        float y0 = b2 ? y[k][1] : y[k][0], y1 = b2 ? y[k][3] : y[k][2];
        y0 += __shfl_xor_sync(0xffffffffu, b2 ? y[k][0] : y[k][1], 4);
        y1 += __shfl_xor_sync(0xffffffffu, b2 ? y[k][2] : y[k][3], 4);
        if constexpr (LPC == 8) {
          dst[b2 ? 4 : 0] = y0;
          dst[b2 ? 12 : 8] = y1;
        } else {
          const bool b3 = q & 8;
          float r = b3 ? y1 : y0;
          r += __shfl_xor_sync(0xffffffffu, b3 ? y0 : y1, 8);
          dst[(b2 ? 4 : 0) + (b3 ? 8 : 0)] = r;
        }
      }
    }
  };

  for (int i = 0; i < tiles; ++i) {
    const int t0 = t_begin + i * kTile;
    const float* const s_du = s_stage + (i & 1) * Sh::kStage;
    float* const s_y = s_stage + (i & 1) * Sh::kStage + kCh * kLdu;
    const float* const s_bc = s_y + kCh * kLdy;
    const uint32_t resets = a.seq ? reset_mask(a, b, t0, tid & 31) : 0u;
    bar_sync<1, NT>(i & 1);
    const int stop = min(kTile, t_end - t0);
    for (int half = 0; half < stop; half += SSD_TOKEN_SCAN_CHECKPOINT) {
      if (!STATE && a.ckpt) {
        const int64_t nck = (a.seqlen + SSD_TOKEN_SCAN_CHECKPOINT - 1) / SSD_TOKEN_SCAN_CHECKPOINT;
        store_state(a.ckpt + (((int64_t)b * nck + (t0 + half) / SSD_TOKEN_SCAN_CHECKPOINT) * a.channels + c0) * a.dstate);
      }
      const int end = min(stop, half + SSD_TOKEN_SCAN_CHECKPOINT);
      if (resets == 0u) {
#pragma unroll kUnroll
        for (int t = half; t < end; t += 4) four(t, s_du, s_bc, s_y, std::false_type(), 0u);
      } else {
#pragma unroll 1
        for (int t = half; t < end; t += 4) four(t, s_du, s_bc, s_y, std::true_type(), resets >> t);
      }
    }
    if (STATE) dropped |= resets != 0u;
    bar_arrive<3, NT>(i & 1);
  }

  if (STATE) {
    const int64_t at = ((int64_t)b * a.segments + seg) * a.channels + c0;
    store_state(a.seg_state + at * a.dstate);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (q == 0 && ch + k * CK < nch) a.seg_decay[at + ch + k * CK] = make_float2(sum_dt[k], dropped ? 0.0f : 1.0f);
  } else if (t_end == a.seqlen) {
    store_state(a.final_states + ((int64_t)b * a.channels + c0) * a.dstate);
  }
}

// How a problem is laid out over the GPU.
struct ScanPlan {
  int lpc, ns, k, tiles_per_group, segments, seg_len;
};

ScanPlan plan_scan(const ssd_token_scan_params_t& p) {
  ScanPlan s;
  const int per_group = p.channels / p.ngroups;
  s.tiles_per_group = (per_group + kCh - 1) / kCh;
  const int64_t blocks = (int64_t)p.batch * p.ngroups * s.tiles_per_group;
  const int n = p.dstate <= 8 ? 8 : p.dstate <= 16 ? 16 : p.dstate <= 32 ? 32 : p.dstate <= 64 ? 64 : p.dstate <= 128 ? 128 : 256;
  s.lpc = n <= 16 ? 4 : n <= 32 ? 8 : 16;
  s.k = SSD_SCAN_K;
  s.ns = n / s.lpc;
  // segments: only where the blocks leave most of the GPU idle, and none shorter than 256 positions
  s.segments = 1;
  const int64_t warps = blocks * s.lpc / (2 * s.k);
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

template <typename T, int LPC, int NS, int K, bool VEC>
int launch_vec(const ScanArgs& a, int batch, cudaStream_t stream) {
  using Sh = ScanShape<LPC, NS, K>;
  constexpr size_t smem = Sh::kSmem;
  dim3 grid(a.ngroups * a.tiles_per_group, a.segments, batch);
  if (smem > 48 * 1024) {
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_kernel<T, LPC, NS, K, false, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_kernel<T, LPC, NS, K, true, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  }
  if (a.segments > 1) {
    grid.y = a.segments - 1;                     // nothing starts from the last segment's state
    token_scan_kernel<T, LPC, NS, K, true, VEC><<<grid, Sh::kThreads, smem, stream>>>(a);
    SSD_CUDA_OK(cudaGetLastError());
    grid.y = a.segments;
  }
  token_scan_kernel<T, LPC, NS, K, false, VEC><<<grid, Sh::kThreads, smem, stream>>>(a);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

template <typename T, int LPC, int NS, int K>
int launch_plan(const ScanArgs& a, const ssd_token_scan_params_t& p, cudaStream_t stream) {
  using Sh = ScanShape<LPC, NS, K>;
  constexpr int CB = Sh::kChunk, EV = kVec;
  // a thread's vector of channels begins at a multiple of its length within a group
  constexpr size_t kMost = EV * sizeof(T) < 16 ? EV * sizeof(T) : 16;
  const int ds = dtype_size(p.dt_dtype);
  const size_t dt_most = EV * ds < 16 ? EV * ds : 16;
  const bool vec = a.per_group % EV == 0 && rows_aligned(p.x, p.x_stride, 2, sizeof(T), kMost) && rows_aligned(p.dt, p.dt_stride, 2, ds, dt_most) &&
                   (p.z == nullptr || rows_aligned(p.z, p.z_stride, 2, sizeof(T), kMost)) && aligned_to(p.out, kMost) && aligned_to(p.out_x, kMost) &&
                   p.dstate % CB == 0 && rows_aligned(p.B, p.B_stride, 3, sizeof(T), CB * sizeof(T)) &&
                   rows_aligned(p.C, p.C_stride, 3, sizeof(T), CB * sizeof(T));
  return vec ? launch_vec<T, LPC, NS, K, true>(a, p.batch, stream) : launch_vec<T, LPC, NS, K, false>(a, p.batch, stream);
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
    switch ((s.k * 100 + s.lpc) * 100 + s.ns) {
      case 10402: return launch_plan<T, 4, 2, 1>(a, p, stream);
      case 10404: return launch_plan<T, 4, 4, 1>(a, p, stream);
      case 10804: return launch_plan<T, 8, 4, 1>(a, p, stream);
      case 11604: return launch_plan<T, 16, 4, 1>(a, p, stream);
      case 11608: return launch_plan<T, 16, 8, 1>(a, p, stream);
      case 11616: return launch_plan<T, 16, 16, 1>(a, p, stream);
      case 20402: return launch_plan<T, 4, 2, 2>(a, p, stream);
      case 20404: return launch_plan<T, 4, 4, 2>(a, p, stream);
      case 20804: return launch_plan<T, 8, 4, 2>(a, p, stream);
      case 21604: return launch_plan<T, 16, 4, 2>(a, p, stream);
      case 21608: return launch_plan<T, 16, 8, 2>(a, p, stream);
      default: return launch_plan<T, 16, 16, 2>(a, p, stream);
    }
  });
}

}  // namespace ssd
