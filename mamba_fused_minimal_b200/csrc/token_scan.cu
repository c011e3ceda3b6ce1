// Selective scan, position by position: h[n] = a h[n] + dt' x B[n], a = exp(dt' A[n]), y = C . h + D x.
//
// Each (position, channel, component) needs one exponential and four multiply-adds, and nothing of it can
// be shared between channels, so at dstate 16 the special function units (16 exponentials per clock and
// SM) bound the kernel, ahead of memory (x, dt, z and out once).  A thread holds NS components of K
// channels' states in registers and LPC adjacent lanes share a channel: the recurrence along the positions
// never leaves a thread, and only y is summed over the LPC lanes.
//
// A block takes 16 channels and walks the positions in tiles of 32.  dt' is formed once per position and
// channel and put beside dt' x in shared memory, B and C are copied there as they are.  What a lane reads
// back per component and position has to pass the shared memory's 128 bytes a clock, broadcast or not,
// so 16-bit ones are widened in registers (1 x 65537 x 320 channels: 398 to 352 us).  The multiply-adds work on
// pairs of components (packed fp32), which halves their issue slots.
//
// The threads that hold the states do nothing else; two more warps load, form dt' and apply D and the gate, a
// tile ahead and a tile behind (594 to 443 us at 2 x 4096 x 5120 channels of 16).  Measured there: 363 to 367 us,
// against 186 us for its exponentials and 51 us for its bytes; issue slots, shared memory and exponentials are
// each a little over half used, and 640 blocks on 148 SMs leave 14 % of them idle at the end.
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
// Rows in shared memory, in floats: dt' and dt' x of a channel by position, and its four shares of y by
// position.  Eight channels' rows start four banks apart, and channels 8 to 15 sixteen banks further, so
// neither the threads that compute nor those that prepare meet in a bank.
constexpr int kLdu = kTile + 4, kDu = kCh * kLdu + 16;
constexpr int kLdy = 4 * kTile + 4, kY = kCh * kLdy + 16;
__device__ __forceinline__ int du_row(int ch) { return ch * kLdu + (ch >> 3) * 16; }
__device__ __forceinline__ int y_row(int ch) { return ch * kLdy + (ch >> 3) * 16; }

// Threads that load, prepare and store: twice as many where a position's B and C are longer (2048 channels of
// 128: 1764 us with 64).
constexpr int helpers(int lpc) { return lpc == 16 ? 128 : 64; }

constexpr int resident(int threads, int states) {
  return threads <= 128 ? 5 : threads <= 192 ? 3 : states <= 8 ? 2 : 1;
}

// LPC lanes share a channel, a thread holds NS components of K channels.
template <typename T, int LPC, int NS, int K>
struct ScanShape {
  static constexpr int kCompute = kCh * LPC / K;      // threads that hold states
  static constexpr int kHelpers = helpers(LPC);
  static constexpr int kVec = kTile * kCh / kHelpers; // elements of x a preparing thread loads per tile
  static constexpr int kPerRow = kCh / kVec;          // such threads per position
  static constexpr int kThreads = kCompute + kHelpers;
  static constexpr int kState = LPC * NS;             // components, padded
  static constexpr int kChunk = NS < 4 ? NS : 4;      // components that are read together
  static constexpr int kGroups = NS / kChunk;
  static constexpr int kRow = 2 * kState;             // a position's B and C
  static constexpr int kItems = 2 * kTile * kState / kChunk;   // chunks of a tile's B and C
  static constexpr int kPer = kItems / kHelpers;
  static constexpr bool kAhead = kPer <= 16;          // B and C of the next tile wait in registers, too
  static constexpr int kStage = 2 * kDu + kY + kTile * kRow * (int)sizeof(T) / 4;   // a tile in shared memory, in 4-byte words
  static constexpr size_t kSmem = 2 * sizeof(float) * kStage;
  // blocks an SM should hold, what leaves a thread the registers that its states need
  static constexpr int kResident = resident(kThreads, NS * K);
};

// CB components of B and CB of C that lie side by side in shared memory, as pairs of fp32
template <int CB, bool C>
__device__ __forceinline__ void load_bc_pairs(const float* p, f32x2 (&B)[CB / 2], f32x2 (&Cv)[CB / 2]) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  B[0] = v.x;
  if constexpr (CB == 2) {
    Cv[0] = v.y;
  } else {
    B[1] = v.y;
    if constexpr (C) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p + 4);
      Cv[0] = w.x, Cv[1] = w.y;
    }
  }
}
template <int CB, bool C, typename T>
__device__ __forceinline__ void load_bc_pairs(const T* p, f32x2 (&B)[CB / 2], f32x2 (&Cv)[CB / 2]) {
  const Pack<uint32_t, CB> w = *reinterpret_cast<const Pack<uint32_t, CB>*>(p);
#pragma unroll
  for (int i = 0; i < CB / 2; ++i) {
    B[i] = widen_pair<T>(w.e[i]);
    if constexpr (C) Cv[i] = widen_pair<T>(w.e[CB / 2 + i]);
  }
}

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
__global__ void __launch_bounds__(ScanShape<T, LPC, NS, K>::kThreads, ScanShape<T, LPC, NS, K>::kResident) token_scan_kernel(ScanArgs a) {
  using Sh = ScanShape<T, LPC, NS, K>;
  constexpr int NT = Sh::kThreads, EV = Sh::kVec, CB = Sh::kChunk, GR = Sh::kGroups, CK = kCh / K;
  extern __shared__ float4 smem4[];
  // a stage: dt' rows, dt' x rows, y rows, bc [kTile][GR][LPC][B: CB, C: CB]
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
    const int lt = tid / Sh::kPerRow, lc = (tid % Sh::kPerRow) * EV;
    const int lcount = max(0, min(EV, nch - lc));
    const int lfrom = c0 + (lcount > 0 ? lc : 0);
    const T* xp = static_cast<const T*>(a.x) + b * a.x_sb + lfrom;
    const T* zp = static_cast<const T*>(a.z) + b * a.z_sb + lfrom;
    const int64_t dt_off = b * a.dt_sb + lfrom;
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_sb + g * a.B_sg;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_sb + g * a.C_sg;
    f32x2 dv[EV / 2], bv[EV / 2];
#pragma unroll
    for (int e = 0; e < EV; e += 2) {
      float u[2], v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u[i] = a.D && e + i < lcount ? load_f(a.D, a.D_dtype, c0 + lc + e + i) : 0.0f;
        v[i] = a.bias && e + i < lcount ? load_f(a.bias, a.bias_dtype, c0 + lc + e + i) : 0.0f;
      }
      dv[e / 2] = pack2(u[0], u[1]);
      bv[e / 2] = pack2(v[0], v[1]);
    }

    Pack<T, EV> xr, dr16;
    Pack<float, EV> dr32;
    Pack<T, CB> bcr[Sh::kAhead ? Sh::kPer : 1];
    // Chunk k of this thread of a tile's B (first half) and C: CB components from `bn` on, of position
    // bt + a multiple of kStep.  A chunk's lane and group: component gl * CB = lane * NS + grp * CB.
    constexpr int kStep = Sh::kHelpers / (GR * LPC), kHalf = Sh::kPer / 2;
    const int gl = tid % (GR * LPC), bt = tid / (GR * LPC), bn = gl * CB;
    const bool bin = bn < a.dstate;
    const T* const Bt = Bp + (VEC && !bin ? 0 : bn);
    const T* const Ct = Cp + (VEC && !bin ? 0 : bn);
    const int bc_at = bt * Sh::kRow + (gl % GR * LPC + gl / GR) * 2 * CB;
    const auto load_bc = [&](int k, int t0) {
      const int t = min(t0 + bt + k % kHalf * kStep, t_end - 1);
      return load_some<CB, VEC>(k < kHalf ? Bt + t * a.B_sl : Ct + t * a.C_sl, a.dstate - bn);
    };
    const auto place_bc = [&](T* s_bc, int k, Pack<T, CB> r) {
      if (a.dstate < Sh::kState) {
#pragma unroll
        for (int i = 0; i < CB; ++i)
          if (bn + i >= a.dstate) r.e[i] = narrow<T>(0.0f);
      }
      *reinterpret_cast<Pack<T, CB>*>(s_bc + bc_at + k % kHalf * kStep * Sh::kRow + (k < kHalf ? 0 : CB)) = r;
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
          if (!STATE || k < kHalf) bcr[k] = load_bc(k, t0);
      }
    };
    const auto prepare = [&](int i) {
      float* const s_d = s_stage + (i & 1) * Sh::kStage + du_row(lc) + lt;
      if (t_begin + i * kTile + lt < t_end) {
        // the branches stand outside the loops: the pairs' chains of operations run side by side
        f32x2 d[EV / 2];
        if (a.dt_f32) {
#pragma unroll
          for (int e = 0; e < EV / 2; ++e) d[e] = add2(pair_of(dr32, e), bv[e]);
        } else {
#pragma unroll
          for (int e = 0; e < EV / 2; ++e) d[e] = add2(pair_of(dr16, e), bv[e]);
        }
        if (a.softplus) {
#pragma unroll
          for (int e = 0; e < EV / 2; ++e) d[e] = softplus2(d[e]);
        }
        if (a.limits) {
#pragma unroll
          for (int e = 0; e < EV / 2; ++e) {
            float v[2];
            unpack2(d[e], v[0], v[1]);
            d[e] = pack2(clamp_f(v[0], a.dt_min, a.dt_max), clamp_f(v[1], a.dt_min, a.dt_max));
          }
        }
#pragma unroll
        for (int e = 0; e < EV / 2; ++e) {
          float v[2], u[2];
          unpack2(d[e], v[0], v[1]);
          unpack2(mul2(d[e], pair_of(xr, e)), u[0], u[1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            s_d[(2 * e + k) * kLdu] = v[k];
            s_d[(2 * e + k) * kLdu + kDu] = u[k];
          }
        }
      } else {
        // positions past the end leave the state as it is
#pragma unroll
        for (int e = 0; e < EV; ++e) s_d[e * kLdu] = s_d[e * kLdu + kDu] = 0.0f;
      }
      T* const s_bc = reinterpret_cast<T*>(s_stage + (i & 1) * Sh::kStage + 2 * kDu + kY);
      constexpr int kMine = STATE ? kHalf : Sh::kPer;
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
    Pack<T, EV> xk = xr, xn = xr, zk;
    if (tiles > 1) fetch(t_begin + kTile);
    for (int i = 0; i < tiles; ++i, xk = xn) {
      const int t0 = t_begin + i * kTile;
      // z of the tile whose y is awaited, read before the next one is prepared
      if (!STATE && a.z) zk = load_some<EV, VEC>(zp + (int64_t)min(t0 + lt, t_end - 1) * a.z_sl, lcount);
      if (i + 1 < tiles) prepare(i + 1);
      xn = xr;
      if (i + 2 < tiles) fetch(t0 + 2 * kTile);
      bar_sync<3, NT>(i & 1);
      const int count = t0 + lt < t_end ? lcount : 0;
      if (!STATE && count > 0) {
        const float* s_y = s_stage + (i & 1) * Sh::kStage + 2 * kDu + y_row(lc) + 4 * lt;
        const int64_t at = ((int64_t)b * a.seqlen + t0 + lt) * a.channels + c0 + lc;
        float o[EV];
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const ulonglong2 y4 = *reinterpret_cast<const ulonglong2*>(s_y + e * kLdy);
          float lo, hi;
          unpack2(add2(y4.x, y4.y), lo, hi);
          o[e] = lo + hi;
        }
#pragma unroll
        for (int e = 0; e < EV; e += 2) unpack2(fma2(dv[e / 2], pair_of(xk, e / 2), pack2(o[e], o[e + 1])), o[e], o[e + 1]);
        if (a.z) {
          if (a.out_x) store_some<EV, VEC>(a.out_x + at, o, count);
#pragma unroll
          for (int e = 0; e < EV; e += 2) unpack2(mul2(pack2(o[e], o[e + 1]), silu2(pair_of(zk, e / 2))), o[e], o[e + 1]);
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
            if (n0 + s + i < a.dstate) v[i] = (keeps ? through_segment(A[i], dec.x, v[i]) : 0.0f) + a.seg_state[at * a.dstate + n0 + s + i];
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
  const auto four = [&](int t, const float* s_du, const T* s_bc, float* s_y, auto reset, uint32_t r4) {
    constexpr bool RESET = decltype(reset)::value;
    float d[K][4], u[K][4], y[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* du = s_du + du_row(ch + k * CK) + t;
      const float4 dd = *reinterpret_cast<const float4*>(du), uu = *reinterpret_cast<const float4*>(du + kDu);
      d[k][0] = dd.x, d[k][1] = dd.y, d[k][2] = dd.z, d[k][3] = dd.w;
      u[k][0] = uu.x, u[k][1] = uu.y, u[k][2] = uu.z, u[k][3] = uu.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 y2[K];
#pragma unroll
      for (int m = 0; m < GR; ++m) {
        const T* row = s_bc + (t + i) * Sh::kRow + (m * LPC + q) * 2 * CB;
        f32x2 Bv[CB / 2], Cv[CB / 2];
        load_bc_pairs<CB, !STATE>(row, Bv, Cv);
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
      float* dst = s_y + y_row(ch + k * CK) + 4 * t + (q & 3);
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
    float* const s_y = s_stage + (i & 1) * Sh::kStage + 2 * kDu;
    const T* const s_bc = reinterpret_cast<const T*>(s_y + kY);
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
        if (end - half == SSD_TOKEN_SCAN_CHECKPOINT) {
#pragma unroll
          for (int k = 0; k < SSD_TOKEN_SCAN_CHECKPOINT; k += 4) four(half + k, s_du, s_bc, s_y, std::false_type(), 0u);
        } else {
#pragma unroll 1
          for (int t = half; t < end; t += 4) four(t, s_du, s_bc, s_y, std::false_type(), 0u);
        }
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

// fp32 B and C pass shared memory in fp32 and need the sharing between two channels of a thread (3 x 777 x
// 1536 channels of 64: 115 us against 167); 16-bit ones need the threads more (2 x 4096 x 5120 channels of
// 16: 387 us against 422).
constexpr int channels_per_thread(int elem) { return elem == 4 ? 2 : 1; }

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
  s.k = channels_per_thread(dtype_size(p.x_dtype));
  s.ns = n / s.lpc;
  // segments: only where less than half of the blocks that fit the GPU at once would run, as many as fill
  // it, and none shorter than 256 positions
  const int64_t fit = kSMs * resident(kCh * s.lpc / s.k + helpers(s.lpc), s.ns * s.k);
  const int64_t want = fit / blocks, room = p.seqlen / 256;
  s.segments = (int)(want < room ? want : room);
  if (s.segments < 3) s.segments = 1;            // the state pass doubles the work
  s.seg_len = ((p.seqlen + s.segments - 1) / s.segments + kTile - 1) / kTile * kTile;
  s.segments = (p.seqlen + s.seg_len - 1) / s.seg_len;
  return s;
}

template <typename T, int LPC, int NS, int K, bool VEC>
int launch_vec(const ScanArgs& a, int batch, cudaStream_t stream) {
  using Sh = ScanShape<T, LPC, NS, K>;
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
  using Sh = ScanShape<T, LPC, NS, K>;
  constexpr int CB = Sh::kChunk, EV = Sh::kVec;
  // a thread's vector of channels begins at a multiple of its length within a group
  constexpr size_t kMost = EV * sizeof(T) < 16 ? EV * sizeof(T) : 16;
  const int ds = dtype_size(p.dt_dtype);
  const size_t dt_most = EV * ds < 16 ? EV * ds : 16;
  const bool vec = a.per_group % EV == 0 && rows_aligned(p.x, p.x_stride, 2, sizeof(T), kMost) && rows_aligned(p.dt, p.dt_stride, 2, ds, dt_most) &&
                   (p.z == nullptr || rows_aligned(p.z, p.z_stride, 2, sizeof(T), kMost)) && aligned_to(p.out, kMost) && aligned_to(p.out_x, 16) &&
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
  // whether clamping changes anything (a softplus is not negative)
  a.limits = p.dt_max < INFINITY || !(p.dt_softplus ? p.dt_min <= 0.0f : p.dt_min == -INFINITY);
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
    constexpr int K = channels_per_thread(sizeof(T));
    switch (s.lpc * 100 + s.ns) {
      case 402: return launch_plan<T, 4, 2, K>(a, p, stream);
      case 404: return launch_plan<T, 4, 4, K>(a, p, stream);
      case 804: return launch_plan<T, 8, 4, K>(a, p, stream);
      case 1604: return launch_plan<T, 16, 4, K>(a, p, stream);
      case 1608: return launch_plan<T, 16, 8, K>(a, p, stream);
      default: return launch_plan<T, 16, 16, K>(a, p, stream);
    }
  });
}

}  // namespace ssd
