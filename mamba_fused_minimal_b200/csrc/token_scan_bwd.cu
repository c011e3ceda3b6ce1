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
//
// Few channels and a long sequence: segments side by side as in the forward pass; a first walk finds what each
// hands to the one before it (18000 positions of 256 channels: 2063 to 356 us).
//
// A block's share of dB and dC takes 2 dstate floats a position, and a block holds 256 / dstate channels, so the
// shares grow with the square of dstate.  Where they pass 512 MB the problem is walked in ranges of positions,
// the last one first, and in parts of the batch; one range's shares are summed before the next one overwrites
// them, and what it hands on waits in memory.
//
// Measured at 2 x 2048 x 5120 channels of 16, bf16: 915 us with the sum of the shares, bound by issue slots (63 %):
// about 50 instructions for each position, channel and component, half of them the exchanges of the two kinds of
// sums.  1 x 4096 x 2048 x 128, in eight ranges: 5.3 ms with the forward pass.
#include "token_scan.cuh"

namespace ssd {
namespace {

constexpr int kBwdThreads = 256;      // two blocks an SM: one loads and sums while the other computes
constexpr int kBwdWarps = kBwdThreads / 32;
constexpr int kT = SSD_TOKEN_SCAN_CHECKPOINT;     // positions of a tile
constexpr int kPitch = kT + 4;                    // row pitch in shared memory

struct ScanBwdArgs {
  ScanArgs f;
  const void* dout;
  const float* carry_in;   // (batch, d, n): what comes from behind the range, or null
  float* carry_out;        // (batch, d, n): what it hands on, or null
  void* dx;
  void* ddt;
  void* dz;
  int b0, r_lo, r_hi;      // the launch's first batch element, its positions r_lo .. r_hi - 1
  // of the launch's batch elements and positions:
  float* part_bc;      // (batch, positions, g, tiles_per_group, 2, n): the blocks' shares of dB and dC
  float* part_A;       // (batch, segments, d, n)
  float* part_D;       // (batch, segments, d)
  float* part_bias;    // (batch, segments, d)
  int64_t d_sb, d_sl;
  int unit, unit32, unit_y, unit_bc, unit_ck;   // bytes copied at a time of x and the like, of an fp32 dt, of out_x, of B and C, of the states
};

template <typename T, int NP>
struct BwdShape {
  static constexpr int kChannels = kBwdThreads / NP;              // channels of a block
  static constexpr int kSlabs = NP > 32 ? NP / 32 : 1;            // warps that share a channel
  static constexpr int kRow = NP == 8 ? 16 : NP == 16 ? 32 : 64;  // a warp's dB and dC of one position
  static constexpr int kItems = kT * kChannels;                   // (position, channel) pairs of a tile
  static constexpr int kPer = kItems > kBwdThreads ? kItems / kBwdThreads : 1;
  static constexpr int kBc = 2 * kT * NP;
  static constexpr int kPerBc = kBc > kBwdThreads ? kBc / kBwdThreads : 1;
  // a tile as it lies in memory: x, dout, z (kItems elements each), B and C (kT rows of dstate), then dt, out_x
  // and the states before the tile (in 4 bytes)
  static constexpr int kBcAt = 3 * kItems, kRaw16 = kBcAt + 2 * kT * NP;
  static constexpr int kYAt = kItems, kStateAt = 2 * kItems, kRaw32 = kStateAt + kBwdThreads;
  static constexpr size_t kRaw = (kRaw16 * sizeof(T) + kRaw32 * 4 + 15) / 16 * 16;
  static constexpr size_t kSmem = 2 * kRaw + sizeof(float) * ((3 * kChannels + 2 * NP) * kPitch + 2 * kChannels * kSlabs * kPitch + kBwdWarps * kT * kRow);
};

// One warp copies `rows` rows of `bytes` bytes, `pitch` bytes apart, to rows of TO bytes in shared memory:
// asynchronously where rows and sizes are multiples of 4, 8 or 16 bytes (`unit`), else by elements of `elem`
// bytes.  Row r stands for row min(r, last).
template <int TO>
__device__ __forceinline__ void copy_rows(char* to, const char* from, int64_t pitch, int rows, int last, int bytes, int unit, int elem, int lane) {
  const int step = unit >= 4 ? unit : elem, shift = __ffs(step) - 1;
  // lanes go over whole rows of TO bytes, a power of two, so that no division is needed
  for (int i = lane << shift; i < rows * TO; i += 32 << shift) {
    const int r = i / TO, k = i % TO;
    if (k >= bytes) continue;
    const char* src = from + min(r, last) * pitch + k;
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to + i));
    if (unit == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else if (unit == 8)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
    else if (unit == 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
    else if (elem == 4)
      *reinterpret_cast<uint32_t*>(to + i) = *reinterpret_cast<const uint32_t*>(src);
    else
      *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(src);
  }
}

// sum += v with the rounding error carried along: the parameters' gradients are sums over every position
__device__ __forceinline__ void add_to(float& sum, float& lost, float v) {
  const float y = v - lost, t = sum + y;
  lost = (t - sum) - y;
  sum = t;
}

// CARRY: only what a segment passes on to the one before it, from zero behind it, and the sum of its dt'.
template <typename T, int NP, bool CARRY>
__global__ void __launch_bounds__(kBwdThreads, 2) token_scan_bwd_kernel(ScanBwdArgs q) {
  using Sh = BwdShape<T, NP>;
  constexpr int NT = kBwdThreads, CH = Sh::kChannels, SL = Sh::kSlabs, ROW = Sh::kRow, PER = Sh::kPer, NBC = Sh::kPerBc;
  constexpr int ES = sizeof(T);
  const ScanArgs& a = q.f;
  extern __shared__ float4 smem4[];
  char* const s_raw = reinterpret_cast<char*>(smem4);        // [2][Sh::kRaw]
  float* s_d = reinterpret_cast<float*>(s_raw + 2 * Sh::kRaw);      // [CH][kPitch] dt'
  float* s_u = s_d + CH * kPitch;                    // dt' x
  float* s_g = s_u + CH * kPitch;                    // dy
  float* s_B = s_g + CH * kPitch;                    // [NP][kPitch]
  float* s_C = s_B + NP * kPitch;
  float* s_p = s_C + NP * kPitch;                    // [2][CH][SL][kPitch]: g . B and the A term
  float* s_bc = s_p + 2 * CH * SL * kPitch;          // [warps][kT][ROW]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int grp = blockIdx.x / a.tiles_per_group, tile_c = blockIdx.x % a.tiles_per_group;
  const int bl = blockIdx.y, b = q.b0 + bl, seg = CARRY ? blockIdx.z + 1 : blockIdx.z;      // nothing needs what the first one passes on
  const int t_lo = q.r_lo + seg * a.seg_len, t_hi = min(q.r_hi, t_lo + a.seg_len);
  const int64_t bs = (int64_t)bl * a.segments + seg;
  const int c0 = grp * a.per_group + tile_c * CH;
  const int nch = min(CH, a.per_group - tile_c * CH);
  const int tiles = (a.seqlen + kT - 1) / kT;
  const int last = t_lo + (t_hi - t_lo - 1) / kT * kT;   // first position of the tile the walk begins with

  // The tiles' values come through two buffers of shared memory: the copies of the next tile are in flight
  // while one is walked (held in registers they did not fit beside the walk: what was loaded was spilled,
  // and so waited for at once).  A warp copies one tensor.
  const auto fetch = [&](int t0, int buf) {
    char* const raw = s_raw + buf * Sh::kRaw;
    constexpr int kOne = Sh::kItems * ES, kBC = kT * NP * ES, k32 = Sh::kRaw16 * ES;
    const int tail = a.seqlen - 1 - t0;
    const int64_t row = (int64_t)b * a.seqlen + t0;
    const auto rows = [&](int at, const void* base, int64_t off, int64_t sl) {
      copy_rows<CH * ES>(raw + at, static_cast<const char*>(base) + (off + (int64_t)t0 * sl + c0) * ES, sl * ES, kT, tail, nch * ES, q.unit, ES, lane);
    };
    const auto states = [&](int at, const void* base, int64_t off, int64_t sl) {
      copy_rows<NP * ES>(raw + at, static_cast<const char*>(base) + (off + (int64_t)t0 * sl) * ES, sl * ES, kT, tail, a.dstate * ES, q.unit_bc, ES, lane);
    };
    switch (warp) {
      case 0: rows(0, a.x, b * a.x_sb, a.x_sl); break;
      case 1: rows(kOne, q.dout, b * q.d_sb, q.d_sl); break;
      case 2:
        if (a.z) rows(2 * kOne, a.z, b * a.z_sb, a.z_sl);
        break;
      case 3:
        if (a.z && !CARRY)
          copy_rows<CH * 4>(raw + k32 + Sh::kYAt * 4, reinterpret_cast<const char*>(a.out_x + row * a.channels + c0), (int64_t)a.channels * 4, kT, tail,
                            nch * 4, q.unit_y, 4, lane);
        break;
      case 4:
        if (a.dt_f32)
          copy_rows<CH * 4>(raw + k32, static_cast<const char*>(a.dt) + (b * a.dt_sb + (int64_t)t0 * a.dt_sl + c0) * 4, a.dt_sl * 4, kT, tail,
                            nch * 4, q.unit32, 4, lane);
        else
          rows(k32, a.dt, b * a.dt_sb, a.dt_sl);
        break;
      case 5:
        if (!CARRY) states(Sh::kBcAt * ES, a.B, b * a.B_sb + grp * a.B_sg, a.B_sl);
        break;
      case 6: states(Sh::kBcAt * ES + kBC, a.C, b * a.C_sb + grp * a.C_sg, a.C_sl); break;
      default:
        if (!CARRY) copy_rows<NP * 4>(raw + k32 + Sh::kStateAt * 4,
                          reinterpret_cast<const char*>(a.ckpt + (((int64_t)b * tiles + t0 / kT) * a.channels + c0) * a.dstate), (int64_t)a.dstate * 4, nch,
                          nch, a.dstate * 4, q.unit_ck, 4, lane);
    }
  };

  // what this thread prepares and stores: positions lt, lt + kStep, ... of the tile, channel lc
  constexpr int kStep = NT / CH;
  const int lt = tid / CH, lc = tid % CH;
  const bool mine = Sh::kItems >= NT || tid < Sh::kItems, inc = lc < nch;
  const int c = c0 + (inc ? lc : 0);
  const float Dv = a.D ? load_f(a.D, a.D_dtype, c) : 0.0f;
  const float bias = a.bias ? load_f(a.bias, a.bias_dtype, c) : 0.0f;
  float sum_D = 0.0f, sum_bias = 0.0f, lost_D = 0.0f, lost_bias = 0.0f;
  const int64_t own = (int64_t)b * a.seqlen * a.channels;       // of the contiguous tensors

  // what this thread computes
  const int n = tid % NP, ch = tid / NP;
  const bool has = ch < nch && n < a.dstate;
  const int at_n = has ? (c0 + ch) * a.dstate + n : 0;            // of a (channels, dstate) tensor
  const int64_t ck_step = (int64_t)a.channels * a.dstate;
  const float A = has ? load_f(a.A, a.A_dtype, at_n) : 0.0f;
  float carry = has && q.carry_in && !CARRY ? q.carry_in[bl * ck_step + at_n] : 0.0f;      // a_{t+1} g_{t+1}
  if (!CARRY && has) {
    // through the segments behind, from the last one on
    for (int j = a.segments - 1; j > seg; --j) {
      const int64_t at = (int64_t)bl * a.segments + j;
      const float2 dec = a.seg_decay[at * a.channels + c0 + ch];
      const bool keeps = dec.y != 0.0f && (j < a.segments - 1 || q.carry_in != nullptr);      // else there is nothing to keep
      carry = (keeps ? through_segment(A * kLog2e, dec.x, carry) : 0.0f) + a.seg_state[at * ck_step + at_n];
    }
  }
  float sum_dt = 0.0f;
  bool dropped = false;
  float sum_A = 0.0f, lost_A = 0.0f;

  // B and C: component bn of positions bt, bt + kBcStep, ...; the first half of the items is B (with eight
  // components the first half of the threads takes B and the other C)
  constexpr bool kOnce = NT / NP > kT;
  constexpr int kBcStep = kOnce ? kT : NT / NP, kHalf = kT / kBcStep;
  static_assert(kOnce ? NBC == 1 && NT / NP == 2 * kT : NBC == 2 * kHalf, "every component of a tile's B and C is taken once");
  const int bn = tid % NP, bt = tid / NP % kT;
  const bool second = kOnce && tid / NP >= kT;
  const bool bin = bn < a.dstate;

  // the block's share of dB and dC: outputs o = k NT + tid; component on of kind oj, in the slabs and
  // positions that k walks through
  constexpr int kOuts = kT * SL * ROW / NT, kQ = NT / ROW, kSum = kBwdWarps / SL;
  const int oq = tid / ROW, oj = tid % ROW;
  const int64_t out_row = (int64_t)a.ngroups * a.tiles_per_group * 2 * a.dstate;
  float* const part = q.part_bc + ((int64_t)bl * (q.r_hi - q.r_lo) - q.r_lo) * out_row + ((int64_t)grp * a.tiles_per_group + tile_c) * 2 * a.dstate;
  const int part_at = (oj / (ROW / 2)) * a.dstate + oj % (ROW / 2);

  fetch(last, 0);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  int buf = 0;
  for (int t0 = last; t0 >= t_lo; t0 -= kT, buf ^= 1) {
    const T* const raw = reinterpret_cast<const T*>(s_raw + buf * Sh::kRaw);
    const float* const raw32 = reinterpret_cast<const float*>(s_raw + buf * Sh::kRaw + Sh::kRaw16 * ES);
    float d[PER], x[PER], dy[PER], slope[PER];         // slope: d dt' / d dt
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int t = t0 + lt + e * kStep;
      const bool in = mine && inc && t < a.seqlen;
      const int item = mine ? (lt + e * kStep) * CH + lc : 0;
      x[e] = in ? widen(raw[item]) : 0.0f;
      d[e] = (a.dt_f32 ? raw32[item] : widen(reinterpret_cast<const T*>(raw32)[item])) + bias;
      slope[e] = 1.0f;
      if (a.softplus) {
        slope[e] = sigmoid_f(d[e]);
        d[e] = softplus_f(d[e]);
      }
      if (a.limits) {
        if (d[e] < a.dt_min || d[e] > a.dt_max) slope[e] = 0.0f;
        d[e] = clamp_f(d[e], a.dt_min, a.dt_max);
      }
      if (!in) d[e] = 0.0f;
      dy[e] = in ? widen(raw[Sh::kItems + item]) : 0.0f;
      if (a.z) {
        const float zv = widen(raw[2 * Sh::kItems + item]), s = sigmoid_f(zv);
        if (in && !CARRY) static_cast<T*>(q.dz)[own + (int64_t)t * a.channels + c] = narrow<T>(dy[e] * raw32[Sh::kYAt + item] * (s * (1.0f + zv * (1.0f - s))));
        dy[e] = in ? dy[e] * (zv * s) : 0.0f;
      }
      if (mine) {
        const int at = lc * kPitch + lt + e * kStep;
        s_d[at] = d[e];
        s_u[at] = d[e] * x[e];
        s_g[at] = dy[e];
      }
      add_to(sum_D, lost_D, dy[e] * x[e]);
    }
#pragma unroll
    for (int k = 0; k < NBC; ++k) {
      const bool is_b = k < kHalf && !second;
      const int t = bt + k % kHalf * kBcStep;
      (is_b ? s_B : s_C)[bn * kPitch + t] = bin ? widen(raw[Sh::kBcAt + (is_b ? t : kT + t) * NP + bn]) : 0.0f;
    }
    float h = has ? raw32[Sh::kStateAt + ch * NP + n] : 0.0f;
    const uint32_t resets = a.seq ? reset_mask(a, b, t0, lane) : 0u;
    __syncthreads();
    if (t0 > t_lo) fetch(t0 - kT, buf ^ 1);

    const auto pass = [&](auto reset) {
      constexpr bool RESET = decltype(reset)::value;
#pragma unroll
      for (int t = kT - 4; t >= 0; t -= 4) {
        const float4 d4 = *reinterpret_cast<const float4*>(&s_d[ch * kPitch + t]);
        const float4 g4 = *reinterpret_cast<const float4*>(&s_g[ch * kPitch + t]);
        const float4 C4 = *reinterpret_cast<const float4*>(&s_C[n * kPitch + t]);
        const float d[4] = {d4.x, d4.y, d4.z, d4.w}, y[4] = {g4.x, g4.y, g4.z, g4.w}, c[4] = {C4.x, C4.y, C4.z, C4.w};
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          carry = fmaf(c[i], y[i], carry) * ex2_approx(d[i] * (A * kLog2e));
          if (RESET && (resets >> (t + i) & 1u)) carry = 0.0f;
        }
        sum_dt += (d[0] + d[1]) + (d[2] + d[3]);
      }
      dropped |= RESET;
    };
    const auto walk = [&](auto reset) {
      constexpr bool RESET = decltype(reset)::value;
      // forwards through the tile: the decays, and what of the state before reaches each position; pairs are
      // two neighbouring positions
      f32x2 dec[kT / 2], kept[kT / 2];
#pragma unroll
      for (int t = 0; t < kT; t += 4) {
        const ulonglong2 d4 = *reinterpret_cast<const ulonglong2*>(&s_d[ch * kPitch + t]);
        const ulonglong2 u4 = *reinterpret_cast<const ulonglong2*>(&s_u[ch * kPitch + t]);
        const ulonglong2 B4 = *reinterpret_cast<const ulonglong2*>(&s_B[n * kPitch + t]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float e[2], k[2], v[2];
          unpack2(mul2(i ? d4.y : d4.x, both(A * kLog2e)), e[0], e[1]);
          unpack2(mul2(i ? u4.y : u4.x, i ? B4.y : B4.x), v[0], v[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            e[j] = ex2_approx(e[j]);
            k[j] = e[j] * h;
            if (RESET && (resets >> (t + 2 * i + j) & 1u)) e[j] = k[j] = 0.0f;
            h = k[j] + v[j];
          }
          dec[t / 2 + i] = pack2(e[0], e[1]);
          kept[t / 2 + i] = pack2(k[0], k[1]);
        }
      }
      // and backwards
      f32x2 sum_A2 = 0;
#pragma unroll
      for (int t = kT - 4; t >= 0; t -= 4) {
        const ulonglong2 d4 = *reinterpret_cast<const ulonglong2*>(&s_d[ch * kPitch + t]);
        const ulonglong2 u4 = *reinterpret_cast<const ulonglong2*>(&s_u[ch * kPitch + t]);
        const ulonglong2 g4 = *reinterpret_cast<const ulonglong2*>(&s_g[ch * kPitch + t]);
        const ulonglong2 B4 = *reinterpret_cast<const ulonglong2*>(&s_B[n * kPitch + t]);
        const ulonglong2 C4 = *reinterpret_cast<const ulonglong2*>(&s_C[n * kPitch + t]);
        float p1[4], p2[4];
#pragma unroll
        for (int i = 1; i >= 0; --i) {
          const f32x2 dd = i ? d4.y : d4.x, uu = i ? u4.y : u4.x, yy = i ? g4.y : g4.x, BB = i ? B4.y : B4.x, CC = i ? C4.y : C4.x;
          float from[2], e[2], g[2], vB[2], vC[2];
          unpack2(mul2(CC, yy), from[0], from[1]);
          unpack2(dec[t / 2 + i], e[0], e[1]);
          // a position that begins a sequence hands nothing on: selected, since what it holds may not be finite
          const int first = RESET ? (int)(resets >> (t + 2 * i)) : 0;
          g[1] = from[1] + carry;
          g[0] = first & 2 ? from[0] : fmaf(g[1], e[1], from[0]);
          carry = first & 1 ? 0.0f : g[0] * e[0];
          const f32x2 gg = pack2(g[0], g[1]);
          const f32x2 m = mul2(gg, kept[t / 2 + i]);
          unpack2(mul2(yy, fma2(uu, BB, kept[t / 2 + i])), vC[0], vC[1]);
          unpack2(mul2(gg, uu), vB[0], vB[1]);
          unpack2(mul2(gg, BB), p1[2 * i], p1[2 * i + 1]);
          unpack2(mul2(m, both(A)), p2[2 * i], p2[2 * i + 1]);
          sum_A2 = fma2(m, dd, sum_A2);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float* row = s_bc + (warp * kT + t + 2 * i + j) * ROW;
            if constexpr (NP >= 32) {
              row[lane] = vB[j];
              row[32 + lane] = vC[j];
            } else {
              // lanes 0..15 keep dB, lanes 16..31 dC, of the channels 16 lanes apart
              float v = (lane < 16 ? vB[j] : vC[j]) + __shfl_xor_sync(0xffffffffu, lane < 16 ? vC[j] : vB[j], 16);
              if constexpr (NP == 8) {
                v += __shfl_xor_sync(0xffffffffu, v, 8);
                if ((lane & 8) == 0) row[(lane >> 4) * 8 + (lane & 7)] = v;
              } else {
                row[lane] = v;
              }
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
      float lo, hi;
      unpack2(sum_A2, lo, hi);
      add_to(sum_A, lost_A, lo + hi);
    };
    // the vote covers 32 positions, of which the tile has the first sixteen
    const bool plain = (resets & 0xffffu) == 0u;
    if constexpr (CARRY) {
      if (plain)
        pass(std::false_type());
      else
        pass(std::true_type());
    } else {
      if (plain)
        walk(std::false_type());
      else
        walk(std::true_type());
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if constexpr (CARRY) continue;

#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int t = t0 + lt + e * kStep;
      if (!mine || !inc || t >= a.seqlen) continue;
      float gB = 0.0f, gA = 0.0f;
#pragma unroll
      for (int s = 0; s < SL; ++s) {
        gB += s_p[(lc * SL + s) * kPitch + lt + e * kStep];
        gA += s_p[((CH + lc) * SL + s) * kPitch + lt + e * kStep];
      }
      const float dd = fmaf(x[e], gB, gA) * slope[e];
      add_to(sum_bias, lost_bias, dd);
      const int64_t at = own + (int64_t)t * a.channels + c;
      static_cast<T*>(q.dx)[at] = narrow<T>(fmaf(d[e], gB, Dv * dy[e]));
      if (a.dt_f32)
        static_cast<float*>(q.ddt)[at] = dd;
      else
        static_cast<T*>(q.ddt)[at] = narrow<T>(dd);
    }
    // over the warps (their channels) in order
#pragma unroll
    for (int k = 0; k < kOuts; ++k) {
      int slab, t;
      if constexpr (kQ % SL == 0) {
        slab = oq % SL;
        t = k * (kQ / SL) + oq / SL;
      } else {
        constexpr int kTurn = SL / kQ;
        slab = k % kTurn * kQ + oq;
        t = k / kTurn;
      }
      if (slab * 32 + oj % (ROW / 2) >= a.dstate || t0 + t >= a.seqlen) continue;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < kSum; ++s) v += s_bc[((s * SL + slab) * kT + t) * ROW + oj];
      part[(int64_t)(t0 + t) * out_row + part_at + slab * 32] = v;
    }
  }

  if constexpr (CARRY) {
    if (has) {
      a.seg_state[bs * ck_step + at_n] = carry;
      if (n == 0) a.seg_decay[bs * a.channels + c0 + ch] = make_float2(sum_dt, dropped ? 0.0f : 1.0f);
    }
    return;
  }
  if (has) {
    q.part_A[bs * ck_step + at_n] = sum_A;
    if (q.carry_out && seg == 0) q.carry_out[bl * ck_step + at_n] = carry;
  }
  // dD and the bias's gradient: over the threads of a channel in order
  __syncthreads();
  s_bc[tid] = sum_D;
  s_bc[NT + tid] = sum_bias;
  __syncthreads();
  if (tid < nch) {
    float u = 0.0f, v = 0.0f;
    for (int s = tid; s < min(NT, Sh::kItems); s += CH) u += s_bc[s], v += s_bc[NT + s];
    q.part_D[bs * a.channels + c0 + tid] = u;
    q.part_bias[bs * a.channels + c0 + tid] = v;
  }
}

// The blocks' shares, joined in a fixed order.  Block i < sums: 32 components of dB and dC of one (position, group)
// over the channel blocks, eight strides side by side (one thread a sum was bound by the latency of its chain of
// loads: 160 us for 4096 positions of 320 blocks).  The blocks behind: dA, dD and the bias's gradient over the batch
// and its segments, one thread an element; `more` adds them to what earlier launches left.
__host__ __device__ constexpr int sum_columns(int dstate) { return (2 * dstate + 31) / 32; }
template <typename T>
__global__ void __launch_bounds__(256) sum_shares_kernel(ScanBwdArgs q, T* dB, T* dC, float* dA, float* dD, float* dbias, int sums, int parts, bool more) {
  __shared__ float s[8][33];
  const int dstate = q.f.dstate, tiles = q.f.tiles_per_group;
  if ((int)blockIdx.x < sums) {
    const int columns = sum_columns(dstate);
    const int64_t row = blockIdx.x / columns;
    const int j = (int)(blockIdx.x % columns) * 32 + threadIdx.x;
    const float* p = q.part_bc + row * tiles * (2 * dstate);
    float v = 0.0f;
    if (j < 2 * dstate) {
#pragma unroll 8
      for (int k = threadIdx.y; k < tiles; k += 8) v += p[(int64_t)k * 2 * dstate + j];
    }
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && j < 2 * dstate) {
      float u = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) u += s[k][threadIdx.x];
      const int64_t each = (int64_t)(q.r_hi - q.r_lo) * q.f.ngroups, bl = row / each;
      const int64_t to = (((q.b0 + bl) * q.f.seqlen + q.r_lo) * q.f.ngroups + (row - bl * each)) * dstate;
      if (j < dstate)
        dB[to + j] = narrow<T>(u);
      else
        dC[to + j - dstate] = narrow<T>(u);
    }
    return;
  }
  const int64_t dn = (int64_t)q.f.channels * dstate, d = q.f.channels;
  int64_t i = (int64_t)(blockIdx.x - sums) * 256 + threadIdx.y * 32 + threadIdx.x;
  const float* p = q.part_A;
  float* out = dA;
  int64_t pitch = dn;
  if (i >= dn) {
    i -= dn;
    p = q.part_D, out = dD, pitch = d;
    if (i >= d) {
      i -= d;
      p = q.part_bias, out = dbias;
      if (i >= d) return;
    }
  }
  if (out == nullptr) return;
  float v = more ? out[i] : 0.0f;
#pragma unroll 4
  for (int b = 0; b < parts; ++b) v += p[b * pitch + i];
  out[i] = v;
}

int padded_state(int n) { return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256; }

int bwd_tiles(const ssd_token_scan_params_t& p) {
  const int ch = kBwdThreads / padded_state(p.dstate);
  return (p.channels / p.ngroups + ch - 1) / ch;
}

constexpr int64_t kShares = 512 << 20;      // bytes of the shares of dB and dC that a launch may leave

// How a problem is walked: `batch` batch elements and `len` positions a launch, in segments of `seg_len`.
struct BwdPlan {
  int batch, len, segments, seg_len;
};
BwdPlan plan_bwd(const ssd_token_scan_params_t& p) {
  BwdPlan s{p.batch, p.seqlen, 1, p.seqlen};
  const int64_t fit = 2 * kSMs, blocks = (int64_t)p.ngroups * bwd_tiles(p);      // of one batch element
  const int64_t bytes = blocks * 2 * p.dstate * sizeof(float);                  // and one position
  if (bytes > kShares / ((int64_t)p.batch * p.seqlen)) {
    // as many batch elements side by side as leave room for 256 positions, so that a launch has many waves of blocks
    // and a block many tiles, then as many positions as there is room for; both evenly
    const int64_t room = kShares / (bytes * 256), most = room < 1 ? 1 : room < p.batch ? room : p.batch;
    const int64_t parts = (p.batch + most - 1) / most;
    s.batch = (int)((p.batch + parts - 1) / parts);
    int64_t len = kShares / (bytes * s.batch) / kT * kT;
    if (len < kT) len = kT;
    if (len < p.seqlen) {
      const int64_t ranges = (p.seqlen + len - 1) / len;
      s.len = (int)(((p.seqlen + ranges - 1) / ranges + kT - 1) / kT * kT);
    }
  }
  // Segments: where less than half of the blocks that fit the GPU would run, as many as fill it, none shorter
  // than 128 positions.  The pass that finds what a segment hands on costs a quarter of the walk.
  const int64_t side = fit / (blocks * s.batch), room = s.len / 128;
  int64_t n = side < room ? side : room;
  if (n < 2) n = 1;
  s.seg_len = (int)(((s.len + n - 1) / n + kT - 1) / kT * kT);
  s.segments = (s.len + s.seg_len - 1) / s.seg_len;
  return s;
}

struct BwdWorkspace {
  size_t bc, A, D, state, carry, decay, total;      // offsets in floats; the bias's shares follow dD's
};
BwdWorkspace bwd_workspace(const ssd_token_scan_params_t& p, const BwdPlan& s) {
  const size_t dn = (size_t)p.channels * p.dstate, each = (size_t)s.batch * s.segments;
  BwdWorkspace w;
  w.decay = 0;                               // pairs: the first, for their alignment
  w.bc = w.decay + (s.segments > 1 ? 2 * each * p.channels : 0);
  w.A = w.bc + (size_t)s.batch * s.len * p.ngroups * bwd_tiles(p) * 2 * p.dstate;
  w.D = w.A + each * dn;
  w.state = w.D + 2 * each * p.channels;
  w.carry = w.state + (s.segments > 1 ? each * dn : 0);
  w.total = w.carry + (s.len < p.seqlen ? 2 * (size_t)s.batch * dn : 0);      // one is read while the other is written
  return w;
}

// the largest of 16, 8 and 4 bytes that `bytes` is a multiple of, else 0
int copy_unit(int64_t bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : bytes % 4 == 0 ? 4 : 0; }
template <typename... Ts>
int copy_unit(int64_t first, int64_t second, Ts... more) {
  const int u = copy_unit(first), v = copy_unit(second, more...);
  return u < v ? u : v;
}

template <typename T, int NP>
int launch_bwd(ScanBwdArgs& q, int batch, cudaStream_t stream) {
  using Sh = BwdShape<T, NP>;
  constexpr size_t smem = Sh::kSmem;
  const ScanArgs& a = q.f;
  const auto at = [](const void* p) { return (int64_t)(reinterpret_cast<uintptr_t>(p) & 15); };
  constexpr int64_t es = sizeof(T);
  // a block's channels begin at a multiple of its own within the group, and its last block ends with it
  const int64_t ch = Sh::kChannels * es, pg = (int64_t)a.per_group * es;
  q.unit = copy_unit(ch, pg, at(a.x), a.x_sb * es, a.x_sl * es, at(q.dout), q.d_sb * es, q.d_sl * es, at(a.z), a.z ? a.z_sb * es : 0, a.z ? a.z_sl * es : 0,
                     a.dt_f32 ? 0 : at(a.dt), a.dt_f32 ? 0 : a.dt_sb * es, a.dt_f32 ? 0 : a.dt_sl * es);
  q.unit32 = copy_unit(Sh::kChannels * 4, (int64_t)a.per_group * 4, at(a.dt), a.dt_sb * 4, a.dt_sl * 4);
  q.unit_y = copy_unit(Sh::kChannels * 4, (int64_t)a.per_group * 4, at(a.out_x), (int64_t)a.channels * 4);
  q.unit_bc = copy_unit(a.dstate * es, at(a.B), a.B_sb * es, a.B_sl * es, a.B_sg * es, at(a.C), a.C_sb * es, a.C_sl * es, a.C_sg * es);
  q.unit_ck = copy_unit(a.dstate * 4, at(a.ckpt));
  if (smem > 48 * 1024)
    SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_bwd_kernel<T, NP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  dim3 grid(a.ngroups * a.tiles_per_group, batch, a.segments);
  if (a.segments > 1) {
    if (smem > 48 * 1024)
      SSD_CUDA_OK(cudaFuncSetAttribute(token_scan_bwd_kernel<T, NP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    grid.z = a.segments - 1;
    token_scan_bwd_kernel<T, NP, true><<<grid, kBwdThreads, smem, stream>>>(q);
    SSD_CUDA_OK(cudaGetLastError());
    grid.z = a.segments;
  }
  token_scan_bwd_kernel<T, NP, false><<<grid, kBwdThreads, smem, stream>>>(q);
  SSD_CUDA_OK(cudaGetLastError());
  return SSD_OK;
}

}  // namespace

size_t token_scan_bwd_workspace(const ssd_token_scan_bwd_params_t& p) { return bwd_workspace(p.scan, plan_bwd(p.scan)).total * sizeof(float); }

int launch_token_scan_bwd(const ssd_token_scan_bwd_params_t& r, cudaStream_t stream) {
  const ssd_token_scan_params_t& p = r.scan;
  SSD_REQUIRE(p.batch <= 65535 && (int64_t)p.batch * p.seqlen * p.ngroups <= 0x3fffffff, SSD_ERR_UNSUPPORTED,
              "token scan: batch %d, seqlen %d or ngroups %d too large", p.batch, p.seqlen, p.ngroups);
  SSD_REQUIRE((int64_t)p.channels * p.dstate <= 0x7fffffff, SSD_ERR_UNSUPPORTED, "token scan: %d channels of %d too many", p.channels, p.dstate);
  const BwdPlan s = plan_bwd(p);
  const BwdWorkspace w = bwd_workspace(p, s);
  const int64_t dn = (int64_t)p.channels * p.dstate;
  ScanBwdArgs q;
  q.f = scan_args(p);
  q.f.tiles_per_group = bwd_tiles(p);
  q.f.seg_len = s.seg_len;
  q.dout = r.dout;
  q.dx = r.dx, q.ddt = r.ddt, q.dz = r.dz;
  float* ws = static_cast<float*>(r.workspace);
  q.part_bc = ws + w.bc;
  q.part_A = ws + w.A;
  q.part_D = ws + w.D;
  q.part_bias = q.part_D + (size_t)s.batch * s.segments * p.channels;
  q.f.seg_state = ws + w.state;
  q.f.seg_decay = reinterpret_cast<float2*>(ws + w.decay);
  q.d_sb = r.dout_stride[0], q.d_sl = r.dout_stride[1];
  return with_type(p.x_dtype, [&](auto t) -> int {
    using T = decltype(t);
    bool more = false;
    for (q.b0 = 0; q.b0 < p.batch; q.b0 += s.batch) {
      const int batch = p.batch - q.b0 < s.batch ? p.batch - q.b0 : s.batch;
      float* carry[2] = {ws + w.carry, ws + w.carry + s.batch * dn};
      for (int range = (p.seqlen - 1) / s.len; range >= 0; --range, more = true) {
        q.r_lo = range * s.len;
        q.r_hi = p.seqlen - q.r_lo < s.len ? p.seqlen : q.r_lo + s.len;
        q.f.segments = (q.r_hi - q.r_lo + s.seg_len - 1) / s.seg_len;
        q.carry_in = q.r_hi < p.seqlen ? carry[range & 1] : r.dfinal_states ? r.dfinal_states + q.b0 * dn : nullptr;
        q.carry_out = range > 0 ? carry[(range - 1) & 1] : r.dinitial_states ? r.dinitial_states + q.b0 * dn : nullptr;
        int rc;
        switch (padded_state(p.dstate)) {
          case 8: rc = launch_bwd<T, 8>(q, batch, stream); break;
          case 16: rc = launch_bwd<T, 16>(q, batch, stream); break;
          case 32: rc = launch_bwd<T, 32>(q, batch, stream); break;
          case 64: rc = launch_bwd<T, 64>(q, batch, stream); break;
          case 128: rc = launch_bwd<T, 128>(q, batch, stream); break;
          default: rc = launch_bwd<T, 256>(q, batch, stream); break;
        }
        if (rc != SSD_OK) return rc;
        const int64_t sums = (int64_t)batch * (q.r_hi - q.r_lo) * p.ngroups * sum_columns(p.dstate), params = ((int64_t)p.channels * (p.dstate + 2) + 255) / 256;
        sum_shares_kernel<T><<<(unsigned)(sums + params), dim3(32, 8), 0, stream>>>(q, static_cast<T*>(r.dB), static_cast<T*>(r.dC), r.dA, r.dD,
                                                                                   r.ddt_bias, (int)sums, batch * q.f.segments, more);
        SSD_CUDA_OK(cudaGetLastError());
      }
    }
    return SSD_OK;
  });
}

}  // namespace ssd
