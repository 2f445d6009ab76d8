// The selective scan: for each channel with its S states
//   step = softplus(delta + bias) (or without the softplus),  a = exp(step A)
//   h_t = a_t h_{t-1} + step_t x_t B_t,   o_t = C_t . h_t + skip x_t,   y_t = o_t silu(gate_t)
// and, with do = dy silu(gate) and g the adjoint of h,
//   g_t = C_t do_t + a_{t+1} g_{t+1},   m_t = g_t a_t h_{t-1}
//   dx = step (g.B) + skip do,   dstep = x (g.B) + m.A,   dA = sum m step
//   dB = sum_channels g step x,   dC = sum_channels do h,   dgate = dy o silu'(gate)
//
// Nothing here is a product of matrices: each (token, channel, state) has a
// decay of its own, one exponential and four multiply-adds forward, and that,
// not memory, bounds the kernels (B15 N2048, 1,024 channels of 16 states: 503
// million of them forward against 252 MB).  So the work is laid out for the
// vector units: LPC adjacent lanes share a channel, SPL states in the registers
// of each, and a wave holds 64 / LPC channels.  The quads of lanes divide what
// a channel has once for each token (softplus, silu, loads, stores) by taking
// one of four tokens each; a token's step reaches the other lanes by DPP.  B
// and C are staged in LDS as fp32, one read for a lane's SPL states.
//
// A sequence is one segment where the channels alone fill the vector units;
// else it is cut into segments, which a launch in front reduces to the state
// that each adds from zero and the sum of its steps (a segment's decay is
// exp(A sum)); the rows' workgroups join the segments in front of their own
// themselves.  The backward does the same with the adjoint, from the end.
//
// The backward walks chunks from the last to the first: it forms a chunk's
// states again from the checkpoint the forward left in front of it, keeps them
// and the decays in registers and walks back through them.  dB and dC are sums
// over channels: over a wave's by lane exchanges, over a workgroup's waves in
// LDS, over workgroups by partial rows that a last launch adds in order.
// Nothing is atomic: the same bits every time.  dA, dskip and the bias's
// gradient, sums over all tokens, run in 64 bits from a chunk on.
#include "selective.h"

namespace dwarf {
namespace {

constexpr int kScanWaves = 4, kScanThreads = kScanWaves * kWave;
constexpr int kTile = 32;           // tokens of B and C in LDS at a time, forward
constexpr int kMaxSegments = 64;
constexpr int kSegmentUnit = 64;    // tokens a segment is a multiple of

// States per lane and lanes per channel for S states.
constexpr int scan_spl(int S) { return S <= 8 ? 2 : S <= 16 ? 4 : 8; }
constexpr int scan_lpc(int S) { return S <= 32 ? 4 : 8; }
// Tokens of a backward chunk, whose states and decays a lane keeps: 64 of each.
constexpr int scan_chunk(int spl) { return 64 / spl; }

struct ScanGeom {
  int segs, seg;             // segments, tokens of each
  int tiles_of_group, tiles; // workgroups' channel tiles
  float* local;              // [B][segs][D][SP]: what a segment adds to the state (or adjoint) from zero
  float* steps;              // [B][segs][D]: the sum of its steps
  float* part;               // [tiles_of_group][B][N][G][2][SP]: dB and dC of a channel tile
  float* part_A;             // [B][segs][D][SP]
  float* part_d;             // [B][segs][2][D]: skip, bias
};

template <int J>
__device__ __forceinline__ float quad_lane(float x) { return dpp_f<J * 0x55>(x); }

// Lane i of each quad receives the sum of p[i] over the LPC lanes of its channel.
template <int LPC>
__device__ __forceinline__ float quad_sums(float p0, float p1, float p2, float p3, int lane) {
  if constexpr (LPC == 8) {   // lane i and lane 7 - i of the eight
    p0 += dpp_f<0x141>(p0);
    p1 += dpp_f<0x141>(p1);
    p2 += dpp_f<0x141>(p2);
    p3 += dpp_f<0x141>(p3);
  }
  const bool odd = lane & 1, high = lane & 2;
  const float a = (odd ? p1 : p0) + dpp_f<0xB1>(odd ? p0 : p1);
  const float b = (odd ? p3 : p2) + dpp_f<0xB1>(odd ? p2 : p3);
  return (high ? b : a) + dpp_f<0x4E>(high ? a : b);
}

__device__ __forceinline__ float step_of(float raw, int softplus) {
  return !softplus ? raw : raw > 20.f ? raw : log1pf(expf(raw));
}

// Where a lane stands.
template <int LPC>
struct ScanLane {
  static constexpr int kCh = kWave / LPC;              // channels of a wave
  static constexpr int kTileCh = kScanWaves * kCh;     // of a workgroup
  int lane, wave, sq, b, seg, tile, g, d;
  bool in;   // the lane's channel is one of the group's; otherwise d is the group's last
  __device__ __forceinline__ ScanLane(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm, int segs) {
    lane = threadIdx.x % kWave;
    wave = threadIdx.x / kWave;
    sq = lane % LPC;
    uint32_t i = blockIdx.x;
    tile = i % static_cast<uint32_t>(gm.tiles);
    i /= static_cast<uint32_t>(gm.tiles);
    seg = i % static_cast<uint32_t>(segs);
    b = i / static_cast<uint32_t>(segs);
    g = tile / gm.tiles_of_group;
    const int per = a.D / a.G, c = tile % gm.tiles_of_group * kTileCh + wave * kCh + lane / LPC;
    in = c < per;
    d = g * per + (in ? c : per - 1);
  }
};

__device__ __forceinline__ int scan_length(const dwarf_selective_scan_fwd_args& a, int b) {
  if (!a.lengths) return a.N;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.N ? a.N : n;
}

// B or C rows of TOK tokens from t on, as the workgroup's threads carry them into LDS: raw in registers between.
template <typename T, int SP, int TOK>
struct BcRows {
  static constexpr int kEach = (TOK * SP + kScanThreads - 1) / kScanThreads;
  T v[kEach];
  __device__ __forceinline__ void load(const T* p, int64_t stride, int t, int end, int S) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kScanThreads + threadIdx.x, s = i % SP;
      int tt = t + i / SP;
      if (tt >= end) tt = end - 1;
      v[e] = p[tt * stride + (s < S ? s : 0)];
    }
  }
  // rows from `end` on and states from S on are zero
  __device__ __forceinline__ void store(float* to, int t, int end, int S) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kScanThreads + threadIdx.x, s = i % SP;
      if (TOK * SP % kScanThreads == 0 || i < TOK * SP) to[i] = s < S && t + i / SP < end ? to_f32(v[e]) : 0.f;
    }
  }
};

template <int SPL>
__device__ __forceinline__ void load_states(const float* p, float* h) {
  if constexpr (SPL == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    h[0] = v.x, h[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < SPL / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      h[4 * i] = v.x, h[4 * i + 1] = v.y, h[4 * i + 2] = v.z, h[4 * i + 3] = v.w;
    }
  }
}
template <int SPL>
__device__ __forceinline__ void store_states(float* p, const float* h) {
  if constexpr (SPL == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(h[0], h[1]);
  } else {
#pragma unroll
    for (int i = 0; i < SPL / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
  }
}

// The user's [..][D][S] states, S as it is.
template <int SPL>
__device__ __forceinline__ void load_user_states(const float* p, int s0, int S, float* h) {
#pragma unroll
  for (int s = 0; s < SPL; ++s) h[s] = p && s0 + s < S ? p[s0 + s] : 0.f;
}
template <int SPL>
__device__ __forceinline__ void store_user_states(float* p, int s0, int S, const float* h) {
#pragma unroll
  for (int s = 0; s < SPL; ++s)
    if (s0 + s < S) p[s0 + s] = h[s];
}

// A in base 2, so that the decay is one exp2.
template <int SPL>
__device__ __forceinline__ void load_rates(const float* A, int64_t d, int s0, int S, float* rate) {
#pragma unroll
  for (int s = 0; s < SPL; ++s) rate[s] = s0 + s < S ? A[d * S + s0 + s] * kLog2e : 0.f;
}

// LOCAL: what a segment adds from zero and its sum of steps, for all segments but the last; otherwise the rows.
template <typename T, int SPL, int LPC, bool LOCAL>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(dwarf_selective_scan_fwd_args a, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kQuads = kTile / 4, kK = scan_chunk(SPL);
  __shared__ __align__(16) float s_b[2][kTile * SP];
  __shared__ __align__(16) float s_c[LOCAL ? 1 : 2][LOCAL ? 4 : kTile * SP];
  const ScanLane<LPC> at(a, gm, LOCAL ? gm.segs - 1 : gm.segs);
  const int s0 = at.sq * SPL, quad = at.lane & 3;
  const int64_t d = at.d;
  const int t0 = at.seg * gm.seg, t1 = min(a.N, t0 + gm.seg);
  const int end = min(t1, scan_length(a, at.b));   // live tokens: [t0, end)
  float rate[SPL], h[SPL];
  load_rates<SPL>(a.A, d, s0, a.S, rate);
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = !LOCAL && a.skip ? a.skip[d] : 0.f;
#pragma unroll
  for (int s = 0; s < SPL; ++s) h[s] = 0.f;
  if constexpr (!LOCAL) {
    if (a.initial) load_user_states<SPL>(a.initial + (static_cast<int64_t>(at.b) * a.D + d) * a.S, s0, a.S, h);
    for (int i = 0; i < at.seg; ++i) {   // the segments in front
      const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + i) * a.D + d;
      float add[SPL];
      load_states<SPL>(gm.local + row * SP + s0, add);
      const float sum = gm.steps[row];
#pragma unroll
      for (int s = 0; s < SPL; ++s) h[s] = fmaf(__builtin_amdgcn_exp2f(sum * rate[s]), h[s], add[s]);
    }
  }
  const T* px = static_cast<const T*>(a.x) + at.b * a.x_stride[0] + d;
  const T* pd = static_cast<const T*>(a.delta) + at.b * a.delta_stride[0] + d;
  const T* pz = static_cast<const T*>(a.gate) + at.b * a.gate_stride[0] + d;
  const T* pB = static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2];
  const T* pC = static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
  T* py = static_cast<T*>(a.y) + at.b * a.y_stride[0] + d;
  const bool gated = !LOCAL && a.gate, writes = at.in && at.sq < 4;
  float* ck = !LOCAL && a.checkpoints && at.in
                  ? a.checkpoints + (static_cast<int64_t>(at.b) * ((a.N + kK - 1) / kK) * a.D + d) * SP + s0 : nullptr;
  float total = 0.f;
  T rx[kQuads], rd[kQuads], rz[kQuads];
  BcRows<T, SP, kTile> rb, rc;
  // a tile's loads: tokens behind the live ones read the last live one again
  auto fetch = [&](int t) {
    rb.load(pB, a.B_stride[1], t, end, a.S);
    if constexpr (!LOCAL) rc.load(pC, a.C_stride[1], t, end, a.S);
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int64_t tt = min(t + 4 * k + quad, end - 1);
      rx[k] = px[tt * a.x_stride[1]];
      rd[k] = pd[tt * a.delta_stride[1]];
      if (gated) rz[k] = pz[tt * a.gate_stride[1]];
    }
  };
  int buf = 0;
  if (t0 < end) {
    fetch(t0);
    rb.store(s_b[0], t0, end, a.S);
    if constexpr (!LOCAL) rc.store(s_c[0], t0, end, a.S);
    __syncthreads();
  }
  for (int t = t0; t < end; t += kTile, buf ^= 1) {
    float u[kQuads], dl[kQuads], z[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      u[k] = to_f32(rx[k]);
      dl[k] = to_f32(rd[k]);
      z[k] = gated ? to_f32(rz[k]) : 0.f;
    }
    const bool more = t + kTile < end;
    if (more) fetch(t + kTile);   // under way while this tile is worked on
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      if (!LOCAL && 4 * k % kK == 0 && ck && t + 4 * k < end)
        store_states<SPL>(ck + static_cast<int64_t>((t + 4 * k) / kK) * a.D * SP, h);
      const int tk = t + 4 * k + quad;
      const bool live = tk < end;
      const float st = live ? step_of(dl[k] + bias, a.softplus) : 0.f;
      const float su = live ? st * u[k] : 0.f;
      if constexpr (LOCAL) total += st;
      const float stj[4] = {quad_lane<0>(st), quad_lane<1>(st), quad_lane<2>(st), quad_lane<3>(st)};
      const float suj[4] = {quad_lane<0>(su), quad_lane<1>(su), quad_lane<2>(su), quad_lane<3>(su)};
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float B[SPL], C[SPL];
        load_states<SPL>(s_b[buf] + (4 * k + j) * SP + s0, B);
        if constexpr (!LOCAL) load_states<SPL>(s_c[buf] + (4 * k + j) * SP + s0, C);
        p[j] = 0.f;
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
          h[s] = fmaf(__builtin_amdgcn_exp2f(stj[j] * rate[s]), h[s], suj[j] * B[s]);
          if constexpr (!LOCAL) p[j] = fmaf(h[s], C[s], p[j]);
        }
      }
      if constexpr (!LOCAL) {
        float o = fmaf(skip, u[k], quad_sums<LPC>(p[0], p[1], p[2], p[3], at.lane));
        if (gated) o *= z[k] * sigmoid_f32(z[k]);
        if (live && writes) py[tk * a.y_stride[1]] = from_f32<T>(o);
      }
    }
    if (more) {
      rb.store(s_b[buf ^ 1], t + kTile, end, a.S);
      if constexpr (!LOCAL) rc.store(s_c[buf ^ 1], t + kTile, end, a.S);
    }
    __syncthreads();
  }
  if constexpr (LOCAL) {
    total = group_sum<4>(total);   // each quad has all tokens
    const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + at.seg) * a.D + d;
    if (at.in) {
      store_states<SPL>(gm.local + row * SP + s0, h);
      if (at.sq == 0) gm.steps[row] = total;
    }
  } else {
    if (writes)
      for (int t = max(t0, end) + quad; t < t1; t += 4) py[t * a.y_stride[1]] = from_f32<T>(0.f);
    if (a.final && at.seg == gm.segs - 1 && at.in)
      store_user_states<SPL>(a.final + (static_cast<int64_t>(at.b) * a.D + d) * a.S, s0, a.S, h);
  }
}

// The adjoint that leaves a segment through its front for none that enters at its end, and the sum of its steps; for all
// segments but the first.
template <typename T, int SPL, int LPC>
__global__ __launch_bounds__(kScanThreads) void scan_adjoint_kernel(dwarf_selective_scan_bwd_args w, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kQuads = kTile / 4;
  __shared__ __align__(16) float s_c[2][kTile * SP];
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  ScanLane<LPC> at(a, gm, gm.segs - 1);
  at.seg += 1;
  const int s0 = at.sq * SPL, quad = at.lane & 3;
  const int64_t d = at.d;
  const int t0 = at.seg * gm.seg, end = min(min(a.N, t0 + gm.seg), scan_length(a, at.b));
  float rate[SPL], ga[SPL];
  load_rates<SPL>(a.A, d, s0, a.S, rate);
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f;
#pragma unroll
  for (int s = 0; s < SPL; ++s) ga[s] = 0.f;
  const T* pd = static_cast<const T*>(a.delta) + at.b * a.delta_stride[0] + d;
  const T* pz = static_cast<const T*>(a.gate) + at.b * a.gate_stride[0] + d;
  const T* pg = static_cast<const T*>(w.dy) + at.b * w.dy_stride[0] + d;
  const T* pC = static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
  const bool gated = a.gate != nullptr;
  float total = 0.f;
  T rg[kQuads], rd[kQuads], rz[kQuads];
  BcRows<T, SP, kTile> rc;
  auto fetch = [&](int t) {
    rc.load(pC, a.C_stride[1], t, end, a.S);
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int64_t tt = min(t + 4 * k + quad, end - 1);
      rg[k] = pg[tt * w.dy_stride[1]];
      rd[k] = pd[tt * a.delta_stride[1]];
      if (gated) rz[k] = pz[tt * a.gate_stride[1]];
    }
  };
  const int tiles = end > t0 ? (end - t0 + kTile - 1) / kTile : 0;
  int buf = 0;
  if (tiles) {
    fetch(t0 + (tiles - 1) * kTile);
    rc.store(s_c[0], t0 + (tiles - 1) * kTile, end, a.S);
    __syncthreads();
  }
  for (int i = tiles - 1; i >= 0; --i, buf ^= 1) {
    const int t = t0 + i * kTile;
    float dy[kQuads], dl[kQuads], z[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      dy[k] = to_f32(rg[k]);
      dl[k] = to_f32(rd[k]);
      z[k] = gated ? to_f32(rz[k]) : 0.f;
    }
    if (i) fetch(t - kTile);
#pragma unroll
    for (int k = kQuads - 1; k >= 0; --k) {
      const bool live = t + 4 * k + quad < end;
      const float st = live ? step_of(dl[k] + bias, a.softplus) : 0.f;
      const float act = gated ? z[k] * sigmoid_f32(z[k]) : 1.f;
      const float go = live ? dy[k] * act : 0.f;
      total += st;
      const float stj[4] = {quad_lane<0>(st), quad_lane<1>(st), quad_lane<2>(st), quad_lane<3>(st)};
      const float goj[4] = {quad_lane<0>(go), quad_lane<1>(go), quad_lane<2>(go), quad_lane<3>(go)};
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        float C[SPL];
        load_states<SPL>(s_c[buf] + (4 * k + j) * SP + s0, C);
#pragma unroll
        for (int s = 0; s < SPL; ++s) ga[s] = __builtin_amdgcn_exp2f(stj[j] * rate[s]) * fmaf(C[s], goj[j], ga[s]);
      }
    }
    if (i) rc.store(s_c[buf ^ 1], t - kTile, end, a.S);
    __syncthreads();
  }
  total = group_sum<4>(total);
  const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + at.seg) * a.D + d;
  if (at.in) {
    store_states<SPL>(gm.local + row * SP + s0, ga);
    if (at.sq == 0) gm.steps[row] = total;
  }
}

// Sums v[0 .. M-1] over the wave's channels (the lane bits above LPC's); lane l keeps value `which(l)` of them.
template <int LPC, int M>
struct ChannelSums {
  static constexpr int kLeft = M >= 8 ? M / 8 : 1;   // values a lane ends with
  static __device__ __forceinline__ float swap_add32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  static __device__ __forceinline__ float swap_add16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  // out[i] is value which(lane) + i: lane bit 5 chooses between the halves of v, bit 4 between the halves of that, bit 3
  // (where there are more than two left) again
  static __device__ __forceinline__ void sum(const float* v, float* out, int lane) {
    float w[M / 2];
#pragma unroll
    for (int i = 0; i < M / 2; ++i) w[i] = swap_add32(v[i], v[i + M / 2]);
    float x[M / 4];
#pragma unroll
    for (int i = 0; i < M / 4; ++i) x[i] = swap_add16(w[i], w[i + M / 4]);
    if constexpr (M >= 8) {
      const bool up = lane & 8;
#pragma unroll
      for (int i = 0; i < M / 8; ++i) out[i] = (up ? x[i + M / 8] : x[i]) + dpp_f<0x128>(up ? x[i] : x[i + M / 8]);
    } else {
      out[0] = x[0] + dpp_f<0x128>(x[0]);   // row_ror:8
    }
    if constexpr (LPC == 4) {
#pragma unroll
      for (int i = 0; i < kLeft; ++i) out[i] += dpp_f<0x104>(out[i]);   // row_shl:4, for the lanes that write
    }
  }
  static __device__ __forceinline__ int which(int lane) {
    return (lane >> 5 & 1) * (M / 2) + (lane >> 4 & 1) * (M / 4) + (M >= 8 ? (lane >> 3 & 1) * (M / 8) : 0);
  }
  // whether the lane is the one that writes its values
  static __device__ __forceinline__ bool writes(int lane) {
    return (LPC == 8 || !(lane & 4)) && (M >= 8 || !(lane & 8));
  }
};

template <typename T, int SPL, int LPC>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_kernel(dwarf_selective_scan_bwd_args w, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kK = scan_chunk(SPL), kQuads = kK / 4;
  using Sums = ChannelSums<LPC, 2 * SPL>;
  __shared__ __align__(16) float s_b[2][kK * SP], s_c[2][kK * SP];
  __shared__ float s_sum[kScanWaves][kK][2 * SP];
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  const ScanLane<LPC> at(a, gm, gm.segs);
  const int s0 = at.sq * SPL, quad = at.lane & 3;
  const int64_t d = at.d;
  const int t0 = at.seg * gm.seg, t1 = min(a.N, t0 + gm.seg), end = min(t1, scan_length(a, at.b));
  float rate[SPL], ga[SPL];   // ga: a_{t+1} g_{t+1}
  load_rates<SPL>(a.A, d, s0, a.S, rate);
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
  load_user_states<SPL>(w.dfinal ? w.dfinal + (static_cast<int64_t>(at.b) * a.D + d) * a.S : nullptr, s0, a.S, ga);
  for (int i = gm.segs - 1; i > at.seg; --i) {   // the segments behind
    const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + i) * a.D + d;
    float add[SPL];
    load_states<SPL>(gm.local + row * SP + s0, add);
    const float sum = gm.steps[row];
#pragma unroll
    for (int s = 0; s < SPL; ++s) ga[s] = fmaf(__builtin_amdgcn_exp2f(sum * rate[s]), ga[s], add[s]);
  }
  if (!at.in)
#pragma unroll
    for (int s = 0; s < SPL; ++s) ga[s] = 0.f;
  const T* px = static_cast<const T*>(a.x) + at.b * a.x_stride[0] + d;
  const T* pd = static_cast<const T*>(a.delta) + at.b * a.delta_stride[0] + d;
  const T* pz = static_cast<const T*>(a.gate) + at.b * a.gate_stride[0] + d;
  const T* pg = static_cast<const T*>(w.dy) + at.b * w.dy_stride[0] + d;
  const T* pB = static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2];
  const T* pC = static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
  T* ox = static_cast<T*>(w.dx) + at.b * w.dx_stride[0] + d;
  T* od = static_cast<T*>(w.ddelta) + at.b * w.ddelta_stride[0] + d;
  T* oz = static_cast<T*>(w.dgate) + at.b * w.dgate_stride[0] + d;
  const float* ck = a.checkpoints + (static_cast<int64_t>(at.b) * ((a.N + kK - 1) / kK) * a.D + d) * SP + s0;
  const int64_t ck_step = static_cast<int64_t>(a.D) * SP;
  const bool gated = a.gate != nullptr, writes = at.in && at.sq < 4;
  float* part = gm.part + ((static_cast<int64_t>(at.tile % gm.tiles_of_group) * a.B + at.b) * a.N * a.G + at.g) * (2 * SP);
  double dA[SPL], dskip = 0., dbias = 0.;
#pragma unroll
  for (int s = 0; s < SPL; ++s) dA[s] = 0.;
  // behind the live tokens everything is zero
  if (writes)
    for (int t = max(t0, end) + quad; t < t1; t += 4) {
      ox[t * w.dx_stride[1]] = from_f32<T>(0.f);
      od[t * w.ddelta_stride[1]] = from_f32<T>(0.f);
      if (gated) oz[t * w.dgate_stride[1]] = from_f32<T>(0.f);
    }
  for (int64_t i = threadIdx.x + static_cast<int64_t>(max(t0, end)) * (2 * SP); i < static_cast<int64_t>(t1) * (2 * SP); i += kScanThreads)
    part[i / (2 * SP) * a.G * (2 * SP) + i % (2 * SP)] = 0.f;

  T rx[kQuads], rd[kQuads], rz[kQuads], rg[kQuads];
  float hn[SPL];
  BcRows<T, SP, kK> rb, rc;
  auto fetch = [&](int t) {
    rb.load(pB, a.B_stride[1], t, end, a.S);
    rc.load(pC, a.C_stride[1], t, end, a.S);
    load_states<SPL>(ck + t / kK * ck_step, hn);
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int64_t tt = min(t + 4 * k + quad, end - 1);
      rx[k] = px[tt * a.x_stride[1]];
      rd[k] = pd[tt * a.delta_stride[1]];
      rg[k] = pg[tt * w.dy_stride[1]];
      if (gated) rz[k] = pz[tt * a.gate_stride[1]];
    }
  };
  const int chunks = end > t0 ? (end - t0 + kK - 1) / kK : 0;
  int buf = 0;
  if (chunks) {
    fetch(t0 + (chunks - 1) * kK);
    rb.store(s_b[0], t0 + (chunks - 1) * kK, end, a.S);
    rc.store(s_c[0], t0 + (chunks - 1) * kK, end, a.S);
    __syncthreads();
  }
  for (int i = chunks - 1; i >= 0; --i, buf ^= 1) {
    const int t = t0 + i * kK;
    float h0[SPL], u[kQuads], raw[kQuads], z[kQuads], dy[kQuads], st[kQuads], su[kQuads], go[kQuads];
#pragma unroll
    for (int s = 0; s < SPL; ++s) h0[s] = hn[s];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const bool live = t + 4 * k + quad < end && at.in;
      u[k] = live ? to_f32(rx[k]) : 0.f;
      raw[k] = to_f32(rd[k]) + bias;
      dy[k] = live ? to_f32(rg[k]) : 0.f;
      z[k] = gated ? to_f32(rz[k]) : 0.f;
    }
    if (i) fetch(t - kK);
    // the chunk's states again
    float dec[kK][SPL], hs[kK][SPL];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const bool live = t + 4 * k + quad < end && at.in;
      st[k] = live ? step_of(raw[k], a.softplus) : 0.f;
      su[k] = live ? st[k] * u[k] : 0.f;
      go[k] = gated ? (live ? dy[k] * (z[k] * sigmoid_f32(z[k])) : 0.f) : dy[k];
      const float stj[4] = {quad_lane<0>(st[k]), quad_lane<1>(st[k]), quad_lane<2>(st[k]), quad_lane<3>(st[k])};
      const float suj[4] = {quad_lane<0>(su[k]), quad_lane<1>(su[k]), quad_lane<2>(su[k]), quad_lane<3>(su[k])};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = 4 * k + j;
        float B[SPL];
        load_states<SPL>(s_b[buf] + n * SP + s0, B);
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
          dec[n][s] = __builtin_amdgcn_exp2f(stj[j] * rate[s]);
          hs[n][s] = fmaf(dec[n][s], n ? hs[n ? n - 1 : 0][s] : h0[s], suj[j] * B[s]);
        }
      }
    }
    // and back through them
    float cA[SPL], cskip = 0.f, cbias = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) cA[s] = 0.f;
#pragma unroll
    for (int k = kQuads - 1; k >= 0; --k) {
      const float stj[4] = {quad_lane<0>(st[k]), quad_lane<1>(st[k]), quad_lane<2>(st[k]), quad_lane<3>(st[k])};
      const float suj[4] = {quad_lane<0>(su[k]), quad_lane<1>(su[k]), quad_lane<2>(su[k]), quad_lane<3>(su[k])};
      const float goj[4] = {quad_lane<0>(go[k]), quad_lane<1>(go[k]), quad_lane<2>(go[k]), quad_lane<3>(go[k])};
      float into[4], mA[4], o[4];
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int n = 4 * k + j;
        float B[SPL], C[SPL], v[2 * SPL], left[Sums::kLeft];
        load_states<SPL>(s_b[buf] + n * SP + s0, B);
        load_states<SPL>(s_c[buf] + n * SP + s0, C);
        into[j] = mA[j] = o[j] = 0.f;
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
          const float g = fmaf(C[s], goj[j], ga[s]);
          v[s] = g * suj[j];
          v[SPL + s] = goj[j] * hs[n][s];
          into[j] = fmaf(g, B[s], into[j]);
          ga[s] = g * dec[n][s];
          const float m = ga[s] * (n ? hs[n ? n - 1 : 0][s] : h0[s]);
          cA[s] = fmaf(m, stj[j], cA[s]);
          mA[j] = fmaf(m, rate[s], mA[j]);
          if (gated) o[j] = fmaf(hs[n][s], C[s], o[j]);
        }
        Sums::sum(v, left, at.lane);
        if (Sums::writes(at.lane)) {
#pragma unroll
          for (int e = 0; e < Sums::kLeft; ++e) {
            const int q = Sums::which(at.lane) + e;   // dB's states, then dC's
            s_sum[at.wave][n][q / SPL * SP + s0 + q % SPL] = left[e];
          }
        }
      }
      const float gB = quad_sums<LPC>(into[0], into[1], into[2], into[3], at.lane);
      const float gA = quad_sums<LPC>(mA[0], mA[1], mA[2], mA[3], at.lane) * (1.f / kLog2e);
      const int tk = t + 4 * k + quad;
      float dd = tk < end ? fmaf(u[k], gB, gA) : 0.f;   // the adjoint goes on through tokens behind the end, unchanged
      if (a.softplus) dd *= sigmoid_f32(raw[k]);
      cskip = fmaf(go[k], u[k], cskip);
      cbias += dd;
      float dz = 0.f;
      if (gated) {
        const float out = fmaf(skip, u[k], quad_sums<LPC>(o[0], o[1], o[2], o[3], at.lane)), e = sigmoid_f32(z[k]);
        dz = dy[k] * out * (e * fmaf(z[k], 1.f - e, 1.f));
      }
      if (writes && tk < end) {
        ox[tk * w.dx_stride[1]] = from_f32<T>(fmaf(st[k], gB, skip * go[k]));
        od[tk * w.ddelta_stride[1]] = from_f32<T>(dd);
        if (gated) oz[tk * w.dgate_stride[1]] = from_f32<T>(dz);
      }
    }
#pragma unroll
    for (int s = 0; s < SPL; ++s) dA[s] += cA[s];
    if (at.in) {   // lanes behind the group's end have computed its last channel's steps
      dskip += cskip;
      dbias += cbias;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kK * 2 * SP; e += kScanThreads) {
      const int n = e / (2 * SP), q = e % (2 * SP);
      if (t + n < end) {
        float x = s_sum[0][n][q];
#pragma unroll
        for (int v = 1; v < kScanWaves; ++v) x += s_sum[v][n][q];
        part[static_cast<int64_t>(t + n) * a.G * (2 * SP) + q] = x;
      }
    }
    if (i) {
      rb.store(s_b[buf ^ 1], t - kK, end, a.S);
      rc.store(s_c[buf ^ 1], t - kK, end, a.S);
    }
    __syncthreads();
  }
  if (!at.in) return;
  const int64_t row = static_cast<int64_t>(at.b) * gm.segs + at.seg;
  if (w.dinitial && at.seg == 0)
    store_user_states<SPL>(w.dinitial + (static_cast<int64_t>(at.b) * a.D + d) * a.S, s0, a.S, ga);
  float sA[SPL];
#pragma unroll
  for (int s = 0; s < SPL; ++s) sA[s] = static_cast<float>(dA[s]);
  store_states<SPL>(gm.part_A + (row * a.D + d) * SP + s0, sA);
  // the quad's tokens, in order; each quad of a channel has them all
  const float ks = group_sum<4>(static_cast<float>(dskip)), kb = group_sum<4>(static_cast<float>(dbias));
  if (at.sq == 0) {
    gm.part_d[(row * 2) * a.D + d] = ks;
    gm.part_d[(row * 2 + 1) * a.D + d] = kb;
  }
}

// dB and dC: the channel tiles' partial rows in order.  One thread to (token, group, B or C, state).
template <typename T>
__global__ __launch_bounds__(256) void scan_sum_rows(const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC,
                                                     int64_t rows, int tiles, int SP, int S) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * 2 * SP) return;
  float x = 0.f;
#pragma unroll 8
  for (int k = 0; k < tiles; ++k) x += part[k * rows * 2 * SP + i];
  const int64_t row = i / (2 * SP);
  const int q = static_cast<int>(i - row * (2 * SP)), s = q < SP ? q : q - SP;
  if (s < S) (q < SP ? dB : dC)[row * S + s] = from_f32<T>(x);
}

// dA, dskip, ddelta_bias: the batches' and segments' partials in order, in 64 bits.
__global__ __launch_bounds__(256) void scan_sum_channels(const float* __restrict__ part_A, const float* __restrict__ part_d,
                                                         float* __restrict__ dA, float* __restrict__ dskip,
                                                         float* __restrict__ dbias, int D, int SP, int S, int parts) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, nA = static_cast<int64_t>(D) * SP;
  double x = 0.;
  if (i < nA) {
    const int s = static_cast<int>(i % SP);
    if (!dA || s >= S) return;
    for (int k = 0; k < parts; ++k) x += part_A[k * nA + i];
    dA[i / SP * S + s] = static_cast<float>(x);
  } else if (i < nA + 2 * D) {
    const int64_t q = i - nA;
    float* out = q < D ? dskip : dbias;
    if (!out) return;
    for (int k = 0; k < parts; ++k) x += part_d[k * 2 * static_cast<int64_t>(D) + q];
    out[q % D] = static_cast<float>(x);
  }
}

// One token of each row.  The first row of a slot takes the slot's later rows after it, in order.
template <typename T, int SPL, int LPC>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(dwarf_selective_scan_step_args a, int tiles_of_group) {
  __shared__ int s_next;
  constexpr int kCh = kWave / LPC;
  const int lane = threadIdx.x % kWave, sq = lane % LPC, s0 = sq * SPL, per = a.D / a.G;
  const int tiles = tiles_of_group * a.G, tile = blockIdx.x % tiles, row0 = blockIdx.x / tiles, g = tile / tiles_of_group;
  const int c = tile % tiles_of_group * (kScanWaves * kCh) + threadIdx.x / kWave * kCh + lane / LPC;
  const bool in = c < per;
  const int64_t d = g * per + (in ? c : per - 1);
  const int slot = a.slots ? a.slots[row0] : row0;
  if (slot < 0 || slot >= a.pool) {   // uniform
    if (in && sq == 0) static_cast<T*>(a.out)[row0 * a.out_stride + d] = from_f32<T>(0.f);
    return;
  }
  const int64_t at = slot * a.slot_stride + d * a.S;
  float h[SPL], rate[SPL], B[SPL], C[SPL], x, raw, z = 0.f;
  load_user_states<SPL>(a.state + at, s0, a.S, h);   // under way while the slots are looked through
  auto fetch = [&](int row) {
    x = to_f32(static_cast<const T*>(a.x)[row * a.x_stride + d]);
    raw = to_f32(static_cast<const T*>(a.delta)[row * a.delta_stride + d]);
    if (a.gate) z = to_f32(static_cast<const T*>(a.gate)[row * a.gate_stride + d]);
    const T* pB = static_cast<const T*>(a.Bm) + row * a.B_stride[0] + g * a.B_stride[1];
    const T* pC = static_cast<const T*>(a.Cm) + row * a.C_stride[0] + g * a.C_stride[1];
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      B[s] = s0 + s < a.S ? to_f32(pB[s0 + s]) : 0.f;
      C[s] = s0 + s < a.S ? to_f32(pC[s0 + s]) : 0.f;
    }
  };
  fetch(row0);
  load_rates<SPL>(a.A, d, s0, a.S, rate);
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
  if (row0 > 0 && a.slots && next_row_of<kScanThreads>(a.slots, slot, 0, a.R, &s_next) < row0) return;   // uniform
  for (int row = row0; row < a.R;) {
    const float st = step_of(raw + bias, a.softplus), su = st * x;
    float p = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      h[s] = fmaf(__builtin_amdgcn_exp2f(st * rate[s]), h[s], su * B[s]);
      p = fmaf(h[s], C[s], p);
    }
    float o = fmaf(skip, x, lanes_sum<LPC>(p));
    if (a.gate) o *= z * sigmoid_f32(z);
    if (in && sq == 0) static_cast<T*>(a.out)[row * a.out_stride + d] = from_f32<T>(o);
    row = a.slots && row + 1 < a.R ? next_row_of<kScanThreads>(a.slots, slot, row + 1, a.R, &s_next) : a.R;
    if (row < a.R) fetch(row);
  }
  if (in) store_user_states<SPL>(a.new_state + at, s0, a.S, h);
}

int scan_tile_channels(int S) { return kScanWaves * (kWave / scan_lpc(S)); }
int scan_padded(int S) { return scan_spl(S) * scan_lpc(S); }

ScanGeom scan_geom(const dwarf_selective_scan_fwd_args& a) {
  ScanGeom gm{};
  const int per = a.D / a.G, ch = scan_tile_channels(a.S);
  gm.tiles_of_group = (per + ch - 1) / ch;
  gm.tiles = gm.tiles_of_group * a.G;
  const int64_t groups = static_cast<int64_t>(a.B) * gm.tiles;
  // One segment where the workgroups (four waves, one for each vector unit of a CU) leave at most a quarter of the 256 CUs
  // without any; otherwise segments for two workgroups a CU, of at least two units.
  int64_t segs = groups >= 192 ? 1 : (512 + groups - 1) / groups;
  const int64_t most = a.N / (2 * kSegmentUnit);
  if (segs > most) segs = most;
  if (segs > kMaxSegments) segs = kMaxSegments;
  if (segs < 1) segs = 1;
  gm.seg = static_cast<int>(((a.N + segs - 1) / segs + kSegmentUnit - 1) / kSegmentUnit * kSegmentUnit);
  if (gm.seg < kSegmentUnit) gm.seg = kSegmentUnit;
  gm.segs = a.N > 0 ? (a.N + gm.seg - 1) / gm.seg : 1;
  return gm;
}

size_t local_floats(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm) {
  return gm.segs > 1 ? static_cast<size_t>(a.B) * gm.segs * a.D * scan_padded(a.S) : 0;
}
size_t step_floats(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm) {
  return gm.segs > 1 ? (static_cast<size_t>(a.B) * gm.segs * a.D + 3) / 4 * 4 : 0;
}

template <typename T, int SPL, int LPC>
void scan_fwd_typed(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm, hipStream_t stream) {
  const unsigned each = static_cast<unsigned>(a.B) * gm.tiles;
  if (gm.segs > 1)
    hipLaunchKernelGGL((scan_fwd_kernel<T, SPL, LPC, true>), dim3(each * (gm.segs - 1)), dim3(kScanThreads), 0, stream, a, gm);
  hipLaunchKernelGGL((scan_fwd_kernel<T, SPL, LPC, false>), dim3(each * gm.segs), dim3(kScanThreads), 0, stream, a, gm);
}

template <typename T, int SPL, int LPC>
void scan_bwd_typed(const dwarf_selective_scan_bwd_args& w, const ScanGeom& gm, hipStream_t stream) {
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  const unsigned each = static_cast<unsigned>(a.B) * gm.tiles;
  constexpr int SP = SPL * LPC;
  if (gm.segs > 1)
    hipLaunchKernelGGL((scan_adjoint_kernel<T, SPL, LPC>), dim3(each * (gm.segs - 1)), dim3(kScanThreads), 0, stream, w, gm);
  hipLaunchKernelGGL((scan_bwd_kernel<T, SPL, LPC>), dim3(each * gm.segs), dim3(kScanThreads), 0, stream, w, gm);
  const int64_t rows = static_cast<int64_t>(a.B) * a.N * a.G;
  if (rows)
    hipLaunchKernelGGL((scan_sum_rows<T>), dim3(static_cast<unsigned>((rows * 2 * SP + 255) / 256)), dim3(256), 0, stream,
                       gm.part, static_cast<T*>(w.dB), static_cast<T*>(w.dC), rows, gm.tiles_of_group, SP, a.S);
  if (w.dA || w.dskip || w.ddelta_bias)
    hipLaunchKernelGGL(scan_sum_channels, dim3(static_cast<unsigned>((static_cast<int64_t>(a.D) * (SP + 2) + 255) / 256)),
                       dim3(256), 0, stream, gm.part_A, gm.part_d, w.dA, w.dskip, w.ddelta_bias, a.D, SP, a.S, a.B * gm.segs);
}

template <typename T, int SPL, int LPC>
void scan_step_typed(const dwarf_selective_scan_step_args& a, hipStream_t stream) {
  const int per = a.D / a.G, ch = scan_tile_channels(a.S), tiles = (per + ch - 1) / ch;
  hipLaunchKernelGGL((scan_step_kernel<T, SPL, LPC>), dim3(static_cast<unsigned>(a.R) * tiles * a.G), dim3(kScanThreads), 0,
                     stream, a, tiles);
}

#define DWARF_SCAN_SHAPES(T, S, CALL)   \
  if ((S) <= 8) CALL(T, 2, 4);          \
  else if ((S) <= 16) CALL(T, 4, 4);    \
  else if ((S) <= 32) CALL(T, 8, 4);    \
  else CALL(T, 8, 8)
#define DWARF_SCAN_TYPES(dtype, S, CALL)                              \
  if ((dtype) == DWARF_F32) { DWARF_SCAN_SHAPES(float, S, CALL); }    \
  else if ((dtype) == DWARF_F16) { DWARF_SCAN_SHAPES(f16, S, CALL); } \
  else { DWARF_SCAN_SHAPES(bf16, S, CALL); }

}  // namespace

int64_t selective_scan_workgroups(const dwarf_selective_scan_fwd_args& a) {
  const ScanGeom gm = scan_geom(a);
  return static_cast<int64_t>(a.B) * gm.tiles * gm.segs;
}

size_t selective_scan_checkpoints(const dwarf_selective_scan_fwd_args& a) {
  const int chunk = scan_chunk(scan_spl(a.S));
  return static_cast<size_t>(a.B) * ((a.N + chunk - 1) / chunk) * a.D * scan_padded(a.S) * sizeof(float);
}

size_t selective_scan_fwd_workspace(const dwarf_selective_scan_fwd_args& a) {
  const ScanGeom gm = scan_geom(a);
  return (local_floats(a, gm) + step_floats(a, gm)) * sizeof(float);
}

hipError_t launch_selective_scan_fwd(const dwarf_selective_scan_fwd_args& a, hipStream_t stream) {
  ScanGeom gm = scan_geom(a);
  gm.local = static_cast<float*>(a.workspace);
  gm.steps = gm.local + local_floats(a, gm);
#define DWARF_SCAN_CALL(T, SPL, LPC) scan_fwd_typed<T, SPL, LPC>(a, gm, stream)
  DWARF_SCAN_TYPES(a.dtype, a.S, DWARF_SCAN_CALL)
#undef DWARF_SCAN_CALL
  return hipGetLastError();
}

size_t selective_scan_bwd_workspace(const dwarf_selective_scan_bwd_args& w) {
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  const ScanGeom gm = scan_geom(a);
  const size_t SP = scan_padded(a.S), parts = static_cast<size_t>(a.B) * gm.segs;
  return (local_floats(a, gm) + step_floats(a, gm) + static_cast<size_t>(gm.tiles_of_group) * a.B * a.N * a.G * 2 * SP +
          parts * a.D * SP + parts * 2 * a.D) * sizeof(float);
}

hipError_t launch_selective_scan_bwd(const dwarf_selective_scan_bwd_args& w, hipStream_t stream) {
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  ScanGeom gm = scan_geom(a);
  const size_t SP = scan_padded(a.S), parts = static_cast<size_t>(a.B) * gm.segs;
  gm.local = static_cast<float*>(w.workspace);
  gm.steps = gm.local + local_floats(a, gm);
  gm.part = gm.steps + step_floats(a, gm);
  gm.part_A = gm.part + static_cast<size_t>(gm.tiles_of_group) * a.B * a.N * a.G * 2 * SP;
  gm.part_d = gm.part_A + parts * a.D * SP;
#define DWARF_SCAN_CALL(T, SPL, LPC) scan_bwd_typed<T, SPL, LPC>(w, gm, stream)
  DWARF_SCAN_TYPES(a.dtype, a.S, DWARF_SCAN_CALL)
#undef DWARF_SCAN_CALL
  return hipGetLastError();
}

hipError_t launch_selective_scan_step(const dwarf_selective_scan_step_args& a, hipStream_t stream) {
#define DWARF_SCAN_CALL(T, SPL, LPC) scan_step_typed<T, SPL, LPC>(a, stream)
  DWARF_SCAN_TYPES(a.dtype, a.S, DWARF_SCAN_CALL)
#undef DWARF_SCAN_CALL
  return hipGetLastError();
}

}  // namespace dwarf
