// The selective scan: for each channel with its S states
//   step = softplus(delta + bias) (or without the softplus),  a = exp(step A)
//   h_t = a_t h_{t-1} + step_t x_t B_t,   o_t = C_t . h_t + skip x_t,   y_t = o_t silu(gate_t)
// and, with do = dy silu(gate) and g the adjoint of h,
//   g_t = C_t do_t + a_{t+1} g_{t+1},   m_t = g_t a_t h_{t-1}
//   dx = step (g.B) + skip do,   dstep = x (g.B) + m.A,   dA = sum m step
//   dB = sum_channels g step x,   dC = sum_channels do h,   dgate = dy o silu'(gate)
//
// Nothing here is a product of matrices: each (token, channel, state) has a
// decay of its own, one exponential and four multiply-adds forward, 13 backward,
// and that, not memory, bounds the kernels.  At B15 N2048, 1,024 channels of 16
// states in bf16 (503 million of them): forward 187 us, 252 MB of rows and 126
// MB of checkpoints; backward 503 us; the vector units issue in 72 and 76% of
// the waves' cycles, and of those 62 and 55% are the operations above (79 and
// 197 us at an instruction every 4 cycles, 8 for the exponential, and 2.34
// GHz).  The clock rises for some 20 passes; the comparisons below are of 12,
// 205 and 540 us in all then.  So the work is laid out for the vector units: LPC adjacent lanes share a channel,
// SPL states in the registers of each, and a wave holds 64 / LPC channels.  The
// quads of lanes divide what a channel has once for each token (softplus, silu,
// loads, stores) by taking one of four tokens each; a token's step reaches the
// other lanes as a DPP operand.  B and C are staged in LDS as fp32, one read for
// a lane's SPL states.  A wave has a vector unit nearly to itself, so waits are
// not hidden by other waves: rows of the next tile are under way and the next
// quad's steps are formed while a quad is worked on, and results are stored
// while the next tile is (forward 403 us without, backward 841).
//
// A sequence is one segment where the channels alone fill the vector units;
// else it is cut into segments, which a launch in front reduces to the state
// that each adds from zero and the sum of its steps (a segment's decay is
// exp(A sum)); the rows' workgroups join the segments in front of their own
// themselves (B1 N65536, 1,024 channels: 32 segments, 233 and 313 us, the vector
// units busy 90 and 87% of that).  The backward does the same with the adjoint,
// from the end.
//
// The backward walks chunks from the last to the first: it forms a chunk's
// states again from the checkpoint the forward left in front of it, keeps them
// and the decays in registers and walks back through them.  dB and dC are sums
// over channels: over a wave's by lane exchanges (by fp32 matrix instructions
// the kernel took 744 us), over a workgroup's waves in LDS, over workgroups by
// partial rows that a last launch adds in order (12 us).
// Nothing is atomic: the same bits every time.  dA, dskip and the bias's
// gradient, sums over all tokens, run in 64 bits from a chunk on.
#include <utility>

#include "selective.h"

namespace dwarf {
namespace {

constexpr int kScanWaves = 4, kScanThreads = kScanWaves * kWave;
constexpr int kTile = 32;           // tokens in LDS at a time, forward
constexpr int kMaxSegments = 64;
constexpr int kSegmentUnit = 32, kSegmentLeast = 64;   // tokens a segment is a multiple of, and has at least

// States per lane and lanes per channel for S states.
constexpr int scan_spl(int S) { return S <= 8 ? 2 : S <= 16 ? 4 : 8; }
constexpr int scan_lpc(int S) { return S <= 32 ? 4 : 8; }
// Tokens of the rows' tiles forward: twice as many where two workgroups still share a CU's LDS with them (a tile's barrier and
// the waits behind it take 3% of the time in 64 tokens, 6 in 32: B15 N2048, 1,024 channels of 16 states in bf16 205 us, not 211;
// the segments' sums have too many registers for it: 340 us, not 260, for B1 N65536).
template <typename T, int SP, bool WIDE>
constexpr int scan_rows_tile() { return WIDE && sizeof(T) == 2 && SP <= 16 ? 2 * kTile : kTile; }
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

// Lane j's value of each quad; j is known once loops are unrolled.  Next to what uses it, it is no instruction of its own
// but an operand's.
__device__ __forceinline__ float quad_lane(float x, int j) {
  if (j == 0) return dpp_f<0x00>(x);
  if (j == 1) return dpp_f<0x55>(x);
  if (j == 2) return dpp_f<0xAA>(x);
  return dpp_f<0xFF>(x);
}

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

// e^x with the argument's rounding to base 2 made up for: 2^-23 off at most (plus the instruction's own last bit).
__device__ __forceinline__ float exp_f32(float x) {
  const float h = x * kLog2e;
  const float lo = fmaf(x, 1.92596299e-8f, fmaf(x, kLog2e, -h));   // log2(e) - kLog2e
  return __builtin_amdgcn_exp2f(h) * fmaf(lo, 0.693147181f, 1.f);
}

// log(1 + e^x) without a branch.  log(w) / (w - 1) changes slowly around the rounded w = 1 + e (and is 1 where w is next to
// 1), so that times the exact e it is right however small e is: 3.5e-7 off at most over [-30, 21], 8e-8 on average.  Above 20
// it is x, below -200, minus infinity included, 0.  (The library's calls, with their branches, took half of the forward's
// instructions.)
struct Softplus {
  float e, above;
  __device__ __forceinline__ explicit Softplus(float x)
      : e(exp_f32(__builtin_amdgcn_fmed3f(x, -200.f, 20.f))), above((x < 20.f ? 20.f : x) - 20.f) {}   // NaN for a NaN
  __device__ __forceinline__ float value() const {
    const float w = fmaxf(1.f + e, 1.00000012f);
    return fmaf(__builtin_amdgcn_logf(w) * 0.693147181f, e * __builtin_amdgcn_rcpf(w - 1.f), above);
  }
  __device__ __forceinline__ float slope() const { return e * __builtin_amdgcn_rcpf(1.f + e); }   // 1 / (1 + e^-x)
};
// Chosen, not branched to: both sides are formed first.  A branch for each quad of tokens keeps the compiler from working on
// several of them at once.
__device__ __forceinline__ float step_of(float raw, bool softplus) {
  const float s = Softplus(raw).value();
  return softplus ? s : raw;
}
// What step_of makes a step of 0 of.
__device__ __forceinline__ float no_step(bool softplus) { return softplus ? -1e4f : 0.f; }
// silu(z), or 1 without a gate.
__device__ __forceinline__ float act_of(float z, bool gated) {
  const float s = z * sigmoid_f32(z);
  return gated ? s : 1.f;
}

// Where a lane stands.
template <int LPC>
struct ScanLane {
  static constexpr int kCh = kWave / LPC;              // channels of a wave
  static constexpr int kTileCh = kScanWaves * kCh;     // of a workgroup
  int lane, wave, sq, b, seg, tile, g, d;
  int local, first, behind;   // the lane's channel in the tile; the tile's first channel, and the one behind its group
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
    const int per = a.D / a.G, c = tile % gm.tiles_of_group * kTileCh;
    local = wave * kCh + lane / LPC;
    first = g * per + c;
    behind = g * per + per;
    in = first + local < behind;
    d = in ? first + local : behind - 1;
  }
};

__device__ __forceinline__ int scan_length(const dwarf_selective_scan_fwd_args& a, int b) {
  if (!a.lengths) return a.N;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.N ? a.N : n;
}

// Rows are addressed by a base that all threads share, which walks with the tiles, and 32-bit byte offsets of the threads
// (the host keeps token strides below 2^22 elements).  Tokens behind the live ones read the last live one again: an offset is
// at most `limit`, one instruction, where a second path for a sequence's last tile would make the compiler wait for its loads
// where the paths meet.
constexpr uint32_t kNoLimit = 0xffffffffu;

// B or C rows of TOK tokens, as the workgroup's threads carry them into LDS: raw in registers between.
template <typename T, int SP, int TOK>
struct BcRows {
  static_assert(TOK * SP % kScanThreads == 0 && kScanThreads % SP == 0, "whole rows, each thread one state");
  static constexpr int kEach = TOK * SP / kScanThreads, kRows = kScanThreads / SP;
  const char* base;   // the tile's first row
  uint32_t stride, state, off;   // bytes: of a token, of the thread's state, of its first row and state
  T v[kEach];
  __device__ __forceinline__ BcRows(const T* p, int64_t stride_, int t, int S)
      : base(reinterpret_cast<const char*>(p + t * stride_)), stride(static_cast<uint32_t>(stride_) * sizeof(T)) {
    const uint32_t s = threadIdx.x % SP;
    state = (s < static_cast<uint32_t>(S) ? s : 0) * sizeof(T);
    off = threadIdx.x / SP * stride + state;
  }
  __device__ __forceinline__ void move(int tiles) { base += tiles * (TOK * static_cast<int64_t>(stride)); }
  __device__ __forceinline__ void load(int live) {   // of the tile's rows
    const uint32_t limit = live < TOK ? (live - 1) * stride + state : kNoLimit;
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = *reinterpret_cast<const T*>(base + min(off + e * (kRows * stride), limit));
  }
  // rows from `live` on and states from S on are zero
  __device__ __forceinline__ void store(float* to, int live, int S) const {
    const bool in = static_cast<int>(threadIdx.x % SP) < S;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      to[e * kScanThreads + threadIdx.x] = in && static_cast<int>(threadIdx.x / SP) + e * kRows < live ? to_f32(v[e]) : 0.f;
  }
};

// A lane's tokens of a channel, one of each quad of a tile of 4 QUADS.
template <typename T, int QUADS>
struct QuadRows {
  char* base;   // the tile's first token
  uint32_t stride, channel, off;   // bytes: of a token, of the channel, of the lane's first token and channel
  __device__ __forceinline__ QuadRows(const void* p, int64_t sequence, int64_t stride_, int64_t d, int t, int quad)
      : base(reinterpret_cast<char*>(static_cast<T*>(const_cast<void*>(p)) + sequence + t * stride_)),
        stride(static_cast<uint32_t>(stride_) * sizeof(T)), channel(static_cast<uint32_t>(d) * sizeof(T)) {
    off = quad * stride + channel;
  }
  __device__ __forceinline__ void move(int tiles) { base += tiles * (4 * QUADS * static_cast<int64_t>(stride)); }
  __device__ __forceinline__ void load(T* v, int live) const {   // of the tile's tokens
    const uint32_t limit = live < 4 * QUADS ? (live - 1) * stride + channel : kNoLimit;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) v[k] = *reinterpret_cast<const T*>(base + min(off + k * (4 * stride), limit));
  }
  __device__ __forceinline__ void store(const float* x) const {
#pragma unroll
    for (int k = 0; k < QUADS; ++k) *reinterpret_cast<T*>(base + (off + k * (4 * stride))) = from_f32<T>(x[k]);
  }
  __device__ __forceinline__ void store(const float* x, int quad, int live) const {
#pragma unroll
    for (int k = 0; k < QUADS; ++k)
      if (4 * k + quad < live) *reinterpret_cast<T*>(base + (off + k * (4 * stride))) = from_f32<T>(x[k]);
  }
};

// Zeros in a channel's tokens `from` to `to`.
template <typename T>
__device__ __forceinline__ void clear_rows(const void* p, int64_t at, int64_t stride, int quad, int from, int to) {
  T* q = static_cast<T*>(const_cast<void*>(p)) + at;
  for (int t = from + quad; t < to; t += 4) q[t * stride] = from_f32<T>(0.f);
}

// A workgroup's tiles [TOK][kCh] of NS inputs, and of NS outputs.
//
// WIDE: the workgroup's threads carry whole rows of the tile between memory and LDS, 16 bytes a thread and access; a lane
// then takes its channel's element from LDS.  A lane's own accesses, where rows are not aligned to 16 bytes, are 2 bytes
// from four rows to a quad, sixteen places a wave's access, which kept the CU's address unit busy for a fifth of the time
// (forward; B15 N2048, 1,024 channels in bf16).  In LDS the vectors of a row are turned by the row, so that the four rows that
// a wave reads together lie in different banks.
template <typename T, int LPC>
struct ScanTile {
  static constexpr int kCh = ScanLane<LPC>::kTileCh, kVe = 16 / sizeof(T), kNv = kCh / kVe;
  static constexpr int kApart = 256 / (kCh * static_cast<int>(sizeof(T)));   // rows until a bank comes again
  static constexpr int kWaveVecs = kCh / kScanWaves / kVe;
  static __device__ __forceinline__ int turned(int row, int vec) {
    return kApart >= 4 ? vec : vec ^ ((row & 3) / (kApart < 4 ? kApart : 4) * kWaveVecs);
  }
  // a lane's element of its first row
  static __device__ __forceinline__ int spot(int quad, int local) {
    return quad * kCh + turned(quad, local / kVe) * kVe + local % kVe;
  }
};

typedef uint32_t Chunk __attribute__((ext_vector_type(4)));   // 16 bytes of a row

struct ScanRows {   // of one input or output
  const void* p;   // nullptr: none
  int64_t sequence, stride;
};

template <typename T, int TOK, int LPC, int NS>
struct WideRows {
  using Tile = ScanTile<T, LPC>;
  static constexpr int kVecs = TOK * Tile::kNv, kAll = NS * kVecs, kEach = (kAll + kScanThreads - 1) / kScanThreads;
  char* at[kEach];       // the thread's vectors of the tile
  int64_t stride[kEach]; // bytes of a token
  int row[kEach], spot[kEach];
  bool ok[kEach];        // the vector is one of the tile's and its group's
  __device__ __forceinline__ WideRows(const ScanRows* rows, const ScanLane<LPC>& lane, int D, int t) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kScanThreads + threadIdx.x, which = min(i / kVecs, NS - 1), vec = i % Tile::kNv;
      row[e] = i % kVecs / Tile::kNv;
      spot[e] = which * (TOK * Tile::kCh) + row[e] * Tile::kCh + Tile::turned(row[e], vec) * Tile::kVe;
      const int c = lane.first + vec * Tile::kVe;
      const void* p = nullptr;
      int64_t sequence = 0, step = 0;
#pragma unroll
      for (int n = 0; n < NS; ++n)
        if (which == n) p = rows[n].p, sequence = rows[n].sequence, step = rows[n].stride;
      ok[e] = i < kAll && p && c < lane.behind;
      if (!p) p = rows[0].p, sequence = rows[0].sequence, step = rows[0].stride;   // loads have to go somewhere
      stride[e] = step * static_cast<int64_t>(sizeof(T));
      at[e] = reinterpret_cast<char*>(static_cast<T*>(const_cast<void*>(p)) + sequence + (t + row[e]) * step + min(c, D - Tile::kVe));
    }
  }
  __device__ __forceinline__ void move(int tiles) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) at[e] += tiles * (TOK * stride[e]);
  }
};

template <typename T, int TOK, int LPC, int NS, bool WIDE>
struct ScanIn {   // WIDE
  WideRows<T, TOK, LPC, NS> rows;
  Chunk v[WideRows<T, TOK, LPC, NS>::kEach];
  T* lds;
  int mine;
  static constexpr int kSpan = NS * TOK * ScanTile<T, LPC>::kCh;   // of one of the two buffers
  __device__ __forceinline__ ScanIn(const ScanRows* in, const ScanLane<LPC>& lane, int D, int t, T* lds_)
      : rows(in, lane, D, t), lds(lds_), mine(ScanTile<T, LPC>::spot(lane.lane & 3, lane.local)) {}
  __device__ __forceinline__ void move(int tiles) { rows.move(tiles); }
  __device__ __forceinline__ void fetch(int live) {
#pragma unroll
    for (int e = 0; e < rows.kEach; ++e) {
      const int over = rows.row[e] - live + 1;   // rows behind the live ones
      v[e] = *reinterpret_cast<const Chunk*>(rows.at[e] - (over > 0 ? over : 0) * rows.stride[e]);
    }
  }
  __device__ __forceinline__ void put(int buf) const {
#pragma unroll
    for (int e = 0; e < rows.kEach; ++e)
      if (rows.kAll % kScanThreads == 0 || e * kScanThreads + static_cast<int>(threadIdx.x) < rows.kAll)
        *reinterpret_cast<Chunk*>(lds + buf * kSpan + rows.spot[e]) = v[e];
  }
  __device__ __forceinline__ float get(int which, int buf, int k) const {
    return to_f32(lds[buf * kSpan + which * (TOK * ScanTile<T, LPC>::kCh) + 4 * k * ScanTile<T, LPC>::kCh + mine]);
  }
};

template <typename T, int TOK, int LPC, int NS>
struct ScanIn<T, TOK, LPC, NS, false> {
  static constexpr int kSpan = 8;   // no LDS
  QuadRows<T, TOK / 4> q[NS];
  bool given[NS];
  T r[NS][TOK / 4];
  float v[NS][TOK / 4];
  template <int... I>
  __device__ __forceinline__ ScanIn(const ScanRows* in, const ScanLane<LPC>& lane, int t, std::integer_sequence<int, I...>)
      : q{QuadRows<T, TOK / 4>(in[I].p, in[I].sequence, in[I].stride, lane.d, t, lane.lane & 3)...}, given{in[I].p != nullptr...} {}
  __device__ __forceinline__ ScanIn(const ScanRows* in, const ScanLane<LPC>& lane, int, int t, T*)
      : ScanIn(in, lane, t, std::make_integer_sequence<int, NS>()) {}
  __device__ __forceinline__ void move(int tiles) {
#pragma unroll
    for (int n = 0; n < NS; ++n) q[n].move(tiles);
  }
  __device__ __forceinline__ void fetch(int live) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (given[n]) q[n].load(r[n], live);   // uniform
  }
  __device__ __forceinline__ void put(int) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int k = 0; k < TOK / 4; ++k) v[n][k] = to_f32(r[n][k]);
  }
  __device__ __forceinline__ float get(int which, int, int k) const { return v[which][k]; }
};

template <typename T, int TOK, int LPC, int NS, bool WIDE>
struct ScanOut {   // WIDE
  WideRows<T, TOK, LPC, NS> rows;
  T* lds;
  int mine;
  static constexpr int kSpan = NS * TOK * ScanTile<T, LPC>::kCh;
  __device__ __forceinline__ ScanOut(const ScanRows* out, const ScanLane<LPC>& lane, int D, int t, T* lds_)
      : rows(out, lane, D, t), lds(lds_), mine(ScanTile<T, LPC>::spot(lane.lane & 3, lane.local)) {}
  __device__ __forceinline__ void move(int tiles) { rows.move(tiles); }
  __device__ __forceinline__ void put(int which, int buf, int k, float x) {
    lds[buf * kSpan + which * (TOK * ScanTile<T, LPC>::kCh) + 4 * k * ScanTile<T, LPC>::kCh + mine] = from_f32<T>(x);
  }
  // Behind a barrier: the tile's live rows, in two parts, so that other work lies between.
  Chunk held[WideRows<T, TOK, LPC, NS>::kEach];
  __device__ __forceinline__ void collect(int buf) {
#pragma unroll
    for (int e = 0; e < rows.kEach; ++e)
      if (rows.kAll % kScanThreads == 0 || rows.ok[e]) held[e] = *reinterpret_cast<const Chunk*>(lds + buf * kSpan + rows.spot[e]);
  }
  __device__ __forceinline__ void send(int live) const {
#pragma unroll
    for (int e = 0; e < rows.kEach; ++e)
      if (rows.ok[e] && rows.row[e] < live) *reinterpret_cast<Chunk*>(rows.at[e]) = held[e];
  }
};

template <typename T, int TOK, int LPC, int NS>
struct ScanOut<T, TOK, LPC, NS, false> {
  static constexpr int kSpan = 8;
  QuadRows<T, TOK / 4> q[NS];
  bool given[NS];
  float v[NS][TOK / 4];
  template <int... I>
  __device__ __forceinline__ ScanOut(const ScanRows* out, const ScanLane<LPC>& lane, int t, std::integer_sequence<int, I...>)
      : q{QuadRows<T, TOK / 4>(out[I].p, out[I].sequence, out[I].stride, lane.d, t, lane.lane & 3)...}, given{out[I].p != nullptr...} {}
  __device__ __forceinline__ ScanOut(const ScanRows* out, const ScanLane<LPC>& lane, int, int t, T*)
      : ScanOut(out, lane, t, std::make_integer_sequence<int, NS>()) {}
  __device__ __forceinline__ void move(int tiles) {
#pragma unroll
    for (int n = 0; n < NS; ++n) q[n].move(tiles);
  }
  __device__ __forceinline__ void put(int which, int, int k, float x) { v[which][k] = x; }
  __device__ __forceinline__ void flush(int live, const ScanLane<LPC>& lane) const {
    if (!lane.in || lane.sq >= 4) return;   // the channel's first quad stores
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (!given[n]) continue;
      if (live >= TOK) q[n].store(v[n]);
      else q[n].store(v[n], lane.lane & 3, live);
    }
  }
};

template <int SPL>
__device__ __forceinline__ void scaled(float f, const float* x, float* y) {
#pragma unroll
  for (int s = 0; s < SPL; ++s) y[s] = f * x[s];
}
template <int SPL>
__device__ __forceinline__ void decays(float step, const float* rate, float* dec) {
  scaled<SPL>(step, rate, dec);
#pragma unroll
  for (int s = 0; s < SPL; ++s) dec[s] = __builtin_amdgcn_exp2f(dec[s]);
}

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

// A in base 2, so that the decay is one exp2; finite where A is minus infinity, so that a step of 0 decays nothing.
__device__ __forceinline__ float rate_of(float A) {
  const float r = A * kLog2e;
  return r < -3.4e38f ? -3.4e38f : r;
}
template <int SPL>
__device__ __forceinline__ void load_rates(const float* A, int64_t d, int s0, int S, float* rate) {
#pragma unroll
  for (int s = 0; s < SPL; ++s) rate[s] = s0 + s < S ? rate_of(A[d * S + s0 + s]) : 0.f;
}

// The state (or adjoint) behind a segment from the one in front: nothing stays nothing, also where a growing segment's
// factor is out of range.
__device__ __forceinline__ float joined(float h, float sum, float rate, float add) {
  return h == 0.f ? add : fmaf(__builtin_amdgcn_exp2f(sum * rate), h, add);
}

// LOCAL: what a segment adds from zero and its sum of steps, for all segments but the last; otherwise the rows.
template <typename T, int SPL, int LPC, bool WIDE, bool LOCAL>
__global__ __launch_bounds__(kScanThreads) __attribute__((amdgpu_waves_per_eu(1, 2))) void scan_fwd_kernel(dwarf_selective_scan_fwd_args a, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kTok = LOCAL ? kTile : scan_rows_tile<T, SP, WIDE>(), kQuads = kTok / 4, kK = scan_chunk(SPL);
  __shared__ __align__(16) float s_b[2][kTok * SP];
  __shared__ __align__(16) float s_c[LOCAL ? 1 : 2][LOCAL ? 4 : kTok * SP];
  constexpr int kIns = LOCAL ? 2 : 3;
  __shared__ __align__(16) T s_in[2 * ScanIn<T, kTok, LPC, kIns, WIDE>::kSpan];
  __shared__ __align__(16) T s_out[LOCAL ? 8 : 2 * ScanOut<T, kTok, LPC, 1, WIDE>::kSpan];
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
      for (int s = 0; s < SPL; ++s) h[s] = joined(h[s], sum, rate[s], add[s]);
    }
  }
  const bool gated = !LOCAL && a.gate, writes = at.in && at.sq < 4;
  const bool softplus = a.softplus;
  const float none = no_step(softplus);
  const ScanRows ins[3] = {{a.x, at.b * a.x_stride[0], a.x_stride[1]}, {a.delta, at.b * a.delta_stride[0], a.delta_stride[1]},
                           {gated ? a.gate : nullptr, at.b * a.gate_stride[0], a.gate_stride[1]}};
  const ScanRows outs[1] = {{a.y, at.b * a.y_stride[0], a.y_stride[1]}};
  ScanIn<T, kTok, LPC, kIns, WIDE> in(ins, at, a.D, t0, s_in);
  ScanOut<T, kTok, LPC, 1, WIDE> out(outs, at, a.D, t0, s_out);
  BcRows<T, SP, kTok> rb(static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2], a.B_stride[1], t0, a.S);
  BcRows<T, SP, kTok> rc(static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2], a.C_stride[1], t0, a.S);
  float* ck = !LOCAL && a.checkpoints && at.in
                  ? a.checkpoints + ((static_cast<int64_t>(at.b) * ((a.N + kK - 1) / kK) + t0 / kK) * a.D + d) * SP + s0 : nullptr;
  const int64_t ck_step = static_cast<int64_t>(a.D) * SP;
  float total = 0.f;
  auto fetch = [&](int live) {   // the tile's first `live` tokens are live
    rb.load(live);
    if constexpr (!LOCAL) rc.load(live);
    in.fetch(live);
  };
  auto take = [&](int to, int live) {
    rb.store(s_b[to], live, a.S);
    if constexpr (!LOCAL) rc.store(s_c[to], live, a.S);
    in.put(to);
  };
  int buf = 0;
  if (t0 < end) {   // around the loop too: one that might not run would wait inside for what is loaded in front of it
    fetch(end - t0);
    take(0, end - t0);
    __syncthreads();
    for (int t = t0; t < end; t += kTok, buf ^= 1) {
      const bool more = t + kTok < end;
      if (more) {   // under way while this tile is worked on
        rb.move(1);
        rc.move(1);
        in.move(1);
        fetch(end - t - kTok);
      }
      // A quad at a time; the next one's rows and steps are formed meanwhile, from values read one quad earlier yet: the compiler
      // waits where it reads.
      float B[2][4 * SPL], C[2][4 * SPL], st[2], su[2], u[2], act[2], vx[2], vd[2], vz[2];
      auto look = [&](int k) {
        const int i = k & 1;
        vx[i] = in.get(0, buf, k), vd[i] = in.get(1, buf, k);
        if constexpr (!LOCAL) vz[i] = in.get(2, buf, k);
      };
      auto begin = [&](int k) {
        const int i = k & 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          load_states<SPL>(s_b[buf] + (4 * k + j) * SP + s0, B[i] + j * SPL);
          if constexpr (!LOCAL) load_states<SPL>(s_c[buf] + (4 * k + j) * SP + s0, C[i] + j * SPL);
        }
        const bool live = t + 4 * k + quad < end;
        u[i] = live ? vx[i] : 0.f;
        st[i] = step_of(live ? vd[i] + bias : none, softplus);
        su[i] = st[i] * u[i];
        if constexpr (LOCAL) total += st[i];
        else act[i] = act_of(vz[i], gated);
      };
      look(0);
      if constexpr (WIDE && !LOCAL)
        if (t > t0) out.collect(buf ^ 1);   // the tile in front, which was whole
      begin(0);
      look(1);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        if (!LOCAL && 4 * k % kK == 0) {
          if (ck && t + 4 * k < end) store_states<SPL>(ck, h);
          ck += ck ? ck_step : 0;
        }
        __builtin_amdgcn_sched_barrier(0);
        if (k + 1 < kQuads) begin(k + 1);
        if (k + 2 < kQuads) look(k + 2);
        const int i = k & 1;
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float dec[SPL], add[SPL];
          decays<SPL>(quad_lane(st[i], j), rate, dec);
          scaled<SPL>(quad_lane(su[i], j), B[i] + j * SPL, add);
          p[j] = 0.f;
#pragma unroll
          for (int s = 0; s < SPL; ++s) {
            h[s] = fmaf(dec[s], h[s], add[s]);
            if constexpr (!LOCAL) p[j] = fmaf(h[s], C[i][j * SPL + s], p[j]);
          }
        }
        if constexpr (!LOCAL)
          out.put(0, buf, k, fmaf(skip, u[i], quad_sums<LPC>(p[0], p[1], p[2], p[3], at.lane)) * act[i]);
      }
      if constexpr (WIDE && !LOCAL)
        if (t > t0) {
          out.send(kTok);
          out.move(1);
        }
      // The next tile's values are waited for in front of this one's stores: loads and stores are counted together, and
      // waiting behind them would wait for the stores too (an eighth of the time).
      if (more) take(buf ^ 1, end - t - kTok);
      __syncthreads();   // one barrier a tile: what it lets through writes the other buffers
      if constexpr (!WIDE && !LOCAL) {
        out.flush(end - t, at);
        out.move(1);
      }
    }
    if constexpr (WIDE && !LOCAL) {
      out.collect(buf ^ 1);
      out.send(end - t0 - (end - t0 - 1) / kTok * kTok);
    }
  }
  if constexpr (LOCAL) {
    total = group_sum<4>(total);   // each quad has all tokens
    const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + at.seg) * a.D + d;
    if (at.in) {
      store_states<SPL>(gm.local + row * SP + s0, h);
      if (at.sq == 0) gm.steps[row] = total;
    }
  } else {
    if (writes) clear_rows<T>(a.y, at.b * a.y_stride[0] + d, a.y_stride[1], quad, max(t0, end), t1);
    if (a.final && at.seg == gm.segs - 1 && at.in)
      store_user_states<SPL>(a.final + (static_cast<int64_t>(at.b) * a.D + d) * a.S, s0, a.S, h);
  }
}

// The adjoint that leaves a segment through its front for none that enters at its end, and the sum of its steps; for all
// segments but the first.
template <typename T, int SPL, int LPC, bool WIDE>
__global__ __launch_bounds__(kScanThreads) __attribute__((amdgpu_waves_per_eu(1, 2))) void scan_adjoint_kernel(dwarf_selective_scan_bwd_args w, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kQuads = kTile / 4;
  __shared__ __align__(16) float s_c[2][kTile * SP];
  __shared__ __align__(16) T s_in[2 * ScanIn<T, kTile, LPC, 3, WIDE>::kSpan];
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
  const bool gated = a.gate != nullptr;
  const bool softplus = a.softplus;
  const float none = no_step(softplus);
  const int tiles = end > t0 ? (end - t0 + kTile - 1) / kTile : 0, last = t0 + (tiles - 1) * kTile;
  const ScanRows ins[3] = {{w.dy, at.b * w.dy_stride[0], w.dy_stride[1]}, {a.delta, at.b * a.delta_stride[0], a.delta_stride[1]},
                           {a.gate, at.b * a.gate_stride[0], a.gate_stride[1]}};
  ScanIn<T, kTile, LPC, 3, WIDE> in(ins, at, a.D, last, s_in);
  BcRows<T, SP, kTile> rc(static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2], a.C_stride[1], last, a.S);
  float total = 0.f;
  int buf = 0;
  if (tiles) {
    rc.load(end - last);
    in.fetch(end - last);
    rc.store(s_c[0], end - last, a.S);
    in.put(0);
    __syncthreads();
    for (int i = tiles - 1; i >= 0; --i, buf ^= 1) {
      const int t = t0 + i * kTile;
      if (i) {   // all tiles in front of the last are whole
        rc.move(-1);
        in.move(-1);
        rc.load(kTile);
        in.fetch(kTile);
      }
      float C[2][4 * SPL], st[2], go[2], vg[2], vd[2], vz[2];
      auto look = [&](int k) {
        const int m = k & 1;
        vg[m] = in.get(0, buf, k), vd[m] = in.get(1, buf, k), vz[m] = in.get(2, buf, k);
      };
      auto begin = [&](int k) {
        const int m = k & 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) load_states<SPL>(s_c[buf] + (4 * k + j) * SP + s0, C[m] + j * SPL);
        const bool live = t + 4 * k + quad < end;
        st[m] = step_of(live ? vd[m] + bias : none, softplus);
        go[m] = (live ? vg[m] : 0.f) * act_of(live && gated ? vz[m] : 0.f, gated);
        total += st[m];
      };
      look(kQuads - 1);
      begin(kQuads - 1);
      look(kQuads - 2);
#pragma unroll
      for (int k = kQuads - 1; k >= 0; --k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k) begin(k - 1);
        if (k > 1) look(k - 2);
        const int m = k & 1;
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          float dec[SPL];
          decays<SPL>(quad_lane(st[m], j), rate, dec);
          const float goj = quad_lane(go[m], j);
#pragma unroll
          for (int s = 0; s < SPL; ++s) ga[s] = fmaf(goj, C[m][j * SPL + s], ga[s]);
#pragma unroll
          for (int s = 0; s < SPL; ++s) ga[s] *= dec[s];
        }
      }
      if (i) {
        rc.store(s_c[buf ^ 1], kTile, a.S);
        in.put(buf ^ 1);
      }
      __syncthreads();
    }
  }
  total = group_sum<4>(total);
  const int64_t row = (static_cast<int64_t>(at.b) * gm.segs + at.seg) * a.D + d;
  if (at.in) {
    store_states<SPL>(gm.local + row * SP + s0, ga);
    if (at.sq == 0) gm.steps[row] = total;
  }
}

template <int N>
__device__ __forceinline__ void store_left(float* p, const float* x) {
  if constexpr (N == 1) p[0] = x[0];
  else if constexpr (N == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  else *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

// Sums v[0 .. 2 SPL - 1] over the wave's channels, the lane bits above LPC's: bit 5 and bit 4 each leave a lane with half of
// the values and add those of two lanes, bit 3 adds.  With four lanes to a channel bit 2 is left to the sum over the waves:
// there an addition takes a thread's, here every lane's turn.
template <int SPL, int LPC>
struct ChannelSums {
  static constexpr int M = 2 * SPL, kLeft = M / 4;   // values a lane ends with
  static constexpr int kParts = LPC == 4 ? 2 : 1;    // partial sums a wave leaves
  static __device__ __forceinline__ float swap_add32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  static __device__ __forceinline__ float swap_add16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  // out[i] is value which(lane) + i
  static __device__ __forceinline__ void sum(const float* v, float* out) {
    float w[M / 2];
#pragma unroll
    for (int i = 0; i < M / 2; ++i) w[i] = swap_add32(v[i], v[i + M / 2]);
#pragma unroll
    for (int i = 0; i < M / 4; ++i) {
      const float x = swap_add16(w[i], w[i + M / 4]);
      out[i] = x + dpp_f<0x128>(x);   // row_ror:8
    }
  }
  static __device__ __forceinline__ int which(int lane) { return (lane >> 5 & 1) * (M / 2) + (lane >> 4 & 1) * (M / 4); }
  static __device__ __forceinline__ int part(int lane) { return kParts == 2 ? lane >> 2 & 1 : 0; }
};

template <typename T, int SPL, int LPC, bool WIDE>
__global__ __launch_bounds__(kScanThreads) __attribute__((amdgpu_waves_per_eu(1, 2))) void scan_bwd_kernel(dwarf_selective_scan_bwd_args w, ScanGeom gm) {
  constexpr int SP = SPL * LPC, kK = scan_chunk(SPL), kQuads = kK / 4;
  using Sums = ChannelSums<SPL, LPC>;
  __shared__ __align__(16) float s_b[2][kK * SP], s_c[2][kK * SP];
  __shared__ __align__(16) float s_sum[2][kScanWaves][kK][Sums::kParts][2 * SP];
  __shared__ __align__(16) T s_in[2 * ScanIn<T, kK, LPC, 4, WIDE>::kSpan];
  __shared__ __align__(16) T s_out[2 * ScanOut<T, kK, LPC, 3, WIDE>::kSpan];
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
    for (int s = 0; s < SPL; ++s) ga[s] = joined(ga[s], sum, rate[s], add[s]);
  }
  if (!at.in)
#pragma unroll
    for (int s = 0; s < SPL; ++s) ga[s] = 0.f;
  const bool gated = a.gate != nullptr, writes = at.in && at.sq < 4;
  const bool softplus = a.softplus;
  const float none = no_step(softplus);
  const int chunks = end > t0 ? (end - t0 + kK - 1) / kK : 0, last = t0 + (chunks - 1) * kK;
  const ScanRows ins[4] = {{a.x, at.b * a.x_stride[0], a.x_stride[1]}, {a.delta, at.b * a.delta_stride[0], a.delta_stride[1]},
                           {w.dy, at.b * w.dy_stride[0], w.dy_stride[1]}, {a.gate, at.b * a.gate_stride[0], a.gate_stride[1]}};
  const ScanRows outs[3] = {{w.dx, at.b * w.dx_stride[0], w.dx_stride[1]}, {w.ddelta, at.b * w.ddelta_stride[0], w.ddelta_stride[1]},
                            {gated ? w.dgate : nullptr, at.b * w.dgate_stride[0], w.dgate_stride[1]}};
  ScanIn<T, kK, LPC, 4, WIDE> in(ins, at, a.D, last, s_in);
  ScanOut<T, kK, LPC, 3, WIDE> out(outs, at, a.D, last, s_out);
  BcRows<T, SP, kK> rb(static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2], a.B_stride[1], last, a.S);
  BcRows<T, SP, kK> rc(static_cast<const T*>(a.Cm) + at.b * a.C_stride[0] + at.g * a.C_stride[2], a.C_stride[1], last, a.S);
  const float* ck = a.checkpoints + ((static_cast<int64_t>(at.b) * ((a.N + kK - 1) / kK) + last / kK) * a.D + d) * SP + s0;
  const int64_t ck_step = static_cast<int64_t>(a.D) * SP;
  float* part = gm.part + ((static_cast<int64_t>(at.tile % gm.tiles_of_group) * a.B + at.b) * a.N * a.G + at.g) * (2 * SP);
  const int64_t part_step = static_cast<int64_t>(a.G) * (2 * SP);   // from token to token
  double dA[SPL], dskip = 0., dbias = 0.;
#pragma unroll
  for (int s = 0; s < SPL; ++s) dA[s] = 0.;
  // behind the live tokens everything is zero
  if (writes) {
    clear_rows<T>(w.dx, outs[0].sequence + d, outs[0].stride, quad, max(t0, end), t1);
    clear_rows<T>(w.ddelta, outs[1].sequence + d, outs[1].stride, quad, max(t0, end), t1);
    if (gated) clear_rows<T>(w.dgate, outs[2].sequence + d, outs[2].stride, quad, max(t0, end), t1);
  }
  for (int i = threadIdx.x / (2 * SP) + max(t0, end); i < t1; i += kScanThreads / (2 * SP))
    part[i * part_step + threadIdx.x % (2 * SP)] = 0.f;

  float hn[SPL];
  // lanes with the same sum write it alike
  const int place = Sums::part(at.lane) * (2 * SP) + Sums::which(at.lane) / SPL * SP + s0 + Sums::which(at.lane) % SPL;
  // A chunk's results go to memory while the next one is worked on: read from LDS behind the barrier, stored later.
  constexpr int kSums = kK * 2 * SP / kScanThreads, kSumTokens = kScanThreads / (2 * SP);   // of a thread; of all at once
  float* sums_to = part + (last + static_cast<int>(threadIdx.x) / (2 * SP)) * part_step + threadIdx.x % (2 * SP);
  float sums[kSums][kScanWaves * Sums::kParts];
  auto collect = [&](int from) {
#pragma unroll
    for (int e = 0; e < kSums; ++e)
#pragma unroll
      for (int v = 0; v < kScanWaves * Sums::kParts; ++v) {
        const int at_ = e * kScanThreads + threadIdx.x;
        sums[e][v] = s_sum[from][v / Sums::kParts][at_ / (2 * SP)][v % Sums::kParts][at_ % (2 * SP)];
      }
    if constexpr (WIDE) out.collect(from);
  };
  auto send = [&](int live) {   // of chunk after chunk, from the last
#pragma unroll
    for (int e = 0; e < kSums; ++e) {
      float x = sums[e][0];
#pragma unroll
      for (int v = 1; v < kScanWaves * Sums::kParts; ++v) x += sums[e][v];
      if (e * kSumTokens + static_cast<int>(threadIdx.x) / (2 * SP) < live) sums_to[e * kSumTokens * part_step] = x;
    }
    sums_to -= kK * part_step;
    if constexpr (WIDE) {
      out.send(live);
      out.move(-1);
    }
  };
  int buf = 0;
  if (chunks) {
    load_states<SPL>(ck, hn);
    rb.load(end - last);
    rc.load(end - last);
    in.fetch(end - last);
    rb.store(s_b[0], end - last, a.S);
    rc.store(s_c[0], end - last, a.S);
    in.put(0);
    __syncthreads();
    for (int i = chunks - 1; i >= 0; --i, buf ^= 1) {
      const int t = t0 + i * kK;
      float h0[SPL], u[kQuads], raw[kQuads], z[kQuads], dy[kQuads], st[kQuads], slope[kQuads], su[kQuads], go[kQuads];
#pragma unroll
      for (int s = 0; s < SPL; ++s) h0[s] = hn[s];
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const bool live = t + 4 * k + quad < end && at.in;
        const float vx = in.get(0, buf, k), vd = in.get(1, buf, k) + bias, vg = in.get(2, buf, k), vz = in.get(3, buf, k);
        u[k] = live ? vx : 0.f;
        raw[k] = live ? vd : none;
        slope[k] = live ? 1.f : 0.f;   // the adjoint goes on through tokens behind the end, unchanged
        dy[k] = live ? vg : 0.f;
        z[k] = live && gated ? vz : 0.f;
      }
      if (i) {   // under way while this chunk is worked on; all chunks in front of the last are whole
        ck -= ck_step;
        rb.move(-1);
        rc.move(-1);
        in.move(-1);
        load_states<SPL>(ck, hn);
        rb.load(kK);
        rc.load(kK);
        in.fetch(kK);
      }
      if (i + 1 < chunks) collect(buf ^ 1);   // the chunk behind
      // the chunk's states again; the next quad's rows are read meanwhile
      float dec[kK][SPL], hs[kK][SPL], R[2][4 * SPL];
      auto begin = [&](int k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load_states<SPL>(s_b[buf] + (4 * k + j) * SP + s0, R[k & 1] + j * SPL);
        const Softplus sp(raw[k]);
        const float s = sp.value(), d = sp.slope();
        st[k] = softplus ? s : raw[k];
        slope[k] = softplus ? d : slope[k];
        su[k] = st[k] * u[k];
        go[k] = dy[k] * act_of(z[k], gated);
      };
      begin(0);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k + 1 < kQuads) begin(k + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = 4 * k + j;
          float add[SPL];
          decays<SPL>(quad_lane(st[k], j), rate, dec[n]);
          scaled<SPL>(quad_lane(su[k], j), R[k & 1] + j * SPL, add);
#pragma unroll
          for (int s = 0; s < SPL; ++s) hs[n][s] = fmaf(dec[n][s], n ? hs[n ? n - 1 : 0][s] : h0[s], add[s]);
        }
      }
#pragma unroll
      for (int s = 0; s < SPL; ++s) asm volatile("" : "+v"(hs[kK - 1][s]));   // the pass ends here, not behind the branch
      if (i + 1 < chunks) send(min(kK, end - t - kK));
      // and back through them; the rows of the two tokens in front are read meanwhile
      float cA[SPL], cskip = 0.f, cbias = 0.f, B[2][2 * SPL], C[2][2 * SPL];
#pragma unroll
      for (int s = 0; s < SPL; ++s) cA[s] = 0.f;
      auto rows = [&](int pair) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          load_states<SPL>(s_b[buf] + (2 * pair + j) * SP + s0, B[pair & 1] + j * SPL);
          load_states<SPL>(s_c[buf] + (2 * pair + j) * SP + s0, C[pair & 1] + j * SPL);
        }
      };
      rows(kK / 2 - 1);
#pragma unroll
      for (int k = kQuads - 1; k >= 0; --k) {
        // other values to the compiler than the first pass's: their way to a quad's lanes is an operand's again, not kept
        asm("" : "+v"(st[k]), "+v"(su[k]));
        float into[4], mA[4], o[4];
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const int n = 4 * k + j, pair = n / 2;
          if (n % 2) {
            __builtin_amdgcn_sched_barrier(0);
            if (pair) rows(pair - 1);
          }
          const float* Bn = B[pair & 1] + n % 2 * SPL;
          const float* Cn = C[pair & 1] + n % 2 * SPL;
          float g[SPL], m[SPL], v[2 * SPL], left[Sums::kLeft];
          const float goj = quad_lane(go[k], j);
#pragma unroll
          for (int s = 0; s < SPL; ++s) g[s] = fmaf(goj, Cn[s], ga[s]);
          scaled<SPL>(goj, hs[n], v + SPL);
          scaled<SPL>(quad_lane(su[k], j), g, v);
#pragma unroll
          for (int s = 0; s < SPL; ++s) {
            ga[s] = g[s] * dec[n][s];
            m[s] = ga[s] * (n ? hs[n ? n - 1 : 0][s] : h0[s]);
          }
          const float stj = quad_lane(st[k], j);
#pragma unroll
          for (int s = 0; s < SPL; ++s) cA[s] = fmaf(stj, m[s], cA[s]);
          into[j] = mA[j] = o[j] = 0.f;
#pragma unroll
          for (int s = 0; s < SPL; ++s) {
            into[j] = fmaf(g[s], Bn[s], into[j]);
            mA[j] = fmaf(m[s], rate[s], mA[j]);
            o[j] = fmaf(hs[n][s], Cn[s], o[j]);
          }
          Sums::sum(v, left);
          store_left<Sums::kLeft>(&s_sum[buf][at.wave][n][0][0] + place, left);   // dB's states, then dC's
        }
        const float gB = quad_sums<LPC>(into[0], into[1], into[2], into[3], at.lane);
        const float gA = quad_sums<LPC>(mA[0], mA[1], mA[2], mA[3], at.lane) * (1.f / kLog2e);
        const float scanned = fmaf(skip, u[k], quad_sums<LPC>(o[0], o[1], o[2], o[3], at.lane)), e = sigmoid_f32(z[k]);
        // Chosen, not multiplied by a slope of 0: a token without a step passes its state on, whose share in the step's gradient
        // is out of range where a rate is minus infinity.  (A delta that is not a number has a slope of 0 too, but no step of 0.)
        const bool still = st[k] == 0.f && slope[k] == 0.f;
        const float dd = still ? 0.f : fmaf(u[k], gB, gA) * slope[k];
        cskip = fmaf(go[k], u[k], cskip);
        cbias += dd;
#pragma unroll
        for (int s = 0; s < SPL; ++s) asm("" : "+v"(cA[s]));   // summed here, not behind the chunk from products kept until then
        out.put(0, buf, k, fmaf(st[k], gB, skip * go[k]));
        out.put(1, buf, k, dd);
        out.put(2, buf, k, dy[k] * scanned * (e * fmaf(z[k], 1.f - e, 1.f)));
      }
      // the next chunk's values are waited for in front of this one's stores, as forward
      if (i) {
        rb.store(s_b[buf ^ 1], kK, a.S);
        rc.store(s_c[buf ^ 1], kK, a.S);
        in.put(buf ^ 1);
      }
#pragma unroll
      for (int s = 0; s < SPL; ++s) dA[s] += cA[s];
      dskip += cskip;
      dbias += cbias;
      __syncthreads();   // one barrier a chunk: what it lets through writes the other buffers
      if constexpr (!WIDE) {
        out.flush(end - t, at);
        out.move(-1);
      }
    }
    collect(buf ^ 1);
    send(min(kK, end - t0));
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

// The last launch, in two parts.  The first row_blocks workgroups add dB and dC, the channel tiles' partial rows in order, a
// thread to (token, group, B or C, state).  The others add dA, dskip and the bias's gradient, the batches' and segments'
// partials, in 64 bits: 32 values each, eight threads to a value, each every eighth partial in order, then the eight (by one
// thread B1 N2048, 128 partials, took 8 us).
constexpr int kSumCols = 32, kSumRows = 256 / kSumCols;
struct ScanSums {
  const float* part; const float* part_A; const float* part_d;
  void* dB; void* dC;
  float* dA; float* dskip; float* dbias;
  int64_t rows;
  int tiles, row_blocks, parts, D, SP, S;
};
template <typename T>
__global__ __launch_bounds__(256) void scan_sum_kernel(ScanSums a) {
  __shared__ double s_part[kSumRows][kSumCols];
  if (static_cast<int>(blockIdx.x) < a.row_blocks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, each = a.rows * 2 * a.SP;
    if (i >= each) return;
    float x = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.tiles; ++k) x += a.part[k * each + i];
    const int64_t row = i / (2 * a.SP);
    const int q = static_cast<int>(i - row * (2 * a.SP)), s = q < a.SP ? q : q - a.SP;
    if (s < a.S) static_cast<T*>(q < a.SP ? a.dB : a.dC)[row * a.S + s] = from_f32<T>(x);
    return;
  }
  const int col = threadIdx.x % kSumCols, first = threadIdx.x / kSumCols;
  const int64_t i = static_cast<int64_t>(blockIdx.x - a.row_blocks) * kSumCols + col, nA = static_cast<int64_t>(a.D) * a.SP;
  const bool in_A = i < nA, in = i < nA + 2 * static_cast<int64_t>(a.D);
  const int64_t q = i - nA, step = in_A ? nA : 2 * static_cast<int64_t>(a.D);
  const float* p = in_A ? a.part_A + i : a.part_d + q;
  double x = 0.;
  if (in)
#pragma unroll 8
    for (int k = first; k < a.parts; k += kSumRows) x += p[k * step];
  s_part[first][col] = x;
  __syncthreads();
  if (first || !in) return;
#pragma unroll
  for (int r = 1; r < kSumRows; ++r) x += s_part[r][col];
  const int s = static_cast<int>(i % a.SP);
  if (in_A) {
    if (a.dA && s < a.S) a.dA[i / a.SP * a.S + s] = static_cast<float>(x);
  } else if (float* out = q < a.D ? a.dskip : a.dbias) {
    out[q % a.D] = static_cast<float>(x);
  }
}

// One token of each row, bound by the pool's memory (256 rows of 1,024 channels of 16 states: 11.6 us, 34 MB at 3.0 TB/s; one
// row 3.4 us): a lane reads and writes its SPL states of a channel as 16-byte vectors
// where the pool allows them (WHOLE: S states to a channel fill the lanes, slots are aligned), B and C likewise.  The first
// row of a slot takes the slot's later rows after it, in order.
template <typename T, int SPL, int LPC, bool WHOLE>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(dwarf_selective_scan_step_args a, int tiles_of_group) {
  __shared__ int s_found[2];
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
  if constexpr (WHOLE) load_states<SPL>(a.state + at + s0, h);   // under way while the slots are looked through
  else load_user_states<SPL>(a.state + at, s0, a.S, h);
  auto fetch = [&](int row) {
    x = to_f32(static_cast<const T*>(a.x)[row * a.x_stride + d]);
    raw = to_f32(static_cast<const T*>(a.delta)[row * a.delta_stride + d]);
    if (a.gate) z = to_f32(static_cast<const T*>(a.gate)[row * a.gate_stride + d]);
    const T* pB = static_cast<const T*>(a.Bm) + row * a.B_stride[0] + g * a.B_stride[1] + s0;
    const T* pC = static_cast<const T*>(a.Cm) + row * a.C_stride[0] + g * a.C_stride[1] + s0;
    if constexpr (WHOLE) {
      T vB[SPL], vC[SPL];
      __builtin_memcpy(vB, pB, sizeof(vB));   // gfx950 loads vectors from any address
      __builtin_memcpy(vC, pC, sizeof(vC));
#pragma unroll
      for (int s = 0; s < SPL; ++s) B[s] = to_f32(vB[s]), C[s] = to_f32(vC[s]);
    } else {
#pragma unroll
      for (int s = 0; s < SPL; ++s) {
        B[s] = s0 + s < a.S ? to_f32(pB[s]) : 0.f;
        C[s] = s0 + s < a.S ? to_f32(pC[s]) : 0.f;
      }
    }
  };
  fetch(row0);
  if constexpr (WHOLE) {
    __builtin_memcpy(rate, a.A + d * a.S + s0, sizeof(rate));
#pragma unroll
    for (int s = 0; s < SPL; ++s) rate[s] = rate_of(rate[s]);
  } else {
    load_rates<SPL>(a.A, d, s0, a.S, rate);
  }
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
  const bool softplus = a.softplus, gated = a.gate != nullptr;
  SameSlot same{false, a.R};
  if (a.slots) same = same_slot<kScanThreads>(a.slots, slot, row0, a.R, s_found);
  if (same.before) return;   // uniform
  for (int row = row0; row < a.R;) {
    const float st = step_of(raw + bias, softplus), su = st * x;
    float p = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      h[s] = fmaf(__builtin_amdgcn_exp2f(st * rate[s]), h[s], su * B[s]);
      p = fmaf(h[s], C[s], p);
    }
    const float o = fmaf(skip, x, lanes_sum<LPC>(p)) * act_of(z, gated);
    if (in && sq == 0) static_cast<T*>(a.out)[row * a.out_stride + d] = from_f32<T>(o);
    row = same.next;
    if (row < a.R) {
      same = same_slot<kScanThreads>(a.slots, slot, row, a.R, s_found);
      fetch(row);
    }
  }
  if (!in) return;
  if constexpr (WHOLE) store_states<SPL>(a.new_state + at + s0, h);
  else store_user_states<SPL>(a.new_state + at, s0, a.S, h);
}

int scan_tile_channels(int S) { return kScanWaves * (kWave / scan_lpc(S)); }
int scan_padded(int S) { return scan_spl(S) * scan_lpc(S); }

ScanGeom scan_geom(const dwarf_selective_scan_fwd_args& a) {
  ScanGeom gm{};
  const int per = a.D / a.G, ch = scan_tile_channels(a.S);
  gm.tiles_of_group = (per + ch - 1) / ch;
  gm.tiles = gm.tiles_of_group * a.G;
  const int64_t groups = static_cast<int64_t>(a.B) * gm.tiles;
  // One segment from three quarters of a workgroup (four waves, one for each vector unit) a CU on: more cost most of the
  // forward's work a second time.  Below that, segments for two workgroups a CU, which share it up to 256 registers: the
  // forward's rows of up to 16 states (of 32 where they are aligned and of 16 bits), the segments' sums of up to 8 (of 16 where
  // aligned and of 16 bits).  The others, every backward kernel among them, run in two rounds.  Against segments for one
  // workgroup a CU, 1,024 channels, us:
  //   states, type   B1 N65536 forward   B2 N2048 with gradients
  //   16 bf16         544 against   642   150 against 150
  //   16 fp32         613 against   668   160 against 151
  //   32 bf16         992 against 1,076   252 against 244
  //   32 fp32       1,104 against 1,094   270 against 247
  //   64 bf16       2,182 against 2,175   490 against 474
  //   64 fp32       2,174 against 2,162   483 against 467
  int64_t segs = groups >= 192 ? 1 : 512 / groups;
  if (segs > kMaxSegments) segs = kMaxSegments;
  gm.seg = static_cast<int>((a.N + segs - 1) / segs + kSegmentUnit - 1) / kSegmentUnit * kSegmentUnit;
  if (gm.seg < kSegmentLeast) gm.seg = kSegmentLeast;
  gm.segs = a.N > 0 ? (a.N + gm.seg - 1) / gm.seg : 1;
  return gm;
}

size_t local_floats(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm) {
  return gm.segs > 1 ? static_cast<size_t>(a.B) * gm.segs * a.D * scan_padded(a.S) : 0;
}
size_t step_floats(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm) {
  return gm.segs > 1 ? (static_cast<size_t>(a.B) * gm.segs * a.D + 3) / 4 * 4 : 0;
}

// Whether rows can be taken 16 bytes at a time: all of them aligned, the groups' channels whole vectors.
bool wide_rows(const void* p, const int64_t (&stride)[2], int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride[0] * es % 16 == 0 && stride[1] * es % 16 == 0;
}
bool scan_wide(const dwarf_selective_scan_fwd_args& a) {
  const int es = a.dtype == DWARF_F32 ? 4 : 2;
  return (a.D / a.G) % (16 / es) == 0 && wide_rows(a.x, a.x_stride, es) && wide_rows(a.delta, a.delta_stride, es) &&
         (!a.gate || wide_rows(a.gate, a.gate_stride, es));
}

template <typename T, int SPL, int LPC, bool WIDE>
void scan_fwd_laid(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm, hipStream_t stream) {
  const unsigned each = static_cast<unsigned>(a.B) * gm.tiles;
  if (gm.segs > 1)
    hipLaunchKernelGGL((scan_fwd_kernel<T, SPL, LPC, WIDE, true>), dim3(each * (gm.segs - 1)), dim3(kScanThreads), 0, stream, a, gm);
  hipLaunchKernelGGL((scan_fwd_kernel<T, SPL, LPC, WIDE, false>), dim3(each * gm.segs), dim3(kScanThreads), 0, stream, a, gm);
}
template <typename T, int SPL, int LPC>
void scan_fwd_typed(const dwarf_selective_scan_fwd_args& a, const ScanGeom& gm, hipStream_t stream) {
  if (scan_wide(a) && wide_rows(a.y, a.y_stride, sizeof(T))) scan_fwd_laid<T, SPL, LPC, true>(a, gm, stream);
  else scan_fwd_laid<T, SPL, LPC, false>(a, gm, stream);
}

template <typename T, int SPL, int LPC, bool WIDE>
void scan_bwd_laid(const dwarf_selective_scan_bwd_args& w, const ScanGeom& gm, hipStream_t stream) {
  const unsigned each = static_cast<unsigned>(w.fwd.B) * gm.tiles;
  if (gm.segs > 1)
    hipLaunchKernelGGL((scan_adjoint_kernel<T, SPL, LPC, WIDE>), dim3(each * (gm.segs - 1)), dim3(kScanThreads), 0, stream, w, gm);
  hipLaunchKernelGGL((scan_bwd_kernel<T, SPL, LPC, WIDE>), dim3(each * gm.segs), dim3(kScanThreads), 0, stream, w, gm);
}
template <typename T, int SPL, int LPC>
void scan_bwd_typed(const dwarf_selective_scan_bwd_args& w, const ScanGeom& gm, hipStream_t stream) {
  const dwarf_selective_scan_fwd_args& a = w.fwd;
  constexpr int SP = SPL * LPC, es = sizeof(T);
  if (scan_wide(a) && wide_rows(w.dy, w.dy_stride, es) && wide_rows(w.dx, w.dx_stride, es) && wide_rows(w.ddelta, w.ddelta_stride, es) &&
      (!a.gate || wide_rows(w.dgate, w.dgate_stride, es)))
    scan_bwd_laid<T, SPL, LPC, true>(w, gm, stream);
  else
    scan_bwd_laid<T, SPL, LPC, false>(w, gm, stream);
  const int64_t rows = static_cast<int64_t>(a.B) * a.N * a.G;
  const int row_blocks = static_cast<int>((rows * 2 * SP + 255) / 256);
  const int sum_blocks = w.dA || w.dskip || w.ddelta_bias
                             ? static_cast<int>((static_cast<int64_t>(a.D) * (SP + 2) + kSumCols - 1) / kSumCols) : 0;
  if (row_blocks + sum_blocks)
    hipLaunchKernelGGL((scan_sum_kernel<T>), dim3(row_blocks + sum_blocks), dim3(256), 0, stream,
                       ScanSums{gm.part, gm.part_A, gm.part_d, w.dB, w.dC, w.dA, w.dskip, w.ddelta_bias, rows,
                                gm.tiles_of_group, row_blocks, a.B * gm.segs, a.D, SP, a.S});
}

template <typename T, int SPL, int LPC>
void scan_step_typed(const dwarf_selective_scan_step_args& a, hipStream_t stream) {
  const int per = a.D / a.G, ch = scan_tile_channels(a.S), tiles = (per + ch - 1) / ch;
  const dim3 grid(static_cast<unsigned>(a.R) * tiles * a.G), block(kScanThreads);
  const bool whole = a.S == SPL * LPC && a.slot_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(a.new_state) % 16 == 0;
  if (whole) hipLaunchKernelGGL((scan_step_kernel<T, SPL, LPC, true>), grid, block, 0, stream, a, tiles);
  else hipLaunchKernelGGL((scan_step_kernel<T, SPL, LPC, false>), grid, block, 0, stream, a, tiles);
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
