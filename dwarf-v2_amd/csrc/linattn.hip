// Linear attention with a decay for each head (g = exp(log_decay), at most 1):
//   S_t = g S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
// in chunks of 64 tokens.  With a chunk's n live tokens counted from 0,
//   o_i = scale [ sum_{j <= i} g^{i-j} (q_i.k_j) v_j + g^{i+1} q_i S_in ]
//   S_out = g^n S_in + sum_j g^{n-1-j} k_j v_j^T
// so only non-negative powers of g appear.  The backward is the same sum in
// other roles: with G the adjoint of the state behind a chunk,
//   dq_i = scale [ sum_{j <= i} g^{i-j} (do_i.v_j) k_j + g^{i+1} do_i S_in^T ]
//   dv_j = scale sum_{i >= j} g^{i-j} (k_j.q_i) do_i + g^{n-1-j} k_j G
//   dk_j = scale sum_{i >= j} g^{i-j} (v_j.do_i) q_i + g^{n-1-j} v_j G^T
//   G_in = g^n G + scale sum_i g^{i+1} q_i do_i^T
// and, with tau the token's place in its segment counted from 1, R and K the
// shares of q.dq and k.dk that come from other chunks, and D the pairs within a
// chunk, weighted with their gap,
//   dlog_decay = sum_segments [ D + sum_t tau (R - K) + n <S_out, G_out> ].
// A segment of one chunk takes each part by its own distance instead,
//   D + sum_t tau R + sum_t (n - tau) K + n g^n <S_in, G_out>,
// where nothing cancels (one token alone has exactly 0); longer ones count tau
// from their middle, so that the two sums, which nearly cancel, stay small.
//
// A sequence is cut into segments.  The local launch forms each segment's own
// sum; up to eight segments the rows' launch joins the sums in front of its
// own, above that a scan launch does; the rows' launch walks a segment's chunks
// with the state in registers.  One segment needs the rows alone.  The backward
// is the same in reverse: dq together with the adjoint's segment sums (they
// read the same rows), a scan (also for the boundary terms), dk and dv, and the
// sums of dlog_decay.
//
// Least traffic is one read of q, k, v and one write of o (backward: q, k, v,
// do read, dq, dk, dv written); two passes read k and v twice.  Measured in
// bf16: B1 N65536 H8, 268 MB at least and 403 MB here, 101 us of launches (rows
// 55, local 39, scan 6.6: 4.0 TB/s); training at B15 N2048 H8 (346 MB at least,
// 566 MB here), 148 us: local 23.9, rows 28.7, dq 41.8, scan 6.5, dk and dv 43.4,
// dlog_decay 3.9.  The rows, dq and dk/dv are bound by a CU's issue slots as much
// as by memory: with k and v from the L2 and nothing stored, the rows of the
// long prompt still take 41 us.
#include <type_traits>

#include "gather.h"
#include "mfma.h"
#include "mixer.h"

namespace dwarf {
namespace {

constexpr int kHd = 64;
constexpr int kChunk = 64;
constexpr int kLaThreads = 256;
constexpr int kState = kHd * kHd;
constexpr int kRowStride = 68;   // LDS rows read as 16-byte vectors
constexpr int kColStride = 65;   // LDS rows read down the columns: rows 16 apart lie 16 banks apart

struct LaRows {
  const void* p;
  int64_t s0, s1, s2;
};
struct LaGeom {
  int B, H, Hkv, N, seg, segs;
  float scale;
  const float* log_decay;
  const int32_t* lengths;
};

// log2 of the head's decay: values above 0 count as 0, and the smallest keep g^0 = 1 (-inf would make it NaN).
__device__ __forceinline__ float la_log2_decay(const LaGeom& gm, int h) {
  const float ld = gm.log_decay[h];
  const float x = ld > 0.f ? 0.f : ld;
  return (x < -1e4f ? -1e4f : x) * kLog2e;
}
__device__ __forceinline__ float la_power(float lg, int n) { return __builtin_amdgcn_exp2f(lg * static_cast<float>(n)); }

// The terms of dlog_decay nearly cancel.  A lane's share of one chunk is formed in fp32; its weight and every sum behind it
// (over a lane's chunks, lanes, segments and sequences) are kept in 64 bits: two instructions a chunk and lane.
__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) x += __shfl_xor(x, o);
  return x;
}
template <int WAVES>
__device__ __forceinline__ double workgroup_sum_f64(double x, double* s_red) {
  x = wave_sum_f64(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) s_red[threadIdx.x / kWave] = x;
  __syncthreads();
  double t = s_red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) t += s_red[i];
  return t;
}

// Where the weights of dlog_decay's two sides count from in a segment of n tokens.
struct LaMid {
  float rows, keys;
};
__device__ __forceinline__ LaMid la_mid(int n) {
  const float f = static_cast<float>(n);
  return n <= kChunk ? LaMid{0.f, f} : LaMid{0.5f * f, 0.5f * f};
}

__device__ __forceinline__ int la_length(const LaGeom& gm, int b) {
  if (!gm.lengths) return gm.N;
  const int n = gm.lengths[b];
  return n < 0 ? 0 : n > gm.N ? gm.N : n;
}

// Sixteen elements from column 16 (threadIdx.x % 4) of row r, zeros where it is not live.
template <typename T>
__device__ __forceinline__ void la_load16(const T* row, bool live, float* x) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 16 / kPer; ++i) {
    if (live) {
      load_vec<T, kPer>(row + i * kPer, x + i * kPer);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[i * kPer + e] = 0.f;
    }
  }
}

// The same on its way: as it is in memory until it is needed, so that a chunk's loads are under way while the one in front
// of it is worked on.
template <typename T>
struct LaRaw16 {
  static constexpr int kPer = 16 / sizeof(T);
  Vec<T, kPer> v[16 / kPer];
  __device__ __forceinline__ void load(const T* row, bool live) {
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) v[i] = live ? *reinterpret_cast<const Vec<T, kPer>*>(row + i * kPer) : Vec<T, kPer>{};
  }
  __device__ __forceinline__ void widen(float* x) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = to_f32(v[i / kPer].e[i % kPer]);
  }
};
// A thread's part of a 64-row tile, row tid / 4 from column 16 (tid % 4), and the tile into LDS rows of STRIDE floats.
template <typename T>
__device__ __forceinline__ void la_tile_fetch(LaRaw16<T>& x, const T* base, int64_t stride, int n) {
  const int r = threadIdx.x / 4;
  x.load(base + r * stride + 16 * (threadIdx.x % 4), r < n);
}
template <typename T, int STRIDE>
__device__ __forceinline__ void la_tile_put(const LaRaw16<T>& t, float* s) {
  float x[16];
  t.widen(x);
#pragma unroll
  for (int i = 0; i < 16; ++i) s[threadIdx.x / 4 * STRIDE + 16 * (threadIdx.x % 4) + i] = x[i];
}

// The chunk's weights in the state's sum, in LDS: forward g^{n-1-j}, reverse g^{j+1}.
template <bool REV>
__device__ __forceinline__ void la_weights(float lg, int n, float* s_w) {
  if (threadIdx.x < kChunk) {
    const int j = threadIdx.x;
    s_w[j] = j < n ? la_power(lg, REV ? j + 1 : n - 1 - j) : 0.f;
  }
}

// acc = g^n acc + us sum_j w_j B_j C_j^T; wave w holds rows [16w, 16w + 16).
template <int BSTRIDE>
__device__ __forceinline__ void la_update(const float* sB, const float* sC, const float* s_w, float shrink, float us,
                                          f32x4* acc) {
  const int l = threadIdx.x % kWave, w = threadIdx.x / kWave, g = l / 16, c = l % 16;
  f32x4 add[4] = {zero4(), zero4(), zero4(), zero4()};
#pragma unroll
  for (int kk = 0; kk < 16; ++kk) {
    const int j = 16 * g + kk;
    const float a = sB[j * BSTRIDE + 16 * w + c] * s_w[j];
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) add[ct] = mfma16_f32(a, sC[j * kColStride + 16 * ct + c], add[ct]);
  }
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[ct][r] = fmaf(shrink, acc[ct][r], us * add[ct][r]);
}

// Segment sums: local[b][h][seg] = sum over the segment of us w B C^T.
template <typename T, bool REV>
__global__ __launch_bounds__(kLaThreads) void la_local_kernel(LaRows B_, int bh, LaRows C_, int ch, LaGeom gm, float us,
                                                              float* __restrict__ local) {
  __shared__ float sB[kChunk * kColStride], sC[kChunk * kColStride], s_w[kChunk];
  const int seg = blockIdx.x % gm.segs, h = blockIdx.x / gm.segs % gm.H, b = blockIdx.x / gm.segs / gm.H;
  const int len = la_length(gm, b), t0 = seg * gm.seg;
  if (t0 >= len) return;
  const int t1 = t0 + gm.seg < len ? t0 + gm.seg : len;
  const float lg = la_log2_decay(gm, h);
  const T* pb = static_cast<const T*>(B_.p) + b * B_.s0 + (h / (gm.H / bh)) * B_.s1;
  const T* pc = static_cast<const T*>(C_.p) + b * C_.s0 + (h / (gm.H / ch)) * C_.s1;
  f32x4 acc[4] = {zero4(), zero4(), zero4(), zero4()};
  const int chunks = (t1 - t0 + kChunk - 1) / kChunk;
  LaRaw16<T> xb, xc;
  auto token = [&](int i) { return t0 + (REV ? chunks - 1 - i : i) * kChunk; };
  auto live = [&](int i) { return i < chunks ? (t1 - token(i) < kChunk ? t1 - token(i) : kChunk) : 0; };
  auto fetch = [&](int i) {   // behind the last chunk: reads nothing
    const int64_t t = i < chunks ? token(i) : t0;
    la_tile_fetch(xb, pb + t * B_.s2, B_.s2, live(i));
    la_tile_fetch(xc, pc + t * C_.s2, C_.s2, live(i));
  };
  fetch(0);
  for (int i = 0; i < chunks; ++i) {
    const int n = live(i);
    __syncthreads();
    la_tile_put<T, kColStride>(xb, sB);
    la_tile_put<T, kColStride>(xc, sC);
    la_weights<REV>(lg, n, s_w);
    __syncthreads();
    fetch(i + 1);
    la_update<kColStride>(sB, sC, s_w, la_power(lg, n), us, acc);
  }
  const int l = threadIdx.x % kWave, w = threadIdx.x / kWave;
  float* out = local + static_cast<int64_t>(blockIdx.x) * kState;
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) out[(16 * w + 4 * (l / 16) + r) * kHd + 16 * ct + l % 16] = acc[ct][r];
}

// Turns the segment sums in place into the state in front of each segment (reverse: the adjoint behind it).  first: the
// state that enters (NULL: zero), last: where the one that leaves goes (NULL: nowhere).  Reverse with dot: the boundary
// terms of dlog_decay, per workgroup.
//
// A thread owns four neighbouring elements of one head's state and up to kScanRun segments in a row, all loaded at once;
// GROUPS threads share the elements, each with a run of its own, and join their runs through LDS.  GROUPS is 1 up to
// kScanRun segments, and 16 above: a long sequence's segments would otherwise be read one memory latency after another.
constexpr int kScanRun = 8;
template <int GROUPS>
constexpr int kScanWgs = kState / 4 * GROUPS / kLaThreads;   // workgroups per head
int scan_wgs(const LaGeom& gm) { return gm.segs > kScanRun ? kScanWgs<16> : kScanWgs<1>; }

template <bool REV, int GROUPS>
__global__ __launch_bounds__(kLaThreads) void la_scan_kernel(float* __restrict__ local, const float* __restrict__ first,
                                                             float* __restrict__ last, LaGeom gm,
                                                             const float* __restrict__ states,
                                                             const float* __restrict__ initial,
                                                             const float* __restrict__ final, double* __restrict__ dot) {
  constexpr int kOwners = kLaThreads / GROUPS;   // threads of a group
  constexpr int kSums = GROUPS == 1;             // states: the segments' own sums (LaEnter), not the states in front
  __shared__ f32x4 s_run[GROUPS][kOwners];
  __shared__ double s_red[kLaThreads / kWave];
  const int bh = blockIdx.x / kScanWgs<GROUPS>, owner = threadIdx.x % kOwners, group = threadIdx.x / kOwners;
  const int e = 4 * (blockIdx.x % kScanWgs<GROUPS> * kOwners + owner);
  const int b = bh / gm.H, h = bh % gm.H;
  const int len = la_length(gm, b), active = (len + gm.seg - 1) / gm.seg;
  const float lg = la_log2_decay(gm, h);
  const int n_last = active ? len - (active - 1) * gm.seg : 0;
  const float full = la_power(lg, gm.seg), tail = la_power(lg, n_last), run_full = la_power(lg, gm.seg * kScanRun);
  float* x = local + static_cast<int64_t>(bh) * gm.segs * kState + e;
  const float* st = states ? states + static_cast<int64_t>(bh) * gm.segs * kState + e : nullptr;
  const int64_t at = static_cast<int64_t>(bh) * kState + e;
  auto load = [](const float* p) { return *reinterpret_cast<const f32x4*>(p); };
  const bool one_chunk = n_last <= kChunk;   // the last segment, and with gm.seg one chunk every one
  const float mid = gm.seg > kChunk ? 0.5f * static_cast<float>(gm.seg) : 0.f;
  const float mid_last = one_chunk ? 0.f : 0.5f * static_cast<float>(n_last);
  f32x4 m = first ? load(first + at) : zero4();
  double sum = 0.;
  auto add_dot = [&](float weight, f32x4 a, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fma(static_cast<double>(weight) * a[i], static_cast<double>(c[i]), sum);
  };
  if (REV && dot && final && active && !one_chunk && group == 0) add_dot(mid_last, m, load(final + at));
  // a pass takes GROUPS runs; position p counts segments in the direction of the scan
  for (int p0 = 0; p0 < active; p0 += GROUPS * kScanRun) {
    const int base = p0 + group * kScanRun;
    const int cnt = active - base < kScanRun ? (active - base < 0 ? 0 : active - base) : kScanRun;
    auto segment = [&](int i) { return static_cast<int64_t>(REV ? active - 1 - base - i : base + i); };
    f32x4 in[kScanRun], sv[kScanRun];
#pragma unroll
    for (int i = 0; i < kScanRun; ++i) {
      in[i] = i < cnt ? load(x + segment(i) * kState) : zero4();
      sv[i] = !(REV && dot && i < cnt) ? zero4()
              : segment(i) > 0         ? load(st + (segment(i) - kSums) * kState)
              : initial                ? load(initial + at)
                                       : zero4();
    }
    auto shrink = [&](int i) { return segment(i) == active - 1 ? tail : full; };
    if constexpr (REV && kSums) {   // all of the head's segments are here: the sums become the states in front
      f32x4 u = dot && initial ? load(initial + at) : zero4();   // and sv of segment 0
#pragma unroll
      for (int i = kScanRun - 1; i >= 0; --i)
        if (i < cnt && segment(i) > 0) u = sv[i] = u * full + sv[i];
    }
    f32x4 enter = m;
    if constexpr (GROUPS > 1) {
      f32x4 r = zero4();   // the run's own sum
#pragma unroll
      for (int i = 0; i < kScanRun; ++i)
        if (i < cnt) r = r * shrink(i) + in[i];
      __syncthreads();   // the pass before has been read
      s_run[group][owner] = r;
      __syncthreads();
      for (int q = 0; q < GROUPS; ++q) {   // the runs in front are whole but for the sequence's last segment
        if (q == group) enter = m;
        const int behind = active - (p0 + q * kScanRun);   // segments from run q on
        if (behind <= 0) break;
        const bool whole = behind >= kScanRun;
        // decay over run q: in the forward direction its last segment may be the tail, in reverse its first one is
        float over = whole ? run_full : 1.f;
        if (!whole)
          for (int i = 0; i < behind; ++i) over *= full;
        const bool has_tail = REV ? p0 + q * kScanRun == 0 : behind <= kScanRun;
        if (has_tail) {
          over = 1.f;
          const int n = behind < kScanRun ? behind : kScanRun;
          for (int i = 0; i + 1 < n; ++i) over *= full;
          over *= tail;
        }
        m = m * over + s_run[q][owner];
      }
    }
    f32x4 v = enter;
#pragma unroll
    for (int i = 0; i < kScanRun; ++i) {
      if (i < cnt) {
        *reinterpret_cast<f32x4*>(x + segment(i) * kState) = v;
        const bool tail_segment = segment(i) == active - 1;
        if (REV && dot && (gm.seg <= kChunk || (tail_segment && one_chunk)))   // uniform
          add_dot(static_cast<float>(tail_segment ? n_last : gm.seg) * shrink(i), sv[i], v);   // <S in front of it, G behind it>
        v = v * shrink(i) + in[i];
        // <S in front of it, G in front of it>, with its own part and that of the segment in front
        if (REV && dot) add_dot((tail_segment ? mid_last : mid) + (segment(i) > 0 ? mid : 0.f), sv[i], v);
      }
    }
    if constexpr (GROUPS == 1) m = v;
  }
  if (last && group == 0) *reinterpret_cast<f32x4*>(last + at) = m;
  if (REV && dot) {
    sum = workgroup_sum_f64<kLaThreads / kWave>(sum, s_red);
    if (threadIdx.x == 0) dot[blockIdx.x] = sum;
  }
}

template <bool REV>
void la_scan(float* local, const float* first, float* last, const LaGeom& gm, const float* states, const float* initial,
             const float* final, double* dot, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(gm.B) * gm.H * scan_wgs(gm));
  if (gm.segs > kScanRun)
    hipLaunchKernelGGL((la_scan_kernel<REV, 16>), grid, dim3(kLaThreads), 0, stream, local, first, last, gm, states, initial,
                       final, dot);
  else
    hipLaunchKernelGGL((la_scan_kernel<REV, 1>), grid, dim3(kLaThreads), 0, stream, local, first, last, gm, states, initial,
                       final, dot);
}

// Where the state in front of a segment comes from: the scan's array (or, for the adjoint of one segment, dfinal), or,
// up to kScanRun segments, the head's first state (NULL: zero) and the sums of the segments in front (NULL: none are),
// joined by the workgroup itself: a few more reads of 16 KB in place of a launch between the sums and the rows.
struct LaEnter {
  const float *scanned, *first, *sums;
};

// One call of la_rows_kernel: rows of A against rows of B and C, the state that enters (trans: read transposed), the result, and with dot the decay's gradient's rows D.
template <typename TO>
struct LaRowsCall {
  LaRows A, B, C, D;
  int ah, bh, ch, dh;    // heads of each
  LaEnter enter;
  bool trans;
  TO* out;
  int64_t o0, o1, o2;
  double* dot;
};

// out_i = intra sum_j W_ij (A_i.B_j) C_j + cs W_i A_i M over a segment's chunks, M updated behind each (in front, in
// reverse); in fp32 throughout, for fp32 and fp16 rows (the fp16 matrix instructions would multiply fp16 rows exactly, but
// what is formed here, scores and states, fits fp16's range only after a power of two for each tile; that is not built, and
// bf16 parts of fp16 rows would double the tiles and the products).  B15 N2048 H8, forward and backward: 124 and 343 us in
// fp16, 133 and 396 in fp32.  Bound by the fp32 matrix rate, of which the forward's rows reach half: 232 instructions of 32
// cycles a wave and chunk, 46 of 92 us.
// leave: where the state behind the last token goes (NULL: nowhere, or the scan has written it).
// dot, forward: sum tau D_i.(out_i's part that comes from M); in reverse the same less (i - j) times each pair's share
// within a chunk, W_ij (A_i.B_j) (D_i.C_j).  blockIdx.y picks the call (dv and dk go in one launch).
template <typename T, typename TO, bool REV>
__global__ __launch_bounds__(kLaThreads) void la_rows_kernel(LaRowsCall<TO> call0, LaRowsCall<TO> call1, LaGeom gm,
                                                             float intra, float cs, float us, float* __restrict__ leave) {
  __shared__ __align__(16) float sB[kChunk * kRowStride];
  __shared__ float sC[kChunk * kColStride], sM[kHd * kColStride], sP[kChunk * kColStride], s_w[kChunk];
  __shared__ double s_red[kLaThreads / kWave];
  const LaRowsCall<TO>& call = blockIdx.y ? call1 : call0;
  const LaRows A_ = call.A, B_ = call.B, C_ = call.C, D_ = call.D;
  const int64_t o2 = call.o2;
  const int seg = blockIdx.x % gm.segs, h = blockIdx.x / gm.segs % gm.H, b = blockIdx.x / gm.segs / gm.H;
  const int l = threadIdx.x % kWave, w = uniform(threadIdx.x / kWave), g = l / 16, c = l % 16;
  const int len = la_length(gm, b), t0 = seg * gm.seg;
  const int tend = t0 + gm.seg < gm.N ? t0 + gm.seg : gm.N;
  const int t1 = tend < len ? tend : len;
  TO* po = call.out + b * call.o0 + h * call.o1;
  // rows behind the sequence are zero
  for (int i = (t1 > t0 ? t1 : t0) * kHd + threadIdx.x; i < tend * kHd; i += kLaThreads)
    po[static_cast<int64_t>(i / kHd) * o2 + i % kHd] = from_f32<TO>(0.f);
  const float lg = la_log2_decay(gm, h);
  const T* pa = static_cast<const T*>(A_.p) + b * A_.s0 + (h / (gm.H / call.ah)) * A_.s1;
  const T* pb = static_cast<const T*>(B_.p) + b * B_.s0 + (h / (gm.H / call.bh)) * B_.s1;
  const T* pc = static_cast<const T*>(C_.p) + b * C_.s0 + (h / (gm.H / call.ch)) * C_.s1;
  const T* pd = call.dot ? static_cast<const T*>(D_.p) + b * D_.s0 + (h / (gm.H / call.dh)) * D_.s1 : nullptr;
  const int64_t head = static_cast<int64_t>(b) * gm.H + h;
  const bool leaves = leave && (len ? t0 < len && len <= t0 + gm.seg : seg == 0);
  f32x4 M[4] = {zero4(), zero4(), zero4(), zero4()};
  auto join = [&](const float* en, float shrink) {
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * w + 4 * g + r, j = 16 * ct + c;
        M[ct][r] = fmaf(M[ct][r], shrink, en[call.trans ? j * kHd + i : i * kHd + j]);
      }
  };
  if (t1 > t0 || leaves) {
    const LaEnter& e = call.enter;
    if (e.scanned) join(e.scanned + static_cast<int64_t>(blockIdx.x) * kState, 0.f);
    if (e.first) join(e.first + head * kState, 0.f);
    if (e.sums)
      for (int p = 0; p < seg; ++p) join(e.sums + (head * gm.segs + p) * kState, la_power(lg, gm.seg));
  }
  const float mid = REV ? la_mid(t1 - t0).keys : la_mid(t1 - t0).rows;
  double total = 0.;
  const int chunks = t1 > t0 ? (t1 - t0 + kChunk - 1) / kChunk : 0;
  LaRaw16<T> xa, xb, xc;
  auto token = [&](int i) { return t0 + (REV ? chunks - 1 - i : i) * kChunk; };
  auto live = [&](int i) { return i < chunks ? (t1 - token(i) < kChunk ? t1 - token(i) : kChunk) : 0; };
  auto fetch = [&](int i) {   // behind the last chunk: reads nothing
    const int64_t t = i < chunks ? token(i) : t0;
    const int n = live(i);
    la_tile_fetch(xb, pb + t * B_.s2, B_.s2, n);
    la_tile_fetch(xc, pc + t * C_.s2, C_.s2, n);
    // row 16w + c of A, elements [16g, 16g + 16): the k index of step kk is 16g + kk in both operands
    xa.load(pa + (t + 16 * w + c) * A_.s2 + 16 * g, 16 * w + c < n);
  };
  fetch(0);
  for (int i = 0; i < chunks; ++i) {
    const int t = token(i), n = live(i);
    __syncthreads();
    la_tile_put<T, kRowStride>(xb, sB);
    la_tile_put<T, kColStride>(xc, sC);
    la_weights<REV>(lg, n, s_w);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) sM[(16 * w + 4 * g + r) * kColStride + 16 * ct + c] = M[ct][r];
    float a[16];
    xa.widen(a);
    __syncthreads();
    fetch(i + 1);
    f32x4 p[4];
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      p[ct] = zero4();
      const float* row = sB + (16 * ct + c) * kRowStride + 16 * g;
      if (REV ? ct >= w : ct <= w) {   // uniform: the others lie on the wrong side of the wave's rows
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const float4 x = *reinterpret_cast<const float4*>(row + 4 * k4);
          p[ct] = mfma16_f32(a[4 * k4], x.x, p[ct]);
          p[ct] = mfma16_f32(a[4 * k4 + 1], x.y, p[ct]);
          p[ct] = mfma16_f32(a[4 * k4 + 2], x.z, p[ct]);
          p[ct] = mfma16_f32(a[4 * k4 + 3], x.w, p[ct]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ii = 16 * w + 4 * g + r, jj = 16 * ct + c, gap = REV ? jj - ii : ii - jj;
        p[ct][r] = gap >= 0 ? intra * p[ct][r] * la_power(lg, gap) : 0.f;
        sP[ii * kColStride + jj] = p[ct][r];
      }
    }
    if (REV && call.dot) {   // uniform
      float d[16];
      la_load16<T>(pd + (t + 16 * w + c) * D_.s2 + 16 * g, 16 * w + c < n, d);
      float pairs = 0.f;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        if (ct < w) continue;
        f32x4 y = zero4();
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) y = mfma16_f32(d[kk], sC[(16 * ct + c) * kColStride + 16 * g + kk], y);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int gap = 16 * ct + c - (16 * w + 4 * g + r);
          pairs = fmaf(static_cast<float>(gap) * p[ct][r], y[r], pairs);   // p is 0 where the gap is negative
        }
      }
      total -= pairs;
    }
    __syncthreads();
    f32x4 o[4] = {zero4(), zero4(), zero4(), zero4()}, x[4] = {zero4(), zero4(), zero4(), zero4()};
#pragma unroll
    for (int kk = 0; kk < 16; ++kk) {
      const float pk = sP[(16 * w + c) * kColStride + 16 * g + kk];
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        o[ct] = mfma16_f32(pk, sC[(16 * g + kk) * kColStride + 16 * ct + c], o[ct]);
        x[ct] = mfma16_f32(a[kk], sM[(16 * g + kk) * kColStride + 16 * ct + c], x[ct]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ii = 16 * w + 4 * g + r;
      if (ii < n) {
        const float carry = cs * la_power(lg, REV ? n - 1 - ii : ii + 1);
        const float tau = static_cast<float>(t - t0 + ii + 1) - mid;
        float s = 0.f;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const float v = carry * x[ct][r];
          po[(t + ii) * o2 + 16 * ct + c] = from_f32<TO>(v + o[ct][r]);
          if (call.dot) s = fmaf(v, to_f32(pd[(t + ii) * D_.s2 + 16 * ct + c]), s);
        }
        total = fma(static_cast<double>(tau), static_cast<double>(s), total);
      }
    }
    la_update<kRowStride>(sB, sC, s_w, la_power(lg, n), us, M);
  }
  if (leaves) {
    float* lv = leave + head * kState;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) lv[(16 * w + 4 * g + r) * kHd + 16 * ct + c] = M[ct][r];
  }
  if (call.dot) {
    total = workgroup_sum_f64<kLaThreads / kWave>(total, s_red);
    if (threadIdx.x == 0) call.dot[blockIdx.x] = total;
  }
}

// ---- bf16 --------------------------------------------------------------------------------------
// The same sums on v_mfma_f32_16x16x32_bf16.  Products of two inputs are exact in fp32; what the kernel forms itself
// (weighted scores, the state, weighted keys) is split into bf16 parts before it meets the matrix cores, two parts
// (2^-17 relative) where the result is rounded to bf16 anyway and three (2^-24, fp32 itself) where it goes into the
// state, so that no intermediate rounding is coarser than the output's.  The sums are bound by memory, and the matrix
// cores have the room, busy a third of the time: instructions of a wave and chunk, on average over the waves, 28 in the
// forward's rows, 37 in dq and 41 in dk and dv, with dlog_decay 44 and 52.
//
// LDS holds tiles as 64 rows of 128 bytes; 16-byte piece p of row r sits at piece p ^ tile_key(r).  Of the 4,096 keys that
// are linear in a row's four low bits this is one of the best: no bank conflicts in whole pieces read down 16 rows and
// written along a row, in 8-byte halves read down 16 rows and in the transposed reads of four rows; the state's 8-byte
// halves written down 16 rows (state_put) take 8 cycles for the 4 of consecutive addresses, which is all of the conflicts
// that SQ_LDS_BANK_CONFLICT shows, 10 to 13% of the LDS's busy cycles.  (The lanes that one cycle of a 16-byte read serves
// are not consecutive ones; measured cycles for 1,024 instructions of a workgroup, with this key and with twice the
// conflicts: 4,160 and 8,252 for whole pieces read, 8,324 and 16,472 for halves written.)
// Scores are formed transposed (rows: the other side's tokens): a lane then holds four consecutive tokens of one own
// row, which is the next product's operand as it stands.  Its tokens are slots in the order 4 g + e, 16 + 4 g + e of
// each 32 (g the lane's group of 16), and a transposed read of four rows gives the other operand in the same order.
// Results come out transposed too: a lane holds four consecutive elements of one row.
constexpr int kTileBytes = kChunk * kHd * 2;

__device__ __forceinline__ int tile_key(int r) { return ((r ^ (r >> 1)) & 4) | (r & 2) | ((r ^ (r >> 2)) & 1); }
__device__ __forceinline__ int tile_at(int r, int byte) { return r * 128 + ((((byte >> 4) ^ tile_key(r)) << 4) | (byte & 15)); }

// A chunk's rows on their way through registers: rows tid / 8 and tid / 8 + 32, piece tid % 8.
struct TileRegs {
  uint4 x[2];
};
__device__ __forceinline__ void tile_fetch(TileRegs& t, const bf16* base, int64_t stride, int n, int tid) {
  const int ld = static_cast<int>(stride) * 2;
  const __amdgpu_buffer_rsrc_t r = rows_rsrc(base, ld, n, 128);   // rows behind the n live ones read zeros
  const uint32_t off = (tid >> 3) * static_cast<uint32_t>(ld) + (tid & 7) * 16;
  t.x[0] = buf_load16(r, off);
  t.x[1] = buf_load16(r, off + 32u * static_cast<uint32_t>(ld));
}
// Where a lane (group g, place c in it) reads and writes in a tile.  A tile_key takes bits 0 to 3 of a row, so steps of
// 16 rows are plain offsets and steps along a row are exclusive ors: everything else is fixed once per launch.
struct TileMap {
  int row;      // row c, elements 8 g + [0, 8)                    (^ 64: 32 elements on, + 2048: 16 rows on)
  int slots;    // row c, elements 4 g + [0, 4)                    (^ 32: 16 elements on, ^ 64: 32)
  int column;   // rows 4 g + [0, 4), column c of the first 16     (^ 32 ct: column 16 ct + c, + 2048: 16 rows on)
  int state;    // row c, elements 16 w + 4 g + [0, 4)             (+ 2048: 16 rows on)
  int put;      // row tid / 8, piece tid % 8                       (+ 4096: 32 rows on)
  __device__ __forceinline__ explicit TileMap(int tid) {
    const int l = threadIdx.x % kWave, w = threadIdx.x / kWave % 4, g = l / 16, c = l % 16;
    row = tile_at(c, 16 * g);
    slots = tile_at(c, 8 * g);
    column = tile_at(4 * g + c / 4, 8 * (c % 4));
    state = tile_at(c, 32 * w + 8 * g);
    put = tile_at(tid >> 3, (tid & 7) * 16);
  }
};
__device__ __forceinline__ void tile_put(const TileRegs& t, char* s, const TileMap& m) {
  *reinterpret_cast<uint4*>(s + m.put) = t.x[0];
  *reinterpret_cast<uint4*>(s + m.put + 4096) = t.x[1];
}
// The same for a workgroup of 512 threads: row tid / 8, piece tid % 8.
__device__ __forceinline__ uint4 tile_fetch_wide(const bf16* base, int64_t stride, int n) {
  const int ld = static_cast<int>(stride) * 2;
  return buf_load16(rows_rsrc(base, ld, n, 128), (threadIdx.x >> 3) * static_cast<uint32_t>(ld) + (threadIdx.x & 7) * 16);
}
__device__ __forceinline__ void tile_put_wide(uint4 x, char* s, const TileMap& m) { *reinterpret_cast<uint4*>(s + m.put) = x; }
// Row 16 rt + c, elements 32 ks + 8 g + [0, 8).
__device__ __forceinline__ bf16x8 tile_row(const char* s, const TileMap& m, int rt, int ks) {
  return bf16x8_from_bits(*reinterpret_cast<const uint4*>(s + (m.row ^ 64 * ks) + 2048 * rt));
}
// Row 16 rt + c, elements in slot order: 32 ks + 4 g + [0, 4) and 32 ks + 16 + 4 g + [0, 4).
__device__ __forceinline__ bf16x8 tile_row_slots(const char* s, const TileMap& m, int rt, int ks) {
  const uint2 lo = *reinterpret_cast<const uint2*>(s + (m.slots ^ 64 * ks) + 2048 * rt);
  const uint2 hi = *reinterpret_cast<const uint2*>(s + (m.slots ^ 64 * ks ^ 32) + 2048 * rt);
  return bf16x8_from_bits(uint4{lo.x, lo.y, hi.x, hi.y});
}
// Column 16 ct + c of the 32 rows from 32 ks, in slot order.
__device__ __forceinline__ bf16x8 tile_column(const char* s, const TileMap& m, int ct, int ks) {
  typedef short i16x8 __attribute__((ext_vector_type(8)));
  const char* p = s + (m.column ^ 32 * ct) + 4096 * ks;
  const i16x4 lo = lds_read_tr16(p), hi = lds_read_tr16(p + 2048);
  const i16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}

__device__ __forceinline__ void unpack8(bf16x8 v, float* x) {
  const uint4 w = __builtin_bit_cast(uint4, v);
  x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z); x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
}
// Two values' bf16 parts: the pair's high parts, and what they leave in x.
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
  const uint32_t h = pack_bf16x2(a, b);
  a -= bf16_lo(h);
  b -= bf16_hi(h);
  return h;
}
template <int PARTS>
__device__ __forceinline__ void split8(float* x, bf16x8* parts) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint4 w;
    if (p + 1 < PARTS) {
      w.x = split_pair(x[0], x[1]); w.y = split_pair(x[2], x[3]);
      w.z = split_pair(x[4], x[5]); w.w = split_pair(x[6], x[7]);
    } else {
      w = uint4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
    parts[p] = bf16x8_from_bits(w);
  }
}

// The wave's 16 rows of the state (rows 16 w + 4 g + r, column 16 ct + c) into PARTS LDS tiles of the transposed state: its
// high parts, behind them what those leave, and so on.
template <int PARTS>
__device__ __forceinline__ void state_put(const f32x4* M, char* s, const TileMap& m) {
#pragma unroll
  for (int ct = 0; ct < 4; ++ct) {
    float x[4] = {M[ct][0], M[ct][1], M[ct][2], M[ct][3]};
    char* at = s + m.state + 2048 * ct;
#pragma unroll
    for (int p = 0; p + 1 < PARTS; ++p)
      *reinterpret_cast<uint2*>(at + p * kTileBytes) = uint2{split_pair(x[0], x[1]), split_pair(x[2], x[3])};
    *reinterpret_cast<uint2*>(at + (PARTS - 1) * kTileBytes) = uint2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  }
}

// A chunk's weights in the adjoint's sum, us g^{j+1}, in factors: token 32 ks + 16 h + 4 g + r has base[r] tile[2 ks + h],
// the second uniform.
struct AdjointWeights {
  float base[4], tile[4];
  __device__ __forceinline__ AdjointWeights(float lg, float us) {
    const int g = (threadIdx.x % kWave) / 16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      base[r] = us * la_power(lg, 4 * g + r + 1);
      tile[r] = __uint_as_float(uniform(__float_as_uint(la_power(lg, 16 * r))));
    }
  }
  __device__ __forceinline__ void apply(int ks, float factor, float* x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= base[e & 3] * (tile[2 * ks + (e >> 2)] * factor);
  }
};
// In the state's sum, g^{n-1-j}, from LDS tables: of a whole chunk, and of the last chunk of n tokens behind it (its dead
// rows are zero, their weight only has to be finite).
constexpr int kTableBytes = 2 * kChunk * 4;
__device__ __forceinline__ void state_weights_put(float lg, int n_last, float* s) {
  const int j = threadIdx.x;
  if (j < 2 * kChunk) {
    const int n = j < kChunk ? kChunk : n_last, p = n - 1 - (j & (kChunk - 1));
    s[j] = la_power(lg, p < 0 ? 0 : p);
  }
}
struct StateWeights {
  const float* s;   // the chunk's table
  __device__ __forceinline__ StateWeights(const float* tables, int n) : s(tables + (n < kChunk ? kChunk : 0)) {}
  __device__ __forceinline__ void apply(int ks, float, float* x) const {
    const float* p = s + 32 * ks + 4 * ((threadIdx.x % kWave) / 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 w = *reinterpret_cast<const float4*>(p + 16 * h);
      x[4 * h] *= w.x; x[4 * h + 1] *= w.y; x[4 * h + 2] *= w.z; x[4 * h + 3] *= w.w;
    }
  }
};

// M = shrink M + factor sum_j weight_j X_j Y_j^T for the wave's 16 columns of X and all of Y.  PARTS: of the weighted X,
// three where the sum goes into an fp32 result, two where it only goes into rows that are rounded to bf16.  The chunk's sum
// is formed from zero and then joins M by rounded arithmetic: the matrix instructions round each addition towards zero, and
// over a state's many chunks that would be a bias.
template <int PARTS, typename W>
__device__ __forceinline__ void state_update(const char* sX, const char* sY, const TileMap& m, int w, const W& weights,
                                             float factor, float shrink, f32x4* M) {
  bf16x8 parts[2][PARTS];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    float x[8];
    unpack8(tile_column(sX, m, w, ks), x);
    weights.apply(ks, factor, x);
    split8<PARTS>(x, parts[ks]);
  }
#pragma unroll
  for (int ct = 0; ct < 4; ++ct) {   // one tile of M at a time: all four at once spill (dq 61 us for 47 at B8 N2048 H8)
    f32x4 add = zero4();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const bf16x8 y = tile_column(sY, m, ct, ks);
#pragma unroll
      for (int p = 0; p < PARTS; ++p) add = mfma16_bf16(parts[ks][p], y, add);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) M[ct][r] = fmaf(M[ct][r], shrink, add[r]);
  }
}
__device__ __forceinline__ void rows_scale(f32x4* M, float shrink) {
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) M[ct][r] *= shrink;
}

// Work item of a workgroup: the heads of one segment next to each other on one XCD (token-major rows of the heads lie
// side by side in memory, and query heads share their K/V head's rows), then the segments.
struct LaItem {
  int b, h, seg;
  int64_t at;   // (b, h, seg) in the state arrays
};
__device__ __forceinline__ LaItem la_item(const LaGeom& gm) {
  const int i = xcd_remap(blockIdx.x, gridDim.x);
  LaItem it;
  it.h = i % gm.H;
  it.seg = i / gm.H % gm.segs;
  it.b = i / gm.H / gm.segs;
  it.at = (static_cast<int64_t>(it.b) * gm.H + it.h) * gm.segs + it.seg;
  return it;
}

__device__ __forceinline__ void state_load(const float* en, bool trans, f32x4* M) {
  const int l = threadIdx.x % kWave, w = threadIdx.x / kWave % 4, g = l / 16, c = l % 16;
#pragma unroll
  for (int ct = 0; ct < 4; ++ct) {
    const int i = 16 * w + 4 * g, j = 16 * ct + c;
    if (!en) M[ct] = zero4();
    else if (trans) M[ct] = *reinterpret_cast<const f32x4*>(en + j * kHd + i);
    else
#pragma unroll
      for (int r = 0; r < 4; ++r) M[ct][r] = en[(i + r) * kHd + j];
  }
}
__device__ __forceinline__ void state_enter(const LaEnter& e, bool trans, const LaGeom& gm, const LaItem& it, float lg,
                                            f32x4* M) {
  const int64_t head = it.b * static_cast<int64_t>(gm.H) + it.h;
  state_load(e.scanned ? e.scanned + it.at * kState : e.first ? e.first + head * kState : nullptr, trans, M);
  if (!e.sums) return;
  const float full = la_power(lg, gm.seg);
#pragma unroll 1
  for (int p = 0; p < it.seg; ++p) {
    f32x4 L[4];
    state_load(e.sums + (head * gm.segs + p) * kState, trans, L);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) M[ct][r] = fmaf(M[ct][r], full, L[ct][r]);
  }
}
__device__ __forceinline__ void state_store(const f32x4* M, float* out) {
  const int l = threadIdx.x % kWave, w = threadIdx.x / kWave % 4, g = l / 16, c = l % 16;
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int r = 0; r < 4; ++r) out[(16 * w + 4 * g + r) * kHd + 16 * ct + c] = M[ct][r];
}

// Four consecutive elements of a row.
__device__ __forceinline__ void put4(bf16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
__device__ __forceinline__ void put4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// Rows as the lanes hold them (row c, elements 16 ct + 4 g + [0, 4) of the wave's 16) to memory, `at` the row's start.
// bf16: the lanes of a row trade halves, so that each holds eight consecutive elements and a store covers 64 bytes of each
// row, not 32: every lane of the wave takes part.
__device__ __forceinline__ void put_rows(bf16* at, bool live, const f32x4* o) {
  const int g = (threadIdx.x % kWave) / 16;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      a[i] = pack_bf16x2(o[2 * s][2 * i], o[2 * s][2 * i + 1]);
      b[i] = pack_bf16x2(o[2 * s + 1][2 * i], o[2 * s + 1][2 * i + 1]);
      const auto x = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);   // trades ct's low bit for g's high one
      const auto y = __builtin_amdgcn_permlane16_swap(x[0], x[1], false, false);   // and that one for g's low one
      a[i] = y[0];
      b[i] = y[1];
    }
    if (live) *reinterpret_cast<uint4*>(at + 32 * s + 8 * g) = uint4{a[0], a[1], b[0], b[1]};
  }
}
__device__ __forceinline__ void put_rows(float* at, bool live, const f32x4* o) {
  const int g = (threadIdx.x % kWave) / 16;
  if (live)
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) *reinterpret_cast<f32x4*>(at + 16 * ct + 4 * g) = o[ct];
}

__device__ __forceinline__ const bf16* la_rows_of(const LaRows& x, int heads, const LaGeom& gm, const LaItem& it) {
  return static_cast<const bf16*>(x.p) + it.b * x.s0 + (it.h / (gm.H / heads)) * x.s1;
}

template <typename TO>
__device__ __forceinline__ void la_zero_rows(TO* po, int64_t o2, int from, int to) {
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = from * (kHd / 4) + threadIdx.x; i < to * (kHd / 4); i += blockDim.x)
    put4(po + static_cast<int64_t>(i / (kHd / 4)) * o2 + i % (kHd / 4) * 4, zero);
}

// Segment sums of the forward (see la_local_kernel).  The loads of two chunks are issued at once.
constexpr int kLocalAhead = 2;
__global__ __launch_bounds__(kLaThreads, 4) void la_local_bf16(LaRows X_, int xh, LaRows Y_, int yh, LaGeom gm,
                                                               float* __restrict__ local) {
  __shared__ __align__(16) char smem[4 * kTileBytes + kTableBytes];   // two chunks of X and Y
  const LaItem it = la_item(gm);   // the rows' launch has the same items on the same XCDs and finds k and v in their L2
  const int len = la_length(gm, it.b), t0 = it.seg * gm.seg;
  if (t0 >= len) return;
  const int t1 = t0 + gm.seg < len ? t0 + gm.seg : len;
  const float lg = la_log2_decay(gm, it.h), full = la_power(lg, kChunk);
  const bf16 *px = la_rows_of(X_, xh, gm, it), *py = la_rows_of(Y_, yh, gm, it);
  const int chunks = (t1 - t0 + kChunk - 1) / kChunk, w = uniform(threadIdx.x / kWave);
  const TileMap m(threadIdx.x);
  f32x4 M[4] = {zero4(), zero4(), zero4(), zero4()};
  const float* tables = reinterpret_cast<const float*>(smem + 4 * kTileBytes);   // written before the first barrier
  state_weights_put(lg, t1 - t0 - (chunks - 1) * kChunk, reinterpret_cast<float*>(smem + 4 * kTileBytes));
  for (int i0 = 0; i0 < chunks; i0 += kLocalAhead) {
    TileRegs x[kLocalAhead], y[kLocalAhead];
#pragma unroll
    for (int u = 0; u < kLocalAhead; ++u) {
      const int64_t t = t0 + static_cast<int64_t>(i0 + u) * kChunk;
      const int n = i0 + u < chunks ? (t1 - t < kChunk ? static_cast<int>(t1 - t) : kChunk) : 0;   // 0: reads nothing
      tile_fetch(x[u], px + t * X_.s2, X_.s2, n, threadIdx.x);
      tile_fetch(y[u], py + t * Y_.s2, Y_.s2, n, threadIdx.x);
    }
#pragma unroll
    for (int u = 0; u < kLocalAhead; ++u) {
      if (i0 + u < chunks) {   // uniform
        char* s = smem + (u & 1) * 2 * kTileBytes;
        tile_put(x[u], s, m);
        tile_put(y[u], s + kTileBytes, m);
        __syncthreads();   // also: every wave is done with the other buffer
        const int t = t0 + (i0 + u) * kChunk, n = t1 - t < kChunk ? t1 - t : kChunk;
        state_update<3>(s, s + kTileBytes, m, w, StateWeights(tables, n), 1.f, n < kChunk ? la_power(lg, n) : full, M);
      }
    }
  }
  state_store(M, local + it.at * kState);
}

// Scores' weights of a lane: rows 4 g + r of a tile of the other side's tokens against its own token c.  near: one
// tile away (gap 1 and up), diagonal: the same tile, 0 where the other token lies on the wrong side.
struct ScoreWeights {
  float diagonal[4], near[4], tile;   // tile: 16 tokens' decay
  __device__ __forceinline__ ScoreWeights(float lg, float scale, bool other_behind) {
    const int l = threadIdx.x % kWave, g = l / 16, c = l % 16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = other_behind ? 4 * g + r - c : c - 4 * g - r;
      diagonal[r] = d >= 0 ? scale * la_power(lg, d) : 0.f;
      near[r] = scale * la_power(lg, d + 16);
    }
    tile = la_power(lg, 16);
  }
  // scores against a tile `away` tiles off (uniform), weighted; away < 0: none of it counts
  __device__ __forceinline__ void apply(f32x4 s, int away, float* p) const {
    const float far = away <= 1 ? 1.f : away == 2 ? tile : tile * tile;
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = away == 0 ? s[r] * diagonal[r] : s[r] * (near[r] * far);
  }
};

// The workgroups that form rows have eight waves: four with 16 rows each, and four that keep the state (forward, dq)
// or form the other gradient (dk beside dv), so that neither part's registers keep a CU from holding sixteen waves.
constexpr int kWideThreads = 512;

// out_i = scale (sum_{j <= i} g^{i-j} (q_i.k_j) v_j + g^{i+1} q_i S) over a segment's chunks.  LDS: two chunks of k and v
// and the two parts of the state in front of each.  leave: see la_rows_kernel.
__global__ __launch_bounds__(kWideThreads, 4) void la_rows_bf16(LaRows Q_, LaRows K_, LaRows V_, LaGeom gm,
                                                                LaEnter enter, bf16* __restrict__ out,
                                                                int64_t o0, int64_t o1, int64_t o2,
                                                                float* __restrict__ leave) {
  __shared__ __align__(16) char smem[8 * kTileBytes + kTableBytes];
  const LaItem it = la_item(gm);
  const int l = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), w = wave % 4, g = l / 16, c = l % 16;
  const bool keeps = wave >= 4;   // this wave keeps the state
  const int len = la_length(gm, it.b), t0 = it.seg * gm.seg;
  const int tend = t0 + gm.seg < gm.N ? t0 + gm.seg : gm.N;
  const int t1 = tend < len ? tend : len;
  bf16* po = out + it.b * o0 + it.h * o1;
  la_zero_rows(po, o2, t1 > t0 ? t1 : t0, tend);
  const float lg = la_log2_decay(gm, it.h);
  const bf16 *pq = la_rows_of(Q_, gm.H, gm, it), *pk = la_rows_of(K_, gm.Hkv, gm, it), *pv = la_rows_of(V_, gm.Hkv, gm, it);
  const TileMap m(threadIdx.x);
  const int chunks = t1 > t0 ? (t1 - t0 + kChunk - 1) / kChunk : 0;
  auto live = [&](int i) { return i < chunks ? (t1 - t0 - i * kChunk < kChunk ? t1 - t0 - i * kChunk : kChunk) : 0; };
  uint4 x, y;
  auto fetch = [&](int i) {   // behind the last chunk: reads nothing
    const int64_t t = t0 + static_cast<int64_t>(i) * kChunk;
    x = tile_fetch_wide(pk + t * K_.s2, K_.s2, live(i));
    y = tile_fetch_wide(pv + t * V_.s2, V_.s2, live(i));
  };
  const float* tables = reinterpret_cast<const float*>(smem + 8 * kTileBytes);   // written before the first barrier
  state_weights_put(lg, live(chunks - 1), reinterpret_cast<float*>(smem + 8 * kTileBytes));
  fetch(0);
  if (keeps) {
    const bool leaves = leave && (len ? t0 < len && len <= t0 + gm.seg : it.seg == 0);
    if (!chunks && !leaves) return;
    f32x4 M[4];
    state_enter(enter, false, gm, it, lg, M);
    state_put<2>(M, smem + 2 * kTileBytes, m);
    const float full = la_power(lg, kChunk);
    for (int i = 0; i < chunks; ++i) {
      char *s = smem + (i & 1) * 4 * kTileBytes, *other = smem + (~i & 1) * 4 * kTileBytes;
      tile_put_wide(x, s, m);
      tile_put_wide(y, s + kTileBytes, m);
      __syncthreads();   // also: every wave is done with the other buffer
      fetch(i + 1);
      const int n = live(i);
      const StateWeights wt(tables, n);
      state_update<3>(s, s + kTileBytes, m, w, wt, 1.f, n < kChunk ? la_power(lg, n) : full, M);   // (two parts would do where nothing leaves: no faster)
      state_put<2>(M, other + 2 * kTileBytes, m);
    }
    if (leaves) state_store(M, leave + (static_cast<int64_t>(it.b) * gm.H + it.h) * kState);
    return;
  }
  const ScoreWeights sw(lg, gm.scale, false);
  const float carry = gm.scale * la_power(lg, 16 * w + c + 1);
  uint4 qn[2];
  auto fetch_q = [&](int i) {
    const int ld = static_cast<int>(Q_.s2) * 2;
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(pq + (t0 + static_cast<int64_t>(i) * kChunk) * Q_.s2, ld, live(i), 128);
    const uint32_t off = static_cast<uint32_t>(16 * w + c) * static_cast<uint32_t>(ld) + 16 * g;
    qn[0] = buf_load16(r, off);
    qn[1] = buf_load16(r, off + 64);
  };
  fetch_q(0);
  for (int i = 0; i < chunks; ++i) {
    char* s = smem + (i & 1) * 4 * kTileBytes;
    tile_put_wide(x, s, m);
    tile_put_wide(y, s + kTileBytes, m);
    const bf16x8 a[2] = {bf16x8_from_bits(qn[0]), bf16x8_from_bits(qn[1])};
    __syncthreads();
    fetch(i + 1);
    fetch_q(i + 1);
    const char *sK = s, *sV = s + kTileBytes, *sM = s + 2 * kTileBytes;
    f32x4 o[4] = {zero4(), zero4(), zero4(), zero4()};
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        o[ct] = mfma16_bf16(tile_row(sM, m, ct, ks), a[ks], o[ct]);
        o[ct] = mfma16_bf16(tile_row(sM + kTileBytes, m, ct, ks), a[ks], o[ct]);
      }
    rows_scale(o, carry);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (2 * ks <= w) {   // uniform: some of the 32 tokens are not behind the wave's rows
        float p[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int jt = 2 * ks + half;
          f32x4 z = zero4();
          if (jt <= w) {
            z = mfma16_bf16(tile_row(sK, m, jt, 0), a[0], z);
            z = mfma16_bf16(tile_row(sK, m, jt, 1), a[1], z);
          }
          sw.apply(z, w - jt, p + 4 * half);
        }
        bf16x8 parts[2];
        split8<2>(p, parts);
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const bf16x8 v = tile_column(sV, m, ct, ks);
          o[ct] = mfma16_bf16(v, parts[0], o[ct]);
          o[ct] = mfma16_bf16(v, parts[1], o[ct]);
        }
      }
    }
    put_rows(po + (t0 + static_cast<int64_t>(i) * kChunk + 16 * w + c) * o2, 16 * w + c < live(i), o);
  }
}

// dq_i = scale (sum_{j <= i} g^{i-j} (do_i.v_j) k_j + g^{i+1} do_i S^T), and from the same tiles the segment's own sum
// of the adjoint, local = sum_i scale g^{i+1} q_i do_i^T (NULL: not wanted): one pass over q and do instead of two.  The
// four state waves keep both.  LDS: one chunk of v, k, q and do, and the parts of S^T in front of it.
//
// DECAY: the rows' side of dlog_decay, sum tau q_i.(the share of dq_i that comes from in front of i's chunk), with the
// state in three parts: it nearly cancels against the keys' side, so that two parts' 2^-17 would show.  Pairs within a
// chunk are the keys' side's (la_dkdv_role).
template <bool DECAY>
__global__ __launch_bounds__(kWideThreads, 4) void la_dq_bf16(LaRows Q_, LaRows O_, LaRows K_, LaRows V_, LaGeom gm,
                                                              LaEnter enter, bf16* __restrict__ dq,
                                                              int64_t o0, int64_t o1, int64_t o2,
                                                              float* __restrict__ local, double* __restrict__ dot) {
  constexpr int kParts = DECAY ? 3 : 2;
  __shared__ __align__(16) char smem[(4 + kParts) * kTileBytes + kTableBytes];
  const LaItem it = la_item(gm);
  const int l = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), w = wave % 4, c = l % 16;
  const bool keeps = wave >= 4;
  const int len = la_length(gm, it.b), t0 = it.seg * gm.seg;
  const int tend = t0 + gm.seg < gm.N ? t0 + gm.seg : gm.N;
  const int t1 = tend < len ? tend : len;
  bf16* po = dq + it.b * o0 + it.h * o1;
  la_zero_rows(po, o2, t1 > t0 ? t1 : t0, tend);
  const float lg = la_log2_decay(gm, it.h);
  const bf16 *pq = la_rows_of(Q_, gm.H, gm, it), *pdo = la_rows_of(O_, gm.H, gm, it);
  const bf16 *pk = la_rows_of(K_, gm.Hkv, gm, it), *pv = la_rows_of(V_, gm.Hkv, gm, it);
  const TileMap m(threadIdx.x);
  const int chunks = t1 > t0 ? (t1 - t0 + kChunk - 1) / kChunk : 0;
  auto live = [&](int i) { return i < chunks ? (t1 - t0 - i * kChunk < kChunk ? t1 - t0 - i * kChunk : kChunk) : 0; };
  char *sV = smem, *sK = smem + kTileBytes, *sQ = smem + 2 * kTileBytes, *sO = smem + 3 * kTileBytes, *sM = smem + 4 * kTileBytes;
  uint4 x[4];
  auto fetch = [&](int i) {
    const int64_t t = t0 + static_cast<int64_t>(i) * kChunk;
    x[0] = tile_fetch_wide(pv + t * V_.s2, V_.s2, live(i));
    x[1] = tile_fetch_wide(pk + t * K_.s2, K_.s2, live(i));
    x[2] = tile_fetch_wide(pq + t * Q_.s2, Q_.s2, live(i));
    x[3] = tile_fetch_wide(pdo + t * O_.s2, O_.s2, live(i));
  };
  auto put = [&]() {
#pragma unroll
    for (int u = 0; u < 4; ++u) tile_put_wide(x[u], smem + u * kTileBytes, m);
  };
  const float* tables = reinterpret_cast<const float*>(smem + (4 + kParts) * kTileBytes);   // written before the first barrier
  state_weights_put(lg, live(chunks - 1), reinterpret_cast<float*>(smem + (4 + kParts) * kTileBytes));
  double total = 0.;
  if (keeps) {
    f32x4 M[4], L[4];
    state_enter(enter, true, gm, it, lg, M);
    fetch(0);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) L[ct] = zero4();
    const float full = la_power(lg, kChunk);
    const AdjointWeights wl(lg, gm.scale);
    float past = 1.f;
    for (int i = 0; i < chunks; ++i) {
      put();
      state_put<kParts>(M, sM, m);
      __syncthreads();
      fetch(i + 1);
      const int n = live(i);
      state_update<kParts>(sV, sK, m, w, StateWeights(tables, n), 1.f, n < kChunk ? la_power(lg, n) : full, M);
      if (local) {
        state_update<3>(sQ, sO, m, w, wl, past, 1.f, L);
        past *= full;
      }
      __syncthreads();   // every wave is done with the tiles
    }
    if (local && chunks) state_store(L, local + it.at * kState);
  } else {
    fetch(0);
    const ScoreWeights sw(lg, gm.scale, false);
    const float carry = gm.scale * la_power(lg, 16 * w + c + 1), mid = la_mid(t1 - t0).rows;
    for (int i = 0; i < chunks; ++i) {
      put();
      __syncthreads();
      fetch(i + 1);
      const int row = 16 * w + c;
      const bf16x8 a[2] = {tile_row(sO, m, w, 0), tile_row(sO, m, w, 1)};
      f32x4 o[4] = {zero4(), zero4(), zero4(), zero4()};
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int p = 0; p < kParts; ++p) o[ct] = mfma16_bf16(tile_row(sM + p * kTileBytes, m, ct, ks), a[ks], o[ct]);
      rows_scale(o, carry);
      if constexpr (DECAY) {
        float sum = 0.f;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const uint2 x2 = *reinterpret_cast<const uint2*>(sQ + (m.slots ^ 32 * ct) + 2048 * w);
          sum = fmaf(o[ct][0], bf16_lo(x2.x), fmaf(o[ct][1], bf16_hi(x2.x), fmaf(o[ct][2], bf16_lo(x2.y), fmaf(o[ct][3], bf16_hi(x2.y), sum))));
        }
        total = fma(static_cast<double>(static_cast<float>(i * kChunk + row + 1) - mid), static_cast<double>(sum), total);   // dead rows of q are zero
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (2 * ks <= w) {
          float p[8];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int jt = 2 * ks + half;
            f32x4 z = zero4();
            if (jt <= w) {
              z = mfma16_bf16(tile_row(sV, m, jt, 0), a[0], z);
              z = mfma16_bf16(tile_row(sV, m, jt, 1), a[1], z);
            }
            sw.apply(z, w - jt, p + 4 * half);
          }
          bf16x8 parts[2];
          split8<2>(p, parts);
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) {
            const bf16x8 k = tile_column(sK, m, ct, ks);
            o[ct] = mfma16_bf16(k, parts[0], o[ct]);
            o[ct] = mfma16_bf16(k, parts[1], o[ct]);
          }
        }
      }
      put_rows(po + (t0 + static_cast<int64_t>(i) * kChunk + row) * o2, row < live(i), o);
      __syncthreads();   // every wave is done with the tiles
    }
  }
  if constexpr (DECAY) {
    const double sum = workgroup_sum_f64<kWideThreads / kWave>(total, reinterpret_cast<double*>(smem));
    if (threadIdx.x == 0) dot[it.at] = sum;
  }
}

// One gradient of la_dkdv_bf16: dv, with its rows of k from LDS, or (KEYS) dk, with its rows of v in registers.  DECAY: the
// keys' side of dlog_decay (see la_dq_bf16), returned by the dk waves.  Without it a chunk's tiles and G's two parts have
// two LDS buffers each; with it G has three parts, and all have one buffer and a second barrier.
template <bool KEYS, bool DECAY, typename TO>
__device__ __forceinline__ double la_dkdv_role(char* smem, const LaRows& Q_, const LaRows& O_, const LaRows& K_, const LaRows& V_,
                                              const LaGeom& gm, const LaItem& it, int t0, int t1,
                                              const float* __restrict__ enter, TO* __restrict__ pr, int64_t stride) {
  constexpr int kParts = DECAY ? 3 : 2;        // of G in LDS
  constexpr int kRead = KEYS ? kParts : 2;     // that this wave's rows take
  const int l = threadIdx.x % kWave, w = uniform(threadIdx.x / kWave) % 4, g = l / 16, c = l % 16;
  const float lg = la_log2_decay(gm, it.h), full = la_power(lg, kChunk);
  const bf16 *pq = la_rows_of(Q_, gm.H, gm, it), *pdo = la_rows_of(O_, gm.H, gm, it);
  const bf16 *pv = la_rows_of(V_, gm.Hkv, gm, it), *pk = la_rows_of(K_, gm.Hkv, gm, it);
  const TileMap m(threadIdx.x);
  f32x4 G[4];
  if constexpr (!KEYS) state_load(enter ? enter + it.at * kState : nullptr, false, G);
  const int chunks = t1 > t0 ? (t1 - t0 + kChunk - 1) / kChunk : 0;
  // chunk i counts from the end; behind the first one nothing is live
  auto live = [&](int i) { return i >= chunks ? 0 : i > 0 ? kChunk : t1 - t0 - (chunks - 1) * kChunk; };
  auto token = [&](int i) { return t0 + static_cast<int64_t>(i < chunks ? chunks - 1 - i : 0) * kChunk; };
  uint4 xq, xo, xk, own[2];
  auto fetch = [&](int i) {
    const int64_t t = token(i);
    xq = tile_fetch_wide(pq + t * Q_.s2, Q_.s2, live(i));
    xo = tile_fetch_wide(pdo + t * O_.s2, O_.s2, live(i));
    xk = tile_fetch_wide(pk + t * K_.s2, K_.s2, live(i));
    if constexpr (KEYS) {   // v in slot order: elements 32 p + 4 g + [0, 4) and 16 on
      const int ld = static_cast<int>(V_.s2) * 2;
      const __amdgpu_buffer_rsrc_t r = rows_rsrc(pv + t * V_.s2, ld, live(i), 128);
      const uint32_t row = static_cast<uint32_t>(16 * w + c) * static_cast<uint32_t>(ld) + 8 * g;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const auto a = __builtin_amdgcn_raw_buffer_load_b64(r, row + 64 * p, 0, 0);
        const auto b = __builtin_amdgcn_raw_buffer_load_b64(r, row + 64 * p + 32, 0, 0);
        own[p] = uint4{a[0], a[1], b[0], b[1]};
      }
    }
  };
  const ScoreWeights sw(lg, gm.scale, true);
  const AdjointWeights wt(lg, gm.scale);
  const float mid = la_mid(t1 - t0).keys;
  double total = 0.;
  fetch(0);
  for (int i = 0; i < chunks; ++i) {
    const int n = live(i);
    char *sQ = smem + (DECAY ? 0 : (i & 1) * 5 * kTileBytes), *sO = sQ + kTileBytes, *sK = sQ + 2 * kTileBytes, *sG = sQ + 3 * kTileBytes;
    tile_put_wide(xq, sQ, m);
    tile_put_wide(xo, sO, m);
    tile_put_wide(xk, sK, m);
    if constexpr (!KEYS) state_put<kParts>(G, sG, m);
    bf16x8 a[2] = {bf16x8_from_bits(own[0]), bf16x8_from_bits(own[1])};
    __syncthreads();   // without DECAY also: every wave is done with the other buffer
    fetch(i + 1);
    if constexpr (!KEYS) {
      a[0] = tile_row(sK, m, w, 0);
      a[1] = tile_row(sK, m, w, 1);
    }
    const int row = 16 * w + c;
    f32x4 acc[4] = {zero4(), zero4(), zero4(), zero4()};
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int part = 0; part < kRead; ++part) {
          const char* s = sG + part * kTileBytes;
          acc[ct] = mfma16_bf16(KEYS ? tile_column(s, m, ct, ks) : tile_row(s, m, ct, ks), a[ks], acc[ct]);
        }
    rows_scale(acc, la_power(lg, n - 1 - row < 0 ? 0 : n - 1 - row));
    if constexpr (KEYS && DECAY) {
      float sum = 0.f;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        const uint2 k = *reinterpret_cast<const uint2*>(sK + (m.slots ^ 32 * ct) + 2048 * w);
        sum = fmaf(acc[ct][0], bf16_lo(k.x), fmaf(acc[ct][1], bf16_hi(k.x), fmaf(acc[ct][2], bf16_lo(k.y), fmaf(acc[ct][3], bf16_hi(k.y), sum))));
      }
      total = fma(static_cast<double>(static_cast<float>(token(i) + row - t0 + 1) - mid), static_cast<double>(sum), total);   // dead rows of k are zero
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (2 * ks + 1 >= w) {   // uniform: some of the 32 tokens are not before the wave's rows
        float p[8];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int tt = 2 * ks + hf;
          f32x4 z = zero4();
          if (tt >= w) {
            z = mfma16_bf16(KEYS ? tile_row_slots(sO, m, tt, 0) : tile_row(sQ, m, tt, 0), a[0], z);
            z = mfma16_bf16(KEYS ? tile_row_slots(sO, m, tt, 1) : tile_row(sQ, m, tt, 1), a[1], z);
          }
          sw.apply(z, tt - w, p + 4 * hf);
          if constexpr (KEYS && DECAY) {
            if (tt >= w) {
              f32x4 y = zero4();
              y = mfma16_bf16(tile_row(sQ, m, tt, 0), tile_row(sK, m, w, 0), y);
              y = mfma16_bf16(tile_row(sQ, m, tt, 1), tile_row(sK, m, w, 1), y);
              const float gap = static_cast<float>(16 * (tt - w) + 4 * g - c);
              float pairs = 0.f;
#pragma unroll
              for (int r = 0; r < 4; ++r) pairs = fmaf((gap + static_cast<float>(r)) * p[4 * hf + r], y[r], pairs);
              total -= pairs;
            }
          }
        }
        bf16x8 parts[2];
        split8<2>(p, parts);
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const bf16x8 v = tile_column(KEYS ? sQ : sO, m, ct, ks);
          acc[ct] = mfma16_bf16(v, parts[0], acc[ct]);
          acc[ct] = mfma16_bf16(v, parts[1], acc[ct]);
        }
      }
    }
    put_rows(pr + (token(i) + row) * stride, row < n, acc);
    if constexpr (!KEYS) {
      state_update<kParts>(sQ, sO, m, w, wt, 1.f, n < kChunk ? la_power(lg, n) : full, G);
    }
    if constexpr (DECAY) __syncthreads();   // every wave is done with the tiles
  }
  return total;
}

// dk and dv of a segment, chunks from its end, G the adjoint of the state behind the chunk:
//   dv_j = scale sum_{i >= j} g^{i-j} (k_j.q_i) do_i + g^{n-1-j} k_j G,  dk_j the same with v, do, q and G^T.
// Four waves form dv and keep G, and four form dk.  The q and do tiles serve as rows and as columns; G lies in LDS
// transposed, read by rows for dv and transposed for dk.  Both roles pass the same barriers.
template <bool DECAY, typename TO>
__global__ __launch_bounds__(kWideThreads, 4) void la_dkdv_bf16(LaRows Q_, LaRows O_, LaRows K_, LaRows V_, LaGeom gm,
                                                                const float* __restrict__ enter, TO* __restrict__ dk,
                                                                int64_t k0, int64_t k1, int64_t k2, TO* __restrict__ dv,
                                                                int64_t v0, int64_t v1, int64_t v2, int outh,
                                                                double* __restrict__ dot) {
  __shared__ __align__(16) char smem[(DECAY ? 6 : 10) * kTileBytes];   // q, do, k and G's parts
  const LaItem it = la_item(gm);
  const int len = la_length(gm, it.b), t0 = it.seg * gm.seg;
  const int tend = t0 + gm.seg < gm.N ? t0 + gm.seg : gm.N;
  const int t1 = tend < len ? tend : len;
  const int oh = it.h / (gm.H / outh);
  TO *pdk = dk + it.b * k0 + oh * k1, *pdv = dv + it.b * v0 + oh * v1;
  la_zero_rows(pdk, k2, t1 > t0 ? t1 : t0, tend);
  la_zero_rows(pdv, v2, t1 > t0 ? t1 : t0, tend);
  double total;
  if (uniform(threadIdx.x / kWave) >= 4) total = la_dkdv_role<true, DECAY>(smem, Q_, O_, K_, V_, gm, it, t0, t1, enter, pdk, k2);
  else total = la_dkdv_role<false, DECAY>(smem, Q_, O_, K_, V_, gm, it, t0, t1, enter, pdv, v2);
  if constexpr (DECAY) {
    const double sum = workgroup_sum_f64<kWideThreads / kWave>(total, reinterpret_cast<double*>(smem));
    if (threadIdx.x == 0) dot[it.at] = sum;
  }
}

// dk (blockIdx.y 0) and dv of a shared head: the query heads' parts in head order.
template <typename T>
struct LaShared {
  const float* part;
  T* out;
  int64_t o0, o1, o2;
};
template <typename T>
__global__ __launch_bounds__(kLaThreads) void la_group_sum(LaShared<T> dk, LaShared<T> dv, LaGeom gm) {
  const LaShared<T>& x = blockIdx.y ? dv : dk;
  const int group = gm.H / gm.Hkv;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kLaThreads + threadIdx.x;   // four elements of a row
  const int d = static_cast<int>(i % (kHd / 4)) * 4;
  const int64_t row = i / (kHd / 4);
  if (row >= static_cast<int64_t>(gm.B) * gm.Hkv * gm.N) return;
  const int64_t n = row % gm.N, kv = row / gm.N % gm.Hkv, b = row / gm.N / gm.Hkv;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q = 0; q < group; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(x.part + ((b * gm.H + kv * group + q) * gm.N + n) * kHd + d);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  const float v[4] = {s.x, s.y, s.z, s.w};
  store_vec<T, 4>(x.out + b * x.o0 + kv * x.o1 + n * x.o2 + d, v);
}

// dlog_decay[h]: the segments' sums over the batch, then the boundary terms; a workgroup per head, fixed order.
__global__ __launch_bounds__(kLaThreads) void la_dlog_kernel(const double* __restrict__ dq_dot,
                                                             const double* __restrict__ dk_dot,
                                                             const double* __restrict__ edge, int edges, LaGeom gm,
                                                             float* __restrict__ dlog) {
  __shared__ double s_red[kLaThreads / kWave];
  const int h = blockIdx.x;
  double t = 0.;
  if (dq_dot) {
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(gm.B) * gm.segs; i += kLaThreads) {
      const int64_t b = i / gm.segs, s = i % gm.segs;
      if (s * gm.seg < la_length(gm, static_cast<int>(b))) {
        const int64_t at = (b * gm.H + h) * gm.segs + s;
        t += dq_dot[at] - dk_dot[at];
      }
    }
  }
  if (edge)
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(gm.B) * edges; i += kLaThreads)
      t += edge[(i / edges * gm.H + h) * edges + i % edges];
  t = workgroup_sum_f64<kLaThreads / kWave>(t, s_red);
  if (threadIdx.x == 0) dlog[h] = gm.log_decay[h] > 0.f ? 0.f : static_cast<float>(t);
}

// One token of each row, S' = g S + k v^T, o = scale q S': a workgroup for each (row, head), whose threads hold four by four
// elements of the state, all of it in flight at once; the rows of the result are added through LDS.  The state is read and
// written once and is all there is: bound by memory.  256 rows of H8 (67 MB): 12.6 us, 5.3 TB/s; one row 3.9 us, a launch's
// own time.  A slot that several rows share is worked by the first one's workgroups, row after row, and the others leave:
// each looks the slots through once, 256 at a time.
constexpr int kStepThreads = 256;
template <typename T>
__global__ __launch_bounds__(kStepThreads) void la_step_kernel(dwarf_linear_attention_step_args a) {
  __shared__ float s_o[kStepThreads / 16][kHd];
  __shared__ int s_next;
  const int h = blockIdx.x % a.H, row0 = blockIdx.x / a.H, kv = h / (a.H / a.H_kv);
  const int c4 = threadIdx.x % 16 * 4, r0 = threadIdx.x / 16 * 4;   // four rows and four columns of the state
  const int slot = a.slots ? a.slots[row0] : row0;
  if (slot < 0 || slot >= a.pool) {
    if (threadIdx.x < kHd)
      static_cast<T*>(a.out)[row0 * a.out_stride[0] + h * a.out_stride[1] + threadIdx.x] = from_f32<T>(0.f);
    return;
  }
  LaGeom gm;
  gm.log_decay = a.log_decay;
  const float decay = la_power(la_log2_decay(gm, h), 1);
  // the first row of a slot takes the slot's later rows after it, in order
  auto next_of = [&](int from) {
    __syncthreads();
    if (threadIdx.x == 0) s_next = a.S;
    __syncthreads();
    for (int i = from + static_cast<int>(threadIdx.x); i < a.S; i += kStepThreads)
      if (a.slots[i] == slot) {
        atomicMin(&s_next, i);
        break;
      }
    __syncthreads();
    return s_next;
  };
  const int64_t at = slot * a.slot_stride + static_cast<int64_t>(h) * kState;
  float4 st[4];   // under way while the slots are looked through
#pragma unroll
  for (int i = 0; i < 4; ++i) st[i] = *reinterpret_cast<const float4*>(a.state + at + (r0 + i) * kHd + c4);
  float qv[4], kx[4], vx[4];
  auto fetch = [&](int row) {
    load_vec<T, 4>(static_cast<const T*>(a.q) + row * a.q_stride[0] + h * a.q_stride[1] + r0, qv);
    load_vec<T, 4>(static_cast<const T*>(a.k) + row * a.k_stride[0] + kv * a.k_stride[1] + r0, kx);
    load_vec<T, 4>(static_cast<const T*>(a.v) + row * a.v_stride[0] + kv * a.v_stride[1] + c4, vx);
  };
  fetch(row0);
  if (row0 > 0 && a.slots && next_of(0) < row0) return;   // uniform
  for (int row = row0; row < a.S;) {
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      st[i].x = fmaf(decay, st[i].x, kx[i] * vx[0]);
      st[i].y = fmaf(decay, st[i].y, kx[i] * vx[1]);
      st[i].z = fmaf(decay, st[i].z, kx[i] * vx[2]);
      st[i].w = fmaf(decay, st[i].w, kx[i] * vx[3]);
      o[0] = fmaf(qv[i], st[i].x, o[0]);
      o[1] = fmaf(qv[i], st[i].y, o[1]);
      o[2] = fmaf(qv[i], st[i].z, o[2]);
      o[3] = fmaf(qv[i], st[i].w, o[3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) s_o[threadIdx.x / 16][c4 + i] = o[i];
    __syncthreads();
    if (threadIdx.x < kHd) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kStepThreads / 16; ++i) t += s_o[i][threadIdx.x];
      static_cast<T*>(a.out)[row * a.out_stride[0] + h * a.out_stride[1] + threadIdx.x] = from_f32<T>(a.scale * t);
    }
    row = a.slots && row + 1 < a.S ? next_of(row + 1) : a.S;
    if (row < a.S) fetch(row);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(a.new_state + at + (r0 + i) * kHd + c4) = st[i];
}

// Tokens of a segment: the longest whose workgroups fill the card.  Long ones (512 and 1,024 tokens) have to leave two for
// each CU, since their rows are bound by what a CU computes: B15 N2048 H8, bf16 forward 45.5 us with 480 workgroups of 512
// tokens, 54.8 with 240 of 1,024.  Short ones one: B4 N2048 H8 20.2 us forward and 42.3 backward with 256 of 256 tokens,
// 24.5 and 45.5 with 512 of 128 (more sums to join).  More of them than that only adds states: B1 N65536 H8 97.7 us with
// 512 of 1,024 tokens, 106 with 1,024 of 512.
int la_segment(int64_t B, int64_t H, int64_t N) {
  for (int seg = 1024; seg > kChunk; seg /= 2)
    if (B * H * ((N + seg - 1) / seg) >= (seg >= 512 ? 448 : 224)) return seg;
  return kChunk;
}

LaGeom la_geom(const dwarf_linear_attention_fwd_args& a) {
  LaGeom gm;
  gm.B = a.B; gm.H = a.H; gm.Hkv = a.H_kv; gm.N = a.N;
  gm.seg = la_segment(a.B, a.H, a.N);
  gm.segs = (a.N + gm.seg - 1) / gm.seg;
  gm.scale = a.scale;
  gm.log_decay = a.log_decay;
  gm.lengths = a.lengths;
  return gm;
}

// The forward's segments are joined by a launch of the scan (also where there are none: the state that enters leaves).
bool la_scanned(const LaGeom& gm) { return gm.segs == 0 || gm.segs > kScanRun; }
LaEnter la_enter(const dwarf_linear_attention_fwd_args& a, const LaGeom& gm) {
  if (la_scanned(gm)) return LaEnter{a.states, nullptr, nullptr};
  return LaEnter{nullptr, a.initial, gm.segs > 1 ? a.states : nullptr};
}

// A single row's stride is whatever the caller's view says: rows behind it must not fall on it.
LaRows la_operand(const void* p, const int64_t* s, int N) { return LaRows{p, s[0], s[1], N > 1 ? s[2] : kHd}; }

void la_fwd_bf16(const dwarf_linear_attention_fwd_args& a, const LaGeom& gm, hipStream_t stream) {
  const LaRows q = la_operand(a.q, a.q_stride, gm.N), k = la_operand(a.k, a.k_stride, gm.N), v = la_operand(a.v, a.v_stride, gm.N);
  const dim3 grid(static_cast<unsigned>(gm.B) * gm.H * gm.segs);
  const bool scanned = la_scanned(gm);
  if (gm.segs > 1)
    hipLaunchKernelGGL(la_local_bf16, grid, dim3(kLaThreads), 0, stream, k, gm.Hkv, v, gm.Hkv, gm, a.states);
  if (scanned) la_scan<false>(a.states, a.initial, a.final, gm, nullptr, nullptr, nullptr, nullptr, stream);
  if (gm.segs == 0) return;
  hipLaunchKernelGGL(la_rows_bf16, grid, dim3(kWideThreads), 0, stream, q, k, v, gm, la_enter(a, gm),
                     static_cast<bf16*>(a.out), a.out_stride[0], a.out_stride[1], a.out_stride[2], scanned ? nullptr : a.final);
}

template <typename T>
void la_fwd_typed(const dwarf_linear_attention_fwd_args& a, const LaGeom& gm, hipStream_t stream) {
  const LaRows q = la_operand(a.q, a.q_stride, gm.N), k = la_operand(a.k, a.k_stride, gm.N), v = la_operand(a.v, a.v_stride, gm.N);
  const dim3 grid(static_cast<unsigned>(gm.B) * gm.H * gm.segs), block(kLaThreads);
  const bool scanned = la_scanned(gm);
  if (gm.segs > 1)
    hipLaunchKernelGGL((la_local_kernel<T, false>), grid, block, 0, stream, k, gm.Hkv, v, gm.Hkv, gm, 1.f, a.states);
  if (scanned) la_scan<false>(a.states, a.initial, a.final, gm, nullptr, nullptr, nullptr, nullptr, stream);
  if (gm.segs == 0) return;
  const LaRowsCall<T> call{q, k, v, LaRows{}, gm.H, gm.Hkv, gm.Hkv, 1, la_enter(a, gm), false, static_cast<T*>(a.out), a.out_stride[0],
                           a.out_stride[1], a.out_stride[2], nullptr};
  hipLaunchKernelGGL((la_rows_kernel<T, T, false>), grid, block, 0, stream, call, call, gm, gm.scale, gm.scale, 1.f,
                     scanned ? nullptr : a.final);
}

// Whether the backward needs the adjoint's scan: several segments, the gradient of the state that enters, or boundary terms
// of dlog_decay.  A single segment has those only where a state enters or its adjoint does; one chunk only where both do.
// Without it a training call of one segment has a launch less (of four), and dq forms no sums.
bool la_joined(const dwarf_linear_attention_bwd_args& a, const LaGeom& gm) {
  if (gm.segs != 1 || a.dinitial) return true;
  if (!a.dlog_decay) return false;
  return gm.N <= kChunk ? a.fwd.initial && a.dfinal : a.fwd.initial || a.dfinal;
}

// Workspace of the backward, in floats: the adjoints per segment, the dlog_decay sums, the shared heads' parts.
struct LaBwdSpace {
  size_t adjoint, dq_dot, dk_dot, edge, dk_part, dv_part, total;
};
LaBwdSpace la_bwd_space(const dwarf_linear_attention_bwd_args& a, const LaGeom& gm) {
  const size_t wgs = static_cast<size_t>(gm.B) * gm.H * gm.segs, rows = static_cast<size_t>(gm.B) * gm.H * gm.N * kHd;
  const bool shared = gm.H != gm.Hkv;
  auto pad = [](size_t n) { return (n + 63) / 64 * 64; };
  LaBwdSpace s;
  size_t at = 0;
  s.adjoint = at; at += wgs * kState;
  s.dq_dot = at; at += a.dlog_decay ? pad(2 * wgs) : 0;   // 64 bits each
  s.dk_dot = at; at += a.dlog_decay ? pad(2 * wgs) : 0;
  s.edge = at; at += a.dlog_decay ? pad(2 * static_cast<size_t>(gm.B) * gm.H * scan_wgs(gm)) : 0;
  s.dk_part = at; at += shared ? rows : 0;
  s.dv_part = at; at += shared ? rows : 0;
  s.total = at;
  return s;
}

template <typename T>
void la_bwd_typed(const dwarf_linear_attention_bwd_args& a, const LaGeom& gm, hipStream_t stream) {
  const dwarf_linear_attention_fwd_args& f = a.fwd;
  const LaRows q = la_operand(f.q, f.q_stride, gm.N), k = la_operand(f.k, f.k_stride, gm.N), v = la_operand(f.v, f.v_stride, gm.N);
  const LaRows dout = la_operand(a.dout, a.dout_stride, gm.N);
  const dim3 grid(static_cast<unsigned>(gm.B) * gm.H * gm.segs), block(kLaThreads);
  const LaBwdSpace sp = la_bwd_space(a, gm);
  float* ws = static_cast<float*>(a.workspace);
  const bool dlog = a.dlog_decay != nullptr;
  float* adj = ws + sp.adjoint;
  double* dq_dot = dlog ? reinterpret_cast<double*>(ws + sp.dq_dot) : nullptr;
  double* dk_dot = dlog ? reinterpret_cast<double*>(ws + sp.dk_dot) : nullptr;
  double* edge = dlog ? reinterpret_cast<double*>(ws + sp.edge) : nullptr;
  const bool joined = la_joined(a, gm);
  const float* enter = joined ? adj : a.dfinal;
  const LaEnter before = la_enter(f, gm), behind = joined ? LaEnter{adj, nullptr, nullptr} : LaEnter{nullptr, a.dfinal, nullptr};
  const bool shared = gm.H != gm.Hkv;
  float *pk = ws + sp.dk_part, *pv = ws + sp.dv_part;
  const int64_t s1 = static_cast<int64_t>(gm.N) * kHd, s0 = s1 * gm.H;   // of the shared heads' parts
  const dim3 wide(kWideThreads);
  if constexpr (std::is_same<T, bf16>::value) {
    if (gm.segs) {
      auto kernel = dlog ? la_dq_bf16<true> : la_dq_bf16<false>;
      hipLaunchKernelGGL(kernel, grid, wide, 0, stream, q, dout, k, v, gm, before, static_cast<bf16*>(a.dq), a.dq_stride[0],
                         a.dq_stride[1], a.dq_stride[2], joined ? adj : nullptr, dq_dot);
    }
  } else if (joined && gm.segs) {
    hipLaunchKernelGGL((la_local_kernel<T, true>), grid, block, 0, stream, q, gm.H, dout, gm.H, gm, gm.scale, adj);
  }
  if (joined)
    la_scan<true>(adj, a.dfinal, a.dinitial, gm, f.states, f.initial, f.final, edge, stream);
  if (gm.segs) {
    if constexpr (std::is_same<T, bf16>::value) {
      if (shared) {
        auto kernel = dlog ? la_dkdv_bf16<true, float> : la_dkdv_bf16<false, float>;
        hipLaunchKernelGGL(kernel, grid, wide, 0, stream, q, dout, k, v, gm, enter, pk, s0, s1, int64_t(kHd), pv, s0, s1,
                           int64_t(kHd), gm.H, dk_dot);
      } else {
        auto kernel = dlog ? la_dkdv_bf16<true, bf16> : la_dkdv_bf16<false, bf16>;
        hipLaunchKernelGGL(kernel, grid, wide, 0, stream, q, dout, k, v, gm, enter, static_cast<bf16*>(a.dk), a.dk_stride[0],
                           a.dk_stride[1], a.dk_stride[2], static_cast<bf16*>(a.dv), a.dv_stride[0], a.dv_stride[1],
                           a.dv_stride[2], gm.Hkv, dk_dot);
      }
    } else {
      const LaRowsCall<T> rows{dout, v, k, q, gm.H, gm.Hkv, gm.Hkv, gm.H, before, true, static_cast<T*>(a.dq), a.dq_stride[0],
                               a.dq_stride[1], a.dq_stride[2], dq_dot};
      hipLaunchKernelGGL((la_rows_kernel<T, T, false>), grid, block, 0, stream, rows, rows, gm, gm.scale, gm.scale, 1.f,
                         nullptr);
      const dim3 both(grid.x, 2);
      if (shared) {
        const LaRowsCall<float> cv{k, q, dout, LaRows{}, gm.Hkv, gm.H, gm.H, 1, behind, false, pv, s0, s1, kHd, nullptr};
        const LaRowsCall<float> ck{v, dout, q, k, gm.Hkv, gm.H, gm.H, gm.Hkv, behind, true, pk, s0, s1, kHd, dk_dot};
        hipLaunchKernelGGL((la_rows_kernel<T, float, true>), both, block, 0, stream, cv, ck, gm, gm.scale, 1.f, gm.scale,
                           nullptr);
      } else {
        const LaRowsCall<T> cv{k, q, dout, LaRows{}, gm.Hkv, gm.H, gm.H, 1, behind, false, static_cast<T*>(a.dv),
                               a.dv_stride[0], a.dv_stride[1], a.dv_stride[2], nullptr};
        const LaRowsCall<T> ck{v, dout, q, k, gm.Hkv, gm.H, gm.H, gm.Hkv, behind, true, static_cast<T*>(a.dk),
                               a.dk_stride[0], a.dk_stride[1], a.dk_stride[2], dk_dot};
        hipLaunchKernelGGL((la_rows_kernel<T, T, true>), both, block, 0, stream, cv, ck, gm, gm.scale, 1.f, gm.scale, nullptr);
      }
    }
    if (shared) {
      const int64_t quads = static_cast<int64_t>(gm.B) * gm.Hkv * gm.N * (kHd / 4);
      const LaShared<T> sk{pk, static_cast<T*>(a.dk), a.dk_stride[0], a.dk_stride[1], a.dk_stride[2]};
      const LaShared<T> sv{pv, static_cast<T*>(a.dv), a.dv_stride[0], a.dv_stride[1], a.dv_stride[2]};
      hipLaunchKernelGGL((la_group_sum<T>), dim3(static_cast<unsigned>((quads + kLaThreads - 1) / kLaThreads), 2), block, 0,
                         stream, sk, sv, gm);
    }
  }
  if (dlog)
    hipLaunchKernelGGL(la_dlog_kernel, dim3(gm.H), block, 0, stream, gm.segs ? dq_dot : nullptr, dk_dot, joined ? edge : nullptr,
                       scan_wgs(gm), gm, a.dlog_decay);
}

}  // namespace

int linear_attention_segment(int B, int H, int N) { return la_segment(B, H, N); }

size_t linear_attention_states_bytes(const dwarf_linear_attention_fwd_args& a) {
  const LaGeom gm = la_geom(a);
  return gm.segs > 1 ? static_cast<size_t>(gm.B) * gm.H * gm.segs * kState * sizeof(float) : 0;
}

size_t linear_attention_bwd_workspace(const dwarf_linear_attention_bwd_args& a) {
  return la_bwd_space(a, la_geom(a.fwd)).total * sizeof(float);
}

hipError_t launch_linear_attention_fwd(const dwarf_linear_attention_fwd_args& a, hipStream_t stream) {
  const LaGeom gm = la_geom(a);
  if (a.dtype == DWARF_F32) la_fwd_typed<float>(a, gm, stream);
  else if (a.dtype == DWARF_F16) la_fwd_typed<f16>(a, gm, stream);
  else la_fwd_bf16(a, gm, stream);
  return hipGetLastError();
}

hipError_t launch_linear_attention_bwd(const dwarf_linear_attention_bwd_args& a, hipStream_t stream) {
  const LaGeom gm = la_geom(a.fwd);
  if (a.fwd.dtype == DWARF_F32) la_bwd_typed<float>(a, gm, stream);
  else if (a.fwd.dtype == DWARF_F16) la_bwd_typed<f16>(a, gm, stream);
  else la_bwd_typed<bf16>(a, gm, stream);
  return hipGetLastError();
}

hipError_t launch_linear_attention_step(const dwarf_linear_attention_step_args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.S) * a.H), block(kStepThreads);
  if (a.dtype == DWARF_F32) hipLaunchKernelGGL((la_step_kernel<float>), grid, block, 0, stream, a);
  else if (a.dtype == DWARF_F16) hipLaunchKernelGGL((la_step_kernel<f16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((la_step_kernel<bf16>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace dwarf
