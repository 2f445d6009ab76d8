// A short causal convolution of each channel, forward, backward and for single
// tokens:
//   p_t = bias + sum_j w_j x_{t-W+1+j},   y_t = p_t or silu(p_t)
//   dp = dy silu'(p),  dx_t = sum_j w_j dp_{t+W-1-j},  dw_j = sum dp_t x_{t-W+1+j},  dbias = sum dp
//
// Forward bound by memory, backward by memory and the vector units (69% of their
// cycles) together.  B15 N2048, 1,024 channels in bf16, W 4, inputs from memory:
// forward 33.5 us (126 MB, 3.8 TB/s), backward 53 (189 MB, 3.6 TB/s), the sums
// 4; from the last-level cache 26 and 48.  B20 of 1,031 channels in fp16, W 3:
// 37 us (169 MB, 4.6 TB/s).
//
// A thread takes VEC adjacent channels (forward 16 bytes of
// them, backward four: with eight, 148 registers left too few waves, 86 us
// where four take 54) and walks a strip of tokens with the last W - 1 inputs in
// registers, four rows on their way (two to eight: the same within 4%): each
// input is loaded once but for the W - 1 rows in front of a strip, which another
// strip's thread loads at about the same time, from the same L2.  Forward the
// threads go over whole rows in order (in rectangles of 32 vectors, as the
// backward's sums have it, the 1,031 channels took 43 us).  Rows need no
// alignment but their elements': gfx950 loads 16 bytes from any address, and a
// width that VEC does not divide has its last vector moved back to the row's
// end, where two threads then store the same values.  The backward forms p
// again from x, which it needs for dw anyway, instead of reading a saved one; a
// strip goes W - 1 tokens further to have the dp that its own dx need.  dw and
// dbias: a thread's sums over its strip in registers, a workgroup's over its
// strips in LDS, then one partial row for each workgroup and a last launch that
// adds those in order, in 64 bits.
#include "selective.h"

namespace dwarf {
namespace {

constexpr int kConvThreads = 256;
constexpr int kConvCols = 32;                              // vectors of channels in a workgroup
constexpr int kConvStrips = kConvThreads / kConvCols;      // strips of tokens in a workgroup
constexpr int kConvAhead = 4;                              // rows of a thread on their way

template <typename T, int VEC>
__device__ __forceinline__ void load_any(const T* p, float* x) {
  T v[VEC];
  __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = to_f32(v[e]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_any(T* p, const float* x) {
  T v[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = from_f32<T>(x[e]);
  __builtin_memcpy(p, v, sizeof(v));
}

struct ConvGeom {
  int cols;        // vectors of channels of a row
  int col_blocks;  // workgroups over them
  int strip;       // tokens of a strip
  int strips;      // strips of a sequence
};

__device__ __forceinline__ int conv_length(const dwarf_causal_conv_fwd_args& a, int b) {
  if (!a.lengths) return a.N;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.N ? a.N : n;
}

// Where a thread stands: its vector's first channel (the last vector lies at the row's end), its sequence and strip.
template <int VEC>
struct ConvAt {
  int d, b, strip, col;
  bool in;
  // FLAT: the threads in order over a strip's vectors, then the next strip's; otherwise a workgroup is a rectangle
  template <bool FLAT>
  static __device__ __forceinline__ ConvAt make(int D, const ConvGeom& gm, int B) {
    ConvAt at;
    // neighbours, which share a strip's first rows and the lines where their vectors meet, on one L2
    const uint32_t block = xcd_remap(blockIdx.x, gridDim.x);
    int64_t s;
    if constexpr (FLAT) {
      const uint32_t i = block * kConvThreads + threadIdx.x;   // a launch has fewer than 2^31 threads
      s = i / static_cast<uint32_t>(gm.cols);
      at.col = i - static_cast<uint32_t>(s) * static_cast<uint32_t>(gm.cols);
    } else {
      at.col = block % static_cast<uint32_t>(gm.col_blocks) * kConvCols + threadIdx.x % kConvCols;
      s = static_cast<int64_t>(block / static_cast<uint32_t>(gm.col_blocks)) * kConvStrips + threadIdx.x / kConvCols;
    }
    at.place(s, D, gm, B);
    return at;
  }
  __device__ __forceinline__ void place(int64_t s, int D, const ConvGeom& gm, int B) {
    in = col < gm.cols && s < static_cast<int64_t>(B) * gm.strips;
    b = in ? static_cast<int>(s / gm.strips) : 0;
    strip = in ? static_cast<int>(s - static_cast<int64_t>(b) * gm.strips) : 0;
    d = col * VEC;
    if (d > D - VEC) d = D - VEC;   // D >= VEC
    if (!in) d = 0;
  }
};

template <int VEC, int W>
__device__ __forceinline__ void conv_weights(const float* weight, const float* bias, int d, float (*w)[VEC], float* c) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = weight[static_cast<int64_t>(d + e) * W + j];
    c[e] = bias ? bias[d + e] : 0.f;
  }
}

// Input row t of a sequence, t >= -(W - 1): the state's in front of the first token.
template <typename T, int VEC, int W>
__device__ __forceinline__ void conv_input(const dwarf_causal_conv_fwd_args& a, const T* x, int b, int d, int t, float* v) {
  if (t >= 0) {
    load_any<T, VEC>(x + t * a.x_stride[1], v);
  } else if (a.initial) {
    load_any<T, VEC>(static_cast<const T*>(a.initial) + (static_cast<int64_t>(b) * (W - 1) + (t + W - 1)) * a.D + d, v);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.f;
  }
}

template <typename T, int VEC, int W>
__global__ __launch_bounds__(kConvThreads) void conv_fwd_kernel(dwarf_causal_conv_fwd_args a, ConvGeom gm) {
  const auto at = ConvAt<VEC>::template make<true>(a.D, gm, a.B);
  if (!at.in) return;
  const int d = at.d, n = conv_length(a, at.b);
  const int t0 = at.strip * gm.strip, t1 = min(a.N, t0 + gm.strip), end = min(t1, n);
  const T* x = static_cast<const T*>(a.x) + at.b * a.x_stride[0] + d;
  T* y = static_cast<T*>(a.y) + at.b * a.y_stride[0] + d;
  if (t0 < end) {
    float w[W][VEC], c[VEC], win[W][VEC];   // win[j]: input t - W + 1 + j
    conv_weights<VEC, W>(a.weight, a.bias, d, w, c);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_input<T, VEC, W>(a, x, at.b, d, t0 - W + 1 + j, win[j + 1]);
    T raw[kConvAhead][VEC];   // rows on the way; behind the sequence's end its last one again
    const T* from = x + t0 * a.x_stride[1];   // the pointers walk: a 64-bit product a row took the backward 49.4 us, not 47.9
    T* to = y + t0 * a.y_stride[1];
    auto fetch = [&](int t, int i) {
      __builtin_memcpy(raw[i], from, sizeof(raw[i]));
      from += t + 1 < end ? a.x_stride[1] : 0;
    };
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i) fetch(t0 + i, i);
    for (int t = t0; t < end; t += kConvAhead) {
#pragma unroll
      for (int i = 0; i < kConvAhead; ++i) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) win[j][e] = win[j + 1][e];
#pragma unroll
        for (int e = 0; e < VEC; ++e) win[W - 1][e] = to_f32(raw[i][e]);
        fetch(t + i + kConvAhead, i);
        float p[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          p[e] = c[e];
#pragma unroll
          for (int j = 0; j < W; ++j) p[e] = fmaf(w[j][e], win[j][e], p[e]);
          const float s = p[e] * sigmoid_f32(p[e]);
          p[e] = a.silu ? s : p[e];
        }
        if (t + i < end) store_any<T, VEC>(to, p);
        to += a.y_stride[1];
      }
    }
  }
  float z[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) z[e] = 0.f;
  for (int t = max(t0, end); t < t1; ++t) store_any<T, VEC>(y + t * a.y_stride[1], z);
  // the last W - 1 inputs, by the sequence's last strip
  if (a.final && at.strip == gm.strips - 1) {
    T* f = static_cast<T*>(a.final) + static_cast<int64_t>(at.b) * (W - 1) * a.D + d;
    for (int j = 0; j < W - 1; ++j) {
      float v[VEC];
      conv_input<T, VEC, W>(a, x, at.b, d, n - (W - 1) + j, v);
      store_any<T, VEC>(f + static_cast<int64_t>(j) * a.D, v);
    }
  }
}

__device__ __forceinline__ float silu_slope(float p) {
  const float e = sigmoid_f32(p);
  return e * fmaf(p, 1.f - e, 1.f);
}

template <typename T, int VEC, int W>
__global__ __launch_bounds__(kConvThreads) void conv_bwd_kernel(dwarf_causal_conv_bwd_args w_, ConvGeom gm, float* __restrict__ part) {
  __shared__ float s_red[kConvStrips][kConvCols * VEC];
  const dwarf_causal_conv_fwd_args& a = w_.fwd;
  const auto at = ConvAt<VEC>::template make<false>(a.D, gm, a.B);
  const int d = at.d;
  float dw[W + 1][VEC];   // dbias last
#pragma unroll
  for (int j = 0; j <= W; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[j][e] = 0.f;
  if (at.in) {
    const int n = conv_length(a, at.b);
    const int t0 = at.strip * gm.strip, t1 = min(a.N, t0 + gm.strip), end = min(t1, n);
    const T* x = static_cast<const T*>(a.x) + at.b * a.x_stride[0] + d;
    const T* dy = static_cast<const T*>(w_.dy) + at.b * w_.dy_stride[0] + d;
    T* dx = static_cast<T*>(w_.dx) + at.b * w_.dx_stride[0] + d;
    const T* df = w_.dfinal ? static_cast<const T*>(w_.dfinal) + static_cast<int64_t>(at.b) * (W - 1) * a.D + d : nullptr;
    T* di = w_.dinitial ? static_cast<T*>(w_.dinitial) + static_cast<int64_t>(at.b) * (W - 1) * a.D + d : nullptr;
    float w[W][VEC], c[VEC], win[W][VEC], dp[W][VEC];   // dp[i]: token t - i
    conv_weights<VEC, W>(a.weight, a.bias, d, w, c);
    // the state's rows get their gradient from the first strip
    const int from = at.strip == 0 && di ? -(W - 1) : t0;
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) dp[j][e] = 0.f;
    if (n == 0 && from < 0) {   // no token is live: the state that enters leaves
      for (int j = 0; j < W - 1; ++j) {
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.f;
        if (df) load_any<T, VEC>(df + static_cast<int64_t>(j) * a.D, f);
        store_any<T, VEC>(di + static_cast<int64_t>(j) * a.D, f);
      }
    } else if (t0 < end || from < 0) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) conv_input<T, VEC, W>(a, x, at.b, d, t0 - W + 1 + j, win[j + 1]);
      // tokens up to W - 1 behind the strip, whose dp its last tokens' dx need; none behind the sequence's end
      const int stop = end + W - 1;
      T rx[kConvAhead][VEC], rg[kConvAhead][VEC];
      const T *px = x + min(t0, n - 1) * a.x_stride[1], *pg = dy + min(t0, n - 1) * w_.dy_stride[1];
      T* pd = dx + (t0 - (W - 1)) * w_.dx_stride[1];   // dx's row of the token W - 1 in front
      auto fetch = [&](int t, int i) {   // behind the sequence's last token: that again
        __builtin_memcpy(rx[i], px, sizeof(rx[i]));
        __builtin_memcpy(rg[i], pg, sizeof(rg[i]));
        px += t + 1 < n ? a.x_stride[1] : 0;
        pg += t + 1 < n ? w_.dy_stride[1] : 0;
      };
#pragma unroll
      for (int i = 0; i < kConvAhead; ++i) fetch(t0 + i, i);
      for (int tb = t0; tb < stop; tb += kConvAhead) {
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i) {
          const int t = tb + i;
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) win[j][e] = win[j + 1][e];
#pragma unroll
          for (int j = W - 1; j > 0; --j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) dp[j][e] = dp[j - 1][e];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            win[W - 1][e] = to_f32(rx[i][e]);
            const float g = to_f32(rg[i][e]);
            float p = c[e];
#pragma unroll
            for (int j = 0; j < W; ++j) p = fmaf(w[j][e], win[j][e], p);
            const float s = g * silu_slope(p), v = a.silu ? s : g;
            dp[0][e] = t < n ? v : 0.f;   // n is also the first token without a dy
            const float own = t < end ? v : 0.f;   // the strip's own tokens
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j][e] = fmaf(own, win[j][e], dw[j][e]);
            dw[W][e] += own;
          }
          fetch(t + kConvAhead, i);
          const int to = t - (W - 1);   // dx_to = sum_j w_j dp_{to + W - 1 - j} = sum_j w_j dp[j]
          if (to >= t0 ? to < end : to >= from) {
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              v[e] = 0.f;
#pragma unroll
              for (int j = 0; j < W; ++j) v[e] = fmaf(w[j][e], dp[j][e], v[e]);
            }
            // the state that leaves holds inputs n - W + 1 .. n - 1
            if (df && to >= n - (W - 1)) {
              float f[VEC];
              load_any<T, VEC>(df + static_cast<int64_t>(to - (n - (W - 1))) * a.D, f);
#pragma unroll
              for (int e = 0; e < VEC; ++e) v[e] += f[e];
            }
            if (to >= 0) store_any<T, VEC>(pd, v);
            else store_any<T, VEC>(di + static_cast<int64_t>(to + W - 1) * a.D, v);
          }
          pd += w_.dx_stride[1];
        }
      }
    }
    float z[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) z[e] = 0.f;
    for (int t = max(t0, end); t < t1; ++t) store_any<T, VEC>(dx + t * w_.dx_stride[1], z);
  }
  if (!part) return;   // uniform
  // the workgroup's strips in order; of channels that two vectors hold the first one's threads write
  const int row = threadIdx.x / kConvCols, col = threadIdx.x % kConvCols;
  const int64_t group = xcd_remap(blockIdx.x, gridDim.x) / static_cast<uint32_t>(gm.col_blocks);
#pragma unroll 1
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int jj = 0; jj <= W; ++jj)
      if (jj == j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_red[row][col * VEC + e] = dw[jj][e];
    __syncthreads();
    for (int i = threadIdx.x; i < kConvCols * VEC; i += kConvThreads) {
      const int cc = static_cast<int>(at.col - col) + i / VEC;   // the vector, of all
      if (cc >= gm.cols) continue;
      int ch = cc * VEC;
      const bool moved = ch > a.D - VEC;
      if (moved) ch = a.D - VEC;
      ch += i % VEC;
      if (moved && ch < cc * VEC) continue;   // the vector in front has it
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < kConvStrips; ++r) t += s_red[r][i];
      part[(group * (W + 1) + j) * a.D + ch] = t;
    }
  }
}

// dweight [D][W] and dbias [D]: 16 channels of one j in a workgroup, 64 threads to a channel, each every 64th partial row
// in order.
constexpr int kConvSumCols = 16, kConvSumRows = 64;
__global__ __launch_bounds__(kConvSumCols * kConvSumRows) void conv_sum_kernel(const float* __restrict__ part, int64_t parts,
                                                                              int D, int W, float* __restrict__ dweight,
                                                                              float* __restrict__ dbias) {
  __shared__ double s_part[kConvSumRows][kConvSumCols + 1];
  const int j = blockIdx.y, col = threadIdx.x % kConvSumCols, row = threadIdx.x / kConvSumCols;
  const int d = blockIdx.x * kConvSumCols + col;
  float* out = j < W ? dweight : dbias;
  if (!out) return;   // uniform
  double t = 0.;
  if (d < D)
#pragma unroll 4
    for (int64_t p = row; p < parts; p += kConvSumRows) t += part[(p * (W + 1) + j) * D + d];
  s_part[row][col] = t;
  __syncthreads();
  if (row == 0 && d < D) {
    double s = 0.;
#pragma unroll 8
    for (int r = 0; r < kConvSumRows; ++r) s += s_part[r][col];
    if (j < W) dweight[static_cast<int64_t>(d) * W + j] = static_cast<float>(s);
    else dbias[d] = static_cast<float>(s);
  }
}

// One token of each row, bound by the launch (256 rows of 1,024 channels: 4.8 us, one row 2.9).  The first row of a slot takes the slot's later rows after it, in order.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(kConvThreads) void conv_step_kernel(dwarf_causal_conv_step_args a, int col_blocks) {
  __shared__ int s_found[2];
  const int row0 = blockIdx.x / col_blocks, col = blockIdx.x % col_blocks * kConvThreads + threadIdx.x;
  const bool in = col < (a.D + VEC - 1) / VEC;
  int d = in ? col * VEC : 0;
  // where the last vector lies at the row's end, channels that two vectors hold are the first one's to store: the states may
  // be updated in place, and what the second then reads of those channels it does not use
  int skip = 0;
  if (d > a.D - VEC) skip = d - (a.D - VEC), d = a.D - VEC;
  const int slot = a.slots ? a.slots[row0] : row0;
  T* out = static_cast<T*>(a.out) + d;
  float v[W][VEC], w[W][VEC], c[VEC];
  auto put = [&](T* p, const float* x) {
    if (!skip) store_any<T, VEC>(p, x);
    else
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (e >= skip) p[e] = from_f32<T>(x[e]);
  };
  if (slot < 0 || slot >= a.pool) {   // uniform
#pragma unroll
    for (int e = 0; e < VEC; ++e) c[e] = 0.f;
    if (in) put(out + row0 * a.out_stride, c);
    return;
  }
  const T* st = static_cast<const T*>(a.state) + slot * a.slot_stride + d;
  T* ns = static_cast<T*>(a.new_state) + slot * a.slot_stride + d;
#pragma unroll
  for (int j = 0; j < W - 1; ++j) load_any<T, VEC>(st + static_cast<int64_t>(j) * a.D, v[j]);
  load_any<T, VEC>(static_cast<const T*>(a.x) + row0 * a.x_stride + d, v[W - 1]);
  conv_weights<VEC, W>(a.weight, a.bias, d, w, c);
  SameSlot same{false, a.R};
  if (a.slots) same = same_slot<kConvThreads>(a.slots, slot, row0, a.R, s_found);
  if (same.before) return;   // uniform
  for (int row = row0; row < a.R;) {
    float p[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      p[e] = c[e];
#pragma unroll
      for (int j = 0; j < W; ++j) p[e] = fmaf(w[j][e], v[j][e], p[e]);
      if (a.silu) p[e] *= sigmoid_f32(p[e]);
    }
    if (in) put(out + row * a.out_stride, p);
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = v[j + 1][e];
    row = same.next;
    if (row < a.R) same = same_slot<kConvThreads>(a.slots, slot, row, a.R, s_found);
    if (row < a.R) load_any<T, VEC>(static_cast<const T*>(a.x) + row * a.x_stride + d, v[W - 1]);
  }
  if (in)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) put(ns + static_cast<int64_t>(j) * a.D, v[j]);
}

int conv_vec(int dtype, int D) {
  const int per = dtype == DWARF_F32 ? 4 : 8;
  return D >= per ? per : 1;
}
int conv_bwd_vec(int D) { return D >= 4 ? 4 : 1; }

ConvGeom conv_geom(const dwarf_causal_conv_fwd_args& a, int vec) {
  ConvGeom gm;
  gm.cols = (a.D + vec - 1) / vec;
  gm.col_blocks = (gm.cols + kConvCols - 1) / kConvCols;
  // Strips of 16 to 64 tokens, as long as leave seven workgroups for each four CUs: a thread reads W - 1 rows in front of its
  // strip and its weights once more for each (B15 N2048, 1,024 channels in bf16: forward strips of 16 tokens take 41 us, of 32
  // 34, of 64 36; backward of 16 58, of 64 53).
  gm.strip = 16;
  while (gm.strip < 64 && static_cast<int64_t>(a.B) * a.N / (2 * gm.strip) / kConvStrips * gm.col_blocks >= 448) gm.strip *= 2;
  gm.strips = a.N > 0 ? (a.N + gm.strip - 1) / gm.strip : 1;
  return gm;
}
int64_t conv_groups(const dwarf_causal_conv_fwd_args& a, const ConvGeom& gm) {
  return (static_cast<int64_t>(a.B) * gm.strips + kConvStrips - 1) / kConvStrips;
}

template <typename T, int VEC, int W>
void conv_fwd_typed(const dwarf_causal_conv_fwd_args& a, hipStream_t stream) {
  const ConvGeom gm = conv_geom(a, VEC);
  const int64_t threads = static_cast<int64_t>(a.B) * gm.strips * gm.cols;
  hipLaunchKernelGGL((conv_fwd_kernel<T, VEC, W>), dim3(static_cast<unsigned>((threads + kConvThreads - 1) / kConvThreads)),
                     dim3(kConvThreads), 0, stream, a, gm);
}
template <typename T, int VEC, int W>
void conv_bwd_typed(const dwarf_causal_conv_bwd_args& a, hipStream_t stream) {
  const ConvGeom gm = conv_geom(a.fwd, VEC);
  const int64_t groups = conv_groups(a.fwd, gm);
  float* part = a.dweight || a.dbias ? static_cast<float*>(a.workspace) : nullptr;
  hipLaunchKernelGGL((conv_bwd_kernel<T, VEC, W>), dim3(static_cast<unsigned>(groups * gm.col_blocks)), dim3(kConvThreads), 0,
                     stream, a, gm, part);
  if (part)
    hipLaunchKernelGGL(conv_sum_kernel, dim3((a.fwd.D + kConvSumCols - 1) / kConvSumCols, W + 1),
                       dim3(kConvSumCols * kConvSumRows), 0, stream, part, groups, a.fwd.D, W, a.dweight, a.dbias);
}
template <typename T, int VEC, int W>
void conv_step_typed(const dwarf_causal_conv_step_args& a, hipStream_t stream) {
  const int cols = (a.D + VEC - 1) / VEC, col_blocks = (cols + kConvThreads - 1) / kConvThreads;
  hipLaunchKernelGGL((conv_step_kernel<T, VEC, W>), dim3(static_cast<unsigned>(a.R) * col_blocks), dim3(kConvThreads), 0, stream,
                     a, col_blocks);
}

#define DWARF_CONV_WIDTHS(T, VEC, W, CALL)    \
  switch (W) {                                \
    case 1: CALL(T, VEC, 1); break;           \
    case 2: CALL(T, VEC, 2); break;           \
    case 3: CALL(T, VEC, 3); break;           \
    case 4: CALL(T, VEC, 4); break;           \
    case 5: CALL(T, VEC, 5); break;           \
    case 6: CALL(T, VEC, 6); break;           \
    case 7: CALL(T, VEC, 7); break;           \
    default: CALL(T, VEC, 8); break;          \
  }
#define DWARF_CONV_VECTORS(T, VEC, wide, W, CALL) \
  if (wide) { DWARF_CONV_WIDTHS(T, VEC, W, CALL) } else { DWARF_CONV_WIDTHS(T, 1, W, CALL) }
#define DWARF_CONV_TYPES(dtype, wide, W, VEC16, CALL)                                             \
  if ((dtype) == DWARF_F32) { DWARF_CONV_VECTORS(float, 4, wide, W, CALL) }                       \
  else if ((dtype) == DWARF_F16) { DWARF_CONV_VECTORS(f16, VEC16, wide, W, CALL) }                \
  else { DWARF_CONV_VECTORS(bf16, VEC16, wide, W, CALL) }

}  // namespace

int64_t causal_conv_workgroups(const dwarf_causal_conv_fwd_args& a) {
  const ConvGeom gm = conv_geom(a, conv_bwd_vec(a.D));   // the backward's: its vectors are the shorter ones
  return conv_groups(a, gm) * gm.col_blocks;
}

size_t causal_conv_bwd_workspace(const dwarf_causal_conv_bwd_args& a) {
  if (!a.dweight && !a.dbias) return 0;
  return static_cast<size_t>(conv_groups(a.fwd, conv_geom(a.fwd, conv_bwd_vec(a.fwd.D)))) * (a.fwd.W + 1) * a.fwd.D * sizeof(float);
}

hipError_t launch_causal_conv_fwd(const dwarf_causal_conv_fwd_args& a, hipStream_t stream) {
#define DWARF_CONV_CALL(T, VEC, W) conv_fwd_typed<T, VEC, W>(a, stream)
  DWARF_CONV_TYPES(a.dtype, conv_vec(a.dtype, a.D) > 1, a.W, 8, DWARF_CONV_CALL)
#undef DWARF_CONV_CALL
  return hipGetLastError();
}

hipError_t launch_causal_conv_bwd(const dwarf_causal_conv_bwd_args& a, hipStream_t stream) {
#define DWARF_CONV_CALL(T, VEC, W) conv_bwd_typed<T, VEC, W>(a, stream)
  DWARF_CONV_TYPES(a.fwd.dtype, conv_bwd_vec(a.fwd.D) > 1, a.fwd.W, 4, DWARF_CONV_CALL)
#undef DWARF_CONV_CALL
  return hipGetLastError();
}

hipError_t launch_causal_conv_step(const dwarf_causal_conv_step_args& a, hipStream_t stream) {
#define DWARF_CONV_CALL(T, VEC, W) conv_step_typed<T, VEC, W>(a, stream)
  DWARF_CONV_TYPES(a.dtype, conv_vec(a.dtype, a.D) > 1, a.W, 8, DWARF_CONV_CALL)
#undef DWARF_CONV_CALL
  return hipGetLastError();
}

}  // namespace dwarf
