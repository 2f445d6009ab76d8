// RMS norm with the residual's addition, forward and backward, and with rows in
// 8 bits.
//   s = x + residual (rounded to the stream's type),  r = 1 / sqrt(mean(s^2) + eps),  y = s r w
//   ds = r (gw - s r^2 mean(gw s)) + ds_out,  gw = g w;  dw = sum g s r over the rows
// In 8 bits y is divided by its row's max|y| / 448 and rounded once to e4m3.
//
// Bound by memory, as layer norm is, and laid out as it (norm_rows.h): a row is
// read once into the registers of 8 to 512 threads, the sum is formed and
// stored on the way, so that the stream is not read a second time for the norm.
// The norm is taken of the sum as it is stored: what the backward reads again
// is then exactly what the forward normalised.  30,720 rows of 512 in bf16, with
// a residual of bf16: forward 23.6 us (126 MB, 5.3 TB/s), backward 24.2 (126 MB,
// 5.2 TB/s), the weight's sum 3.9.  40,960 rows with an fp32 residual into e4m3:
// 39.9 us (231 MB, 5.8 TB/s).  Seven rows of 1,031 in fp32: 3.3 us.
//
// Wider rows, forward and backward with the sums: 8,192 of 4,096 in bf16 44 and
// 52 us (268 MB each), with an fp32 stream 75 (403 MB) and 108 (537 MB).  The
// backward of four 16-bit vectors a thread (1,025 to 2,048 and 8,193 to 16,384
// elements) does not fit its 256 registers: it holds the next row of three
// inputs, and spills 27 to 40, with an fp32 stream 129 to 156.  16,384 rows of 2,048
// in bf16: 66 us (268 MB, 4.1 TB/s), with an fp32 stream 173 (537 MB, 3.1
// TB/s); 2,048 of 16,384 86 and 200.  Streamed rows, read twice or three times:
// 1,024 of 20,000 in bf16 58 and 111 us (164 MB each).
#include "norm_rows.h"
#include "selective.h"

namespace dwarf {
namespace {

static_assert(alignof(Vec<float, 8>) == 16, "norm_vec_ok checks a stream's rows for 16 bytes");

__device__ __forceinline__ float max2(float a, float b) { return a > b ? a : b; }

template <int LANES>
__device__ __forceinline__ float lanes_max(float x) {
  if constexpr (LANES >= 2) x = max2(x, dpp_f<0xB1>(x));
  if constexpr (LANES >= 4) x = max2(x, dpp_f<0x4E>(x));
  if constexpr (LANES >= 8) x = max2(x, dpp_f<0x141>(x));
  if constexpr (LANES >= 16) x = max2(x, dpp_f<0x140>(x));
  if constexpr (LANES >= 32) x = max2(x, __shfl_xor(x, 16));
  if constexpr (LANES >= 64) x = max2(x, __shfl_xor(x, 32));
  return x;
}
template <int TPR, int THREADS>
__device__ __forceinline__ float row_max(float x, float* s_red) {
  if constexpr (TPR <= kWave) {
    return lanes_max<TPR>(x);
  } else {
    x = lanes_max<kWave>(x);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s_red[threadIdx.x / kWave] = x;
    __syncthreads();
    float t = s_red[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWave; ++w) t = max2(t, s_red[w]);
    return t;
  }
}

// The row's scale: a row of zeros has the smallest normal number, so that no row is divided by zero.
__device__ __forceinline__ float eight_scale(float most) { return max2(most * (1.f / 448.f), 1.17549435e-38f); }

// VEC values in e4m3.  |o| <= 448 (1 + 2^-21) rounds to 448; what is not a number stays none.
template <int VEC>
__device__ __forceinline__ void store_eights(uint8_t* p, const float* o) {
  if constexpr (VEC >= 4) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(o[4 * i], o[4 * i + 1], 0, false);
      v = __builtin_amdgcn_cvt_pk_fp8_f32(o[4 * i + 2], o[4 * i + 3], v, true);
      w[i] = static_cast<uint32_t>(v);
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    *p = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(o[0], 0.f, 0, false));
  }
}

struct RmsFwd {
  const void* x; int64_t xs0, xs1;
  const void* residual; int64_t rs0, rs1;
  const float* weight;
  void* sum; int64_t ss0, ss1;
  void* y; int64_t ys0, ys1;
  float* scale;
};

template <typename T, typename R, int VEC, int TPR, int K>
__global__ __launch_bounds__(norm_fwd_threads(TPR)) void rms_fwd_kernel(RmsFwd a, NormGeom gm) {
  constexpr int kThreads = norm_fwd_threads(TPR), kRows = kThreads / TPR;
  __shared__ float s_red[kThreads / kWave];
  const int sub = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;   // a multiple of the groups
  const NormWalk walk(kRows, threadIdx.x / TPR, gm.groups);
  if (walk.first >= gm.rows) return;   // a row's threads together
  const float fd = static_cast<float>(gm.D);
  const T* px = walk.at(static_cast<const T*>(a.x), a.xs0, a.xs1);
  const R* pr = walk.at(static_cast<const R*>(a.residual), a.rs0, a.rs1);
  R* ps = walk.at(static_cast<R*>(a.sum), a.ss0, a.ss1);
  T* py = walk.at(static_cast<T*>(a.y), a.ys0, a.ys1);
  uint8_t* pq = walk.at(static_cast<uint8_t*>(a.y), a.ys0, a.ys1);
  const bool added = a.residual != nullptr, eights = a.scale != nullptr;   // uniform
  NormRaw<T, VEC, TPR, K> nx;
  NormRaw<R, VEC, TPR, K> nr;
  nx.load(px, sub, gm.D);
  if (added) nr.load(pr, sub, gm.D);
  float w[K * VEC];
  norm_table<VEC, TPR, K>(a.weight, walk.group, sub, gm.D, 1.f, w);
  for (int64_t r = walk.first; r < gm.rows; r += step) {
    float v[K * VEC];
    nx.widen(sub, gm.D, v);
    if (added) {
      float t[K * VEC];
      nr.widen(sub, gm.D, t);
#pragma unroll
      for (int i = 0; i < K * VEC; ++i) v[i] = to_f32(from_f32<R>(v[i] + t[i]));
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int d = (k * TPR + sub) * VEC;
        if (d < gm.D) store_vec<R, VEC>(ps + d, v + k * VEC);
      }
      ps += walk.by * a.ss0;
    }
    // the next row's loads are under way while this one is summed (behind the last row: this one again)
    if (r + step < gm.rows) {
      px += walk.by * a.xs0;
      pr += walk.by * a.rs0;
    }
    nx.load(px, sub, gm.D);
    if (added) nr.load(pr, sub, gm.D);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) q = fmaf(v[i], v[i], q);
    const float rs = 1.f / sqrtf(row_sum<TPR, kThreads>(q, s_red) / fd + gm.eps);
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) v[i] = v[i] * rs * w[i];
    if (eights) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < K * VEC; ++i) m = max2(fabsf(v[i]), m);   // elements behind the row's end are 0
      const float sc = eight_scale(row_max<TPR, kThreads>(m, s_red)), inv = 1.f / sc;
#pragma unroll
      for (int i = 0; i < K * VEC; ++i) v[i] *= inv;
      if (sub == 0) a.scale[r] = sc;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int d = (k * TPR + sub) * VEC;
        if (d < gm.D) store_eights<VEC>(pq + d, v + k * VEC);
      }
      pq += walk.by * a.ys0;
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int d = (k * TPR + sub) * VEC;
        if (d < gm.D) store_vec<T, VEC>(py + d, v + k * VEC);
      }
      py += walk.by * a.ys0;
    }
  }
}

struct RmsBwd {
  const void* s; int64_t xs0, xs1;
  const void* dy; int64_t gs0, gs1;
  const void* dsum; int64_t us0, us1;
  const float* weight;
  void* dx; int64_t ds0, ds1;
  void* dr; int64_t rs0, rs1;
};

template <typename T, typename R, int VEC, int TPR, int K>
__global__ __launch_bounds__(kNormBwdThreads) void rms_bwd_kernel(RmsBwd a, float* __restrict__ part_w, NormGeom gm) {
  constexpr int kRows = kNormBwdThreads / TPR;
  extern __shared__ __align__(16) float n_smem[];   // [kRows][D] where partials are kept
  __shared__ float s_red[kNormBwdThreads / kWave];
  const int sub = threadIdx.x % TPR, row = threadIdx.x / TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;   // a multiple of the groups
  const NormWalk walk(kRows, row, gm.groups);
  const float fd = static_cast<float>(gm.D);
  const bool any = walk.first < gm.rows, more = a.dsum != nullptr;   // threads without a row read the first and add nothing
  const R* px = any ? walk.at(static_cast<const R*>(a.s), a.xs0, a.xs1) : static_cast<const R*>(a.s);
  const T* pg = any ? walk.at(static_cast<const T*>(a.dy), a.gs0, a.gs1) : static_cast<const T*>(a.dy);
  const R* pu = any ? walk.at(static_cast<const R*>(a.dsum), a.us0, a.us1) : static_cast<const R*>(a.dsum);
  T* dx = walk.at(static_cast<T*>(a.dx), a.ds0, a.ds1);
  R* dr = walk.at(static_cast<R*>(a.dr), a.rs0, a.rs1);
  NormRaw<R, VEC, TPR, K> nx, nu;
  NormRaw<T, VEC, TPR, K> ng;
  nx.load(px, sub, gm.D);
  ng.load(pg, sub, gm.D);
  if (more) nu.load(pu, sub, gm.D);
  float w[K * VEC], dw[K * VEC];
  norm_table<VEC, TPR, K>(a.weight, walk.group, sub, gm.D, 1.f, w);
#pragma unroll
  for (int i = 0; i < K * VEC; ++i) dw[i] = 0.f;
  for (int64_t r = walk.first; r < gm.rows; r += step, dx += walk.by * a.ds0, dr += walk.by * a.rs0) {
    float v[K * VEC], g[K * VEC], u[K * VEC];
    nx.widen(sub, gm.D, v);
    ng.widen(sub, gm.D, g);
    if (more) nu.widen(sub, gm.D, u);
    else
#pragma unroll
      for (int i = 0; i < K * VEC; ++i) u[i] = 0.f;
    if (r + step < gm.rows) {   // behind the last row: this one again
      px += walk.by * a.xs0;
      pg += walk.by * a.gs0;
      pu += walk.by * a.us0;
    }
    nx.load(px, sub, gm.D);
    ng.load(pg, sub, gm.D);
    if (more) nu.load(pu, sub, gm.D);
    float q = 0.f, sgv = 0.f;
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) {
      q = fmaf(v[i], v[i], q);
      sgv = fmaf(g[i] * w[i], v[i], sgv);
    }
    q = row_sum<TPR, kNormBwdThreads>(q, s_red);
    sgv = row_sum<TPR, kNormBwdThreads>(sgv, s_red);
    const float rs = 1.f / sqrtf(q / fd + gm.eps);
    const float m2 = sgv / fd * rs * rs;
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) {
      u[i] = fmaf(rs, fmaf(-v[i], m2, g[i] * w[i]), u[i]);
      dw[i] = fmaf(g[i], v[i] * rs, dw[i]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = (k * TPR + sub) * VEC;
      if (d >= gm.D) continue;
      if (a.dx) store_vec<T, VEC>(dx + d, u + k * VEC);
      if (a.dr) store_vec<R, VEC>(dr + d, u + k * VEC);
    }
  }
  if (!part_w) return;   // uniform
  // the workgroup's rows of one group, in row order
  const int parts = norm_parts(gm.groups, kRows);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = (k * TPR + sub) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (d < gm.D) n_smem[row * gm.D + d + e] = dw[k * VEC + e];
  }
  __syncthreads();
  float* out = part_w + static_cast<int64_t>(blockIdx.x) * parts * gm.D;
  for (int i = threadIdx.x; i < parts * gm.D; i += kNormBwdThreads) {
    float t = 0.f;
    for (int rr = i / gm.D; rr < kRows; rr += gm.groups) t += n_smem[rr * gm.D + i % gm.D];
    out[i] = t;
  }
}

// Rows longer than the registers hold: a workgroup per row.  The sum is stored in the first pass and read again from the
// caches, each value by the thread that stored it.
template <typename T, typename R, int VEC>
__global__ __launch_bounds__(kNormThreads) void rms_fwd_stream(RmsFwd a, NormGeom gm) {
  __shared__ float s_red[kNormThreads / kWave];
  const float fd = static_cast<float>(gm.D);
  const bool added = a.residual != nullptr;   // uniform
  for (int64_t r = blockIdx.x; r < gm.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + norm_at(r, gm.groups, a.xs0, a.xs1);
    const R* rr = static_cast<const R*>(a.residual) + norm_at(r, gm.groups, a.rs0, a.rs1);
    R* sr = static_cast<R*>(a.sum) + norm_at(r, gm.groups, a.ss0, a.ss1);
    const int64_t at = norm_at(r, gm.groups, a.ys0, a.ys1);
    const float* wg = a.weight + (r % gm.groups) * gm.D;
    float q = 0.f, m = 0.f, v[VEC], t[VEC];
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
      if (added) {
        load_vec<R, VEC>(rr + d, t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = to_f32(from_f32<R>(v[e] + t[e]));
        store_vec<R, VEC>(sr + d, v);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) q = fmaf(v[e], v[e], q);
    }
    const float rs = 1.f / sqrtf(row_sum<kNormThreads, kNormThreads>(q, s_red) / fd + gm.eps);
    auto normalised = [&](int64_t d) {
      if (added) load_vec<R, VEC>(sr + d, v);
      else load_vec<T, VEC>(xr + d, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = v[e] * rs * (a.weight ? wg[d + e] : 1.f);
    };
    float inv = 1.f;
    if (a.scale) {
      for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
        normalised(d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max2(fabsf(v[e]), m);
      }
      const float sc = eight_scale(row_max<kNormThreads, kNormThreads>(m, s_red));
      inv = 1.f / sc;
      if (threadIdx.x == 0) a.scale[r] = sc;
    }
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      normalised(d);
      if (a.scale) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= inv;
        store_eights<VEC>(static_cast<uint8_t*>(a.y) + at + d, v);
      } else {
        store_vec<T, VEC>(static_cast<T*>(a.y) + at + d, v);
      }
    }
  }
}

// The gradients of such rows, and each row's r for the columns' pass behind it.
template <typename T, typename R, int VEC>
__global__ __launch_bounds__(kNormThreads) void rms_bwd_stream(RmsBwd a, float* __restrict__ stats, NormGeom gm) {
  __shared__ float s_red[kNormThreads / kWave];
  const float fd = static_cast<float>(gm.D);
  for (int64_t r = blockIdx.x; r < gm.rows; r += gridDim.x) {
    const R* xr = static_cast<const R*>(a.s) + norm_at(r, gm.groups, a.xs0, a.xs1);
    const T* gr = static_cast<const T*>(a.dy) + norm_at(r, gm.groups, a.gs0, a.gs1);
    const R* ur = static_cast<const R*>(a.dsum) + norm_at(r, gm.groups, a.us0, a.us1);
    T* dx = static_cast<T*>(a.dx) + norm_at(r, gm.groups, a.ds0, a.ds1);
    R* dr = static_cast<R*>(a.dr) + norm_at(r, gm.groups, a.rs0, a.rs1);
    const float* wg = a.weight + (r % gm.groups) * gm.D;
    float q = 0.f, sgv = 0.f, v[VEC], g[VEC], u[VEC];
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<R, VEC>(xr + d, v);
      load_vec<T, VEC>(gr + d, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        q = fmaf(v[e], v[e], q);
        sgv = fmaf(g[e] * (a.weight ? wg[d + e] : 1.f), v[e], sgv);
      }
    }
    q = row_sum<kNormThreads, kNormThreads>(q, s_red);
    sgv = row_sum<kNormThreads, kNormThreads>(sgv, s_red);
    const float rs = 1.f / sqrtf(q / fd + gm.eps);
    const float m2 = sgv / fd * rs * rs;
    if (stats && threadIdx.x == 0) stats[r] = rs;
    if (!a.dx && !a.dr) continue;   // uniform
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<R, VEC>(xr + d, v);
      load_vec<T, VEC>(gr + d, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[e] = 0.f;
      if (a.dsum) load_vec<R, VEC>(ur + d, u);
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[e] = fmaf(rs, fmaf(-v[e], m2, g[e] * (a.weight ? wg[d + e] : 1.f)), u[e]);
      if (a.dx) store_vec<T, VEC>(dx + d, u);
      if (a.dr) store_vec<R, VEC>(dr + d, u);
    }
  }
}

// dw partials of such rows: workgroup (c, p, group) adds column block c over the group's rows p, p + P, ...
template <typename T, typename R>
__global__ __launch_bounds__(kNormThreads) void rms_bwd_columns(RmsBwd a, const float* __restrict__ stats,
                                                                float* __restrict__ part_w, NormGeom gm) {
  const int d = blockIdx.x * kNormThreads + threadIdx.x;
  if (d >= gm.D) return;
  const int group = blockIdx.z;
  float w = 0.f;
  for (int64_t r = static_cast<int64_t>(blockIdx.y) * gm.groups + group; r < gm.rows;
       r += static_cast<int64_t>(gridDim.y) * gm.groups) {
    const float v = to_f32(static_cast<const R*>(a.s)[norm_at(r, gm.groups, a.xs0, a.xs1) + d]);
    const float g = to_f32(static_cast<const T*>(a.dy)[norm_at(r, gm.groups, a.gs0, a.gs1) + d]);
    w = fmaf(g, v * stats[r], w);
  }
  part_w[(static_cast<int64_t>(blockIdx.y) * gm.groups + group) * gm.D + d] = w;
}

int elem_bytes(int dtype) { return dtype == DWARF_F32 ? 4 : 2; }

NormPlan rms_fwd_plan(const dwarf_rms_norm_fwd_args& a) {
  const int es = elem_bytes(a.dtype);
  bool vec = norm_vec_ok(a.x, a.x_stride, es);
  if (a.scale) {   // as many bytes as x's vectors have elements
    const int per = 16 / es;
    vec = vec && reinterpret_cast<uintptr_t>(a.y) % per == 0 && a.y_stride[0] % per == 0 && a.y_stride[1] % per == 0;
  } else {
    vec = vec && norm_vec_ok(a.y, a.y_stride, es);
  }
  if (a.residual) {
    const int rs = elem_bytes(a.residual_dtype);
    vec = vec && norm_vec_ok(a.residual, a.residual_stride, rs) && norm_vec_ok(a.sum, a.sum_stride, rs);
  }
  return norm_plan(a.rows, a.groups, a.D, 16 / es, vec, kNormThreads);
}

NormPlan rms_bwd_plan(const dwarf_rms_norm_bwd_args& a) {
  const int es = elem_bytes(a.dtype), rs = elem_bytes(a.stream_dtype);
  bool vec = norm_vec_ok(a.stream, a.stream_stride, rs) && norm_vec_ok(a.dy, a.dy_stride, es);
  if (a.dsum) vec = vec && norm_vec_ok(a.dsum, a.dsum_stride, rs);
  if (a.dx) vec = vec && norm_vec_ok(a.dx, a.dx_stride, es);
  if (a.dresidual) vec = vec && norm_vec_ok(a.dresidual, a.dresidual_stride, rs);
  NormPlan p = norm_plan(a.rows, a.groups, a.D, 16 / es, vec, kNormBwdThreads);
  const int64_t rows = a.rows * a.groups;
  const int most = p.k >= 2 ? kNormBwdBlocks / 2 : kNormBwdBlocks;   // as layer norm's backward
  p.blocks = static_cast<int>(norm_blocks(rows, a.groups, p.block_rows, most));
  if (!p.tpr) {
    p.blocks = static_cast<int>(rows < 2048 ? rows : 2048);
    p.columns_y = static_cast<int>(a.rows < 64 ? a.rows : 64);
  }
  return p;
}

template <typename T, typename R, int VEC>
void rms_fwd_typed(const RmsFwd& f, const NormPlan& p, const NormGeom& gm, hipStream_t stream) {
  constexpr int kThr = kNormThreads;
  if (!p.tpr) {
    const int64_t blocks = gm.rows < 2048 ? gm.rows : 2048;
    hipLaunchKernelGGL((rms_fwd_stream<T, R, VEC>), dim3(static_cast<unsigned>(blocks)), dim3(kThr), 0, stream, f, gm);
    return;
  }
#define DWARF_RMS_LAUNCH(TPR, K) \
  hipLaunchKernelGGL((rms_fwd_kernel<T, R, VEC, TPR, K>), dim3(p.blocks), dim3(norm_fwd_threads(TPR)), 0, stream, f, gm)
  if (p.tpr == kNormBwdThreads) { DWARF_RMS_LAUNCH(kNormBwdThreads, 4); return; }
  DWARF_NORM_SHAPES(DWARF_RMS_LAUNCH)
#undef DWARF_RMS_LAUNCH
}

template <typename T, typename R, int VEC>
void rms_bwd_typed(const RmsBwd& b, const dwarf_rms_norm_bwd_args& a, const NormPlan& p, const NormGeom& gm,
                   hipStream_t stream) {
  constexpr int kThr = kNormBwdThreads;
  float* ws = static_cast<float*>(a.workspace);
  const int sum_blocks = (a.D + kNormSumCols - 1) / kNormSumCols * a.groups;
  if (!p.tpr) {
    float* stats = a.dweight ? ws : nullptr;
    hipLaunchKernelGGL((rms_bwd_stream<T, R, VEC>), dim3(p.blocks), dim3(kNormThreads), 0, stream, b, stats, gm);
    if (!a.dweight) return;
    float* part = ws + gm.rows;
    hipLaunchKernelGGL((rms_bwd_columns<T, R>), dim3((a.D + kNormThreads - 1) / kNormThreads, p.columns_y, a.groups),
                       dim3(kNormThreads), 0, stream, b, stats, part, gm);
    hipLaunchKernelGGL(norm_sum_kernel, dim3(sum_blocks), dim3(kNormSumCols * kNormSumRows), 0, stream, part,
                       static_cast<const float*>(nullptr), p.columns_y, a.groups, a.groups, a.D, a.dweight,
                       static_cast<float*>(nullptr));
    return;
  }
  float* part = a.dweight ? ws : nullptr;
  const size_t lds = a.dweight ? static_cast<size_t>(p.block_rows) * a.D * sizeof(float) : 0;
#define DWARF_RMS_LAUNCH(TPR, K) \
  hipLaunchKernelGGL((rms_bwd_kernel<T, R, VEC, TPR, K>), dim3(p.blocks), dim3(kThr), lds, stream, b, part, gm)
  DWARF_NORM_SHAPES(DWARF_RMS_LAUNCH)
#undef DWARF_RMS_LAUNCH
  if (a.dweight)
    hipLaunchKernelGGL(norm_sum_kernel, dim3(sum_blocks), dim3(kNormSumCols * kNormSumRows), 0, stream, part,
                       static_cast<const float*>(nullptr), p.blocks, p.block_rows, a.groups, a.D, a.dweight,
                       static_cast<float*>(nullptr));
}

// The element types (row, stream) and whether vectors are taken.
#define DWARF_RMS_TYPES(dtype, stream_dtype, CALL)                                            \
  if ((dtype) == DWARF_F32) p.vec ? CALL(float, float, 4) : CALL(float, float, 1);            \
  else if ((dtype) == DWARF_F16 && (stream_dtype) == DWARF_F32) p.vec ? CALL(f16, float, 8) : CALL(f16, float, 1); \
  else if ((dtype) == DWARF_F16) p.vec ? CALL(f16, f16, 8) : CALL(f16, f16, 1);               \
  else if ((stream_dtype) == DWARF_F32) p.vec ? CALL(bf16, float, 8) : CALL(bf16, float, 1);  \
  else p.vec ? CALL(bf16, bf16, 8) : CALL(bf16, bf16, 1)

}  // namespace

size_t rms_norm_bwd_workspace(const dwarf_rms_norm_bwd_args& a) {
  if (!a.dweight) return 0;
  const NormPlan p = rms_bwd_plan(a);
  if (!p.tpr)
    return (static_cast<size_t>(a.rows) * a.groups + static_cast<size_t>(p.columns_y) * a.groups * a.D) * sizeof(float);
  return static_cast<size_t>(p.blocks) * norm_parts(a.groups, p.block_rows) * a.D * sizeof(float);
}

hipError_t launch_rms_norm_fwd(const dwarf_rms_norm_fwd_args& a, hipStream_t stream) {
  const NormPlan p = rms_fwd_plan(a);
  const NormGeom gm{a.rows * a.groups, a.groups, a.D, a.eps};
  const RmsFwd f{a.x, a.x_stride[0], a.x_stride[1], a.residual, a.residual_stride[0], a.residual_stride[1], a.weight,
                 a.sum, a.sum_stride[0], a.sum_stride[1], a.y, a.y_stride[0], a.y_stride[1], a.scale};
  const int sd = a.residual ? a.residual_dtype : a.dtype;
#define DWARF_RMS_CALL(T, R, VEC) rms_fwd_typed<T, R, VEC>(f, p, gm, stream)
  DWARF_RMS_TYPES(a.dtype, sd, DWARF_RMS_CALL);
#undef DWARF_RMS_CALL
  return hipGetLastError();
}

hipError_t launch_rms_norm_bwd(const dwarf_rms_norm_bwd_args& a, hipStream_t stream) {
  const NormPlan p = rms_bwd_plan(a);
  const NormGeom gm{a.rows * a.groups, a.groups, a.D, a.eps};
  const RmsBwd b{a.stream, a.stream_stride[0], a.stream_stride[1], a.dy, a.dy_stride[0], a.dy_stride[1],
                 a.dsum, a.dsum_stride[0], a.dsum_stride[1], a.weight, a.dx, a.dx_stride[0], a.dx_stride[1],
                 a.dresidual, a.dresidual_stride[0], a.dresidual_stride[1]};
#define DWARF_RMS_CALL(T, R, VEC) rms_bwd_typed<T, R, VEC>(b, a, p, gm, stream)
  DWARF_RMS_TYPES(a.dtype, a.stream_dtype, DWARF_RMS_CALL);
#undef DWARF_RMS_CALL
  return hipGetLastError();
}

}  // namespace dwarf
