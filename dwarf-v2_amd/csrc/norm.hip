// Layer norm, forward and backward, with the weight's and bias's gradients.
//   y = (x - mu) r w + b,  r = 1 / sqrt(var + eps),  h = (x - mu) r
//   dx = r (gw - mean(gw) - h mean(gw h)),  gw = g w;  dw = sum g h, db = sum g over the rows
// Rows are [rows][groups][D], group g with its own weights: groups 1 is a norm
// over the model's width, groups H and D 64 a norm of each head's row.
//
// Both directions are bound by memory: each row is read once into registers
// (mean, then the variance of the centred values, then the result), and the
// backward forms the statistics again from the row it reads anyway instead of
// reading saved ones.  TPR adjacent threads share a row, K vectors each; rows
// too long for the registers (16,384 elements of 16 bits) take the streaming
// kernels, one workgroup per row, whose second and third pass read the caches.
//
// The grid's stride over the rows is a multiple of the groups, so a thread
// keeps one group: its weights and its part of dw and db stay in registers
// over all its rows, and its place moves by one step (with a division by the
// groups for each row and weights read one by one, B15 T2048 D512 took 19.4 us
// forward and 23.5 backward where it takes 12.6 and 21.9).  A workgroup adds its threads' parts in LDS and writes
// one partial row per group that it holds; a second launch adds those in a
// fixed order.
#include "norm_rows.h"

namespace dwarf {
namespace {

template <typename T, int VEC, int TPR, int K>
__global__ __launch_bounds__(norm_fwd_threads(TPR)) void norm_fwd_kernel(
    const T* __restrict__ x, int64_t xs0, int64_t xs1, const float* __restrict__ weight, const float* __restrict__ bias,
    T* __restrict__ y, int64_t ys0, int64_t ys1, NormGeom gm) {
  constexpr int kThreads = norm_fwd_threads(TPR), kRows = kThreads / TPR;
  __shared__ float s_red[kThreads / kWave];
  const int sub = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;   // a multiple of the groups
  const NormWalk walk(kRows, threadIdx.x / TPR, gm.groups);
  if (walk.first >= gm.rows) return;   // a row's threads together
  const float fd = static_cast<float>(gm.D);   // sums are divided, so that a row of one value has it as its mean
  const T* px = walk.at(x, xs0, xs1);
  T* yr = walk.at(y, ys0, ys1);
  NormRaw<T, VEC, TPR, K> next;
  next.load(px, sub, gm.D);
  float w[K * VEC], b[K * VEC];
  norm_table<VEC, TPR, K>(weight, walk.group, sub, gm.D, 1.f, w);
  norm_table<VEC, TPR, K>(bias, walk.group, sub, gm.D, 0.f, b);
  for (int64_t r = walk.first; r < gm.rows; r += step, yr += walk.by * ys0) {
    float v[K * VEC];
    next.widen(sub, gm.D, v);
    // the next row's loads are under way while this one is summed (behind the last row: this one again)
    if (r + step < gm.rows) px += walk.by * xs0;
    next.load(px, sub, gm.D);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) s += v[i];
    const float mu = row_sum<TPR, kThreads>(s, s_red) / fd;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = (k * TPR + sub) * VEC < gm.D;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[k * VEC + e] = in ? v[k * VEC + e] - mu : 0.f;
        q = fmaf(v[k * VEC + e], v[k * VEC + e], q);
      }
    }
    const float rs = 1.f / sqrtf(row_sum<TPR, kThreads>(q, s_red) / fd + gm.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = (k * TPR + sub) * VEC;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = fmaf(v[k * VEC + e] * rs, w[k * VEC + e], b[k * VEC + e]);
      if (d < gm.D) store_vec<T, VEC>(yr + d, o);
    }
  }
}

template <typename T, int VEC, int TPR, int K>
__global__ __launch_bounds__(kNormBwdThreads) void norm_bwd_kernel(
    const T* __restrict__ x, int64_t xs0, int64_t xs1, const T* __restrict__ dy, int64_t gs0, int64_t gs1,
    const float* __restrict__ weight, T* __restrict__ dx, int64_t ds0, int64_t ds1, float* __restrict__ part_w,
    float* __restrict__ part_b, NormGeom gm) {
  constexpr int kRows = kNormBwdThreads / TPR;
  extern __shared__ __align__(16) float n_smem[];   // [kRows][D] where partials are kept
  __shared__ float s_red[kNormBwdThreads / kWave];
  const int sub = threadIdx.x % TPR, row = threadIdx.x / TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;   // a multiple of the groups
  const NormWalk walk(kRows, row, gm.groups);
  const float fd = static_cast<float>(gm.D);   // sums are divided, so that a row of one value has it as its mean
  const bool any = walk.first < gm.rows;   // threads without a row read the first one and add nothing
  const T* px = any ? walk.at(x, xs0, xs1) : x;
  const T* pg = any ? walk.at(dy, gs0, gs1) : dy;
  T* dr = walk.at(dx, ds0, ds1);
  NormRaw<T, VEC, TPR, K> nx, ng;
  nx.load(px, sub, gm.D);
  ng.load(pg, sub, gm.D);
  float w[K * VEC], dw[K * VEC], db[K * VEC];
  norm_table<VEC, TPR, K>(weight, walk.group, sub, gm.D, 1.f, w);
#pragma unroll
  for (int i = 0; i < K * VEC; ++i) dw[i] = db[i] = 0.f;
  for (int64_t r = walk.first; r < gm.rows; r += step, dr += walk.by * ds0) {
    float v[K * VEC], g[K * VEC];
    float s = 0.f;
    nx.widen(sub, gm.D, v);
    ng.widen(sub, gm.D, g);
    if (r + step < gm.rows) {   // behind the last row: this one again
      px += walk.by * xs0;
      pg += walk.by * gs0;
    }
    nx.load(px, sub, gm.D);
    ng.load(pg, sub, gm.D);
#pragma unroll
    for (int i = 0; i < K * VEC; ++i) s += v[i];
    const float mu = row_sum<TPR, kNormBwdThreads>(s, s_red) / fd;
    float q = 0.f, sg = 0.f, sgv = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = (k * TPR + sub) * VEC < gm.D;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = k * VEC + e;
        v[i] = in ? v[i] - mu : 0.f;
        q = fmaf(v[i], v[i], q);
        const float gw = norm_weighted(g[i], w[i]);
        sg += gw;
        sgv = fmaf(gw, v[i], sgv);
      }
    }
    q = row_sum<TPR, kNormBwdThreads>(q, s_red);
    sg = row_sum<TPR, kNormBwdThreads>(sg, s_red);
    sgv = row_sum<TPR, kNormBwdThreads>(sgv, s_red);
    const float rs = 1.f / sqrtf(q / fd + gm.eps);
    const float m1 = sg / fd, m2 = sgv / fd * rs * rs;   // mean(gw), mean(gw h) r
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = (k * TPR + sub) * VEC;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = k * VEC + e;
        o[e] = rs * (norm_weighted(g[i], w[i]) - m1 - v[i] * m2);
        dw[i] = fmaf(g[i], v[i] * rs, dw[i]);
        db[i] += g[i];
      }
      if (dx && d < gm.D) store_vec<T, VEC>(dr + d, o);
    }
  }
  // the workgroup's rows of one group, in row order
  const int parts = norm_parts(gm.groups, kRows);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    float* part = which ? part_b : part_w;   // uniform
    if (!part) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = (k * TPR + sub) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (d < gm.D) n_smem[row * gm.D + d + e] = which ? db[k * VEC + e] : dw[k * VEC + e];
    }
    __syncthreads();
    float* out = part + static_cast<int64_t>(blockIdx.x) * parts * gm.D;
    for (int i = threadIdx.x; i < parts * gm.D; i += kNormBwdThreads) {
      float t = 0.f;
      for (int rr = i / gm.D; rr < kRows; rr += gm.groups) t += n_smem[rr * gm.D + i % gm.D];
      out[i] = t;
    }
  }
}

// Rows longer than the registers hold: a workgroup per row, which reads it once for each pass.
template <typename T, int VEC>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_stream(const T* __restrict__ x, int64_t xs0, int64_t xs1,
                                                                const float* __restrict__ weight,
                                                                const float* __restrict__ bias, T* __restrict__ y,
                                                                int64_t ys0, int64_t ys1, NormGeom gm) {
  __shared__ float s_red[kNormThreads / kWave];
  const float fd = static_cast<float>(gm.D);   // sums are divided, so that a row of one value has it as its mean
  for (int64_t r = blockIdx.x; r < gm.rows; r += gridDim.x) {
    const T* xr = x + norm_at(r, gm.groups, xs0, xs1);
    T* yr = y + norm_at(r, gm.groups, ys0, ys1);
    const float* wg = weight + (r % gm.groups) * gm.D;
    const float* bg = bias + (r % gm.groups) * gm.D;
    float s = 0.f, q = 0.f, v[VEC];
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[e];
    }
    const float mu = row_sum<kNormThreads, kNormThreads>(s, s_red) / fd;
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) q = fmaf(v[e] - mu, v[e] - mu, q);
    }
    const float rs = 1.f / sqrtf(row_sum<kNormThreads, kNormThreads>(q, s_red) / fd + gm.eps);
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fmaf((v[e] - mu) * rs, weight ? wg[d + e] : 1.f, bias ? bg[d + e] : 0.f);
      store_vec<T, VEC>(yr + d, v);
    }
  }
}

// dx of such rows, and the row's mean and r for the columns' pass behind it.
template <typename T, int VEC>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_stream(const T* __restrict__ x, int64_t xs0, int64_t xs1,
                                                                const T* __restrict__ dy, int64_t gs0, int64_t gs1,
                                                                const float* __restrict__ weight, T* __restrict__ dx,
                                                                int64_t ds0, int64_t ds1, float* __restrict__ stats,
                                                                NormGeom gm) {
  __shared__ float s_red[kNormThreads / kWave];
  const float fd = static_cast<float>(gm.D);   // sums are divided, so that a row of one value has it as its mean
  for (int64_t r = blockIdx.x; r < gm.rows; r += gridDim.x) {
    const T* xr = x + norm_at(r, gm.groups, xs0, xs1);
    const T* gr = dy + norm_at(r, gm.groups, gs0, gs1);
    const float* wg = weight + (r % gm.groups) * gm.D;
    float s = 0.f, q = 0.f, sg = 0.f, sgv = 0.f, v[VEC], g[VEC];
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[e];
    }
    const float mu = row_sum<kNormThreads, kNormThreads>(s, s_red) / fd;
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
      load_vec<T, VEC>(gr + d, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float c = v[e] - mu, gw = norm_weighted(g[e], weight ? wg[d + e] : 1.f);
        q = fmaf(c, c, q);
        sg += gw;
        sgv = fmaf(gw, c, sgv);
      }
    }
    q = row_sum<kNormThreads, kNormThreads>(q, s_red);
    sg = row_sum<kNormThreads, kNormThreads>(sg, s_red);
    sgv = row_sum<kNormThreads, kNormThreads>(sgv, s_red);
    const float rs = 1.f / sqrtf(q / fd + gm.eps);
    const float m1 = sg / fd, m2 = sgv / fd * rs * rs;
    if (stats && threadIdx.x == 0) {
      stats[2 * r] = mu;
      stats[2 * r + 1] = rs;
    }
    if (!dx) continue;
    T* dr = dx + norm_at(r, gm.groups, ds0, ds1);
    for (int64_t d = threadIdx.x * VEC; d < gm.D; d += kNormThreads * VEC) {
      load_vec<T, VEC>(xr + d, v);
      load_vec<T, VEC>(gr + d, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = rs * (norm_weighted(g[e], weight ? wg[d + e] : 1.f) - m1 - (v[e] - mu) * m2);
      store_vec<T, VEC>(dr + d, v);
    }
  }
}

// dw and db partials of such rows: workgroup (c, p, group) adds column block c over the group's rows p, p + P, ...
template <typename T>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_columns(const T* __restrict__ x, int64_t xs0, int64_t xs1,
                                                                 const T* __restrict__ dy, int64_t gs0, int64_t gs1,
                                                                 const float* __restrict__ stats,
                                                                 float* __restrict__ part_w, float* __restrict__ part_b,
                                                                 NormGeom gm) {
  const int d = blockIdx.x * kNormThreads + threadIdx.x;
  if (d >= gm.D) return;
  const int group = blockIdx.z;
  float w = 0.f, b = 0.f;
  for (int64_t r = static_cast<int64_t>(blockIdx.y) * gm.groups + group; r < gm.rows;
       r += static_cast<int64_t>(gridDim.y) * gm.groups) {
    const float v = to_f32(x[norm_at(r, gm.groups, xs0, xs1) + d]), g = to_f32(dy[norm_at(r, gm.groups, gs0, gs1) + d]);
    w = fmaf(g, (v - stats[2 * r]) * stats[2 * r + 1], w);
    b += g;
  }
  const int64_t at = (static_cast<int64_t>(blockIdx.y) * gm.groups + group) * gm.D + d;
  if (part_w) part_w[at] = w;
  if (part_b) part_b[at] = b;
}

// The backward's grid: up to two workgroups per CU, which leave at most 512 partial rows per group to the sum.
NormPlan norm_bwd_plan(const dwarf_layer_norm_bwd_args& a) {
  const int es = a.fwd.dtype == DWARF_F32 ? 4 : 2;
  bool vec = norm_vec_ok(a.fwd.x, a.fwd.x_stride, es) && norm_vec_ok(a.dy, a.dy_stride, es);
  if (a.dx) vec = vec && norm_vec_ok(a.dx, a.dx_stride, es);
  NormPlan p = norm_plan(a.fwd.rows, a.fwd.groups, a.fwd.D, 16 / es, vec, kNormBwdThreads);
  const int64_t rows = a.fwd.rows * a.fwd.groups;
  // Threads with several vectors of a row have enough loads in flight with one workgroup on their CU, and each workgroup
  // leaves a partial row.  33.5 MB in bf16, with 256 and with 512 workgroups: rows of 1,024 25.6 and 30.7 us, of 2,048 28.5
  // and 38.4, of 8,192 39.6 and 52.8; with one vector to a thread, rows of 4,096 37.0 and 35.2.
  const int most = p.k >= 2 ? kNormBwdBlocks / 2 : kNormBwdBlocks;
  p.blocks = static_cast<int>(norm_blocks(rows, a.fwd.groups, p.block_rows, most));
  if (!p.tpr) {
    p.blocks = static_cast<int>(rows < 2048 ? rows : 2048);
    p.columns_y = static_cast<int>(a.fwd.rows < 64 ? a.fwd.rows : 64);
  }
  return p;
}

template <typename T, int VEC>
void norm_fwd_typed(const dwarf_layer_norm_fwd_args& f, const NormPlan& p, const NormGeom& gm, hipStream_t stream) {
  constexpr int kThr = kNormThreads;
  const T* x = static_cast<const T*>(f.x);
  T* y = static_cast<T*>(f.y);
  if (!p.tpr) {
    const int64_t blocks = gm.rows < 2048 ? gm.rows : 2048;
    hipLaunchKernelGGL((norm_fwd_stream<T, VEC>), dim3(static_cast<unsigned>(blocks)), dim3(kThr), 0, stream, x,
                       f.x_stride[0], f.x_stride[1], f.weight, f.bias, y, f.y_stride[0], f.y_stride[1], gm);
    return;
  }
#define DWARF_NORM_LAUNCH(TPR, K)                                                                               \
  hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, TPR, K>), dim3(p.blocks), dim3(norm_fwd_threads(TPR)), 0, stream, \
                     x, f.x_stride[0], f.x_stride[1], f.weight, f.bias, y, f.y_stride[0], f.y_stride[1], gm)
  if (p.tpr == kNormBwdThreads) { DWARF_NORM_LAUNCH(kNormBwdThreads, 4); return; }
  DWARF_NORM_SHAPES(DWARF_NORM_LAUNCH)
#undef DWARF_NORM_LAUNCH
}

template <typename T, int VEC>
void norm_bwd_typed(const dwarf_layer_norm_bwd_args& a, const NormPlan& p, const NormGeom& gm, hipStream_t stream) {
  constexpr int kThr = kNormBwdThreads;
  const dwarf_layer_norm_fwd_args& f = a.fwd;
  const T* x = static_cast<const T*>(f.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  float* ws = static_cast<float*>(a.workspace);
  const bool sums = a.dweight || a.dbias;
  if (!p.tpr) {
    float* stats = sums ? ws : nullptr;
    float* pw = a.dweight ? ws + 2 * gm.rows : nullptr;
    float* pb = a.dbias ? ws + 2 * gm.rows + (a.dweight ? static_cast<int64_t>(p.columns_y) * f.groups * f.D : 0) : nullptr;
    hipLaunchKernelGGL((norm_bwd_stream<T, VEC>), dim3(p.blocks), dim3(kNormThreads), 0, stream, x, f.x_stride[0],
                       f.x_stride[1], dy, a.dy_stride[0], a.dy_stride[1], f.weight, dx, a.dx_stride[0], a.dx_stride[1],
                       stats, gm);
    if (!sums) return;
    hipLaunchKernelGGL((norm_bwd_columns<T>), dim3((f.D + kNormThreads - 1) / kNormThreads, p.columns_y, f.groups),
                       dim3(kNormThreads), 0, stream, x, f.x_stride[0], f.x_stride[1], dy, a.dy_stride[0],
                       a.dy_stride[1], stats, pw, pb, gm);
    hipLaunchKernelGGL(norm_sum_kernel, dim3((f.D + kNormSumCols - 1) / kNormSumCols * f.groups, 2), dim3(kNormSumCols * kNormSumRows), 0,
                       stream, pw, pb, p.columns_y, f.groups, f.groups, f.D, a.dweight, a.dbias);
    return;
  }
  const int64_t span = static_cast<int64_t>(p.blocks) * norm_parts(f.groups, p.block_rows) * f.D;
  float* pw = a.dweight ? ws : nullptr;
  float* pb = a.dbias ? ws + (a.dweight ? span : 0) : nullptr;
  const size_t lds = sums ? static_cast<size_t>(p.block_rows) * f.D * sizeof(float) : 0;
#define DWARF_NORM_LAUNCH(TPR, K)                                                                                  \
  hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, TPR, K>), dim3(p.blocks), dim3(kThr), lds, stream, x, f.x_stride[0], \
                     f.x_stride[1], dy, a.dy_stride[0], a.dy_stride[1], f.weight, dx, a.dx_stride[0],              \
                     a.dx_stride[1], pw, pb, gm)
  DWARF_NORM_SHAPES(DWARF_NORM_LAUNCH)
#undef DWARF_NORM_LAUNCH
  if (sums)
    hipLaunchKernelGGL(norm_sum_kernel, dim3((f.D + kNormSumCols - 1) / kNormSumCols * f.groups, 2), dim3(kNormSumCols * kNormSumRows), 0,
                       stream, pw, pb, p.blocks, p.block_rows, f.groups, f.D, a.dweight, a.dbias);
}

NormGeom norm_geom(const dwarf_layer_norm_fwd_args& f) {
  return NormGeom{f.rows * f.groups, f.groups, f.D, f.eps};
}

}  // namespace

size_t layer_norm_bwd_workspace(const dwarf_layer_norm_bwd_args& a) {
  if (!a.dweight && !a.dbias) return 0;
  const NormPlan p = norm_bwd_plan(a);
  const size_t sums = (a.dweight ? 1 : 0) + (a.dbias ? 1 : 0);
  if (!p.tpr)
    return (2 * static_cast<size_t>(a.fwd.rows) * a.fwd.groups + sums * p.columns_y * a.fwd.groups * a.fwd.D) * sizeof(float);
  return sums * p.blocks * norm_parts(a.fwd.groups, p.block_rows) * a.fwd.D * sizeof(float);
}

hipError_t launch_layer_norm_fwd(const dwarf_layer_norm_fwd_args& f, hipStream_t stream) {
  const int es = f.dtype == DWARF_F32 ? 4 : 2;
  const bool vec = norm_vec_ok(f.x, f.x_stride, es) && norm_vec_ok(f.y, f.y_stride, es);
  const NormPlan p = norm_plan(f.rows, f.groups, f.D, 16 / es, vec, kNormThreads);
  const NormGeom gm = norm_geom(f);
  if (f.dtype == DWARF_F32) p.vec ? norm_fwd_typed<float, 4>(f, p, gm, stream) : norm_fwd_typed<float, 1>(f, p, gm, stream);
  else if (f.dtype == DWARF_F16) p.vec ? norm_fwd_typed<f16, 8>(f, p, gm, stream) : norm_fwd_typed<f16, 1>(f, p, gm, stream);
  else p.vec ? norm_fwd_typed<bf16, 8>(f, p, gm, stream) : norm_fwd_typed<bf16, 1>(f, p, gm, stream);
  return hipGetLastError();
}

hipError_t launch_layer_norm_bwd(const dwarf_layer_norm_bwd_args& a, hipStream_t stream) {
  const NormPlan p = norm_bwd_plan(a);
  const NormGeom gm = norm_geom(a.fwd);
  if (a.fwd.dtype == DWARF_F32) p.vec ? norm_bwd_typed<float, 4>(a, p, gm, stream) : norm_bwd_typed<float, 1>(a, p, gm, stream);
  else if (a.fwd.dtype == DWARF_F16) p.vec ? norm_bwd_typed<f16, 8>(a, p, gm, stream) : norm_bwd_typed<f16, 1>(a, p, gm, stream);
  else p.vec ? norm_bwd_typed<bf16, 8>(a, p, gm, stream) : norm_bwd_typed<bf16, 1>(a, p, gm, stream);
  return hipGetLastError();
}

}  // namespace dwarf
