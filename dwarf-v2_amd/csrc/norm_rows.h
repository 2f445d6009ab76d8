// What the norms of rows share (norm.hip, rms.hip): how threads share and walk
// rows of [rows][groups][D], the rows' sums, and the weight gradients' partial
// rows and their sum.
#pragma once

#include "mixer.h"

namespace dwarf {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormBwdThreads = 512;
constexpr int kNormBlocks = 2048;   // 768: 14.4 us for B15 T2048 D512 in bf16, 1,536: 13.1, 2,048: 12.6 (63 MB: 5.0 TB/s)
constexpr int kNormBwdBlocks = 512;   // with the sums' launch behind it, 256: 27.6 us there, 512: 25.9, 768: 27.5, 1,024: 29.0

struct NormGeom {
  int64_t rows;   // rows * groups of the call
  int groups, D;
  float eps;
};

// Row r of the [rows][groups] grid.
__device__ __forceinline__ int64_t norm_at(int64_t r, int groups, int64_t s0, int64_t s1) {
  if (groups == 1) return r * s0;
  const int64_t o = r / groups;
  return o * s0 + (r - o * groups) * s1;
}

// g w, rounded the same in the row's mean and in what the mean is taken from: a row of one value then has a gradient of
// exactly 0, where a fused product would leave the rounding's residue times r.
__device__ __forceinline__ float norm_weighted(float g, float w) {
#pragma clang fp contract(off)
  return g * w;
}

// Sum over the TPR threads of a row.  TPR above the wave: the whole workgroup of THREADS is one row's.
template <int TPR, int THREADS>
__device__ __forceinline__ float row_sum(float x, float* s_red) {
  if constexpr (TPR <= kWave) {
    return lanes_sum<TPR>(x);
  } else {
    static_assert(TPR == THREADS, "a row is shared by one workgroup");
    x = lanes_sum<kWave>(x);
    __syncthreads();   // the previous sum has been read
    if (threadIdx.x % kWave == 0) s_red[threadIdx.x / kWave] = x;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) t += s_red[w];
    return t;
  }
}

// A row's vectors of one thread, as they are in memory; vectors behind the row's end are the row's first one again (no
// branch stands around a load) and are zeroed when they are widened.
template <typename T, int VEC, int TPR, int K>
struct NormRaw {
  Vec<T, VEC> v[K];
  __device__ __forceinline__ void load(const T* row, int sub, int D) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = (k * TPR + sub) * VEC;
      v[k] = *reinterpret_cast<const Vec<T, VEC>*>(row + (d < D ? d : 0));
    }
  }
  __device__ __forceinline__ void widen(int sub, int D, float* x) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[k * VEC + e] = (k * TPR + sub) * VEC < D ? to_f32(v[k].e[e]) : 0.f;
  }
};

// The rows of a thread in the register kernels: row `first` and every row a grid's stride behind it, all of one group, so
// that its place moves by one fixed step and no row is divided by the groups.
struct NormWalk {
  uint32_t first, group;   // both kernels' grids hold fewer than 2^32 rows
  int64_t outer, by;       // first / groups, and the stride over the outer rows
  __device__ __forceinline__ NormWalk(int block_rows, int row, int groups) {
    first = blockIdx.x * static_cast<uint32_t>(block_rows) + static_cast<uint32_t>(row);
    const uint32_t o = first / static_cast<uint32_t>(groups);
    group = first - o * static_cast<uint32_t>(groups);
    outer = o;
    by = gridDim.x * static_cast<uint32_t>(block_rows) / static_cast<uint32_t>(groups);   // a whole number
  }
  template <typename T>
  __device__ __forceinline__ T* at(T* p, int64_t s0, int64_t s1) const { return p + outer * s0 + group * s1; }
};

// A thread's part of a group's weights (or biases), `none` where there are none; aligned to their elements only.
template <int VEC, int TPR, int K>
__device__ __forceinline__ void norm_table(const float* t, uint32_t group, int sub, int D, float none, float* w) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = (k * TPR + sub) * VEC;
    if (t) __builtin_memcpy(w + k * VEC, t + static_cast<int64_t>(group) * D + (d < D ? d : 0), VEC * sizeof(float));
    else
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[k * VEC + e] = none;
  }
}

constexpr int norm_fwd_threads(int tpr) { return tpr > kNormThreads ? tpr : kNormThreads; }

// Partial rows a workgroup of the backward writes: one per group among its kRows rows.
__host__ __device__ inline int norm_parts(int groups, int block_rows) { return groups < block_rows ? groups : block_rows; }

// dw (blockIdx.y 0) and db from the partials: 16 columns of one group per workgroup, 64 threads to a column, which add
// every 64th partial row in order and are then added in order themselves.  Partial row i of workgroup b belongs to group
// (b block_rows + i) % groups: one row of each workgroup where its rows hold every group, of some where they do not.
constexpr int kNormSumCols = 16, kNormSumRows = 64;
__global__ __launch_bounds__(kNormSumCols * kNormSumRows) void norm_sum_kernel(const float* __restrict__ part_w,
                                                                              const float* __restrict__ part_b, int blocks,
                                                                              int block_rows, int groups, int D,
                                                                              float* __restrict__ dweight,
                                                                              float* __restrict__ dbias) {
  __shared__ float s_part[kNormSumRows][kNormSumCols + 1];
  const float* part = blockIdx.y ? part_b : part_w;
  float* out = blockIdx.y ? dbias : dweight;
  if (!out) return;   // uniform
  const int col_blocks = (D + kNormSumCols - 1) / kNormSumCols;
  const int group = blockIdx.x / col_blocks, col = threadIdx.x % kNormSumCols, row = threadIdx.x / kNormSumCols;
  const int d = blockIdx.x % col_blocks * kNormSumCols + col;
  const int parts = norm_parts(groups, block_rows);
  float t = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int b = row; b < blocks; b += kNormSumRows) {
      const uint32_t behind = static_cast<uint32_t>(b) * static_cast<uint32_t>(block_rows) % static_cast<uint32_t>(groups);
      const int i = group >= static_cast<int>(behind) ? group - static_cast<int>(behind) : group + groups - static_cast<int>(behind);
      const float v = part[(static_cast<int64_t>(b) * parts + (i < parts ? i : 0)) * D + d];
      t += i < parts ? v : 0.f;
    }
  }
  s_part[row][col] = t;
  __syncthreads();
  if (row < 4) {   // 16 rows each, then the four
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < kNormSumRows / 4; ++r) s += s_part[row * (kNormSumRows / 4) + r][col];
    s += __shfl_down(s, 2 * kNormSumCols);
    s += __shfl_down(s, kNormSumCols);
    if (row == 0 && d < D) out[static_cast<int64_t>(group) * D + d] = s;
  }
}

// How a row is shared: vectors of 16 bytes where the layout allows them, single elements otherwise.
struct NormPlan {
  bool vec;
  int tpr, k;        // tpr 0: the streaming kernels
  int block_rows;    // backward
  int blocks;        // backward
  int columns_y;     // streaming backward: row parts of the columns' pass
};

inline int gcd(int a, int b) {
  while (b) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

inline bool norm_vec_ok(const void* p, const int64_t* s, int esize) {
  const int per = 16 / esize;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % per == 0 && s[1] % per == 0;
}

inline int64_t norm_blocks(int64_t rows, int groups, int block_rows, int most) {
  int64_t want = (rows + block_rows - 1) / block_rows;
  if (want > most) want = most;
  const int unit = groups / gcd(groups, block_rows);   // the grid's stride is a multiple of the groups
  return (want + unit - 1) / unit * unit;
}

// A row goes to as many threads as take one vector each, up to the wave, then to a wave with up to four each, then to the
// workgroup: its sums need barriers, which a row of a wave does not (33.5 MB in bf16, forward and backward with the sums:
// 16,384 rows of 1,024 by waves 12.2 and 25.6 us, by workgroups 18.6 and 70; 8,192 of 2,048 13.2 and 28.5 against 12.9 and
// 42).  Longer rows are read three times: 1,024 of 16,384 19.6 us forward in the registers of 512 threads, 66 streamed.
inline NormPlan norm_plan(int64_t rows, int groups, int D, int per, bool vec, int threads) {
  NormPlan p;
  p.vec = vec && D % per == 0;
  const int units = p.vec ? D / per : D;
  p.k = 1;
  if (units <= 8) p.tpr = 8;
  else if (units <= 16) p.tpr = 16;
  else if (units <= 32) p.tpr = 32;
  else if (units <= 64) p.tpr = 64;
  else if (units <= 128) p.tpr = 64, p.k = 2;
  else if (units <= 256) p.tpr = 64, p.k = 4;
  else if (units <= 4 * threads) p.tpr = threads, p.k = units <= threads ? 1 : units <= 2 * threads ? 2 : 4;
  else if (units <= 4 * kNormBwdThreads) p.tpr = kNormBwdThreads, p.k = 4;   // forward: a larger workgroup
  else p.tpr = 0;
  p.block_rows = p.tpr && p.tpr < threads ? threads / p.tpr : 1;
  p.blocks = static_cast<int>(norm_blocks(rows * groups, groups, p.block_rows, kNormBlocks));
  p.columns_y = 0;
  return p;
}

#define DWARF_NORM_SHAPES(LAUNCH)                                                                        \
  switch (p.tpr) {                                                                                       \
    case 8: LAUNCH(8, 1); break;                                                                         \
    case 16: LAUNCH(16, 1); break;                                                                       \
    case 32: LAUNCH(32, 1); break;                                                                       \
    case 64: if (p.k == 1) { LAUNCH(64, 1); } else if (p.k == 2) { LAUNCH(64, 2); } else { LAUNCH(64, 4); } break; \
    default: if (p.k == 1) { LAUNCH(kThr, 1); } else if (p.k == 2) { LAUNCH(kThr, 2); } else { LAUNCH(kThr, 4); } \
  }

}  // namespace
}  // namespace dwarf
