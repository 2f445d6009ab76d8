// What the kernels of dwarf_selective.h share (rms.hip, conv.hip, selscan.hip):
// their launches, and the sigmoid.
#pragma once

#include "dwarf_selective.h"
#include "mixer.h"

namespace dwarf {

hipError_t launch_rms_norm_fwd(const dwarf_rms_norm_fwd_args& a, hipStream_t stream);
size_t rms_norm_bwd_workspace(const dwarf_rms_norm_bwd_args& a);
hipError_t launch_rms_norm_bwd(const dwarf_rms_norm_bwd_args& a, hipStream_t stream);

int64_t causal_conv_workgroups(const dwarf_causal_conv_fwd_args& a);
hipError_t launch_causal_conv_fwd(const dwarf_causal_conv_fwd_args& a, hipStream_t stream);
size_t causal_conv_bwd_workspace(const dwarf_causal_conv_bwd_args& a);
hipError_t launch_causal_conv_bwd(const dwarf_causal_conv_bwd_args& a, hipStream_t stream);
hipError_t launch_causal_conv_step(const dwarf_causal_conv_step_args& a, hipStream_t stream);

int64_t selective_scan_workgroups(const dwarf_selective_scan_fwd_args& a);
size_t selective_scan_checkpoints(const dwarf_selective_scan_fwd_args& a);
size_t selective_scan_fwd_workspace(const dwarf_selective_scan_fwd_args& a);
hipError_t launch_selective_scan_fwd(const dwarf_selective_scan_fwd_args& a, hipStream_t stream);
size_t selective_scan_bwd_workspace(const dwarf_selective_scan_bwd_args& a);
hipError_t launch_selective_scan_bwd(const dwarf_selective_scan_bwd_args& a, hipStream_t stream);
hipError_t launch_selective_scan_step(const dwarf_selective_scan_step_args& a, hipStream_t stream);

constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + e^-x).  The exponential's argument is rounded once, so the result is |x| 2^-24 off at most where it matters:
// for large -x the exponential is the result's inverse, and x e^x is small next to what it is added to.
__device__ __forceinline__ float sigmoid_f32(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// The rows of a step that share `slot`: whether one lies in front of row `row`, and the next one behind it (`rows` if there
// is none).  Every thread of the workgroup calls it; s_found is the workgroup's own.
struct SameSlot {
  bool before;
  int next;
};
template <int THREADS>
__device__ __forceinline__ SameSlot same_slot(const int32_t* slots, int slot, int row, int rows, int* s_found) {
  if (threadIdx.x == 0) s_found[0] = 0, s_found[1] = rows;
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += THREADS)
    if (i != row && slots[i] == slot) {
      if (i < row) s_found[0] = 1;
      else atomicMin(&s_found[1], i);
    }
  __syncthreads();
  const SameSlot r{s_found[0] != 0, s_found[1]};
  __syncthreads();   // read before it is written again
  return r;
}

}  // namespace dwarf
