// Element types, vectors and lane reductions of the mixer kernels (norm.hip,
// rotary.hip, linattn.hip).
#pragma once

#include "common.h"
#include "dsqg_internal.h"
#include "dwarf_mixer.h"

namespace dwarf {

typedef _Float16 f16;

__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float(static_cast<uint32_t>(x.bits) << 16); }
__device__ __forceinline__ float to_f32(f16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return bf16{f32_to_bf16_bits(x)}; }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) { return static_cast<f16>(x); }
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }

// VEC consecutive elements as one access: the whole vector is aligned to its size, and to 16 bytes where it is longer (eight fp32
// of a stream beside rows of 16 bits).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Vec {
  T e[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = to_f32(v.e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  Vec<T, VEC> v;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v.e[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Vec<T, VEC>*>(p) = v;
}

// Sum over groups of LANES adjacent lanes (a power of two up to the wave), in
// every lane of the group.  The quads and rows of 16 go through DPP.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (LANES >= 2) x += dpp_f<0xB1>(x);    // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) x += dpp_f<0x4E>(x);    // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) x += dpp_f<0x141>(x);   // row_half_mirror: the other quad of eight lanes
  if constexpr (LANES >= 16) x += dpp_f<0x140>(x);  // row_mirror: the other eight of sixteen
  if constexpr (LANES >= 32) x += __shfl_xor(x, 16);
  if constexpr (LANES >= 64) x += __shfl_xor(x, 32);
  return x;
}

}  // namespace dwarf
