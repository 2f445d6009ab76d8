// Rotary positions of q and k in one launch.  Pair i of a row at position p is
// turned by the angle 2 pi p turns[i] / 2^64,
//   (a, b) -> magnitude (a cos - b sin, b cos + a sin),
// the gradient's pass by the negative angle; elements behind the pairs are
// copied.
//
// The angle in turns is the integer product p * turns[i] modulo 2^64: whole
// turns drop out exactly, so a position of 2^31 has an angle as exact as
// position 1 (2^-32 turns are kept; an fp32 product p f is off by 0.03 rad at
// p = 2^20).  Sine and cosine of the fraction are the hardware's (v_sin_f32
// takes turns) where the result is rounded to 16 bits: the fraction in fp32 is
// off by up to 2^-22.3 rad, less than the instruction is.  For fp32 results the
// nearest quarter turn is taken off as an integer first: fp32 holds the rest, an
// eighth of a turn at most, to 2^-25.3 rad, angles near a quarter turn are as
// exact as near 0, and sincospif takes it (40.7 us for q and k of B15 T2048 H8,
// with and without; 16-bit decode steps would take 3.25 us for 3.13).
//
// Bound by memory: each row is read and written once.  A thread owns one
// vector of pairs (16 bytes of a row; in the half layout two) of one token and
// walks over heads, so that an angle is formed once for several heads; adjacent
// threads own the row's other vectors and then the next heads.  Where the
// layout allows no 16-byte vectors a thread owns single pairs.
#include "mixer.h"

namespace dwarf {
namespace {

constexpr int kRotThreads = 256;

struct RotGeom {
  int64_t tokens;   // B * N
  int N, H, heads;  // query heads, query and key heads together
  int D, pairs;
  int units;        // work units of a row
  int turn_units;   // of which turn pairs (half layout; the interleaved units decide by pair)
  int slices;       // threads that share a token's unit, each with every slices-th head
  bool small;
  float magnitude;
};
struct RotTensor {
  const void* in;
  void* out;
  int64_t i0, i1, i2, o0, o1, o2;
};

template <typename T>
__device__ __forceinline__ void turn_sincos(uint32_t frac, float magnitude, bool inverse, float* s, float* c) {
  float sn, cs;
  if constexpr (sizeof(T) == 4) {
    const uint32_t up = frac + (1u << 29), quarter = up >> 30;   // the nearest quarter turn, and the rest in [-1/8, 1/8)
    const float rest = static_cast<float>(static_cast<int32_t>((up & 0x3fffffffu) - (1u << 29))) * 0x1p-32f;
    float y, x;
    sincospif(2.f * rest, &y, &x);
    sn = quarter & 1 ? x : y;   // a quarter more: (cos, -sin); a half more: both negated
    cs = quarter & 1 ? y : x;
    sn = quarter & 2 ? -sn : sn;
    cs = (quarter + 1) & 2 ? -cs : cs;
  } else {
    // the fraction as a signed number of turns in [-1/2, 1/2)
    const float turn = static_cast<float>(static_cast<int32_t>(frac)) * 0x1p-32f;
    sn = __builtin_amdgcn_sinf(turn);
    cs = __builtin_amdgcn_cosf(turn);
  }
  *s = (inverse ? -sn : sn) * magnitude;
  *c = cs * magnitude;
}

template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotTensor q, RotTensor k, const void* __restrict__ positions,
                                                             int64_t p0, int64_t p1, int narrow, int inverse,
                                                             const uint64_t* __restrict__ turns, RotGeom gm) {
  constexpr int kPairs = INTERLEAVED ? VEC / 2 : VEC;   // pairs of a unit
  const int64_t id = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kRotThreads + threadIdx.x;
  const uint32_t per_token = static_cast<uint32_t>(gm.units) * static_cast<uint32_t>(gm.slices);
  int64_t token, b;
  if (gm.small) {   // uniform: the whole grid counts in 32 bits
    token = static_cast<uint32_t>(id) / per_token;
    b = static_cast<uint32_t>(token) / static_cast<uint32_t>(gm.N);
  } else {
    token = id / per_token;
    b = token / gm.N;
  }
  if (token >= gm.tokens) return;
  const uint32_t rest = static_cast<uint32_t>(id - token * per_token);
  const int slice = static_cast<int>(rest / static_cast<uint32_t>(gm.units)), unit = static_cast<int>(rest) - slice * gm.units;
  const int64_t n = token - b * gm.N;
  const bool copy = !INTERLEAVED && unit >= gm.turn_units;
  const int first = INTERLEAVED ? unit * kPairs : unit * VEC;   // first pair
  float sn[kPairs], cs[kPairs];
  if (!copy) {
    const int64_t at = b * p0 + n * p1;
    const uint64_t pos = static_cast<uint64_t>(narrow ? static_cast<int64_t>(static_cast<const int32_t*>(positions)[at])
                                                      : static_cast<const int64_t*>(positions)[at]);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      sn[i] = 0.f;
      cs[i] = 1.f;
      if (first + i < gm.pairs)
        turn_sincos<T>(static_cast<uint32_t>((pos * turns[first + i]) >> 32), gm.magnitude, inverse, &sn[i], &cs[i]);
    }
  }
  for (int h = slice; h < gm.heads; h += gm.slices) {
    const bool key = h >= gm.H;
    const RotTensor& t = key ? k : q;
    const int hh = key ? h - gm.H : h;
    const T* x = static_cast<const T*>(t.in) + b * t.i0 + hh * t.i1 + n * t.i2;
    T* y = static_cast<T*>(t.out) + b * t.o0 + hh * t.o1 + n * t.o2;
    if constexpr (INTERLEAVED) {
      const int d = unit * VEC;
      float v[VEC], o[VEC];
      load_vec<T, VEC>(x + d, v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const bool turned = first + i < gm.pairs;   // a copied element takes nothing from its neighbour, NaN or not
        o[2 * i] = turned ? v[2 * i] * cs[i] - v[2 * i + 1] * sn[i] : v[2 * i];
        o[2 * i + 1] = turned ? v[2 * i + 1] * cs[i] + v[2 * i] * sn[i] : v[2 * i + 1];
      }
      store_vec<T, VEC>(y + d, o);
    } else if (copy) {
      const int d = 2 * gm.pairs + (unit - gm.turn_units) * VEC;
      *reinterpret_cast<Vec<T, VEC>*>(y + d) = *reinterpret_cast<const Vec<T, VEC>*>(x + d);
    } else {
      float a[VEC], c[VEC], oa[VEC], oc[VEC];
      load_vec<T, VEC>(x + first, a);
      load_vec<T, VEC>(x + gm.pairs + first, c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        oa[i] = a[i] * cs[i] - c[i] * sn[i];
        oc[i] = c[i] * cs[i] + a[i] * sn[i];
      }
      store_vec<T, VEC>(y + first, oa);
      store_vec<T, VEC>(y + gm.pairs + first, oc);
    }
  }
}

bool rot_vec_ok(const void* p, const int64_t* s, int esize) {
  const int per = 16 / esize;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % per == 0 && s[1] % per == 0 && s[2] % per == 0;
}

RotTensor rot_tensor(const void* in, const int64_t* is, void* out, const int64_t* os) {
  return RotTensor{in, out, is[0], is[1], is[2], os[0], os[1], os[2]};
}

template <typename T, int VEC, bool INTERLEAVED>
void rot_launch(const dwarf_rotary_args& a, hipStream_t stream) {
  RotGeom gm;
  gm.tokens = static_cast<int64_t>(a.B) * a.N;
  gm.N = a.N;
  gm.H = a.H;
  gm.heads = a.H + (a.k ? a.H_kv : 0);
  gm.D = a.D;
  gm.pairs = a.pairs;
  gm.turn_units = a.pairs / VEC;
  gm.units = INTERLEAVED ? a.D / VEC : gm.turn_units + (a.D - 2 * a.pairs) / VEC;
  gm.magnitude = a.magnitude;
  // Four heads to a thread where that leaves 1,024 threads for each CU, one where it does not.  q and k of B15 T2048 H8
  // each, bf16: one head 37.4 us, two 31.1, four 30.1 (126 MB: 4.2 TB/s).
  const int64_t each = gm.tokens * gm.units;
  const int four = (gm.heads + 3) / 4;
  gm.slices = each * four >= 256 * 1024 ? four : gm.heads;
  const int64_t threads = each * gm.slices;
  gm.small = threads < (int64_t(1) << 31);
  // a grid's dimension counts its threads in 32 bits
  const int64_t blocks = (threads + kRotThreads - 1) / kRotThreads, most = 1 << 22, wide = blocks < most ? blocks : most;
  const dim3 grid(static_cast<unsigned>(wide), static_cast<unsigned>((blocks + wide - 1) / wide));
  hipLaunchKernelGGL((rotary_kernel<T, VEC, INTERLEAVED>), grid, dim3(kRotThreads), 0, stream,
                     rot_tensor(a.q, a.q_stride, a.q_out, a.q_out_stride), rot_tensor(a.k, a.k_stride, a.k_out, a.k_out_stride),
                     a.positions, a.position_stride[0], a.position_stride[1], a.position_bytes == 4, a.inverse, a.turns, gm);
}

template <typename T>
void rot_typed(const dwarf_rotary_args& a, hipStream_t stream) {
  constexpr int kPer = 16 / sizeof(T);
  bool vec = rot_vec_ok(a.q, a.q_stride, sizeof(T)) && rot_vec_ok(a.q_out, a.q_out_stride, sizeof(T));
  if (a.k) vec = vec && rot_vec_ok(a.k, a.k_stride, sizeof(T)) && rot_vec_ok(a.k_out, a.k_out_stride, sizeof(T));
  if (a.interleaved) {
    if (vec && a.D % kPer == 0) rot_launch<T, kPer, true>(a, stream);
    else rot_launch<T, 2, true>(a, stream);
  } else {
    if (vec && a.D % kPer == 0 && a.pairs % kPer == 0) rot_launch<T, kPer, false>(a, stream);
    else rot_launch<T, 1, false>(a, stream);
  }
}

}  // namespace

hipError_t launch_rotary(const dwarf_rotary_args& a, hipStream_t stream) {
  if (a.dtype == DWARF_F32) rot_typed<float>(a, stream);
  else if (a.dtype == DWARF_F16) rot_typed<f16>(a, stream);
  else rot_typed<bf16>(a, stream);
  return hipGetLastError();
}

}  // namespace dwarf
