// What the policy operators' kernels share: element types, 16-byte vectors at any address, and reductions over the
// lanes of a wave by DPP and lane swaps.
#pragma once
#include <hip/hip_runtime.h>

namespace pol {

enum Type { F32 = 0, BF16 = 1, F16 = 2 };
constexpr int bytes_of(int type) { return type == F32 ? 4 : 2; }

template <typename T>
struct Vec {  // 16 bytes of T
  static constexpr int E = 16 / sizeof(T);
  T v[E];
};

// 16 bytes at an address of the element type's alignment only: the global memory path takes them in one instruction
// (unaligned access is on for this target), so rows of any length and views at any offset are read as aligned ones are
template <typename T>
__device__ __forceinline__ Vec<T> load16(const T* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const Vec<T>& v) {
  __builtin_memcpy(p, &v, 16);
}

// N floats from N elements of W at p
template <int N, typename W>
__device__ __forceinline__ void load_floats(float* f, const W* p) {
  constexpr int E = Vec<W>::E;
#pragma unroll
  for (int i = 0; i < N; i += E) {
    const Vec<W> v = load16(p + i);
#pragma unroll
    for (int e = 0; e < E; ++e) f[i + e] = (float)v.v[e];
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// x of the lane in the neighbouring row of 16 (rows 0/1, 2/3), and of the other half of the wave, added to x
__device__ __forceinline__ float add_rows(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_halves(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_halves(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// the sum of x over each aligned group of L lanes (a power of two, at most 64), in every lane of the group
template <int L>
__device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (L >= 2) x += dpp<0xB1>(x);   // lanes 1 0 3 2 of each four
  if constexpr (L >= 4) x += dpp<0x4E>(x);   // lanes 2 3 0 1 of each four
  if constexpr (L >= 8) x += dpp<0x141>(x);  // each eight mirrored
  if constexpr (L >= 16) x += dpp<0x140>(x); // each sixteen mirrored
  if constexpr (L >= 32) x = add_rows(x);
  if constexpr (L >= 64) x = add_halves(x);
  return x;
}

constexpr float LOG2E_GATE = 1.4426950408889634f, LOG2E_REST = 1.925963e-8f;  // log2(e) to 24 bits, and what is left of it
// a = 1 / (1 + exp(-f)) and 1 - a of a gate in T. In float32 the smaller one is within 7 2^-24 of itself, down to 2^-126, below which
// they are 0; in 16 bits the exponent's own rounding stays, 1.3 |f| 2^-24 more, far below what the last place of such an f tells.
template <typename T>
__device__ __forceinline__ void gates(float f, float& keep, float& take) {
  float e;
  if constexpr (sizeof(T) == 4) {  // with what the exponent's rounding and the constant's take off, which is felt by far gates
    f = f > 200.0f ? 200.0f : f;
    const float t = -f * LOG2E_GATE, rest = fmaf(-f, LOG2E_REST, fmaf(-f, LOG2E_GATE, -t));
    e = __builtin_amdgcn_exp2f(t);
    e = t > 126.0f ? INFINITY : fmaf(e, rest * 0.6931472f, e);
  } else {
    e = __builtin_amdgcn_exp2f(-f * LOG2E_GATE);
  }
  keep = __builtin_amdgcn_rcpf(1.0f + e);
  take = f >= 0.0f ? e * keep : 1.0f - keep;
}

// the sum of x over this lane and those before it in the wave
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned shifted(unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ unsigned scan_wave(unsigned x) {
  x += shifted<0x111, 0xf>(x);  // within each sixteen: from 1, 2, 4 and 8 lanes before
  x += shifted<0x112, 0xf>(x);
  x += shifted<0x114, 0xf>(x);
  x += shifted<0x118, 0xf>(x);
  x += shifted<0x142, 0xa>(x);  // the first and third sixteen's last lane to the next sixteen
  x += shifted<0x143, 0xc>(x);  // the first half's last lane to the second half
  return x;
}

}  // namespace pol
