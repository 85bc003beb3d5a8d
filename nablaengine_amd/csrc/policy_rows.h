// What the kernels that take rows share: a row in registers, vectors of 16 bytes spread over a group of lanes, the sums over
// such a group, and the group that a row's length chooses.
#pragma once
#include "policy_device.h"

namespace pol {

// Rows that no register variant holds: each pass reads the row again (it stays in the L2 cache: at most a few MB).
constexpr int WIDE = 1024;  // lanes of the largest groups, and of the wide rows'

// the vectors of E that hold n elements, n up to 2^31 - 1
__host__ __device__ __forceinline__ int vectors_in(int n, int e) { return n / e + (n % e != 0); }

// A row of n elements in vectors of E. The last one ends with the row: where n is no multiple of E it holds elements of the
// one before again, which both write, with the same values, and only the first counts in sums. A tail of single elements
// cost the waves that hold it as much again as the row: 2^27 elements in rows of 99 bfloat16 211 us forward and 307
// backward, now 107 and 182.
template <int E>
__device__ __forceinline__ int first_of(int v, int n) { return v * E <= n - E || n < E ? v * E : n - E; }
// whether element e of vector v counts
template <int E>
__device__ __forceinline__ bool own(int v, int n, int e) {
  const int at = first_of<E>(v, n) + e;
  return at >= v * E && at < n;
}

// vector v of a row (of parameters), `none` where there is no row, vector or element
template <int E, typename T>
__device__ __forceinline__ void row_load(const T* p, int v, int n, float none, float* f) {
  if (p && v * E < n && n >= E) {
    load_floats<E>(f, p + first_of<E>(v, n));
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = p && n < E && v == 0 && e < n ? (float)p[e] : none;
  }
}
template <typename T>
__device__ __forceinline__ void row_store(T* p, int v, int n, const float* f) {
  constexpr int E = Vec<T>::E;
  if (v * E >= n) return;
  if (n >= E) {
    Vec<T> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = (T)f[e];
    store16(p + first_of<E>(v, n), o);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < n) p[e] = (T)f[e];
  }
}

// the sum over a group's L lanes; `red` has a float a wave. Every thread of the workgroup calls it where L > 64.
template <int L>
__device__ __forceinline__ float group_sum(float x, float* red) {
  if constexpr (L <= 64) {
    return sum_lanes<L>(x);
  } else {
    x = sum_lanes<64>(x);
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = x;
    __syncthreads();
    const int first = threadIdx.x / L * (L / 64);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) s += red[first + i];
    return s;
  }
}

constexpr int vjp_block(int lanes) { return lanes > 512 ? lanes : 512; }  // work-items of a backward's workgroup

constexpr int CUS = 256;

// f(L, C) for a row of nv vectors of E elements: the smallest group that holds it. Returns false where none does. Two vectors
// a lane save barriers where a vector is 4 float32 (rows of 2048: 203 us forward and 304 backward for 233 and 327 with one);
// with 8 elements of 16 bits they take the registers of other waves (rows of 4096 bfloat16: 180 us backward with one a lane,
// 270 with two; of 768: 109 forward for 132), but where only groups of 1024, two a CU, would hold the row with one (8192:
// 126 and 198 us for 167 and 252).
template <int E, typename F>
bool by_width(int nv, F f) {
#define POL_CASE(L, C) \
  if (nv <= L * C) { f(std::integral_constant<int, L>{}, std::integral_constant<int, C>{}); return true; }
  POL_CASE(8, 1) POL_CASE(16, 1) POL_CASE(32, 1) POL_CASE(64, 1)
  if constexpr (E == 8) {
    POL_CASE(128, 1) POL_CASE(256, 1) POL_CASE(512, 1) POL_CASE(512, 2)
  } else {
    POL_CASE(64, 2) POL_CASE(256, 1) POL_CASE(256, 2)
  }
  POL_CASE(1024, 1) POL_CASE(1024, 2)
#undef POL_CASE
  return false;
}
inline int vectors_of(int n, int type) { return vectors_in(n, 16 / bytes_of(type)); }

#define POL_BY_TYPES(CALL)                                                                      \
  switch (type * 3 + wtype) {                                                                   \
    case F32 * 3 + F32: return CALL(float, float);                                              \
    case BF16 * 3 + F32: return CALL(__bf16, float);                                            \
    case BF16 * 3 + BF16: return CALL(__bf16, __bf16);                                          \
    case F16 * 3 + F32: return CALL(_Float16, float);                                           \
    case F16 * 3 + F16: return CALL(_Float16, _Float16);                                        \
  }                                                                                             \
  return (int)hipErrorInvalidValue;

}  // namespace pol
