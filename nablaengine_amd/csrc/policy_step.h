// What the single-token attention kernels share: 16-bit dot products, the joining of what a workgroup's lanes and waves have of
// a unit (one world, key/value head, up to GC of its query heads and stretch of its history), and of a history's stretches.
#pragma once
#include "policy_device.h"

namespace pol {

typedef __bf16 B2 __attribute__((ext_vector_type(2)));
typedef _Float16 H2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float dot2(const __bf16* a, const __bf16* b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(*(const B2*)a, *(const B2*)b, c, false);
}
__device__ __forceinline__ float dot2(const _Float16* a, const _Float16* b, float c) {
  return __builtin_amdgcn_fdot2(*(const H2*)a, *(const H2*)b, c, false);
}

constexpr float LOG2E_STEP = 1.4426950408889634f;
constexpr int UNROLL = 2;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: 0

// A unit's outputs o and running maxima and sums, which each group of LPR lanes has of the keys it read, from W waves of the
// workgroup's four; to the output, or to the unit's part where there are several stretches. none: the world has no tokens.
template <typename T, int LPR, int GC, int W, typename A>
__device__ __forceinline__ void finish_unit(const A& a, int world, int kv, int g0, int stretch, bool exists, bool none, const float* m,
                                            float* sum, float (*o)[8]) {
  __shared__ float wm[4][GC], wl[4][GC];
  __shared__ float wo[4][GC][LPR * 8];
  const int l = threadIdx.x % 64, w = threadIdx.x / 64, part = l % LPR, rg = l / LPR, d0 = part * 8;
  // join the row groups of the wave, then the waves
  auto put = [&](int g, int d, float top, float total, float x) {
    const long long head = (long long)world * a.heads + kv * a.group + g0 + g;
    if (a.stretches == 1) {
      ((T*)a.out)[head * a.dim + d] = (T)(none ? 0.0f : x / total);
    } else {
      float* to_part = a.part + ((long long)stretch * a.worlds * a.heads + head) * (a.dim + 2);
      to_part[d] = x;
      if (d == 0) {
        to_part[a.dim] = top;
        to_part[a.dim + 1] = total;
      }
    }
  };
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    float top = m[g];
#pragma unroll
    for (int d = LPR; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float f = m[g] == -INFINITY ? 0.0f : exp2_fast(m[g] - top);
    sum[g] *= f;
    if (LPR <= 8) sum[g] += __shfl_xor(sum[g], 8);
    sum[g] = add_halves(add_rows(sum[g]));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[g][e] *= f;
      if (LPR <= 8) o[g][e] += __shfl_xor(o[g][e], 8);
      o[g][e] = add_halves(add_rows(o[g][e]));
    }
    if (rg == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) wo[w][g][d0 + e] = o[g][e];
      if (part == 0) {
        wm[w][g] = top;
        wl[w][g] = sum[g];
      }
    }
  }
  if constexpr (W == 1) {  // the wave's own LDS: what it wrote it reads
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int i = l; i < GC * LPR * 8; i += 64) {
      const int g = i / (LPR * 8), d = i % (LPR * 8);
      if (g0 + g < a.group && d < a.dim) put(g, d, wm[w][g], wl[w][g], wo[w][g][d]);
    }
  } else {
    __syncthreads();
    if (!exists) return;
    for (int i = threadIdx.x; i < GC * LPR * 8; i += 256) {
      const int g = i / (LPR * 8), d = i % (LPR * 8);
      if (g0 + g >= a.group || d >= a.dim) continue;
      const float top = fmaxf(fmaxf(wm[0][g], wm[1][g]), fmaxf(wm[2][g], wm[3][g]));
      float total = 0.0f, x = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = wm[j][g] == -INFINITY ? 0.0f : exp2_fast(wm[j][g] - top);
        total += f * wl[j][g];
        x += f * wo[j][g][d];
      }
      put(g, d, top, total, x);
    }
  }
}

// One workgroup a head: the stretches' factors from their maxima, then their sums in their order, JW of them at once and
// those joined at the end. With one wave a head, one stretch after another, the join took as long as the reading.
constexpr int MOST_STRETCHES = 2048;
template <typename T, int LPR, typename A>
__global__ __launch_bounds__(1024) void k_step_join(A a) {
  constexpr int D = LPR * 8, JW = 1024 / D;
  __shared__ float factor[MOST_STRETCHES];
  __shared__ float red[16];
  __shared__ float sums[JW][D];
  const long long all = (long long)a.worlds * a.heads, head = blockIdx.x;
  const int n = a.dim + 2, wave = threadIdx.x / 64;
  const float* p = a.part + head * n;
  const long long step = all * n;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < a.stretches; s += 1024) {
    factor[s] = p[s * step + a.dim];
    top = fmaxf(top, factor[s]);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (threadIdx.x % 64 == 0) red[wave] = top;
  __syncthreads();
  for (int w = 0; w < 16; ++w) top = fmaxf(top, red[w]);
  __syncthreads();
  float total = 0.0f;
  for (int s = threadIdx.x; s < a.stretches; s += 1024) {
    factor[s] = factor[s] == -INFINITY ? 0.0f : exp2_fast(factor[s] - top);
    total += factor[s] * p[s * step + a.dim + 1];
  }
  total = sum_lanes<64>(total);
  if (threadIdx.x % 64 == 0) red[wave] = total;
  __syncthreads();
  total = 0.0f;
  for (int w = 0; w < 16; ++w) total += red[w];
  const int d = threadIdx.x % D, j = threadIdx.x / D;
  float x = 0.0f;
  if (d < a.dim) {
#pragma unroll 8
    for (int s = j; s < a.stretches; s += JW) x += factor[s] * p[s * step + d];
  }
  sums[j][d] = x;
  __syncthreads();
  if (j == 0 && d < a.dim) {
    x = 0.0f;
#pragma unroll
    for (int i = 0; i < JW; ++i) x += sums[i][d];
    ((T*)a.out)[head * a.dim + d] = (T)(a.lengths[head / a.heads] <= 0 ? 0.0f : x / total);
  }
}

// Stretches. Many worlds or long histories: enough workgroups for the 256 CUs twice over, none under 512 keys. Few: up to a
// workgroup a CU of stretches down to 128 keys, where there are four of them at least, since the join takes 4 us. 8 heads
// on 2 of 64, stretches of 512 and of 128: one world of 1000 tokens 13.6 and 9.2 us, of 8000 13.9 and 10.3, 16 worlds of 1000
// 13.7 and 9.6; but one of 257 8.1 and 8.8, 64 of 500 10.9 and 11.9, 256 of 333 14 and 28, one of 131072 22.6 and 32.7.
inline int step_heads_a_group(int group) { return group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8; }
inline int step_stretches(int worlds, int kv_heads, int group, int capacity) {
  const int gc = step_heads_a_group(group);
  const long long blocks = (long long)worlds * kv_heads * ((group + gc - 1) / gc);
  auto of = [&](int fill, int least) {
    const long long want = (fill + blocks - 1) / blocks, most = (capacity + least - 1) / least;
    return want < most ? want : most;
  };
  const long long many = of(2048, 512), few = of(256, 128), n = few >= 4 && few > many ? few : many;
  return (int)(n < 1 ? 1 : n < MOST_STRETCHES ? n : MOST_STRETCHES);
}

// Where there are many units, a wave takes one alone: nothing is joined over LDS, and short histories do not leave three
// waves of four idle. Histories of 256, 8 heads on 2 of 64, alone and by four waves: 1024 units 21.4 and 20.1 us, 2048 28.5
// and 34.0, 4096 53.0 and 62.6, 8192 107 and 131; of 511, 1024 units 36.8 and 30.1. Stretches are long: 2048 of 1024 keys and
// heads of 128 take 215 us alone, 180 by four.
constexpr int ALONE = 2048;

}  // namespace pol
