// Attention of one new query a world over that world's cached history: the control loop's form.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the world's first `length` cached tokens; zeros where there are none, NaN (0 / 0) where
//       every score is -inf
//
// Memory bounds it: each cached key and value is read once, for all the query heads that share it. A workgroup takes
// one world, one key/value head and one stretch of the history. A key's 16-byte chunks lie across LPR lanes, so that a
// wave reads 64 / LPR keys at once in whole lines; the scores come from two-element dot products in 16 bits with
// float32 sums and DPP adds over the LPR lanes, and each group of LPR lanes keeps its own running maximum, sum and
// output in float32 over the keys it reads. The groups are joined at the end in registers and LDS, and stretches (long
// histories of few worlds) by a second kernel in a fixed order.
//
// Measured: 4096 worlds with up to 256 tokens, 8 heads on 2 of 64, 0.39 GB in 96 us (4.1 TB/s, of the 3.9 that a sum over one
// large tensor and the 5.2 that a copy reach); 4 worlds with up to 131072 tokens, 16 heads on 4 of 128, 0.9 GB in 176 us (5.1
// TB/s) and 5 us for the join; one world with 257 tokens 5.4 us, bound by its launch and one read after another. A turn
// reads the next one's keys and values ahead, two a lane: with four a wave less fits (104 us for 100).
#include "../../include/nablaengine_policy.h"
#include "policy_device.h"

namespace pol {

struct Step {
  const void *q, *k, *v;
  long long q_w, q_h, k_w, k_t, k_h, v_w, v_t, v_h;  // elements from world to world, token to token, head to head
  int worlds, heads, kv_heads, group, dim, capacity;
  const int* lengths;
  float scale;
  void* out;  // (worlds, heads, dim)
  int stretches, stretch, units;
  float* part;  // (stretches, worlds, heads, dim + 2): output sums, running maximum, sum
};

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

// W of a workgroup's four waves share a unit (one world, key/value head, up to GC of its query heads and stretch)
template <typename T, int LPR, int GC, int W>
__global__ __launch_bounds__(256) void k_step(Step a) {
  constexpr int RPW = 64 / LPR, BATCH = RPW * UNROLL;  // keys a wave reads at once, and in one turn
  __shared__ float wm[4][GC], wl[4][GC];
  __shared__ float wo[4][GC][LPR * 8];
  const int l = threadIdx.x % 64, w = threadIdx.x / 64, part = l % LPR, rg = l / LPR, d0 = part * 8;
  const int chunks = (a.group + GC - 1) / GC;
  int id = blockIdx.x * (4 / W) + w / W;
  const bool exists = id < a.units;
  if (W == 1 && !exists) return;
  if (!exists) id = 0;
  const int g0 = id % chunks * GC;
  id /= chunks;
  const int kv = id % a.kv_heads;
  id /= a.kv_heads;
  const int stretch = id % a.stretches, world = id / a.stretches;
  int length = exists ? a.lengths[world] : 0;
  length = length < 0 ? 0 : length > a.capacity ? a.capacity : length;
  const long long from = (long long)stretch * a.stretch, to = from + a.stretch;
  const int begin = from < length ? (int)from : length, end = to < length ? (int)to : length;
  const bool in_row = d0 < a.dim;
  int key = begin + w % W * BATCH + rg;  // this lane's next key to read
  const T* kp = (const T*)a.k + (long long)world * a.k_w + (long long)kv * a.k_h + key * a.k_t + d0;
  const T* vp = (const T*)a.v + (long long)world * a.v_w + (long long)kv * a.v_h + key * a.v_t + d0;
  Vec<T> kn[UNROLL], vn[UNROLL];  // one turn ahead
  auto read = [&] {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const bool in = in_row && key + u * RPW < end;
      kn[u] = in ? load16(kp + u * RPW * a.k_t) : Vec<T>{};
      vn[u] = in ? load16(vp + u * RPW * a.v_t) : Vec<T>{};
    }
    key += W * BATCH;
    kp += W * BATCH * a.k_t;
    vp += W * BATCH * a.v_t;
  };
  read();
  Vec<T> q[GC];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    q[g] = Vec<T>{};
    if (in_row && g0 + g < a.group)
      q[g] = load16((const T*)a.q + (long long)world * a.q_w + (long long)(kv * a.group + g0 + g) * a.q_h + d0);
  }
  const float c = a.scale * LOG2E_STEP;
  float m[GC], sum[GC], o[GC][8];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    m[g] = -INFINITY;
    sum[g] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[g][e] = 0.0f;
  }
  for (int key0 = begin + w % W * BATCH; key0 < end; key0 += W * BATCH) {
    Vec<T> k[UNROLL], v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) k[u] = kn[u], v[u] = vn[u];
    read();
    float s[GC][UNROLL];
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      float top = m[g];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) d = dot2(&q[g].v[e], &k[u].v[e], d);
        d = sum_lanes<LPR>(d) * c;
        s[g][u] = key0 + rg + u * RPW < end ? d : -INFINITY;
        top = fmaxf(top, s[g][u]);
      }
      const float base = top == -INFINITY ? 0.0f : top, f = exp2_fast(m[g] - base);
      m[g] = top;
      sum[g] *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[g][e] *= f;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        s[g][u] = exp2_fast(s[g][u] - base);
        sum[g] += s[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (float)v[u].v[e];
#pragma unroll
        for (int g = 0; g < GC; ++g) o[g][e] += s[g][u] * x;
      }
  }
  // join the row groups of the wave, then the waves
  auto put = [&](int g, int d, float top, float total, float x) {
    const long long head = (long long)world * a.heads + kv * a.group + g0 + g;
    if (a.stretches == 1) {
      ((T*)a.out)[head * a.dim + d] = (T)(length == 0 ? 0.0f : x / total);
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
template <typename T, int LPR>
__global__ __launch_bounds__(1024) void k_step_join(Step a) {
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
int step_heads_a_group(int group) { return group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8; }
int step_stretches(int worlds, int kv_heads, int group, int capacity) {
  const int gc = step_heads_a_group(group);
  const long long blocks = (long long)worlds * kv_heads * ((group + gc - 1) / gc);
  auto of = [&](int fill, int least) {
    const long long want = (fill + blocks - 1) / blocks, most = (capacity + least - 1) / least;
    return want < most ? want : most;
  };
  const long long many = of(2048, 512), few = of(256, 128), n = few >= 4 && few > many ? few : many;
  return (int)(n < 1 ? 1 : n < MOST_STRETCHES ? n : MOST_STRETCHES);
}
size_t step_work_bytes(int worlds, int heads, int kv_heads, int dim, int capacity) {
  if (worlds <= 0) return 0;
  const int n = step_stretches(worlds, kv_heads, heads / kv_heads, capacity);
  return n == 1 ? 0 : sizeof(float) * (size_t)n * worlds * heads * (dim + 2);
}

// Where there are many units, a wave takes one alone: nothing is joined over LDS, and short histories do not leave three
// waves of four idle. Histories of 256, 8 heads on 2 of 64, alone and by four waves: 1024 units 21.4 and 20.1 us, 2048 28.5
// and 34.0, 4096 53.0 and 62.6, 8192 107 and 131; of 511, 1024 units 36.8 and 30.1. Stretches are long: 2048 of 1024 keys and
// heads of 128 take 215 us alone, 180 by four.
constexpr int ALONE = 2048;
template <typename T, int LPR, int GC>
void step_units(hipStream_t st, const Step& a) {
  if (a.stretches == 1 && a.units >= ALONE) k_step<T, LPR, GC, 1><<<(a.units + 3) / 4, 256, 0, st>>>(a);
  else k_step<T, LPR, GC, 4><<<a.units, 256, 0, st>>>(a);
}
template <typename T, int LPR>
int step(hipStream_t st, Step a) {
  const int gc = step_heads_a_group(a.group);
  const long long units = (long long)a.worlds * a.kv_heads * ((a.group + gc - 1) / gc) * a.stretches;
  if (units >= 1LL << 24) return (int)hipErrorInvalidValue;
  a.units = (int)units;
  switch (gc) {
    case 1: step_units<T, LPR, 1>(st, a); break;
    case 2: step_units<T, LPR, 2>(st, a); break;
    case 4: step_units<T, LPR, 4>(st, a); break;
    default: step_units<T, LPR, 8>(st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.stretches == 1) return (int)e;
  k_step_join<T, LPR><<<(unsigned)(a.worlds * a.heads), 1024, 0, st>>>(a);
  return (int)hipGetLastError();
}

int launch_step(hipStream_t st, int type, Step a) {
  a.stretches = step_stretches(a.worlds, a.kv_heads, a.group, a.capacity);
  a.stretch = (a.capacity + a.stretches - 1) / a.stretches;
  if (type == BF16) return a.dim <= 64 ? step<__bf16, 8>(st, a) : step<__bf16, 16>(st, a);
  return a.dim <= 64 ? step<_Float16, 8>(st, a) : step<_Float16, 16>(st, a);
}

}  // namespace pol

extern "C" {

int dk_attention_step(hipStream_t st, int type, int worlds, int heads, int kv_heads, int dim, int capacity,
                      const void* q, long long q_w, long long q_h, const void* k, long long k_w, long long k_t,
                      long long k_h, const void* v, long long v_w, long long v_t, long long v_h, const int* lengths,
                      float scale, void* out, void* work) {
  if ((type != pol::BF16 && type != pol::F16) || worlds < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 ||
      dim > 128 || dim % 8 || capacity < 0 || capacity >= 1 << 30 || !(scale > 0.0f))
    return (int)hipErrorInvalidValue;
  if (worlds == 0) return 0;
  if (!q || !lengths || !out || (capacity && (!k || !v)) ||
      (!work && pol::step_work_bytes(worlds, heads, kv_heads, dim, capacity)))
    return (int)hipErrorInvalidValue;
  pol::Step a = {};
  a.q = q, a.k = k, a.v = v, a.q_w = q_w, a.q_h = q_h;
  a.k_w = k_w, a.k_t = k_t, a.k_h = k_h, a.v_w = v_w, a.v_t = v_t, a.v_h = v_h;
  a.worlds = worlds, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim;
  a.capacity = capacity, a.lengths = lengths, a.scale = scale, a.out = out, a.part = (float*)work;
  return pol::launch_step(st, type, a);
}

long long dk_attention_step_work_bytes(int worlds, int heads, int kv_heads, int dim, int capacity) {
  if (worlds < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || capacity < 0) return 0;
  return (long long)pol::step_work_bytes(worlds, heads, kv_heads, dim, capacity);
}

}  // extern "C"
