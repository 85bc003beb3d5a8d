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
#include "policy_step.h"

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

// W of a workgroup's four waves share a unit (one world, key/value head, up to GC of its query heads and stretch)
template <typename T, int LPR, int GC, int W>
__global__ __launch_bounds__(256) void k_step(Step a) {
  constexpr int RPW = 64 / LPR, BATCH = RPW * UNROLL;  // keys a wave reads at once, and in one turn
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
  finish_unit<T, LPR, GC, W>(a, world, kv, g0, stretch, exists, length == 0, m, sum, o);
}

size_t step_work_bytes(int worlds, int heads, int kv_heads, int dim, int capacity) {
  if (worlds <= 0) return 0;
  const int n = step_stretches(worlds, kv_heads, heads / kv_heads, capacity);
  return n == 1 ? 0 : sizeof(float) * (size_t)n * worlds * heads * (dim + 2);
}

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
