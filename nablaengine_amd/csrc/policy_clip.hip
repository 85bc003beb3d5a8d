// The global norm of many gradients, and their clipping.
//
//   norm = sqrt(sum over tensors and elements of g^2),  f = min(1, limit / (norm + 1e-6)),  out = g f
//
// Memory bounds both passes: the first reads every gradient, the second reads it again and writes it, in place or into
// other tensors (an optimizer's float32 buffers). The tensors' addresses travel as kernel arguments, so a call copies
// no table to the GPU, waits for nothing and can be captured in a HIP graph; a launch takes up to TABLE tensors of any
// sizes and types. Each tensor is cut into units of UNIT elements, and a workgroup takes a contiguous run of all units.
//
// The squares are summed in float64. A square of a float32 is exact there and neither overflows nor vanishes:
// backpropagation through contacts can give gradients beyond 1e19, whose squares float32 cannot hold, and a norm of inf
// would zero the step that clipping is there to keep. The sums go to the caller's buffer, one a workgroup, and each
// workgroup of the second pass adds them all in the same fixed order (no atomics), at most 8.5 KB from the L2 cache,
// which saves a launch in between.
//
// Measured: 302 million weights in 196 tensors (bfloat16 matrices, float32 vectors), 0.6 GB read, read again and written as
// 1.2 GB of float32: 513 us, 160 for the squares and 345 for the second pass, together 4.7 TB/s, what a copy of 4 GiB
// reaches (the squares alone 3.8: the cache still writes back the last pass's outputs). More sums in flight, two and four
// accumulators a thread gained nothing. The gradients of a small network, 16 tensors of 256 x 256 and less: 4.3 and 4.7 us of two
// launches and 16 us a call from Python. Units of 8192 or 16384 elements gained nothing.
#include "../../include/nablaengine_policy.h"
#include "policy_device.h"

namespace pol {

constexpr int UNIT = 4096, BLOCK = 256;
constexpr int SUMS = 1024;  // workgroups that sum squares, but for one more a launch where a share rounds up
constexpr int CUS = 256;

struct Grad {
  const void* g;
  void* out;
  long long n;
  int unit;  // this tensor's first unit in its launch
  short type, out_type;
};
// 4 KB of kernel arguments hold the table and the rest
constexpr int TABLE = 124;
struct Grads {
  Grad t[TABLE];
  int count, units;
};
static_assert(sizeof(Grads) <= 4000, "kernel arguments");

// f(tensor, first element, element past the last) for each tensor of this workgroup's share of the units
template <typename F>
__device__ __forceinline__ void my_units(const Grads& a, F f) {
  int u = (int)((long long)blockIdx.x * a.units / gridDim.x);
  const int end = (int)((long long)(blockIdx.x + 1) * a.units / gridDim.x);
  int lo = 0, hi = a.count;  // the tensor of unit u: the last whose first unit is not past it
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.t[mid].unit <= u) lo = mid; else hi = mid;
  }
  for (; u < end; ++lo) {
    const int next = lo + 1 < a.count && a.t[lo + 1].unit < end ? a.t[lo + 1].unit : end;
    const long long at = (long long)(u - a.t[lo].unit) * UNIT, to = (long long)(next - a.t[lo].unit) * UNIT;
    f(a.t[lo], at, to < a.t[lo].n ? to : a.t[lo].n);
    u = next;
  }
}

// f(first element, elements) for steps of `most` vectors a thread, then of one, then of single elements
template <int E, int MOST, typename F>
__device__ __forceinline__ void steps(long long at, long long end, F f) {
  for (; end - at >= (long long)MOST * E * BLOCK; at += MOST * E * BLOCK)
    f(at + threadIdx.x * E, std::integral_constant<int, MOST>{});
  for (; end - at >= E * BLOCK; at += E * BLOCK) f(at + threadIdx.x * E, std::integral_constant<int, 1>{});
  for (at += threadIdx.x; at < end; at += BLOCK) f(at, std::integral_constant<int, 0>{});
}

template <typename T>
__device__ __forceinline__ double squares(const T* g, long long at, long long end) {
  constexpr int E = Vec<T>::E;
  double s = 0.0;
  steps<E, 8>(at, end, [&](long long i, auto count) {
    constexpr int N = decltype(count)::value;
    if constexpr (N == 0) {
      const double d = (double)(float)g[i];
      s = fma(d, d, s);
    } else {
      Vec<T> v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = load16(g + i + k * BLOCK * E);
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const double d = (double)(float)v[k].v[e];
          s = fma(d, d, s);
        }
    }
  });
  return s;
}

__device__ __forceinline__ double block_sum(double s, double* red) {  // in every thread
#pragma unroll
  for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < BLOCK / 64; ++i) s += red[i];
  return s;
}

__global__ __launch_bounds__(BLOCK) void k_squares(Grads a, double* __restrict__ sums) {
  __shared__ double red[BLOCK / 64];
  double s = 0.0;
  my_units(a, [&](const Grad& t, long long at, long long end) {
    if (t.type == F32) s += squares((const float*)t.g, at, end);
    else if (t.type == BF16) s += squares((const __bf16*)t.g, at, end);
    else s += squares((const _Float16*)t.g, at, end);
  });
  s = block_sum(s, red);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// the norm from the workgroups' sums, in every thread
__device__ __forceinline__ double norm_of(const double* sums, int count, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += BLOCK) s += sums[i];
  return sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(BLOCK) void k_grad_norm(const double* __restrict__ sums, int count, float* __restrict__ norm) {
  __shared__ double red[BLOCK / 64];
  const double r = norm_of(sums, count, red);
  if (threadIdx.x == 0) *norm = (float)r;
}

// in place every thread reads what it writes itself, and reads it first
template <typename T, typename O>
__device__ __forceinline__ void scale(const T* g, O* out, long long at, long long end, float f) {
  constexpr int E = Vec<T>::E, OE = Vec<O>::E;
  static_assert(E % OE == 0, "an output element has as many bytes as the gradient's, or more");
  steps<E, 4>(at, end, [&](long long i, auto count) {
    constexpr int N = decltype(count)::value;
    if constexpr (N == 0) {
      out[i] = (O)((float)g[i] * f);
    } else {
      Vec<T> v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = load16(g + i + k * BLOCK * E);
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int j = 0; j < E / OE; ++j) {
          Vec<O> o;
#pragma unroll
          for (int e = 0; e < OE; ++e) o.v[e] = (O)((float)v[k].v[j * OE + e] * f);
          store16(out + i + k * BLOCK * E + j * OE, o);
        }
    }
  });
}

__global__ __launch_bounds__(BLOCK) void k_clip(Grads a, const double* __restrict__ sums, int count, float limit,
                                                float* __restrict__ norm) {
  __shared__ double red[BLOCK / 64];
  const double r = norm_of(sums, count, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)r;
  const double q = (double)limit / (r + 1e-6);
  const float f = q >= 1.0 ? 1.0f : (float)q;  // a norm of NaN gives NaN, as the product with it would
  my_units(a, [&](const Grad& t, long long at, long long end) {
    if (f == 1.0f && t.out == t.g) return;  // x 1 in place: x
    switch (t.type * 3 + t.out_type) {
      case F32 * 3 + F32: return scale((const float*)t.g, (float*)t.out, at, end, f);
      case BF16 * 3 + F32: return scale((const __bf16*)t.g, (float*)t.out, at, end, f);
      case F16 * 3 + F32: return scale((const _Float16*)t.g, (float*)t.out, at, end, f);
      case BF16 * 3 + BF16: return scale((const __bf16*)t.g, (__bf16*)t.out, at, end, f);
      case F16 * 3 + F16: return scale((const _Float16*)t.g, (_Float16*)t.out, at, end, f);
    }
  });
}

// ---- launches -------------------------------------------------------------------------------------------------------

long long units_of(long long n) { return (n + UNIT - 1) / UNIT; }

// f(table) for tables of up to TABLE tensors and 2^30 units; a tensor longer than that is cut
template <typename F>
int by_tables(int count, const void* const* g, void* const* out, const long long* n, const int* type,
              const int* out_type, F f) {
  Grads a;
  a.count = a.units = 0;
  constexpr long long MOST = 1LL << 30;
  for (int i = 0; i < count; ++i) {
    for (long long at = 0; at < n[i];) {
      if (a.count == TABLE || a.units == MOST) {
        if (const int rc = f(a)) return rc;
        a.count = a.units = 0;
      }
      const long long left = n[i] - at, room = (MOST - a.units) * UNIT, m = left < room ? left : room;
      Grad& t = a.t[a.count++];
      t.g = (const char*)g[i] + at * bytes_of(type[i]);
      t.out = out ? (char*)out[i] + at * bytes_of(out_type[i]) : nullptr;
      t.n = m;
      t.unit = a.units;
      t.type = (short)type[i];
      t.out_type = (short)(out ? out_type[i] : 0);
      a.units += (int)units_of(m);
      at += m;
    }
  }
  return a.count ? f(a) : 0;
}

// the workgroups that sum a table's squares: their share of SUMS by units, at least one
int sums_of(int units, long long all) {
  const long long share = all <= SUMS ? units : ((long long)units * SUMS + all - 1) / all;
  return (int)(share < 1 ? 1 : share);
}
// most sums a call of `count` tensors writes: SUMS and one a table for the roundings (a table ends with its 124th
// tensor, or at 2^30 units, which no memory holds twice)
size_t clip_work_bytes(int count) { return count > 0 ? sizeof(double) * (size_t)(SUMS + count / TABLE + 64) : 0; }

int launch_clip(hipStream_t st, int count, const void* const* g, void* const* out, const long long* n, const int* type,
                const int* out_type, float limit, float* norm, void* work) {
  double* sums = (double*)work;
  long long all = 0;
  for (int i = 0; i < count; ++i) all += units_of(n[i]);
  int at = 0;
  int rc = by_tables(count, g, nullptr, n, type, nullptr, [&](const Grads& a) {
    const int blocks = sums_of(a.units, all);
    k_squares<<<blocks, BLOCK, 0, st>>>(a, sums + at);
    at += blocks;
    return (int)hipGetLastError();
  });
  if (rc) return rc;
  if (!out || all == 0) {
    k_grad_norm<<<1, BLOCK, 0, st>>>(sums, at, norm);
    return (int)hipGetLastError();
  }
  return by_tables(count, g, out, n, type, out_type, [&](const Grads& a) {
    const int most = 8 * CUS, blocks = a.units < most ? a.units : most;
    k_clip<<<blocks, BLOCK, 0, st>>>(a, sums, at, limit, norm);
    norm = nullptr;  // the first launch writes it
    return (int)hipGetLastError();
  });
}

}  // namespace pol

extern "C" {

int dk_clip(hipStream_t st, int count, const void* const* g, const long long* n, const int* type, void* const* out,
            const int* out_type, float limit, float* norm, void* work) {
  if (count < 0 || !norm || (count > 0 && (!g || !n || !type || !work || (out && !out_type))))
    return (int)hipErrorInvalidValue;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || type[i] < 0 || type[i] > 2 || (n[i] > 0 && !g[i])) return (int)hipErrorInvalidValue;
    if (out && ((n[i] > 0 && !out[i]) || (out_type[i] != type[i] && out_type[i] != pol::F32)))
      return (int)hipErrorInvalidValue;
  }
  return pol::launch_clip(st, count, g, out, n, type, out_type, limit, norm, work);
}

long long dk_clip_work_bytes(int count) { return (long long)pol::clip_work_bytes(count); }

}  // extern "C"
