// Layer norm of rows, forward and backward.
//
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean g - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Memory bounds both: the forward reads x and writes y, the backward reads x and dy and writes dx. A row is read once
// into the registers of a group of L lanes (C vectors of 16 bytes each) and everything is computed from there: the
// mean, then the squares about it (no cancellation), then the outputs, in float32 whatever the row's type; each output
// is rounded once. The backward's groups walk over rows and keep their columns' dw and db sums in registers; at the end
// a workgroup adds its groups' sums in LDS and writes one partial row, and a second small kernel adds the partial rows
// in a fixed order (no atomics: bitwise the same on every run).
#include "../../include/nablaengine_policy.h"
#include "policy_device.h"

namespace pol {

// Rows that no register variant holds: each pass reads the row again (it stays in the L2 cache: at most a few MB).
constexpr int WIDE = 1024;  // lanes of the largest groups, and of the wide rows'

template <typename T>
__device__ __forceinline__ void row_load(const T* p, int v, int n, float* f) {  // vector v of a row of n elements
  constexpr int E = Vec<T>::E;
  const int at = v * E;
  if (at + E <= n) {
    load_floats<E>(f, p + at);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = at + e < n ? (float)p[at + e] : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void row_store(T* p, int v, int n, const float* f) {
  constexpr int E = Vec<T>::E;
  const int at = v * E;
  if (at + E <= n) {
    Vec<T> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = (T)f[e];
    store16(p + at, o);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (at + e < n) p[at + e] = (T)f[e];
  }
}
// the E parameters of vector v (`none` where there is no such parameter, and past the row's end)
template <int E, typename W>
__device__ __forceinline__ void param_load(const W* p, int v, int n, float none, float* f) {
  const int at = v * E;
  if (p && at + E <= n) {
    load_floats<E>(f, p + at);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = p && at + e < n ? (float)p[at + e] : none;
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

template <typename T, typename W, int L, int C>
__global__ __launch_bounds__(L > 256 ? L : 256) void k_norm(long long rows, int n, const T* __restrict__ x, long long xs,
                                                            const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                            T* __restrict__ y, float* __restrict__ stats) {
  constexpr int E = Vec<T>::E, BLOCK = L > 256 ? L : 256, GROUPS = BLOCK / L;
  __shared__ float red[BLOCK / 64];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  for (long long row = (long long)blockIdx.x * GROUPS + group; row < rows; row += (long long)gridDim.x * GROUPS) {
    float f[C][E];
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      row_load(x + row * xs, lane + c * L, n, f[c]);
#pragma unroll
      for (int e = 0; e < E; ++e) s += f[c][e];
    }
    const float mu = group_sum<L>(s, red) / (float)n;
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[c][e] = (lane + c * L) * E + e < n ? f[c][e] - mu : 0.0f;
        q += f[c][e] * f[c][e];
      }
    const float r = 1.0f / sqrtf(group_sum<L>(q, red) / (float)n + eps);
    if (stats && lane == 0) {
      stats[row] = mu;
      stats[rows + row] = r;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if ((lane + c * L) * E >= n) continue;
      float wf[E], bf[E];
      param_load<E>(w, lane + c * L, n, 1.0f, wf);
      param_load<E>(b, lane + c * L, n, 0.0f, bf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[c][e] = f[c][e] * r * wf[e] + bf[e];
      row_store(y + row * n, lane + c * L, n, f[c]);
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(WIDE) void k_norm_wide(long long rows, int n, const T* __restrict__ x, long long xs,
                                                    const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                    T* __restrict__ y, float* __restrict__ stats) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[WIDE / 64];
  const int nv = (n + E - 1) / E;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    float f[E], s = 0.0f, q = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      row_load(xr, v, n, f);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += f[e];
      s += t;
    }
    const float mu = group_sum<WIDE>(s, red) / (float)n;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      row_load(xr, v, n, f);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = v * E + e < n ? f[e] - mu : 0.0f;
        t += d * d;
      }
      q += t;
    }
    const float r = 1.0f / sqrtf(group_sum<WIDE>(q, red) / (float)n + eps);
    if (stats && threadIdx.x == 0) {
      stats[row] = mu;
      stats[rows + row] = r;
    }
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      float wf[E], bf[E];
      row_load(xr, v, n, f);
      param_load<E>(w, v, n, 1.0f, wf);
      param_load<E>(b, v, n, 0.0f, bf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = (f[e] - mu) * r * wf[e] + bf[e];
      row_store(y + row * n, v, n, f);
    }
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------

// part: (blocks, 2, n) float32, each workgroup's sums of dy xh and of dy over its rows
constexpr int vjp_block(int lanes) { return lanes > 512 ? lanes : 512; }

template <typename T, typename W, int L, int C>
__global__ __launch_bounds__(vjp_block(L)) void k_norm_vjp(long long rows, int n, const T* __restrict__ x, long long xs,
                                                   const T* __restrict__ dy, long long dys, const W* __restrict__ w,
                                                   const float* __restrict__ stats, T* __restrict__ dx,
                                                   float* __restrict__ part) {
  constexpr int E = Vec<T>::E, GROUPS = vjp_block(L) / L, CE = C * E;
  constexpr int SLOTS = L >= 64 ? GROUPS : 8;  // the sums left after those inside each wave
  __shared__ float red[16];
  __shared__ float add[SLOTS > 1 ? SLOTS / 2 * L * CE : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  float aw[CE], ab[CE];
#pragma unroll
  for (int i = 0; i < CE; ++i) aw[i] = ab[i] = 0.0f;
  // groups of several waves meet at barriers: the workgroup stays together, a group past the last row has none of it
  for (long long row = (long long)blockIdx.x * GROUPS + group;; row += (long long)gridDim.x * GROUPS) {
    if (L > 64 ? row - group >= rows : row >= rows) break;
    const int m = row < rows ? n : 0;
    float f[CE], g[CE];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      row_load(x + row * xs, lane + c * L, m, f + c * E);
      row_load(dy + row * dys, lane + c * L, m, g + c * E);
    }
    const float mu = m ? stats[row] : 0.0f, r = m ? stats[rows + row] : 0.0f;
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float wf[E];
      param_load<E>(w, lane + c * L, n, 1.0f, wf);
#pragma unroll
      for (int e = 0; e < E; ++e) {  // past the row's end x and dy were read as 0: g stays 0 there, xh is not used
        const int i = c * E + e;
        f[i] = (f[i] - mu) * r;
        aw[i] += g[i] * f[i];
        ab[i] += g[i];
        g[i] *= wf[e];
        s += g[i];
        q += g[i] * f[i];
      }
    }
    if (dx) {
      const float ms = group_sum<L>(s, red) / (float)n, mq = group_sum<L>(q, red) / (float)n;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if ((lane + c * L) * E >= m) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) f[c * E + e] = r * (g[c * E + e] - ms - f[c * E + e] * mq);
        row_store(dx + row * n, lane + c * L, m, f + c * E);
      }
    }
  }
  if (!part) return;
  // the lanes of a wave that hold the same columns, then the waves (or groups) by halves: a fixed order
  float* out = part + (long long)blockIdx.x * 2 * n;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* a = which ? ab : aw;
#pragma unroll
    for (int i = 0; i < CE; ++i) {
      if constexpr (L <= 8) a[i] += __shfl_xor(a[i], 8);
      if constexpr (L <= 16) a[i] = add_rows(a[i]);
      if constexpr (L <= 32) a[i] = add_halves(a[i]);
    }
    const int slot = L >= 64 ? group : threadIdx.x / 64;
    const bool holds = L >= 64 || threadIdx.x % 64 < L;
#pragma unroll
    for (int half = SLOTS / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (holds && slot >= half && slot < 2 * half)
#pragma unroll
        for (int i = 0; i < CE; ++i) add[((slot - half) * CE + i) * L + lane] = a[i];
      __syncthreads();
      if (holds && slot < half)
#pragma unroll
        for (int i = 0; i < CE; ++i) a[i] += add[(slot * CE + i) * L + lane];
    }
    if (holds && slot == 0)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int col = (lane + c * L) * E + e;
          if (col < n) out[which * n + col] = a[c * E + e];
        }
  }
}

// wide rows: a workgroup takes a contiguous share of the rows and adds its columns' sums in its partial row, which is
// its own (each column's thread is the same one throughout)
template <typename T, typename W>
__global__ __launch_bounds__(WIDE) void k_norm_vjp_wide(long long rows, int n, const T* __restrict__ x, long long xs,
                                                        const T* __restrict__ dy, long long dys,
                                                        const W* __restrict__ w, const float* __restrict__ stats,
                                                        T* __restrict__ dx, float* __restrict__ part) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[WIDE / 64];
  const int nv = (n + E - 1) / E;
  float* out = part ? part + (long long)blockIdx.x * 2 * n : nullptr;
  bool first = true;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, first = false) {
    const float mu = stats[row], r = stats[rows + row];
    float s = 0.0f, q = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      float f[E], g[E], wf[E];
      row_load(x + row * xs, v, n, f);
      row_load(dy + row * dys, v, n, g);
      param_load<E>(w, v, n, 1.0f, wf);
      float ts = 0.0f, tq = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[e] = (f[e] - mu) * r;
        const int col = v * E + e;
        if (out && col < n) {
          out[col] = (first ? 0.0f : out[col]) + g[e] * f[e];
          out[n + col] = (first ? 0.0f : out[n + col]) + g[e];
        }
        ts += g[e] * wf[e];
        tq += g[e] * wf[e] * f[e];
      }
      s += ts;
      q += tq;
    }
    if (!dx) continue;
    const float ms = group_sum<WIDE>(s, red) / (float)n, mq = group_sum<WIDE>(q, red) / (float)n;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      float f[E], g[E], wf[E];
      row_load(x + row * xs, v, n, f);
      row_load(dy + row * dys, v, n, g);
      param_load<E>(w, v, n, 1.0f, wf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = r * (g[e] * wf[e] - ms - (f[e] - mu) * r * mq);
      row_store(dx + row * n, v, n, f);
    }
  }
}

// dw, db from the partial rows: 64 columns a workgroup, 16 waves each adding every 16th row, then the waves' sums
template <typename W>
__global__ __launch_bounds__(1024) void k_norm_params(int blocks, int n, const float* __restrict__ part,
                                                      W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float add[16][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const long long col = (long long)blockIdx.x * 64 + lane;  // of the 2 n columns
  float s = 0.0f;
  if (col < 2LL * n) {
#pragma unroll 8
    for (int i = wave; i < blocks; i += 16) s += part[(long long)i * 2 * n + col];
  }
  add[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < 2LL * n) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += add[i][lane];
    W* out = col < n ? dw : db;
    if (out) out[col < n ? col : col - n] = (W)s;
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------

constexpr int CUS = 256;

// f(L, C) for a row of nv vectors: the smallest group that holds it. Returns false where none does.
template <typename F>
bool by_width(int nv, F f) {
#define POL_CASE(L, C) \
  if (nv <= L * C) { f(std::integral_constant<int, L>{}, std::integral_constant<int, C>{}); return true; }
  POL_CASE(8, 1) POL_CASE(16, 1) POL_CASE(32, 1) POL_CASE(64, 1) POL_CASE(64, 2) POL_CASE(256, 1) POL_CASE(256, 2)
  POL_CASE(1024, 1) POL_CASE(1024, 2)
#undef POL_CASE
  return false;
}
// lanes a row, and vectors a lane
void group_of(int nv, int& lanes, int& vectors) {
  lanes = WIDE, vectors = 2;
  by_width(nv, [&](auto l, auto c) { lanes = decltype(l)::value, vectors = decltype(c)::value; });
}
int vectors_of(int n, int type) { const int e = 16 / bytes_of(type); return (n + e - 1) / e; }

// The backward's workgroups: each row in flight at once at most, and what the CUs hold at once (of 8 waves: three with one
// vector a lane, two with two; more would only write more partial rows). 524288 x 256 bfloat16: 174 us with two a CU, 151
// with three, 194 with four, which take a second round.
int vjp_blocks(long long rows, int n, int type) {
  int lanes, vectors;
  group_of(vectors_of(n, type), lanes, vectors);
  const int groups = vjp_block(lanes) / lanes;
  const long long need = (rows + groups - 1) / groups, most = (vectors == 1 && lanes <= 512 ? 3 : 2) * CUS;
  return (int)(need < most ? need : most);
}

template <typename T, typename W>
int norm(hipStream_t st, long long rows, int n, int type, const void* x, long long xs, const void* w, const void* b,
         float eps, void* y, float* stats) {
  auto launch = [&](auto kernel, int block, int groups) {
    const long long need = (rows + groups - 1) / groups, most = 32LL * CUS;
    kernel<<<(unsigned)(need < most ? need : most), block, 0, st>>>(rows, n, (const T*)x, xs, (const W*)w, (const W*)b,
                                                                    eps, (T*)y, stats);
  };
  if (!by_width(vectors_of(n, type), [&](auto l, auto c) {
        constexpr int L = decltype(l)::value, C = decltype(c)::value, BLOCK = L > 256 ? L : 256;
        launch(k_norm<T, W, L, C>, BLOCK, BLOCK / L);
      }))
    launch(k_norm_wide<T, W>, WIDE, 1);
  return (int)hipGetLastError();
}

template <typename T, typename W>
int norm_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long xs, const void* dy,
             long long dys, const void* w, const float* stats, void* dx, void* dw, void* db, void* work) {
  const int blocks = vjp_blocks(rows, n, type);
  float* part = dw || db ? (float*)work : nullptr;
  if (rows > 0) {
    auto launch = [&](auto kernel, int block) {
      kernel<<<blocks, block, 0, st>>>(rows, n, (const T*)x, xs, (const T*)dy, dys, (const W*)w, stats, (T*)dx, part);
    };
    if (!by_width(vectors_of(n, type), [&](auto l, auto c) {
          launch(k_norm_vjp<T, W, decltype(l)::value, decltype(c)::value>, vjp_block(decltype(l)::value));
        }))
      launch(k_norm_vjp_wide<T, W>, WIDE);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (dw || db)  // no rows: no partial rows, and zeros
    k_norm_params<W><<<(2LL * n + 63) / 64, 1024, 0, st>>>(rows > 0 ? blocks : 0, n, part, (W*)dw, (W*)db);
  return (int)hipGetLastError();
}

size_t norm_work_bytes(long long rows, int n, int type) {
  return rows > 0 ? (size_t)vjp_blocks(rows, n, type) * 2 * n * sizeof(float) : 0;
}

#define POL_BY_TYPES(CALL)                                                                      \
  switch (type * 3 + wtype) {                                                                   \
    case F32 * 3 + F32: return CALL(float, float);                                              \
    case BF16 * 3 + F32: return CALL(__bf16, float);                                            \
    case BF16 * 3 + BF16: return CALL(__bf16, __bf16);                                          \
    case F16 * 3 + F32: return CALL(_Float16, float);                                           \
    case F16 * 3 + F16: return CALL(_Float16, _Float16);                                        \
  }                                                                                             \
  return (int)hipErrorInvalidValue;

int launch_norm(hipStream_t st, long long rows, int n, int type, const void* x, long long xs, int wtype, const void* w,
                const void* b, float eps, void* y, float* stats) {
#define CALL(T, W) norm<T, W>(st, rows, n, type, x, xs, w, b, eps, y, stats)
  POL_BY_TYPES(CALL)
#undef CALL
}
int launch_norm_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long xs, const void* dy,
                    long long dys, int wtype, const void* w, const float* stats, void* dx, void* dw, void* db,
                    void* work) {
#define CALL(T, W) norm_vjp<T, W>(st, rows, n, type, x, xs, dy, dys, w, stats, dx, dw, db, work)
  POL_BY_TYPES(CALL)
#undef CALL
}

}  // namespace pol

extern "C" {

int dk_layer_norm(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, int w_type,
                  const void* w, const void* b, float eps, void* y, float* stats) {
  if (rows < 0 || n < 1 || type < 0 || type > 2 || (w_type != pol::F32 && w_type != type))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y) return (int)hipErrorInvalidValue;
  return pol::launch_norm(st, rows, n, type, x, x_row, w_type, w, b, eps, y, stats);
}

int dk_layer_norm_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* dy,
                      long long dy_row, int w_type, const void* w, const float* stats, void* dx, void* dw, void* db,
                      void* work) {
  if (rows < 0 || n < 1 || type < 0 || type > 2 || (w_type != pol::F32 && w_type != type))
    return (int)hipErrorInvalidValue;
  if (rows > 0 && (!x || !dy || !stats || ((dw || db) && !work))) return (int)hipErrorInvalidValue;
  return pol::launch_norm_vjp(st, rows, n, type, x, x_row, dy, dy_row, w_type, w, stats, dx, dw, db, work);
}

long long dk_layer_norm_work_bytes(long long rows, int n, int type) {
  return rows > 0 && n > 0 && type >= 0 && type <= 2 ? (long long)pol::norm_work_bytes(rows, n, type) : 0;
}

}  // extern "C"
