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
//
// Measured, 2^27 elements, of the 5.2 TB/s of a large copy: forward 5.0 to 5.6 TB/s in float32 at widths 32 to 8192, odd
// ones (99, 331, 1331) among them, and in bfloat16 at 64 to 4096 (4.1 to 5.0 at odd ones); backward 4.8 to 5.4 TB/s in
// float32, in bfloat16 4.5 to 5.2 at powers of two and 3.5 to 4.4 at odd widths, where a vector's conversions bound it.
// Up to a few thousand rows a call is bound by its launch (2 us a kernel).
#include "../../include/nablaengine_policy.h"
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

template <typename T, typename W, int L, int C>
__global__ __launch_bounds__(L > 256 ? L : 256) void k_norm(long long rows, int n, const T* __restrict__ x, long long xs,
                                                            const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                            T* __restrict__ y, float* __restrict__ stats) {
  constexpr int E = Vec<T>::E, BLOCK = L > 256 ? L : 256, GROUPS = BLOCK / L;
  __shared__ float red[BLOCK / 64];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  // A lane's parameters, the same for all its rows, stay in registers and are read beside its first row, not after the
  // sums: rows of 4096 float32 193 us for 317. For 16 and more too few waves would fit.
  constexpr bool KEEP = C * E <= 8;
  float wf[KEEP ? C : 1][E], bf[KEEP ? C : 1][E];
  auto params = [&](int c, int to) {
    row_load<E>(w, lane + c * L, n, 1.0f, wf[to]);
    row_load<E>(b, lane + c * L, n, 0.0f, bf[to]);
  };
  if (KEEP)
#pragma unroll
    for (int c = 0; c < C; ++c) params(c, c);
  // groups of several waves meet at barriers: the workgroup stays together, a group past the last row has none of it
  for (long long row = (long long)blockIdx.x * GROUPS + group;; row += (long long)gridDim.x * GROUPS) {
    if (L > 64 ? row - group >= rows : row >= rows) break;
    const int m = row < rows ? n : 0;
    float f[C][E];
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      row_load<E>(x + row * xs, lane + c * L, m, 0.0f, f[c]);
#pragma unroll
      for (int e = 0; e < E; ++e) s += own<E>(lane + c * L, n, e) ? f[c][e] : 0.0f;
    }
    const float mu = group_sum<L>(s, red) / (float)n;
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[c][e] -= mu;
        const float d = own<E>(lane + c * L, n, e) ? f[c][e] : 0.0f;
        q += d * d;
      }
    const float r = 1.0f / sqrtf(group_sum<L>(q, red) / (float)n + eps);
    if (stats && lane == 0 && m) {
      stats[row] = mu;
      stats[rows + row] = r;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if ((lane + c * L) * E >= m) continue;
      const int at = KEEP ? c : 0;
      if (!KEEP) params(c, at);
#pragma unroll
      for (int e = 0; e < E; ++e) f[c][e] = f[c][e] * r * wf[at][e] + bf[at][e];
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
  const int nv = vectors_in(n, E);
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    float f[E], s = 0.0f, q = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      row_load<E>(xr, v, n, 0.0f, f);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += own<E>(v, n, e) ? f[e] : 0.0f;
      s += t;
    }
    const float mu = group_sum<WIDE>(s, red) / (float)n;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      row_load<E>(xr, v, n, 0.0f, f);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = own<E>(v, n, e) ? f[e] - mu : 0.0f;
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
      row_load<E>(xr, v, n, 0.0f, f);
      row_load<E>(w, v, n, 1.0f, wf);
      row_load<E>(b, v, n, 0.0f, bf);
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
  // as the forward (rows of 331 float32 316 us for 365), but for 16-bit rows of several waves, which have the registers for
  // three workgroups a CU only without: rows of 4096 bfloat16 180 us for 248
  constexpr bool KEEP = CE <= 8 && (E == 4 || L <= 64);
  float wf[KEEP ? C : 1][E];
  if (KEEP)
#pragma unroll
    for (int c = 0; c < C; ++c) row_load<E>(w, lane + c * L, n, 1.0f, wf[c]);
  // as in the forward, groups of several waves stay together
  for (long long row = (long long)blockIdx.x * GROUPS + group;; row += (long long)gridDim.x * GROUPS) {
    if (L > 64 ? row - group >= rows : row >= rows) break;
    const int m = row < rows ? n : 0;
    float f[CE], g[CE];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      row_load<E>(x + row * xs, lane + c * L, m, 0.0f, f + c * E);
      row_load<E>(dy + row * dys, lane + c * L, m, 0.0f, g + c * E);
    }
    const float mu = m ? stats[row] : 0.0f, r = m ? stats[rows + row] : 0.0f;
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = KEEP ? c : 0;
      if (!KEEP) row_load<E>(w, lane + c * L, n, 1.0f, wf[at]);
#pragma unroll
      for (int e = 0; e < E; ++e) {  // past the row's end x and dy were read as 0: g stays 0 there, xh is not used
        const int i = c * E + e;
        f[i] = (f[i] - mu) * r;
        aw[i] += g[i] * f[i];
        ab[i] += g[i];
        g[i] *= wf[at][e];
        const float t = own<E>(lane + c * L, n, e) ? g[i] : 0.0f;
        s += t;
        q += t * f[i];
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
          if (own<E>(lane + c * L, n, e)) out[which * n + first_of<E>(lane + c * L, n) + e] = a[c * E + e];
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
  const int nv = vectors_in(n, E);
  float* out = part ? part + (long long)blockIdx.x * 2 * n : nullptr;
  float* out_b = part ? out + n : nullptr;  // 2 n may pass 2^31
  bool first = true;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, first = false) {
    const float mu = stats[row], r = stats[rows + row];
    float s = 0.0f, q = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      float f[E], g[E], wf[E];
      row_load<E>(x + row * xs, v, n, 0.0f, f);
      row_load<E>(dy + row * dys, v, n, 0.0f, g);
      row_load<E>(w, v, n, 1.0f, wf);
      float ts = 0.0f, tq = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[e] = (f[e] - mu) * r;
        if (!own<E>(v, n, e)) continue;
        const int col = first_of<E>(v, n) + e;
        if (out) {
          out[col] = (first ? 0.0f : out[col]) + g[e] * f[e];
          out_b[col] = (first ? 0.0f : out_b[col]) + g[e];
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
      row_load<E>(x + row * xs, v, n, 0.0f, f);
      row_load<E>(dy + row * dys, v, n, 0.0f, g);
      row_load<E>(w, v, n, 1.0f, wf);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = r * (g[e] * wf[e] - ms - (f[e] - mu) * r * mq);
      row_store(dx + row * n, v, n, f);
    }
  }
}

// dw, db from the partial rows: 64 columns a workgroup at a time, 16 waves each adding every 16th row, then the waves' sums
constexpr int MOST_BLOCKS = 1 << 21;  // a launch's work-items stay below 2^32
template <typename W>
__global__ __launch_bounds__(1024) void k_norm_params(int blocks, int n, const float* __restrict__ part,
                                                      W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float add[16][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  for (long long first = (long long)blockIdx.x * 64; first < 2LL * n; first += (long long)gridDim.x * 64) {
    const long long col = first + lane;  // of the 2 n columns
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
    __syncthreads();
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------

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
// lanes a row, and vectors a lane
void group_of(int nv, int type, int& lanes, int& vectors) {
  lanes = WIDE, vectors = 2;
  auto f = [&](auto l, auto c) { lanes = decltype(l)::value, vectors = decltype(c)::value; };
  if (bytes_of(type) == 2) by_width<8>(nv, f);
  else by_width<4>(nv, f);
}
int vectors_of(int n, int type) { return vectors_in(n, 16 / bytes_of(type)); }

// The backward's workgroups: each row in flight at once at most, and what the CUs hold at once (of 8 waves: three with one
// vector a lane, two with two; more would only write more partial rows). 524288 x 256 bfloat16: 174 us with two a CU, 151
// with three, 194 with four, which are not all held at once.
int vjp_blocks(long long rows, int n, int type) {
  int lanes, vectors;
  group_of(vectors_of(n, type), type, lanes, vectors);
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
  if (!by_width<Vec<T>::E>(vectors_of(n, type), [&](auto l, auto c) {
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
    if (!by_width<Vec<T>::E>(vectors_of(n, type), [&](auto l, auto c) {
          launch(k_norm_vjp<T, W, decltype(l)::value, decltype(c)::value>, vjp_block(decltype(l)::value));
        }))
      launch(k_norm_vjp_wide<T, W>, WIDE);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (dw || db) {  // no rows: no partial rows, and zeros
    const long long need = (2LL * n + 63) / 64;
    k_norm_params<W><<<(unsigned)(need < MOST_BLOCKS ? need : MOST_BLOCKS), 1024, 0, st>>>(rows > 0 ? blocks : 0, n, part,
                                                                                           (W*)dw, (W*)db);
  }
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
