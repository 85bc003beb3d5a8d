// The gated residual between two blocks: a block's output normed, gated and scaled onto the residual stream, and the stream
// normed for the next block; forward and backward, a row at a time.
//
//   r = 1 / sqrt(mean u^2 + eps),  uh = u r,  n = uh w,  y = x + s sg n,  sg = 1 / (1 + exp(-gate))
//   r' = 1 / sqrt(mean y^2 + eps),  yh = y r',  z = yh w'
//   e = dy + r' (dz w' - yh mean(dz w' yh)),  dx = e,  dgate = e s n sg (1 - sg),  c = e s sg w,  du = r (c - uh mean(c uh))
//   m = sum over rows of e sg uh:  dw = s m,  ds = w m;  dw' = sum over rows of dz yh
//
// Memory bounds the forward: it reads three rows and writes two, and of 131072 rows of 512 bfloat16 takes 125 us, 5.4 TB/s, more
// than a large copy's 5.0 to 5.2. The backward reads five and writes three, 251 us, 4.3 TB/s: beside that its vector instructions
// take 56 % of the SIMDs' cycles (two gates' exponentials and reciprocals and some 60 others an element). A row is read once into the registers of a group of L lanes and all
// is computed there in float32; z comes of the y that is not rounded yet, and the backward computes y again from x, u and gate,
// which it needs anyway, instead of reading a rounded one. The backward's groups keep their columns' m and dw' in registers; at
// the end a workgroup adds its groups' sums in LDS and writes one partial row, and a second kernel adds those in a fixed order.
#include "../../include/nablaengine_memory.h"
#include "policy_device.h"
#include "policy_rows.h"

namespace pol {

struct Residual {
  long long rows;
  int n;
  const void *x, *u, *gate;  // gate NULL: sg = 1
  long long x_r, u_r, g_r;   // elements from row to row
  const void *w, *w2, *s;    // each NULL: ones
  float eps;
  void *y, *z;
  float* stats;  // (2, rows): r and r', or NULL
  // the backward's
  const void *dy, *dz;  // each NULL: zeros
  long long dy_r, dz_r;
  void *dx, *du, *dgate;  // each NULL: not wanted
  float* part;            // (blocks, 2, n): each workgroup's m and dw', or NULL
};

// how many of vector v's first elements the vector before it holds too; elements past the row are 0 and count as nothing
template <int E>
__device__ __forceinline__ int repeated(int v, int n) {
  return n >= E && v < vectors_in(n, E) ? v * E - first_of<E>(v, n) : 0;
}
// vector v of a row of activations that may not be there
template <typename T>
__device__ __forceinline__ void given(const void* p, long long row, long long stride, int v, int n, float* f) {
  row_load<Vec<T>::E>(p ? (const T*)p + row * stride : (const T*)nullptr, v, n, 0.0f, f);
}
// the same as it is
template <typename T>
__device__ __forceinline__ Vec<T> row_vector(const T* p, int v, int n) {
  constexpr int E = Vec<T>::E;
  Vec<T> r = {};
  if (p && v * E < n) {
    if (n >= E) {
      r = load16(p + first_of<E>(v, n));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < n) r.v[e] = p[e];
    }
  }
  return r;
}
// The compiler takes its 16 bytes for new ones: what was computed of them before is not kept in registers for later.
template <typename T>
__device__ __forceinline__ void anew(Vec<T>& v) {
  unsigned x[4];
  __builtin_memcpy(x, &v, 16);
  asm("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
  __builtin_memcpy(&v, x, 16);
}
__device__ __forceinline__ float of_wave(float x) {  // one for all lanes
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}
template <typename T>
__device__ __forceinline__ float open_gate(const Residual& a, float f, float& shut) {
  float open;
  gates<T>(f, open, shut);
  if (!a.gate) open = 1.0f, shut = 0.0f;
  return open;
}

template <typename T, typename W, int L, int C>
__global__ __launch_bounds__(L > 256 ? L : 256) void k_residual(Residual a) {
  constexpr int E = Vec<T>::E, BLOCK = L > 256 ? L : 256, GROUPS = BLOCK / L;
  constexpr bool KEEP = C * E <= 8;  // a lane's parameters, the same for all its rows, in registers
  __shared__ float red[BLOCK / 64];
  const int lane = threadIdx.x % L, group = threadIdx.x / L, n = a.n;
  float w[KEEP ? C : 1][E], w2[KEEP ? C : 1][E], sc[KEEP ? C : 1][E];
  auto params = [&](int c, int to) {
    row_load<E>((const W*)a.w, lane + c * L, n, 1.0f, w[to]);
    row_load<E>((const W*)a.s, lane + c * L, n, 1.0f, sc[to]);
  };
  int repeats[C];  // elements of this lane's vectors that the one before has: the row's last vector ends with it
#pragma unroll
  for (int c = 0; c < C; ++c) repeats[c] = repeated<E>(lane + c * L, n);
  auto next_params = [&](int c, int to) { row_load<E>((const W*)a.w2, lane + c * L, n, 1.0f, w2[to]); };
  if (KEEP)
#pragma unroll
    for (int c = 0; c < C; ++c) params(c, c), next_params(c, c);
  // groups of several waves meet at barriers: the workgroup stays together, a group past the last row has none of it
  for (long long row = (long long)blockIdx.x * GROUPS + group;; row += (long long)gridDim.x * GROUPS) {
    if (L > 64 ? row - group >= a.rows : row >= a.rows) break;
    const int m = row < a.rows ? n : 0;
    float x[C][E], u[C][E], g[C][E], q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      given<T>(a.u, row, a.u_r, lane + c * L, m, u[c]);
      given<T>(a.x, row, a.x_r, lane + c * L, m, x[c]);
      given<T>(a.gate, row, a.g_r, lane + c * L, m, g[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) q += e >= repeats[c] ? u[c][e] * u[c][e] : 0.0f;
    const float r = 1.0f / sqrtf(group_sum<L>(q, red) / (float)n + a.eps);
    q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = KEEP ? c : 0;
      if (!KEEP) params(c, at);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float shut;
        const float sg = open_gate<T>(a, g[c][e], shut);
        x[c][e] += sc[at][e] * sg * (u[c][e] * r * w[at][e]);
        q += e >= repeats[c] ? x[c][e] * x[c][e] : 0.0f;
      }
    }
    const float r2 = 1.0f / sqrtf(group_sum<L>(q, red) / (float)n + a.eps);
    if (a.stats && lane == 0 && m) {
      a.stats[row] = r;
      a.stats[a.rows + row] = r2;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if ((lane + c * L) * E >= m) continue;
      const int at = KEEP ? c : 0;
      if (!KEEP) next_params(c, at);
      row_store((T*)a.y + row * n, lane + c * L, n, x[c]);
#pragma unroll
      for (int e = 0; e < E; ++e) x[c][e] *= r2 * w2[at][e];
      row_store((T*)a.z + row * n, lane + c * L, n, x[c]);
    }
  }
}

// rows that no group holds are read once for each sum and once more
template <typename T, typename W>
__global__ __launch_bounds__(WIDE) void k_residual_wide(Residual a) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[WIDE / 64];
  const int n = a.n, nv = vectors_in(n, E);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float x[E], u[E], g[E], w[E], s[E], q = 0.0f, r = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      given<T>(a.u, row, a.u_r, v, n, u);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += own<E>(v, n, e) ? u[e] * u[e] : 0.0f;
      q += t;
    }
    r = 1.0f / sqrtf(group_sum<WIDE>(q, red) / (float)n + a.eps);
    auto stream = [&](int v) {
      given<T>(a.x, row, a.x_r, v, n, x);
      given<T>(a.u, row, a.u_r, v, n, u);
      given<T>(a.gate, row, a.g_r, v, n, g);
      row_load<E>((const W*)a.w, v, n, 1.0f, w);
      row_load<E>((const W*)a.s, v, n, 1.0f, s);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float shut;
        const float sg = open_gate<T>(a, g[e], shut);
        x[e] += s[e] * sg * (u[e] * r * w[e]);
      }
    };
    q = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      stream(v);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += own<E>(v, n, e) ? x[e] * x[e] : 0.0f;
      q += t;
      row_store((T*)a.y + row * n, v, n, x);
    }
    const float r2 = 1.0f / sqrtf(group_sum<WIDE>(q, red) / (float)n + a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[row] = r;
      a.stats[a.rows + row] = r2;
    }
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      stream(v);
      row_load<E>((const W*)a.w2, v, n, 1.0f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= r2 * w[e];
      row_store((T*)a.z + row * n, v, n, x);
    }
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------

template <typename T, typename W, int L>
__global__ __launch_bounds__(vjp_block(L), 4) void k_residual_vjp(Residual a) {
  constexpr int E = Vec<T>::E, GROUPS = vjp_block(L) / L;
  constexpr int SLOTS = L >= 64 ? GROUPS : 8;  // the sums left after those inside each wave
  __shared__ float red[16];
  __shared__ float add[SLOTS > 1 ? SLOTS / 2 * L * E : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L, n = a.n;
  // the parameters as the lanes of a group use them, the same for all rows; in LDS, since a lane's 24 floats would be the
  // registers of the second workgroup (neighbouring lanes' 16 bytes side by side: lanes 32 bytes apart conflict)
  __shared__ __align__(16) float params[3][L * E];
  float am[E], an[E];
#pragma unroll
  for (int e = 0; e < E; ++e) am[e] = an[e] = 0.0f;
  for (int v = threadIdx.x; v < L; v += vjp_block(L)) {
    float f[E];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      row_load<E>((const W*)(i == 0 ? a.w : i == 1 ? a.w2 : a.s), v, n, 1.0f, f);
#pragma unroll
      for (int e = 0; e < E; ++e) params[i][(e / 4 * L + v) * 4 + e % 4] = f[e];
    }
  }
  __syncthreads();
  const int repeats = repeated<E>(lane, n);
  // as in the forward, groups of several waves stay together
  for (long long row = (long long)blockIdx.x * GROUPS + group;; row += (long long)gridDim.x * GROUPS) {
    if (L > 64 ? row - group >= a.rows : row >= a.rows) break;
    const int m = row < a.rows ? n : 0;
    int place = lane;  // anew for each row, so that the parameters are not read to registers once and for all
    asm volatile("" : "+v"(place));
    auto param = [&](int which, int e) { return params[which][(e / 4 * L + place) * 4 + e % 4]; };
    // What is read stays as it is, half the registers of its floats in 16 bits; of the products only those that the sums between
    // them need are kept: 114 to 119 registers a lane instead of 163, two workgroups a compute unit instead of one.
    const Vec<T> xr = row_vector((const T*)a.x + row * a.x_r, lane, m);
    Vec<T> ur = row_vector((const T*)a.u + row * a.u_r, lane, m);
    const Vec<T> gr = row_vector(a.gate ? (const T*)a.gate + row * a.g_r : nullptr, lane, m);
    Vec<T> yr = row_vector(a.dy ? (const T*)a.dy + row * a.dy_r : nullptr, lane, m);
    Vec<T> zr = row_vector(a.dz ? (const T*)a.dz + row * a.dz_r : nullptr, lane, m);
    float r = m ? a.stats[row] : 0.0f, r2 = m ? a.stats[a.rows + row] : 0.0f;
    if (L >= 64) r = of_wave(r), r2 = of_wave(r2);
    float q = 0.0f, yh[E], sg[E], shut[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {  // past the row's end all five were read as 0
      sg[e] = open_gate<T>(a, (float)gr.v[e], shut[e]);
      yh[e] = ((float)xr.v[e] + param(2, e) * sg[e] * ((float)ur.v[e] * r * param(0, e))) * r2;
      const float dz = (float)zr.v[e];
      an[e] += dz * yh[e];
      q += e >= repeats ? dz * param(1, e) * yh[e] : 0.0f;
    }
    q = group_sum<L>(q, red) / (float)n;
    anew(ur), anew(yr), anew(zr);
    float p = 0.0f, c[E], dx[E], dg[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float uh = (float)ur.v[e] * r;
      dx[e] = (float)yr.v[e] + r2 * ((float)zr.v[e] * param(1, e) - yh[e] * q);
      c[e] = dx[e] * param(2, e) * sg[e] * param(0, e);
      am[e] += dx[e] * sg[e] * uh;
      dg[e] = c[e] * uh * shut[e];
      p += e >= repeats ? c[e] * uh : 0.0f;
    }
    const bool mine = lane * E < m;
    if (mine && a.dx) row_store((T*)a.dx + row * n, lane, n, dx);
    if (mine && a.dgate) row_store((T*)a.dgate + row * n, lane, n, dg);
    if (a.du) {
      p = group_sum<L>(p, red) / (float)n;
      anew(ur);
#pragma unroll
      for (int e = 0; e < E; ++e) c[e] = r * (c[e] - (float)ur.v[e] * r * p);
      if (mine) row_store((T*)a.du + row * n, lane, n, c);
    }
  }
  if (!a.part) return;
  // the lanes of a wave that hold the same columns, then the waves (or groups) by halves: a fixed order
  float* out = a.part + (long long)blockIdx.x * 2 * n;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* s = which ? an : am;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (L <= 8) s[e] += __shfl_xor(s[e], 8);
      if constexpr (L <= 16) s[e] = add_rows(s[e]);
      if constexpr (L <= 32) s[e] = add_halves(s[e]);
    }
    const int slot = L >= 64 ? group : threadIdx.x / 64;
    const bool holds = L >= 64 || threadIdx.x % 64 < L;
#pragma unroll
    for (int half = SLOTS / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (holds && slot >= half && slot < 2 * half)
#pragma unroll
        for (int e = 0; e < E; ++e) add[((slot - half) * E + e) * L + lane] = s[e];
      __syncthreads();
      if (holds && slot < half)
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += add[(slot * E + e) * L + lane];
    }
    if (holds && slot == 0)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (own<E>(lane, n, e)) out[(long long)which * n + first_of<E>(lane, n) + e] = s[e];
  }
}

// wide rows: a workgroup adds its columns' sums in its partial row, which is its own (each column's thread is the same one
// throughout)
template <typename T, typename W>
__global__ __launch_bounds__(WIDE) void k_residual_vjp_wide(Residual a) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[WIDE / 64];
  const int n = a.n, nv = vectors_in(n, E);
  float* out = a.part ? a.part + (long long)blockIdx.x * 2 * n : nullptr;
  float* out_n = out ? out + n : nullptr;
  bool first = true;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
    const float r = a.stats[row], r2 = a.stats[a.rows + row];
    float uh[E], yh[E], sg[E], shut[E], dz[E], gz[E], w[E], s[E];
    auto load = [&](int v) {
      float x[E], g[E], w2[E];
      given<T>(a.x, row, a.x_r, v, n, x);
      given<T>(a.u, row, a.u_r, v, n, uh);
      given<T>(a.gate, row, a.g_r, v, n, g);
      given<T>(a.dz, row, a.dz_r, v, n, dz);
      row_load<E>((const W*)a.w, v, n, 1.0f, w);
      row_load<E>((const W*)a.w2, v, n, 1.0f, w2);
      row_load<E>((const W*)a.s, v, n, 1.0f, s);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sg[e] = open_gate<T>(a, g[e], shut[e]);
        uh[e] *= r;
        yh[e] = (x[e] + s[e] * sg[e] * (uh[e] * w[e])) * r2;
        gz[e] = dz[e] * w2[e];
      }
    };
    float q = 0.0f, p = 0.0f;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      load(v);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += own<E>(v, n, e) ? gz[e] * yh[e] : 0.0f;
      q += t;
    }
    q = group_sum<WIDE>(q, red) / (float)n;
    float de[E], c[E];
    auto branch = [&](int v) {
      load(v);
      given<T>(a.dy, row, a.dy_r, v, n, de);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        de[e] += r2 * (gz[e] - yh[e] * q);
        c[e] = de[e] * s[e] * sg[e] * w[e];
      }
    };
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      branch(v);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!own<E>(v, n, e)) continue;
        t += c[e] * uh[e];
        if (!out) continue;
        const int col = first_of<E>(v, n) + e;
        out[col] = (first ? 0.0f : out[col]) + de[e] * sg[e] * uh[e];
        out_n[col] = (first ? 0.0f : out_n[col]) + dz[e] * yh[e];
      }
      p += t;
    }
    p = group_sum<WIDE>(p, red) / (float)n;
    for (int v = threadIdx.x; v < nv; v += WIDE) {
      branch(v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        shut[e] *= de[e] * s[e] * (uh[e] * w[e]) * sg[e];
        c[e] = r * (c[e] - uh[e] * p);
      }
      if (a.dx) row_store((T*)a.dx + row * n, v, n, de);
      if (a.dgate) row_store((T*)a.dgate + row * n, v, n, shut);
      if (a.du) row_store((T*)a.du + row * n, v, n, c);
    }
  }
}

// dw = s m, ds = w m and dw' from the partial rows: 64 columns a workgroup at a time, 16 waves each adding every 16th row
constexpr int MOST_BLOCKS = 1 << 21;  // a launch's work-items stay below 2^32
template <typename W>
__global__ __launch_bounds__(1024) void k_residual_params(int blocks, int n, const float* __restrict__ part, const W* __restrict__ w,
                                                          const W* __restrict__ s, W* __restrict__ dw, W* __restrict__ dw2,
                                                          W* __restrict__ ds) {
  __shared__ float add[16][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  for (long long first = (long long)blockIdx.x * 64; first < 2LL * n; first += (long long)gridDim.x * 64) {
    const long long col = first + lane;  // of the 2 n columns
    float t = 0.0f;
    if (col < 2LL * n) {
#pragma unroll 8
      for (int i = wave; i < blocks; i += 16) t += part[(long long)i * 2 * n + col];
    }
    add[wave][lane] = t;
    __syncthreads();
    if (wave == 0 && col < 2LL * n) {
      t = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) t += add[i][lane];
      if (col < n) {
        if (dw) dw[col] = (W)(s ? (float)s[col] * t : t);
        if (ds) ds[col] = (W)(w ? (float)w[col] * t : t);
      } else if (dw2) {
        dw2[col - n] = (W)t;
      }
    }
    __syncthreads();
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------

// The backward's lanes hold one vector each: it keeps ten values for each element.
template <typename F>
bool by_width_vjp(int nv, F f) {
#define POL_CASE(L) \
  if (nv <= L) { f(std::integral_constant<int, L>{}); return true; }
  POL_CASE(8) POL_CASE(16) POL_CASE(32) POL_CASE(64) POL_CASE(128) POL_CASE(256) POL_CASE(512) POL_CASE(1024)
#undef POL_CASE
  return false;
}
int residual_blocks(long long rows, int n, int type) {
  int lanes = WIDE;
  by_width_vjp(vectors_of(n, type), [&](auto l) { lanes = decltype(l)::value; });
  const int groups = vjp_block(lanes) / lanes;
  const long long need = (rows + groups - 1) / groups, most = 2 * CUS;
  return (int)(need < most ? need : most);
}

template <typename T, typename W>
int residual(hipStream_t st, const Residual& a, int type) {
  auto launch = [&](auto kernel, int block, int groups) {
    const long long need = (a.rows + groups - 1) / groups, most = 32LL * CUS;
    kernel<<<(unsigned)(need < most ? need : most), block, 0, st>>>(a);
  };
  if (!by_width<Vec<T>::E>(vectors_of(a.n, type), [&](auto l, auto c) {
        constexpr int L = decltype(l)::value, C = decltype(c)::value, BLOCK = L > 256 ? L : 256;
        if constexpr (L * C * Vec<T>::E > 8192) launch(k_residual_wide<T, W>, WIDE, 1);  // the registers would not do
        else launch(k_residual<T, W, L, C>, BLOCK, BLOCK / L);
      }))
    launch(k_residual_wide<T, W>, WIDE, 1);
  return (int)hipGetLastError();
}
template <typename T, typename W>
int residual_vjp(hipStream_t st, const Residual& a, int type, void* dw, void* dw2, void* ds) {
  const int blocks = residual_blocks(a.rows, a.n, type);
  if (a.rows > 0) {
    if (!by_width_vjp(vectors_of(a.n, type), [&](auto l) {
          constexpr int L = decltype(l)::value;
          k_residual_vjp<T, W, L><<<blocks, vjp_block(L), 0, st>>>(a);
        }))
      k_residual_vjp_wide<T, W><<<blocks, WIDE, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (dw || dw2 || ds) {  // no rows: no partial rows, and zeros
    const long long need = (2LL * a.n + 63) / 64;
    k_residual_params<W><<<(unsigned)(need < MOST_BLOCKS ? need : MOST_BLOCKS), 1024, 0, st>>>(
        a.rows > 0 ? blocks : 0, a.n, a.part, (const W*)a.w, (const W*)a.s, (W*)dw, (W*)dw2, (W*)ds);
  }
  return (int)hipGetLastError();
}
int launch_residual(hipStream_t st, const Residual& a, int type, int wtype) {
#define CALL(T, W) residual<T, W>(st, a, type)
  POL_BY_TYPES(CALL)
#undef CALL
}
int launch_residual_vjp(hipStream_t st, const Residual& a, int type, int wtype, void* dw, void* dw2, void* ds) {
#define CALL(T, W) residual_vjp<T, W>(st, a, type, dw, dw2, ds)
  POL_BY_TYPES(CALL)
#undef CALL
}

bool residual_takes(long long rows, int n, int type, int w_type) {
  return rows >= 0 && n >= 1 && type >= 0 && type <= 2 && (w_type == F32 || w_type == type);
}

}  // namespace pol

extern "C" {

int dk_gated_residual(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* u,
                      long long u_row, const void* gate, long long gate_row, int w_type, const void* w, const void* next_w,
                      const void* scale, float eps, void* y, void* z, float* stats) {
  if (!pol::residual_takes(rows, n, type, w_type)) return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !u || !y || !z) return (int)hipErrorInvalidValue;
  pol::Residual a = {};
  a.rows = rows, a.n = n, a.x = x, a.u = u, a.gate = gate, a.x_r = x_row, a.u_r = u_row, a.g_r = gate_row;
  a.w = w, a.w2 = next_w, a.s = scale, a.eps = eps, a.y = y, a.z = z, a.stats = stats;
  return pol::launch_residual(st, a, type, w_type);
}

int dk_gated_residual_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* u,
                          long long u_row, const void* gate, long long gate_row, int w_type, const void* w, const void* next_w,
                          const void* scale, const float* stats, const void* dy, long long dy_row, const void* dz,
                          long long dz_row, void* dx, void* du, void* dgate, void* dw, void* dnext_w, void* dscale, void* work) {
  const bool params = dw || dnext_w || dscale;
  if (!pol::residual_takes(rows, n, type, w_type) || (rows > 0 && (!x || !u || !stats || (params && !work))))
    return (int)hipErrorInvalidValue;
  pol::Residual a = {};
  a.rows = rows, a.n = n, a.x = x, a.u = u, a.gate = gate, a.x_r = x_row, a.u_r = u_row, a.g_r = gate_row;
  a.w = w, a.w2 = next_w, a.s = scale, a.stats = const_cast<float*>(stats);
  a.dy = dy, a.dz = dz, a.dy_r = dy_row, a.dz_r = dz_row, a.dx = dx, a.du = du, a.dgate = gate ? dgate : nullptr;
  a.part = params ? (float*)work : nullptr;
  return pol::launch_residual_vjp(st, a, type, w_type, dw, dnext_w, dscale);
}

long long dk_gated_residual_work_bytes(long long rows, int n, int type) {
  if (rows <= 0 || n < 1 || type < 0 || type > 2) return 0;
  return (long long)pol::residual_blocks(rows, n, type) * 2 * n * 4;
}

}  // extern "C"
