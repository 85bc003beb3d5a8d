// Causal attention over packed sequences with shared key/value heads: forward and backward.
//
//   S = scale Q K^T, key j <= i + (keys - queries), P = softmax(S), O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta), delta = dO . O a row,  dQ = scale dS K,  dK = scale dS^T Q
//
// A workgroup of four waves takes 128 rows of one key/value head's queries, row = token * group + head, so that the
// heads of a group share each key and value tile and short sequences still fill the rows; a wave takes 32 rows.
#include "../../include/nablaengine_policy.h"
#include "policy_attend.h"

namespace pol {

// ---- the order ------------------------------------------------------------------------------------------------------

// One workgroup lists the tiles, heaviest first (a counting sort by the tiles of the other side that each one reads;
// its place among equals is free, results do not depend on the order). seqs + 1 sequences, LS lanes on each.
__global__ __launch_bounds__(1024) void k_attend_order(int seqs, int tq, int tk, int group, const int* __restrict__ starts_q,
                                                       const int* __restrict__ starts_k, int* __restrict__ order) {
  constexpr int BUCKETS = 1024;
  __shared__ int count[BUCKETS];
  __shared__ int wave_sum[16];
  int ls = 1;
  while (ls < 1024 && ls * 2 * (long long)(seqs + 1) <= 1024) ls *= 2;
  const int lane = threadIdx.x % ls, first_seq = threadIdx.x / ls, stride = 1024 / ls;
  const long long caps[2] = {order_queries(seqs, tq, group), order_keys(seqs, tk)};
  int* list = order + ORDER_HEAD;
  for (int which = 0; which < 2; ++which) {
    auto each_tile = [&](auto f) {
      for (int s = first_seq; s <= seqs; s += stride) {
        int q0, k0, nq, nk;
        sequence(starts_q, s, seqs, tq, q0, nq);
        sequence(starts_k, s, seqs, tk, k0, nk);
        if (s == seqs) (which ? nq : nk) = 0;
        const int rows = which ? nk : nq * group, per = which ? KROWS : QROWS, tiles = (rows + per - 1) / per;
        for (int t = lane; t < tiles; t += ls) {
          int cost;
          if (which) {  // the query rows that see the tile's first key
            const int from = t * KROWS - (nk - nq);
            cost = nq - (from > 0 ? from : 0);
            cost = (int)(((long long)(cost > 0 ? cost : 0) * group + TILE - 1) / TILE);
          } else {  // the keys that the tile's last row sees
            const int last = ((t + 1) * QROWS < rows ? (t + 1) * QROWS : rows) - 1, keys = last / group + nk - nq + 1;
            cost = keys > 0 ? (keys + TILE - 1) / TILE : 0;
          }
          f(s, t, BUCKETS - 1 - (cost < BUCKETS ? cost : BUCKETS - 1));
        }
      }
    };
    count[threadIdx.x] = 0;
    __syncthreads();
    each_tile([&](int, int, int b) { atomicAdd(&count[b], 1); });
    __syncthreads();
    // exclusive prefix over the buckets
    const int mine = count[threadIdx.x];
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(sum, d);
      if (threadIdx.x % 64 >= d) sum += x;
    }
    if (threadIdx.x % 64 == 63) wave_sum[threadIdx.x / 64] = sum;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < (int)threadIdx.x / 64) before += wave_sum[w];
      total += wave_sum[w];
    }
    count[threadIdx.x] = before + sum - mine;
    if (threadIdx.x == 0) order[which] = total < caps[which] ? total : (int)caps[which];
    __syncthreads();
    each_tile([&](int s, int t, int b) {
      const int at = atomicAdd(&count[b], 1);
      if (at < caps[which]) {
        list[2 * at] = s;
        list[2 * at + 1] = t;
      }
    });
    __syncthreads();
    list += 2 * caps[0];
  }
}

// what a workgroup works on
struct Place {
  int tile, kv, q0, nq, k0, nk;
};
__device__ __forceinline__ bool place(const Attend& a, int which, Place& p) {
  const int entry = blockIdx.x / a.kv_heads;
  if (entry >= a.order[which]) return false;
  const int* list = a.order + ORDER_HEAD + (which ? 2 * order_queries(a.seqs, a.tq, a.group) : 0) + 2LL * entry;
  const int s = list[0];
  p.tile = list[1];
  p.kv = blockIdx.x % a.kv_heads;
  sequence(a.starts_q, s, a.seqs, a.tq, p.q0, p.nq);
  sequence(a.starts_k, s, a.seqs, a.tk, p.k0, p.nk);
  if (s == a.seqs) (which ? p.nq : p.nk) = 0;
  return true;
}

// A tile of TILE rows on its way from memory to LDS: 16-byte chunks, the same for each thread of the 256.
template <int DP, typename T>
struct Stage {
  static constexpr int CH = DP / 8, N = TILE * CH / 256;
  V8<T> x[N];
  // row r of the tile is at base + r * stride; rows past `rows` and columns past `dim` are zeros
  __device__ __forceinline__ void load(const T* base, long long stride, int rows, int dim) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * 256 + threadIdx.x, r = at / CH, c = at % CH;
      x[i] = r < rows && 8 * c < dim ? load8(base + r * stride + 8 * c) : zero8<T>();
    }
  }
  __device__ __forceinline__ void write(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * 256 + threadIdx.x;
      *(V8<T>*)(tile + chunk_at<DP>(at / CH, at % CH)) = x[i];
    }
  }
};

// ---- forward --------------------------------------------------------------------------------------------------------

template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void k_attend(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[TILE * DP];
  __shared__ __align__(16) T vs[TILE * DP];
  Place p;
  if (!place(a, 0, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, w = threadIdx.x / 64;
  const int rows = p.nq * a.group, off = p.nk - p.nq, dim = a.dim;
  const int row0 = p.tile * QROWS + 32 * w, row = row0 + n;
  const bool valid = row < rows;
  const int pos = row / a.group, head = p.kv * a.group + row % a.group;
  const int limit = valid ? pos + off : -1;  // the row's last key (below 0: none)
  // of the wave's rows: the last key that all see, and the last that any sees; of the workgroup's
  const int all_see = row0 < rows ? row0 / a.group + off : -1;
  const int any_sees = row0 < rows ? (row0 + 31 < rows ? row0 + 31 : rows - 1) / a.group + off : -1;
  const int end0 = p.tile * QROWS + QROWS < rows ? p.tile * QROWS + QROWS : rows;
  const int last = (end0 - 1) / a.group + off;
  const int tiles = last < 0 ? 0 : last / TILE + 1;

  V8<T> q[KS];
  load_rows<DP>(valid ? (const T*)a.q + (long long)(p.q0 + pos) * a.q_t + (long long)head * a.q_h : nullptr, dim, h, q);
  const T* kb = (const T*)a.k + (long long)p.k0 * a.k_t + (long long)p.kv * a.k_h;
  const T* vb = (const T*)a.v + (long long)p.k0 * a.v_t + (long long)p.kv * a.v_h;

  F16x acc[DT] = {};
  float m = -INFINITY, sum = 0.0f;
  const float c = a.scale * LOG2E;
  Stage<DP, T> ksg, vsg;
  if (tiles) {
    ksg.load(kb, a.k_t, p.nk, dim);
    vsg.load(vb, a.v_t, p.nk, dim);
  }
  for (int t = 0; t < tiles; ++t) {
    const int key0 = t * TILE;
    __syncthreads();
    ksg.write(ks);
    vsg.write(vs);
    __syncthreads();
    if (t + 1 < tiles) {
      ksg.load(kb + (long long)(key0 + TILE) * a.k_t, a.k_t, p.nk - key0 - TILE, dim);
      vsg.load(vb + (long long)(key0 + TILE) * a.v_t, a.v_t, p.nk - key0 - TILE, dim);
    }
    if (key0 > any_sees) continue;
    const bool second = key0 + 32 <= any_sees;
    F16x s[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !second) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[1][r] = -INFINITY;
        break;
      }
#pragma unroll
      for (int x = 0; x < KS; ++x) s[i] = mfma(read_rows<DP>(ks, 32 * i, x, n, h), q[x], s[i]);
      if (key0 + 32 * i + 31 > all_see)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * i + r % 4 + 8 * (r / 4) + 4 * h > limit) s[i][r] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[1][r]);
    const float m1 = fmaxf(m, max_halves(top));
    const float base = m1 == -INFINITY ? 0.0f : m1 * c;  // a row that has seen no key yet
    if (__any(m1 != m)) {
      const float f = m == -INFINITY ? 0.0f : exp2f(m * c - base);
      sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= f;
      m = m1;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[i][r] = exp2f(fmaf(s[i][r], c, -base));
        sum += s[i][r];
      }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x == 2 && !second) break;
      const V8<T> pr = pack<T>(s[x / 2], x % 2);
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = mfma(read_columns<DP>(vs, 16 * x, d, l), pr, acc[d]);
    }
  }
  sum = add_halves(sum);
  if (a.lse && valid && h == 0)
    a.lse[(long long)head * a.tq + p.q0 + pos] = sum == 0.0f ? INFINITY : m * c + log2f(sum);
  store_rows<DP>(valid ? (T*)a.out + ((long long)(p.q0 + pos) * a.heads + head) * dim : nullptr, dim, h, acc,
                 sum == 0.0f ? 0.0f : 1.0f / sum);
}

// ---- backward: the queries' gradient --------------------------------------------------------------------------------

template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void k_attend_dq(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[TILE * DP];
  __shared__ __align__(16) T vs[TILE * DP];
  Place p;
  if (!place(a, 0, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, w = threadIdx.x / 64;
  const int rows = p.nq * a.group, off = p.nk - p.nq, dim = a.dim;
  const int row0 = p.tile * QROWS + 32 * w, row = row0 + n;
  const bool valid = row < rows;
  const int pos = row / a.group, head = p.kv * a.group + row % a.group;
  const int limit = valid ? pos + off : -1;
  const int all_see = row0 < rows ? row0 / a.group + off : -1;
  const int any_sees = row0 < rows ? (row0 + 31 < rows ? row0 + 31 : rows - 1) / a.group + off : -1;
  const int end0 = p.tile * QROWS + QROWS < rows ? p.tile * QROWS + QROWS : rows;
  const int last = (end0 - 1) / a.group + off;
  const int tiles = last < 0 ? 0 : last / TILE + 1;

  V8<T> q[KS], g[KS];
  const long long token = p.q0 + pos;
  load_rows<DP>(valid ? (const T*)a.q + token * a.q_t + (long long)head * a.q_h : nullptr, dim, h, q);
  load_rows<DP>(valid ? (const T*)a.dout + token * a.do_t + (long long)head * a.do_h : nullptr, dim, h, g);
  float delta = 0.0f, lse = INFINITY;
  {
    V8<T> o[KS];
    load_rows<DP>(valid ? (const T*)a.out + (token * a.heads + head) * dim : nullptr, dim, h, o);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)o[s][e] * (float)g[s][e];
    delta = add_halves(delta);
    if (valid) {
      lse = a.lse[(long long)head * a.tq + token];
      if (h == 0) a.delta[(long long)head * a.tq + token] = delta;
    }
  }
  const T* kb = (const T*)a.k + (long long)p.k0 * a.k_t + (long long)p.kv * a.k_h;
  const T* vb = (const T*)a.v + (long long)p.k0 * a.v_t + (long long)p.kv * a.v_h;
  F16x acc[DT] = {};
  const float c = a.scale * LOG2E;
  Stage<DP, T> ksg, vsg;
  if (tiles) {
    ksg.load(kb, a.k_t, p.nk, dim);
    vsg.load(vb, a.v_t, p.nk, dim);
  }
  for (int t = 0; t < tiles; ++t) {
    const int key0 = t * TILE;
    __syncthreads();
    ksg.write(ks);
    vsg.write(vs);
    __syncthreads();
    if (t + 1 < tiles) {
      ksg.load(kb + (long long)(key0 + TILE) * a.k_t, a.k_t, p.nk - key0 - TILE, dim);
      vsg.load(vb + (long long)(key0 + TILE) * a.v_t, a.v_t, p.nk - key0 - TILE, dim);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (key0 + 32 * i > any_sees) break;
      F16x s = {}, dp = {};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        s = mfma(read_rows<DP>(ks, 32 * i, x, n, h), q[x], s);
        dp = mfma(read_rows<DP>(vs, 32 * i, x, n, h), g[x], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2f(fmaf(s[r], c, -lse)) * (dp[r] - delta);
      if (key0 + 32 * i + 31 > all_see)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * i + r % 4 + 8 * (r / 4) + 4 * h > limit) s[r] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const V8<T> ds = pack<T>(s, x);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = mfma(read_columns<DP>(ks, 32 * i + 16 * x, d, l), ds, acc[d]);
      }
    }
  }
  store_rows<DP>(valid ? (T*)a.dq + (token * a.heads + head) * dim : nullptr, dim, h, acc, a.scale);
}

// ---- backward: the keys' and values' gradients ----------------------------------------------------------------------

// A wave keeps 32 keys and their values as B operands and walks over the rows that see them; rows lie in LDS. S = Q K^T
// here, so that a lane holds 16 rows of ONE key and P, dS are the B operands of dV^T = dO^T P and dK^T = Q^T dS.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void k_attend_dkv(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32, CH = DP / 8, N = TILE * CH / 256;
  __shared__ __align__(16) T qs[TILE * DP];
  __shared__ __align__(16) T gs[TILE * DP];
  __shared__ __align__(16) float lses[TILE], deltas[TILE];
  __shared__ __align__(16) int limits[TILE];
  Place p;
  if (!place(a, 1, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, w = threadIdx.x / 64;
  const int rows = p.nq * a.group, off = p.nk - p.nq, dim = a.dim;
  const int key0 = p.tile * KROWS + 32 * w, key = key0 + n;
  const bool valid = key < p.nk;
  V8<T> k[KS], v[KS];
  load_rows<DP>(valid ? (const T*)a.k + (long long)(p.k0 + key) * a.k_t + (long long)p.kv * a.k_h : nullptr, dim, h, k);
  load_rows<DP>(valid ? (const T*)a.v + (long long)(p.k0 + key) * a.v_t + (long long)p.kv * a.v_h : nullptr, dim, h, v);
  F16x dk[DT] = {}, dv[DT] = {};
  const float c = a.scale * LOG2E;
  const int from = p.tile * KROWS - off;  // the first token that sees the tile's first key
  const int first = (from > 0 ? from : 0) * a.group;

  V8<T> qx[N], gx[N];
  float lse = INFINITY, delta = 0.0f;
  int limit = -1;
  auto load = [&](int r0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * 256 + threadIdx.x, r = r0 + at / CH, d = at % CH * 8;
      const bool in = r < rows && d < dim;
      const int pos = r / a.group, head = p.kv * a.group + r % a.group;
      qx[i] = in ? load8((const T*)a.q + (long long)(p.q0 + pos) * a.q_t + (long long)head * a.q_h + d) : zero8<T>();
      gx[i] = in ? load8((const T*)a.dout + (long long)(p.q0 + pos) * a.do_t + (long long)head * a.do_h + d) : zero8<T>();
    }
    if (threadIdx.x < TILE) {
      const int r = r0 + threadIdx.x, pos = r / a.group;
      const long long at = (long long)(p.kv * a.group + r % a.group) * a.tq + p.q0 + pos;
      lse = r < rows ? a.lse[at] : INFINITY;
      delta = r < rows ? a.delta[at] : 0.0f;
      limit = r < rows ? pos + off : -1;
    }
  };
  if (first < rows) load(first);
  for (int r0 = first; r0 < rows; r0 += TILE) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * 256 + threadIdx.x;
      *(V8<T>*)(qs + chunk_at<DP>(at / CH, at % CH)) = qx[i];
      *(V8<T>*)(gs + chunk_at<DP>(at / CH, at % CH)) = gx[i];
    }
    if (threadIdx.x < TILE) {
      lses[threadIdx.x] = lse;
      deltas[threadIdx.x] = delta;
      limits[threadIdx.x] = limit;
    }
    __syncthreads();
    if (r0 + TILE < rows) load(r0 + TILE);
    if (key0 >= p.nk) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ra = r0 + 32 * i, rb = ra + 31 < rows ? ra + 31 : rows - 1;
      if (ra >= rows || rb / a.group + off < key0) continue;  // no row sees a key of the wave
      F16x s = {}, dp = {};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        s = mfma(read_rows<DP>(qs, 32 * i, x, n, h), k[x], s);
        dp = mfma(read_rows<DP>(gs, 32 * i, x, n, h), v[x], dp);
      }
      const bool masked = ra / a.group + off < key0 + 31;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * i + 8 * j + 4 * h;
        const float4 ls = *(const float4*)(lses + at), de = *(const float4*)(deltas + at);
        const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dev[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * j + e;
          s[r] = exp2f(fmaf(s[r], c, -lsv[e]));
          dp[r] = s[r] * (dp[r] - dev[e]);
        }
        if (masked) {
          const int4 li = *(const int4*)(limits + at);
          const int liv[4] = {li.x, li.y, li.z, li.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key > liv[e]) s[4 * j + e] = dp[4 * j + e] = 0.0f;
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const V8<T> pr = pack<T>(s, x), ds = pack<T>(dp, x);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          dv[d] = mfma(read_columns<DP>(gs, 32 * i + 16 * x, d, l), pr, dv[d]);
          dk[d] = mfma(read_columns<DP>(qs, 32 * i + 16 * x, d, l), ds, dk[d]);
        }
      }
    }
  }
  const long long at = ((long long)(p.k0 + key) * a.kv_heads + p.kv) * dim;
  store_rows<DP>(valid ? (T*)a.dk + at : nullptr, dim, h, dk, a.scale);
  store_rows<DP>(valid ? (T*)a.dv + at : nullptr, dim, h, dv, 1.0f);
}

// ---- launches -------------------------------------------------------------------------------------------------------

size_t attend_work_bytes(int seqs, int tq, int tk, int group) {
  return sizeof(int) * (ORDER_HEAD + 2 * (size_t)(order_queries(seqs, tq, group) + order_keys(seqs, tk)));
}

template <typename T, int DP>
int attend(hipStream_t st, const Attend& a) {
  const long long blocks = order_queries(a.seqs, a.tq, a.group) * a.kv_heads;
  k_attend<T, DP><<<(unsigned)blocks, 256, 0, st>>>(a);
  return (int)hipGetLastError();
}
template <typename T, int DP>
int attend_vjp(hipStream_t st, const Attend& a) {
  if (a.tq) k_attend_dq<T, DP><<<(unsigned)(order_queries(a.seqs, a.tq, a.group) * a.kv_heads), 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (a.tk) k_attend_dkv<T, DP><<<(unsigned)(order_keys(a.seqs, a.tk) * a.kv_heads), 256, 0, st>>>(a);
  return (int)hipGetLastError();
}

int launch_attend(hipStream_t st, int type, const Attend& a) {
  k_attend_order<<<1, 1024, 0, st>>>(a.seqs, a.tq, a.tk, a.group, a.starts_q, a.starts_k, (int*)a.order);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.tq) return (int)e;
  if (type == BF16) return a.dim <= 64 ? attend<__bf16, 64>(st, a) : attend<__bf16, 128>(st, a);
  return a.dim <= 64 ? attend<_Float16, 64>(st, a) : attend<_Float16, 128>(st, a);
}
int launch_attend_vjp(hipStream_t st, int type, const Attend& a) {
  if (type == BF16) return a.dim <= 64 ? attend_vjp<__bf16, 64>(st, a) : attend_vjp<__bf16, 128>(st, a);
  return a.dim <= 64 ? attend_vjp<_Float16, 64>(st, a) : attend_vjp<_Float16, 128>(st, a);
}

}  // namespace pol

namespace {
// whether the kernels and their grids hold these sizes
bool attention_takes(int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk) {
  if ((type != pol::BF16 && type != pol::F16) || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 128 ||
      dim % 8 || seqs < 0 || tq < 0 || tk < 0 || tk >= 1 << 30 || (long long)tq * (heads / kv_heads) >= 1 << 30)
    return false;
  const long long most = (1LL << 24) - 1;  // workgroups of 256 work-items a launch
  return pol::order_queries(seqs, tq, heads / kv_heads) * kv_heads <= most && pol::order_keys(seqs, tk) * kv_heads <= most;
}
}  // namespace

extern "C" {

int dk_attention(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                 long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v,
                 long long v_t, long long v_h, const int* starts_q, const int* starts_k, float scale, void* out,
                 float* lse, void* work) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || !starts_q || !starts_k || !work ||
      (tq && (!q || !out)) || (tk && (!k || !v)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.out = out, a.lse = lse, a.order = (const int*)work;
  return pol::launch_attend(st, type, a);
}

int dk_attention_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk,
                     const void* q, long long q_t, long long q_h, const void* k, long long k_t, long long k_h,
                     const void* v, long long v_t, long long v_h, const int* starts_q, const int* starts_k,
                     float scale, const void* out, const float* lse, const void* work, const void* dout,
                     long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || !starts_q || !starts_k || !work ||
      (tq && (!q || !out || !lse || !dout || !delta || !dq)) || (tk && (!k || !v || !dk || !dv)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.order = (const int*)work;
  a.out = const_cast<void*>(out), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.do_t = do_t, a.do_h = do_h, a.delta = delta, a.dq = dq, a.dk = dk, a.dv = dv;
  return pol::launch_attend_vjp(st, type, a);
}

long long dk_attention_work_bytes(int heads, int kv_heads, int seqs, int tq, int tk) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || seqs < 0 || tq < 0 || tk < 0) return 0;
  return (long long)pol::attend_work_bytes(seqs, tq, tk, heads / kv_heads);
}

}  // extern "C"
