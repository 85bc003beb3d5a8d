// Causal attention over packed sequences with shared key/value heads: forward and backward.
//
//   S = scale Q K^T, key j <= i + (keys - queries), P = softmax(S), O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta), delta = dO . O a row,  dQ = scale dS K,  dK = scale dS^T Q
//
// A workgroup of four waves takes 128 rows of one key/value head's queries, row = token * group + head, so that the
// heads of a group share each key and value tile and short sequences still fill the rows; a wave takes 32 rows.
//
// What bounds it. A pair of a query and a key costs the forward 4 dim operations in products and one exponential with some ten
// vector instructions beside it, the backward 10 dim (14 with the scores that two kernels compute for themselves) and two
// exponentials. At heads of 64 the vector instructions take longer than the products (a forward's tile of 32 x 32 issues 132
// for its 8 products: 76 % with their issue and 31 % of the SIMDs' cycles; some 72 would do, the rest are register moves,
// addresses and masks): 256 episodes of up to 1000 tokens, 8 heads on 2, forward 250 us (550 TFLOP/s), dq 350, dkv 450 (610
// with what they compute again). At heads of 128 the products lead: 2 sequences of 8192 and 2752 tokens, 16 heads on 4,
// forward 340 us (900 TFLOP/s; a large library product of 16 bits reaches 1200), dq 440, dkv 955. Short sequences are bound
// by their bytes: 4096 segments of up to 32 tokens, 8 heads on 2, forward 56 us (4.0 TB/s), dq 81 (3.8), dkv 60 (4.4).
#include "../../include/nablaengine_policy.h"
#include "policy_attend.h"

namespace pol {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- the order ------------------------------------------------------------------------------------------------------

// One workgroup lists the tiles by a counting sort (a tile's place among equals is free, results do not depend on the
// order). seqs + 1 sequences, LS lanes on each. Sequence lengths are on the GPU only: without the lists each workgroup would
// have to search the offsets for its tile, and the heaviest tiles would not start first (2 sequences of 8192 and 2800
// tokens: 350 us forward for 470). 4 us for a few sequences, 15 for 4096; the backward takes the forward's lists.
__global__ __launch_bounds__(1024) void k_attend_order(int seqs, int tq, int tk, int group, int key_waves, int by_sequence,
                                                       const int* starts_q, const int* starts_k,
                                                       int* __restrict__ order) {
  constexpr int BUCKETS = 1024;
  // Places are unsigned: offsets that fall make sequences overlap, whose tiles together can pass 2^32. A place past the list
  // is not written. Places that wrap fill the list again, so that an entry may mix two of them: place() looks at it.
  __shared__ unsigned count[2][BUCKETS];
  __shared__ unsigned wave_sum[2][16];
  constexpr int STAGED = 8192;  // sequences whose offsets are read to LDS, all at once: the passes below wait for none
  __shared__ int staged[2][STAGED + 1];
  if (seqs <= STAGED) {
    for (int s = threadIdx.x; s <= seqs; s += 1024) staged[0][s] = starts_q[s], staged[1][s] = starts_k[s];
    starts_q = staged[0], starts_k = staged[1];
    __syncthreads();
  }
  int ls = 1;
  if (by_sequence < 3)
    while (ls < 1024 && ls * 2 * (long long)(seqs + 1) <= 1024) ls *= 2;
  const int lane = threadIdx.x % ls, first_seq = threadIdx.x / ls, stride = 1024 / ls;
  const int bits[2] = {7, key_waves == 1 ? 5 : 7};  // of a tile's rows
  static_assert(QROWS == 128, "");
  const unsigned caps[2] = {(unsigned)order_queries(seqs, tq, group), (unsigned)order_keys(seqs, tk, key_waves)};
  int* const lists[2] = {order + ORDER_HEAD, order + ORDER_HEAD + 2LL * caps[0]};
  auto bucket_of = [](int cost) {  // rows or keys of the other side, below 2^30
    const int tiles = cost > 0 ? (int)((unsigned)(cost + TILE - 1) / TILE) : 0;
    return BUCKETS - 1 - (tiles < BUCKETS ? tiles : BUCKETS - 1);
  };
  // f(list, sequence, first tile, tiles, bucket) for every stretch of tiles that stays together; every lane of a wave takes
  // part each time, with 0 tiles where it has none
  auto each = [&](auto f) {
    for (int s0 = 0; s0 <= seqs; s0 += stride) {
      const int s = s0 + first_seq < seqs ? s0 + first_seq : seqs;
      const bool mine = s0 + first_seq <= seqs;
      int q0, k0, nq, nk;
      sequence(starts_q, s, seqs, tq, q0, nq);
      sequence(starts_k, s, seqs, tk, k0, nk);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int mq = which && s == seqs ? 0 : nq, mk = !which && s == seqs ? 0 : nk;
        const int rows = which ? mk : mq * group, tiles = mine ? (rows + (1 << bits[which]) - 1) >> bits[which] : 0;
        auto bucket = [&](int t) {
          int cost;
          if (which) {  // the query rows that see the tile's first key
            const int from = (t << bits[1]) - (mk - mq);
            cost = mq - (from > 0 ? from : 0);
            cost = (cost > 0 ? cost : 0) * group;
          } else {  // the keys that the tile's last row sees
            const int last = ((t + 1) * QROWS < rows ? (t + 1) * QROWS : rows) - 1;
            cost = last / group + mk - mq + 1;
          }
          return bucket_of(cost);
        };
        if (by_sequence >> which & 1) {  // its heaviest tile: the last row sees every key, the first key almost every row
          f(which, s, 0, lane == 0 ? tiles : 0, bucket_of(which ? (mq < mk ? mq : mk) * group : mk));
        } else {
          for (int t = lane; __any(t < tiles); t += ls) f(which, s, t, t < tiles ? 1 : 0, bucket(t));
        }
      }
    }
  };
  // adds n to a bucket's count and returns what it was; lanes that all add to one bucket (short sequences mostly cost the
  // same) add at once: one after another they took half of this kernel's time
  auto add = [&](int which, int n, int b) -> unsigned {
    const unsigned long long some = __ballot(n > 0);
    if (!some) return 0;
    const int lead = uniform(__builtin_ctzll(some)), b0 = __builtin_amdgcn_readlane(b, lead);
    if (!__all(n == 0 || b == b0)) return n ? atomicAdd(&count[which][b], (unsigned)n) : 0;
    const unsigned before = scan_wave((unsigned)n), all = __builtin_amdgcn_readlane(before, 63);
    unsigned base = 0;
    if ((int)threadIdx.x % 64 == lead) base = atomicAdd(&count[which][b0], all);
    return __builtin_amdgcn_readlane(base, lead) + before - (unsigned)n;
  };
  count[0][threadIdx.x] = count[1][threadIdx.x] = 0;
  __syncthreads();
  each([&](int which, int, int, int n, int b) { add(which, n, b); });
  __syncthreads();
  // exclusive prefixes over the buckets
  unsigned mine[2], sum[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    mine[which] = count[which][threadIdx.x];
    sum[which] = scan_wave(mine[which]);
    if (threadIdx.x % 64 == 63) wave_sum[which][threadIdx.x / 64] = sum[which];
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    unsigned before = 0, total = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < (int)threadIdx.x / 64) before += wave_sum[which][w];
      total += wave_sum[which][w];
    }
    count[which][threadIdx.x] = before + sum[which] - mine[which];
    if (threadIdx.x == 0) order[which] = (int)(total < caps[which] ? total : caps[which]);
  }
  __syncthreads();
  each([&](int which, int s, int t, int n, int b) {
    unsigned at = add(which, n, b);
    for (int i = 0; i < n; ++i, ++at)  // the heaviest of the sequence first
      if (at < caps[which]) {
        lists[which][2LL * at] = s;
        lists[which][2LL * at + 1] = t + (which ? i : n - 1 - i);
      }
  });
}

// what a workgroup works on
struct Place {
  int at, tile, kv, part, q0, nq, k0, nk;
};
// entry `at` of a list times its key/value heads
__device__ __forceinline__ bool place(const Attend& a, int which, int at, Place& p) {
  const int entry = at / a.kv_heads;
  if (entry >= uniform(a.order[which])) return false;
  const int* list = a.order + ORDER_HEAD + (which ? 2 * order_queries(a.seqs, a.tq, a.group) : 0) + 2LL * entry;
  const int s = uniform(list[0]);
  p.at = at;
  p.tile = uniform(list[1]);
  p.kv = at % a.kv_heads;
  sequence(a.starts_q, s, a.seqs, a.tq, p.q0, p.nq);
  sequence(a.starts_k, s, a.seqs, a.tk, p.k0, p.nk);
  p.q0 = uniform(p.q0), p.nq = uniform(p.nq), p.k0 = uniform(p.k0), p.nk = uniform(p.nk);
  if (s == a.seqs) (which ? p.nq : p.nk) = 0;
  return which ? p.tile * 32 * a.key_waves < p.nk : p.tile * QROWS < p.nq * a.group;
}
// this workgroup's, of `parts` a tile and key/value head
__device__ __forceinline__ bool place_of_block(const Attend& a, int which, int parts, Place& p) {
  const int b = blockIdx.x;
  int at;
  if (a.by_sequence >> which & 1) {
    const int all = uniform(a.order[which]) * a.kv_heads * parts, base = b / (WINDOW * XCDS) * (WINDOW * XCDS);
    const int left = all - base, mine = left < WINDOW * XCDS ? (left + XCDS - 1) / XCDS : WINDOW, r = b - base;
    if (left <= 0 || r / XCDS >= mine) return false;
    at = base + r % XCDS * mine + r / XCDS;
    p.part = at % parts, at /= parts;
  } else {  // the heavier part first
    const int n = uniform(a.order[which]) * a.kv_heads;
    if (b >= n * parts) return false;
    p.part = parts > 1 ? b / n : 0, at = b - p.part * n;
  }
  return place(a, which, at, p);
}
// workgroups that cover a list of at most `most` tiles
unsigned blocks_of(const Attend& a, long long most, int parts) {
  return (unsigned)((most * a.kv_heads * parts + XCDS - 1) / XCDS * XCDS);
}

// The keys' side of the forward and of the queries' gradient: tiles of TILE keys and their values, one tile ahead.
template <int DP, typename T>
struct Keys {
  static constexpr int CH = DP / 8, STEP = 256 / CH, N = TILE / STEP;  // chunks a row; rows a turn of the workgroup
  const T *k, *v;  // this thread's chunk of the tile's first rows
  long long k_t, v_t;
  int row, at, left;  // this thread's row; its wave's place in LDS; keys from the tile's first on
  bool in_row;
  __device__ __forceinline__ Keys(const Attend& a, const Place& p, int first) {  // from tile `first` on
    row = threadIdx.x / CH;
    const int c = threadIdx.x % CH ^ swizzle<DP>(row);  // LDS is filled in order: the swizzle is the source's
    in_row = 8 * c < a.dim;
    k_t = a.k_t, v_t = a.v_t;
    k = (const T*)a.k + (long long)(p.k0 + first * TILE) * k_t + (long long)p.kv * a.k_h + row * k_t + 8 * c;
    v = (const T*)a.v + (long long)(p.k0 + first * TILE) * v_t + (long long)p.kv * a.v_h + row * v_t + 8 * c;
    at = threadIdx.x / 64 * 64 * 8;
    left = p.nk - first * TILE;
  }
  __device__ __forceinline__ void next(T* ks, T* vs) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool valid = in_row && row + i * STEP < left;
      to_lds(k + i * STEP * k_t, valid, ks + i * 2048 + at);
      to_lds(v + i * STEP * v_t, valid, vs + i * 2048 + at);
    }
    k += TILE * k_t;
    v += TILE * v_t;
    left -= TILE;
  }
};

// The rows' side: a wave's 32 query rows of a workgroup's 128
struct Rows {
  int pos, head, limit, all_see, any_sees, tiles;
  bool valid;
  __device__ __forceinline__ Rows(const Attend& a, const Place& p, int w) {
    const int rows = p.nq * a.group, off = p.nk - p.nq;
    const int row0 = p.tile * QROWS + 32 * w, row = row0 + threadIdx.x % 32;
    valid = row < rows;
    pos = row / a.group;
    head = p.kv * a.group + row % a.group;
    limit = valid ? pos + off : -1;  // the row's last key (below 0: none)
    // of the wave's rows: the last key that all see, and the last that any sees; the workgroup's tiles of keys
    all_see = row0 < rows ? row0 / a.group + off : -1;
    any_sees = row0 < rows ? (row0 + 31 < rows ? row0 + 31 : rows - 1) / a.group + off : -1;
    const int end = p.tile * QROWS + QROWS < rows ? p.tile * QROWS + QROWS : rows, last = (end - 1) / a.group + off;
    tiles = last < 0 ? 0 : last / TILE + 1;
  }
};

// one row of a wave's 32, for all its lanes
struct Sight {
  long long token, head;
  int limit;
  __device__ __forceinline__ Sight(const Attend& a, const Place& p, const Rows& r, int n) {
    token = p.q0 + __builtin_amdgcn_readlane(r.pos, n);
    head = __builtin_amdgcn_readlane(r.head, n);
    limit = __builtin_amdgcn_readlane(r.limit, n);
  }
};

// ---- forward --------------------------------------------------------------------------------------------------------

// One pass over the keys with the running maximum and sum of the softmax, both in float32. The next tile of keys and values is
// sent for before the products of this one, and one barrier a tile orders both. The two buffers are one array, in which the
// compiler cannot tell them apart: it waits for the load before this tile's first operand is read. What covers a load is the
// work of the other workgroups, two a CU (four at heads of 64). Holding a tile's operands in registers one phase ahead cost a workgroup of them
// (258 us to 283, heads of 64). The probabilities are rounded to 16 bits for the second product, as the values are; the sum
// they are divided by is that of the unrounded ones, which the backward needs.

// What a tile's parts hand to the join, in the order of the registers: each lane's N sums, and for N + 2 a row's maximum and
// its sum of probabilities.
template <int N>
struct Part {
  static constexpr size_t SIZE = 256 * N;  // floats of a slot: four waves
  float* at;
  __device__ __forceinline__ Part(const Attend& a, size_t slot, int wave) {
    at = a.scratch + slot * SIZE + wave * 64 * N + threadIdx.x % 64;
  }
  __device__ __forceinline__ void put(int first, const F16x* acc, int n) const {
#pragma unroll
    for (int i = 0; i < n; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) at[64 * (16 * (first + i) + j)] = acc[i][j];
  }
};
template <int DP>
using RowsPart = Part<DP / 2 + 2>;
// One block of the join: 32 rows (keys) and 32 of their elements. Its four waves take every fourth part, f(part) times it,
// and wave 0 gets the sum of all.
template <int N, typename F>
__device__ __forceinline__ F16x add_parts(const Attend& a, size_t slot, int parts, int wave, int block, F f) {
  __shared__ float sums[3][16][64];
  const int w = uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  F16x acc = {};
#pragma unroll 4
  for (int i = w; i < parts; i += 4) {
    const float* from = Part<N>(a, slot + i, wave).at + 64 * 16 * block;
    const float times = f(i);
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = fmaf(times, from[64 * j], acc[j]);
  }
  if (w)
#pragma unroll
    for (int j = 0; j < 16; ++j) sums[w - 1][j][l] = acc[j];
  __syncthreads();
  if (!w)
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[j] += sums[o][j][l];
  return acc;
}

// what a wave's rows come to, from their outputs' sums, the maximum that these lack and the probabilities' sum: zeros where
// a row sees no key, NaN where every score it sees is -inf (0 / 0, as the softmax's definition has it)
template <typename T, int DP, int N>
__device__ __forceinline__ void finish_rows(const Attend& a, const Place& p, const Rows& r, int d0, const F16x* acc, float m,
                                            float sum) {
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const float c = a.scale * LOG2E;
  const long long token = p.q0 + r.pos;
  if (a.lse && r.valid && h == 0 && d0 == 0)
    a.lse[(long long)r.head * a.tq + token] = r.limit < 0 ? INFINITY : m * c + (log2f(sum) - Range<T>::LIFT);
  const unsigned bad = bad_columns(r.valid && not_finite<N>(acc) != 0.0f);
  store_rows<N>(r.valid && !(bad >> n & 1) ? (T*)a.out + (token * a.heads + r.head) * dim : nullptr, d0, dim, h, acc,
                r.limit < 0 ? 0.0f : 1.0f / sum);
  for (unsigned left = bad; left; left &= left - 1) {
    const Sight one(a, p, r, __builtin_ctz(left));
    const Row<DP> qr((const T*)a.q + one.token * a.q_t + one.head * a.q_h, dim);
    Row<DP> o = {};
    float top = -INFINITY, total = 0.0f;
    for (int j = 0; j <= one.limit && total == total; ++j) {
      const float x = qr.dot(Row<DP>((const T*)a.k + (p.k0 + j) * a.k_t + p.kv * a.k_h, dim)) * c, top1 = fmaxf(top, x);
      const float base1 = top1 == -INFINITY ? 0.0f : top1, f = exp2_fast(top - base1), pr = exp2_fast(x - base1);
      total = total * f + pr;
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) o.x[i] *= f;
      o.add(pr, Row<DP>((const T*)a.v + (p.k0 + j) * a.v_t + p.kv * a.v_h, dim));
      top = top1;
    }
    o.store((T*)a.out + (one.token * a.heads + one.head) * dim, d0, d0 + 32 * N < dim ? d0 + 32 * N : dim,
            one.limit < 0 ? 0.0f : 1.0f / total);
  }
}

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(256, 2) void k_attend(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[2][TILE * DP];
  __shared__ __align__(16) T vs[2][TILE * DP];
  Place p;
  if (!place_of_block(a, 0, SPLIT ? a.parts_q : 1, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const Rows r(a, p, uniform(threadIdx.x / 64));
  const Slice my(r.tiles, SPLIT ? a.parts_q : 1, SPLIT ? p.part : 0);
  const int first = SPLIT ? my.first : 0, end = SPLIT ? my.end : r.tiles;
  if (SPLIT && p.part >= my.parts) return;
  Keys<DP, T> keys(a, p, first);
  if (first < end) keys.next(ks[first & 1], vs[first & 1]);
  V8<T> q[KS];
  load_rows<DP>(r.valid ? (const T*)a.q + (long long)(p.q0 + r.pos) * a.q_t + (long long)r.head * a.q_h : nullptr, dim, h,
                q);
  F16x acc[DT] = {};
  float m = -INFINITY, sum = 0.0f;
  const float c = a.scale * LOG2E;
  for (int t = first; t < end; ++t) {
    const int key0 = t * TILE;
    const T *kt = ks[t & 1], *vt = vs[t & 1];
    loads_done();
    __syncthreads();  // this tile is there for all, and all are done with the one before
    if (t + 1 < end) keys.next(ks[(t + 1) & 1], vs[(t + 1) & 1]);
    if (key0 > r.any_sees) continue;
    const bool second = key0 + 32 <= r.any_sees;
    F16x s[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !second) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[1][j] = -INFINITY;
        break;
      }
#pragma unroll
      for (int x = 0; x < KS; ++x) s[i] = mfma(read_rows<DP>(kt, 32 * i, x, n, h), q[x], s[i]);
      if (key0 + 32 * i + 31 > r.all_see)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (key0 + 32 * i + j % 4 + 8 * (j / 4) + 4 * h > r.limit) s[i][j] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, s[0][j]);
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, s[1][j]);
    top = max_halves(top);
    // The subtracted maximum may lag behind the true one by 2^SLACK: sums and products stay far inside float32 and the
    // probabilities, at most 2^(SLACK + LIFT), inside float16; the quotient at the end is the same. The outputs are then
    // hardly ever rescaled.
    if (__any(top * c > m * c + Range<T>::SLACK)) {
      const float m1 = fmaxf(m, top), f = m == -INFINITY ? 0.0f : exp2_fast((m - m1) * c);
      sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[d][j] *= f;
      m = m1;
    }
    const float base = (m == -INFINITY ? 0.0f : m * c) - Range<T>::LIFT;  // 0: a row that has seen no key yet
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        s[i][j] = exp2_fast(fmaf(s[i][j], c, -base));
        sum += s[i][j];
      }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x == 2 && !second) break;
      const V8<T> pr = pack<T>(s[x / 2], x % 2);
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = mfma(read_columns<DP>(vt, 16 * x, d, l), pr, acc[d]);
    }
  }
  sum = add_halves(sum);
  if (SPLIT && my.parts > 1) {
    const RowsPart<DP> mine(a, (size_t)p.at * a.parts_q + p.part, uniform(threadIdx.x / 64));
    mine.put(0, acc, DT);
    mine.at[64 * 16 * DT] = m, mine.at[64 * (16 * DT + 1)] = sum;
    return;
  }
  finish_rows<T, DP, DT>(a, p, r, 0, acc, m, sum);
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attend_join(Attend a) {
  constexpr int DT = DP / 32, N = DP / 2 + 2;
  const int wave = blockIdx.y / DT, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 0, 1, p)) return;
  const Rows r(a, p, wave);
  const int parts = Slice(r.tiles, a.parts_q, 0).parts;
  if (parts == 1) return;
  const size_t slot = (size_t)p.at * a.parts_q;
  auto stat = [&](int part, int which) { return Part<N>(a, slot + part, wave).at[64 * (N - 2 + which)]; };
  const float c = a.scale * LOG2E;
  float m = -INFINITY, sum = 0.0f;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) m = fmaxf(m, stat(i, 0));
  const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) sum += exp2_fast((stat(i, 0) - base) * c) * stat(i, 1);
  const F16x acc = add_parts<N>(a, slot, parts, wave, block, [&](int i) { return exp2_fast((stat(i, 0) - base) * c); });
  if (threadIdx.x < 64) finish_rows<T, DP, 1>(a, p, r, 32 * block, &acc, m, sum);
}

// ---- backward: the queries' gradient --------------------------------------------------------------------------------

// The forward's walk with the stored log-sum: P and dP a tile from two products over the same keys, dS rounded to 16 bits for
// the third. Both gradients from one kernel would need atomics on dq, whose order changes results from run to run, or a
// buffer of float32 a key tile: dq has a kernel of its own, at two products of seven computed again.

template <typename T, int DP, int N>
__device__ __forceinline__ void finish_dq(const Attend& a, const Place& p, const Rows& r, int d0, const F16x* acc, float lse,
                                          float delta) {
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const float c = a.scale * LOG2E;
  const long long token = p.q0 + r.pos;
  const unsigned bad = bad_columns(r.valid && not_finite<N>(acc) != 0.0f);
  store_rows<N>(r.valid && !(bad >> n & 1) ? (T*)a.dq + (token * a.heads + r.head) * dim : nullptr, d0, dim, h, acc,
                a.scale);
  for (unsigned left = bad; left; left &= left - 1) {
    const int i = __builtin_ctz(left);
    const Sight one(a, p, r, i);
    const Row<DP> qr((const T*)a.q + one.token * a.q_t + one.head * a.q_h, dim);
    const Row<DP> gr((const T*)a.dout + one.token * a.do_t + one.head * a.do_h, dim);
    const float lse1 = __shfl(lse, i), delta1 = __shfl(delta, i);
    Row<DP> o = {};
    for (int j = 0; j <= one.limit && !o.all_nan(dim); ++j) {
      const Row<DP> kr((const T*)a.k + (p.k0 + j) * a.k_t + p.kv * a.k_h, dim);
      const float dp = gr.dot(Row<DP>((const T*)a.v + (p.k0 + j) * a.v_t + p.kv * a.v_h, dim));
      o.add(exp2_fast(qr.dot(kr) * c - lse1) * (dp - delta1), kr);
    }
    o.store((T*)a.dq + (one.token * a.heads + one.head) * dim, d0, d0 + 32 * N < dim ? d0 + 32 * N : dim, a.scale);
  }
}

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(256, 2) void k_attend_dq(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[2][TILE * DP];
  __shared__ __align__(16) T vs[2][TILE * DP];
  Place p;
  if (!place_of_block(a, 0, SPLIT ? a.parts_q : 1, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const Rows r(a, p, uniform(threadIdx.x / 64));
  const Slice my(r.tiles, SPLIT ? a.parts_q : 1, SPLIT ? p.part : 0);
  const int first = SPLIT ? my.first : 0, end = SPLIT ? my.end : r.tiles;
  if (SPLIT && p.part >= my.parts) return;
  Keys<DP, T> keys(a, p, first);
  if (first < end) keys.next(ks[first & 1], vs[first & 1]);
  const long long token = p.q0 + r.pos;
  V8<T> q[KS], g[KS];
  load_rows<DP>(r.valid ? (const T*)a.q + token * a.q_t + (long long)r.head * a.q_h : nullptr, dim, h, q);
  load_rows<DP>(r.valid ? (const T*)a.dout + token * a.do_t + (long long)r.head * a.do_h : nullptr, dim, h, g);
  const float lse = r.valid ? a.lse[(long long)r.head * a.tq + token] : INFINITY;
  const float c = a.scale * LOG2E;
  // the row's 32 scores and dP of subtile i; masked probabilities are 0
  auto products = [&](const T* kt, const T* vt, int key0, int i, F16x& s, F16x& dp) {
    s = F16x{}, dp = F16x{};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      s = mfma(read_rows<DP>(kt, 32 * i, x, n, h), q[x], s);
      dp = mfma(read_rows<DP>(vt, 32 * i, x, n, h), g[x], dp);
    }
    if (key0 + 32 * i + 31 > r.all_see)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (key0 + 32 * i + j % 4 + 8 * (j / 4) + 4 * h > r.limit) s[j] = -INFINITY, dp[j] = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = exp2_fast(fmaf(s[j], c, -lse));
  };
  // delta = dout . out from the stored output, whose rounding is felt where few keys share a row: rows whose keys all
  // lie in the first tile take it from that tile's products instead, sum P dP in float32, below
  float delta = 0.0f;
  const bool few = r.any_sees < TILE;
  if (!few) {
    V8<T> o[KS];
    load_rows<DP>(r.valid ? (const T*)a.out + (token * a.heads + r.head) * dim : nullptr, dim, h, o);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)o[s][e] * (float)g[s][e];
    delta = add_halves(delta);
  }
  F16x acc[DT] = {};
  Lift<T> lift;
  for (int t = first; t < end; ++t) {
    const int key0 = t * TILE;
    const T *kt = ks[t & 1], *vt = vs[t & 1];
    loads_done();
    __syncthreads();
    if (t + 1 < end) keys.next(ks[(t + 1) & 1], vs[(t + 1) & 1]);
    if (t == 0 && few) {
#pragma unroll 1
      for (int i = 0; 32 * i <= r.any_sees; ++i) {
        F16x s, dp;
        products(kt, vt, 0, i, s, dp);
#pragma unroll
        for (int j = 0; j < 16; ++j) delta += s[j] * dp[j];
      }
      delta = add_halves(delta);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (key0 + 32 * i > r.any_sees) break;
      F16x s, dp;
      products(kt, vt, key0, i, s, dp);
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] *= dp[j] - delta;
      lift.template scale<DT>(s, acc);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const V8<T> ds = pack<T>(s, x);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = mfma(read_columns<DP>(kt, 32 * i + 16 * x, d, l), ds, acc[d]);
      }
    }
  }
  lift.template unscale<DT>(acc, 1.0f);
  if (r.valid && h == 0 && (!SPLIT || p.part == 0)) a.delta[(long long)r.head * a.tq + token] = delta;
  if (SPLIT && my.parts > 1) {
    RowsPart<DP>(a, (size_t)p.at * a.parts_q + p.part, uniform(threadIdx.x / 64)).put(0, acc, DT);
    return;
  }
  finish_dq<T, DP, DT>(a, p, r, 0, acc, lse, delta);
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attend_dq_join(Attend a) {
  constexpr int DT = DP / 32;
  const int wave = blockIdx.y / DT, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 0, 1, p)) return;
  const Rows r(a, p, wave);
  const int parts = Slice(r.tiles, a.parts_q, 0).parts;
  if (parts == 1) return;
  const F16x acc =
      add_parts<DP / 2 + 2>(a, (size_t)p.at * a.parts_q, parts, wave, block, [](int) { return 1.0f; });
  const long long at = (long long)r.head * a.tq + p.q0 + r.pos;
  if (threadIdx.x < 64)
    finish_dq<T, DP, 1>(a, p, r, 32 * block, &acc, r.valid ? a.lse[at] : INFINITY, r.valid ? a.delta[at] : 0.0f);
}

// ---- backward: the keys' and values' gradients ----------------------------------------------------------------------

// Gradients of shared heads add up in the same sums, since the rows of a key/value head's whole group pass by.
// A wave keeps 32 keys and their values as B operands and walks over the rows that see them; rows lie in LDS, RT at a
// time. S = Q K^T here, so that a lane holds 16 rows of ONE key and P, dS are the B operands of dV^T = dO^T P and dK^T =
// Q^T dS. KW of the waves differ in their keys, the others take every SPLIT-th subtile of 32 rows of the same keys, and
// their sums are added at the end, in order.
template <typename T, int DP, int WAVES>
struct DkvTiles {
  static constexpr int RT = WAVES == 1 ? 32 : DP == 64 ? 64 : 128;
  alignas(16) T tiles[2][2][RT * DP];  // (turn, q or dout)
  alignas(16) float lses[2][RT], deltas[2][RT];
  alignas(16) int places_of[2][RT];  // a row's token from its tile's first
};
// Heads of 128: dk and dv together take 128 registers a lane, with the keys and values more than two waves a SIMD have.
// One workgroup takes dk and another dv (a fourth more products, the scores twice): 1150 us at sequences of 8192 and 2800
// tokens of 16 heads on 4 against 1480 us with both in one and part of the operands in LDS or scratch, and 1230 us with one
// wave a SIMD. Eight waves share a tile of 128 rows, 995 us: twice the products a byte read. Their waves run their products
// at a higher priority than another's exponentials, 955 us; at heads of 64, where those are the longer part, that gains
// nothing (forward 249 us to 260). The wait for the next tile's load stands between the first products and the column
// operands here; the eight waves fill a CU's LDS, so that no other workgroup covers it.
enum Role { BOTH, KEYS, VALUES };
struct RowTiles {  // the rows that see a key tile, in tiles of RT rows or a little less
  int used, first, tiles;
  __device__ __forceinline__ RowTiles(const Attend& a, const Place& p, int kw, int rt) {
    used = a.group <= rt ? rt / a.group * a.group : rt;
    const int rows = p.nq * a.group;
    const int from = p.tile * 32 * kw - (p.nk - p.nq);  // the first token that sees the tile's first key
    first = (from > 0 ? from : 0) * a.group;
    tiles = rows > first ? (rows - 1 - first) / used + 1 : 0;
  }
};
// a key tile's part: dk and dv of its 32 keys a wave in turn (heads of 64), or one of them
constexpr int KEY_PART = 64;
__device__ __forceinline__ size_t key_slot(const Attend& a, const Place& p, int role) {
  return ((size_t)p.at * (role == BOTH ? 1 : 2) + (role == VALUES)) * a.parts_k;
}
template <typename T, int DP, int N, int ROLE>
__device__ __forceinline__ void finish_dkv(const Attend& a, const Place& p, int key0, int d0, const F16x* dk, const F16x* dv) {
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim, group = a.group;
  const int rows = p.nq * group, off = p.nk - p.nq, key = key0 + n;
  const bool valid = key < p.nk;
  const float c = a.scale * LOG2E;
  const float off_dv = ROLE != KEYS ? not_finite<N>(dv) : 0.0f, off_dk = ROLE != VALUES ? not_finite<N>(dk) : 0.0f;
  const unsigned bad = bad_columns(valid && off_dv + off_dk != 0.0f);
  const bool put = valid && !(bad >> n & 1);
  const long long at = ((long long)(p.k0 + key) * a.kv_heads + p.kv) * dim;
  if (ROLE != VALUES) store_rows<N>(put ? (T*)a.dk + at : nullptr, d0, dim, h, dk, a.scale);
  if (ROLE != KEYS) store_rows<N>(put ? (T*)a.dv + at : nullptr, d0, dim, h, dv, 1.0f);
  for (unsigned left = bad; left; left &= left - 1) {
    const int one = key0 + __builtin_ctz(left);
    const Row<DP> kr((const T*)a.k + (long long)(p.k0 + one) * a.k_t + p.kv * a.k_h, dim);
    const Row<DP> vr((const T*)a.v + (long long)(p.k0 + one) * a.v_t + p.kv * a.v_h, dim);
    Row<DP> ok = {}, ov = {};
    for (int r = (one - off > 0 ? one - off : 0) * group;
         r < rows && !((ROLE == VALUES || ok.all_nan(dim)) && (ROLE == KEYS || ov.all_nan(dim))); ++r) {
      const long long token = p.q0 + r / group, head = p.kv * group + r % group;
      const Row<DP> qr((const T*)a.q + token * a.q_t + head * a.q_h, dim);
      const Row<DP> gr((const T*)a.dout + token * a.do_t + head * a.do_h, dim);
      const float pr = exp2_fast(qr.dot(kr) * c - a.lse[head * a.tq + token]);
      if (ROLE != KEYS) ov.add(pr, gr);
      if (ROLE != VALUES) ok.add(pr * (gr.dot(vr) - a.delta[head * a.tq + token]), qr);
    }
    const long long to = ((long long)(p.k0 + one) * a.kv_heads + p.kv) * dim;
    const int d1 = d0 + 32 * N < dim ? d0 + 32 * N : dim;
    if (ROLE != VALUES) ok.store((T*)a.dk + to, d0, d1, a.scale);
    if (ROLE != KEYS) ov.store((T*)a.dv + to, d0, d1, 1.0f);
  }
}
template <typename T, int DP, int KW, int WAVES, int ROLE, bool PARTS>
__device__ __forceinline__ void dkv_tile(const Attend& a, const Place& p, DkvTiles<T, DP, WAVES>& lds) {
  constexpr int RT = DkvTiles<T, DP, WAVES>::RT;
  constexpr int KS = DP / 16, DT = DP / 32, CH = DP / 8, STEP = 64 * WAVES / CH, SPLIT = WAVES / KW;
  // of a subtile's two column operands, those read during the exponentials (heads of 128 in parts: none, no register is left)
  constexpr int AHEAD = DP == 64 ? 2 : !PARTS ? 1 : 0;
  constexpr int SUB = RT / 32, N = RT / STEP;
  auto& tiles = lds.tiles;
  auto &lses = lds.lses, &deltas = lds.deltas;
  auto& places_of = lds.places_of;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim, group = a.group;
  const int tid = threadIdx.x % (64 * WAVES), w = uniform(tid / 64);
  auto meet = [] {  // the waves of the tile; one alone only keeps its own LDS accesses in order
    if constexpr (WAVES > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  const int kw = w % KW, split = w / KW;
  const int rows = p.nq * group, off = p.nk - p.nq;
  const int key0 = p.tile * 32 * KW + 32 * kw, key = key0 + n;
  const bool valid = key < p.nk;
  const float c = a.scale * LOG2E;

  // Row tiles start at whole tokens (but for groups above RT, whose rows' places are computed anew for each tile), so
  // that a thread's rows keep their distance from the tile's first token: RT or a little less rows are used of each.
  const RowTiles all(a, p, KW, RT);
  const int used = all.used, first = all.first, back = used / group;  // back: tokens of a tile
  auto chunk = [&](int i) { return tid % CH ^ swizzle<DP>(tid / CH + i * STEP); };
  const T *qp[N], *gp[N];  // this thread's rows of the next tile to load, and its row's place in lse and delta
  long long stat = 0;
  auto places = [&](int r0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r0 + tid / CH + i * STEP, pos = r / group, head = p.kv * group + r % group;
      qp[i] = (const T*)a.q + (long long)(p.q0 + pos) * a.q_t + (long long)head * a.q_h + 8 * chunk(i);
      gp[i] = (const T*)a.dout + (long long)(p.q0 + pos) * a.do_t + (long long)head * a.do_h + 8 * chunk(i);
    }
    const int r = r0 + tid;
    stat = (long long)(p.kv * group + r % group) * a.tq + p.q0 + r / group;
  };
  float lse = INFINITY, delta = 0.0f;
  auto load = [&](int r0, int turn) {  // the rows from r0, then the places of those before them
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = tid / CH + i * STEP;
      const bool there = 8 * chunk(i) < dim && row < used && r0 + row < rows;
      to_lds(qp[i], there, tiles[turn][0] + (i * WAVES + w) * 512);
      to_lds(gp[i], there, tiles[turn][1] + (i * WAVES + w) * 512);
    }
    if (tid < RT) {
      const bool there = tid < used && r0 + tid < rows;
      lse = there ? a.lse[stat] - Range<T>::LIFT_BACK : INFINITY;
      if (ROLE != VALUES) delta = there ? a.delta[stat] : 0.0f;
    }
    if (group > RT) {
      if (r0 >= used) places(r0 - used);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) qp[i] -= back * a.q_t, gp[i] -= back * a.do_t;
      stat -= back;
    }
  };
  // From the last rows, which every key tile of the sequence reads, to the tile's first: workgroups that run side by
  // side then read the same rows at about the same time, from the L2 cache of their XCD.
  const Slice my(all.tiles, PARTS ? a.parts_k : 1, PARTS ? p.part % a.parts_k : 0);
  const int start = first + (all.tiles - 1 - (PARTS ? my.first : 0)) * used;
  const int last = PARTS ? first + (all.tiles - my.end) * used : first;
  if (PARTS && p.part % a.parts_k >= my.parts) return;
  places(start >= last ? start : 0);
  if (start >= last) load(start, 0);
  V8<T> k[KS], v[KS];
  load_rows<DP>(valid ? (const T*)a.k + (long long)(p.k0 + key) * a.k_t + (long long)p.kv * a.k_h : nullptr, dim, h, k);
  if (ROLE != VALUES)
    load_rows<DP>(valid ? (const T*)a.v + (long long)(p.k0 + key) * a.v_t + (long long)p.kv * a.v_h : nullptr, dim, h, v);
  F16x dk[DT] = {}, dv[DT] = {};
  Lift<T> lift;
  if (tid < RT && group <= RT) places_of[0][tid] = places_of[1][tid] = tid / group;
  // tokens from a tile's first to those of a subtile's first row and, at most, its last: x / group for x < RT as a product
  const int inverse = 65535 / group + 1;
  auto tokens = [&](int x) { return x * inverse >> 16; };
  int turn = 0, sub0 = 0, token0 = start / group;
  for (int r0 = start; r0 >= last; r0 -= used, turn ^= 1, sub0 += SUB) {
    if (tid < RT) {
      lses[turn][tid] = lse;
      deltas[turn][tid] = delta;
      if (group > RT) places_of[turn][tid] = (r0 % group + tid) / group;
    }
    loads_done();
    meet();
    if (r0 - used >= last) load(r0 - used, turn ^ 1);
    if (key0 >= p.nk) continue;
    const int token = group <= RT ? token0 : r0 / group;
    token0 -= back;
    const T *qt = tiles[turn][0], *gt = tiles[turn][1];
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      if (SPLIT > 1 && (sub0 + i) % SPLIT != split) continue;
      // the last keys that the subtile's first row and (at most) its last one see
      const int low = token + (group <= RT ? tokens(32 * i) : 0) + off;
      const int most = token + (group <= RT ? tokens(32 * i + 31 < used ? 32 * i + 31 : used - 1) : 1) + off;
      if (32 * i >= used || r0 + 32 * i >= rows || most < key0) continue;
      F16x s = {}, dp = {};
#pragma unroll
      for (int y = 0; y < KS; y += 4) {
        V8<T> qr[4], gr[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          qr[x] = read_rows<DP>(qt, 32 * i, y + x, n, h);
          if (ROLE != VALUES) gr[x] = read_rows<DP>(gt, 32 * i, y + x, n, h);
        }
        phase();
        if (WAVES == 8) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          s = mfma(qr[x], k[y + x], s);
          if (ROLE != VALUES) dp = mfma(gr[x], v[y + x], dp);
        }
      }
      if (WAVES == 8) __builtin_amdgcn_s_setprio(0);
      V8<T> qc[2][DT], gc[2][DT];  // on their way during the exponentials
#pragma unroll
      for (int x = 0; x < AHEAD; ++x)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (ROLE != KEYS) gc[x][d] = read_columns<DP>(gt, 32 * i + 16 * x, d, l);
          if (ROLE != VALUES) qc[x][d] = read_columns<DP>(qt, 32 * i + 16 * x, d, l);
        }
      phase();
      const bool masked = low < key0 + 31;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * i + 8 * j + 4 * h;
        typedef float F4 __attribute__((ext_vector_type(4)));
        typedef int I4 __attribute__((ext_vector_type(4)));
        const F4 ls = *(const F4*)(lses[turn] + at), de = *(const F4*)(deltas[turn] + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * j + e] = exp2_fast(fmaf(s[4 * j + e], c, -ls[e]));
          if (ROLE != VALUES) dp[4 * j + e] = s[4 * j + e] * (dp[4 * j + e] - de[e]);
        }
        if (masked) {
          const I4 li = *(const I4*)(places_of[turn] + at) + (token + off);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key > li[e]) s[4 * j + e] = dp[4 * j + e] = 0.0f;
        }
      }
      if (ROLE != VALUES) lift.template scale<DT>(dp, dk);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const V8<T> pr = pack<T>(s, x), ds = pack<T>(dp, x);
        if (WAVES == 8) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (ROLE != KEYS) dv[d] = mfma(x < AHEAD ? gc[x][d] : read_columns<DP>(gt, 32 * i + 16 * x, d, l), pr, dv[d]);
          if (ROLE != VALUES) dk[d] = mfma(x < AHEAD ? qc[x][d] : read_columns<DP>(qt, 32 * i + 16 * x, d, l), ds, dk[d]);
        }
        if (WAVES == 8) __builtin_amdgcn_s_setprio(0);
      }
    }
  }
  if (Range<T>::LIFT_BACK != 0.0f) {
    constexpr float back = 1.0f / (1 << (int)Range<T>::LIFT_BACK);
    if (ROLE != VALUES) lift.template unscale<DT>(dk, back);
    if (ROLE != KEYS)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) dv[d][j] *= back;
  }
  // the waves of the same keys: split 0 adds the others' sums, one after another
  if constexpr (SPLIT > 1) {
    float* mine = (float*)&tiles[0][0][0];  // (KW, 16 DT, 64) a turn: dk, then dv; within the tiles
    static_assert(sizeof(tiles) >= sizeof(float) * KW * 16 * DT * 64, "");
#pragma unroll
    for (int o = 1; o < SPLIT; ++o)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if (ROLE == (which ? KEYS : VALUES)) continue;
        F16x* acc = which ? dv : dk;
        meet();
        if (split == o)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 16; ++j) mine[((kw * DT + d) * 16 + j) * 64 + l] = acc[d][j];
        meet();
        if (split == 0)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[d][j] += mine[((kw * DT + d) * 16 + j) * 64 + l];
      }
    if (split) return;
  }
  if (PARTS && my.parts > 1) {
    const Part<KEY_PART> mine(a, key_slot(a, p, ROLE) + p.part % a.parts_k, w);
    if (ROLE != VALUES) mine.put(0, dk, DT);
    if (ROLE != KEYS) mine.put(ROLE == BOTH ? DT : 0, dv, DT);
    return;
  }
  finish_dkv<T, DP, DT, ROLE>(a, p, key0, 0, dk, dv);
}

template <typename T, int DP, int KW, int WAVES, bool PARTS>
__global__ __launch_bounds__(WAVES == 8 ? 512 : 256) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_attend_dkv(Attend a) {
  __shared__ DkvTiles<T, DP, WAVES> lds[WAVES == 1 ? 4 : 1];
  const int parts = PARTS ? a.parts_k : 1;
  Place p;
  if constexpr (WAVES == 1) {  // each wave a tile of its own
    const int w = uniform(threadIdx.x / 64);
    if (place(a, 1, blockIdx.x * 4 + w, p)) dkv_tile<T, DP, KW, WAVES, BOTH, false>(a, p, lds[w]);
  } else if constexpr (DP == 64) {
    if (place_of_block(a, 1, parts, p)) dkv_tile<T, DP, KW, WAVES, BOTH, PARTS>(a, p, lds[0]);
  } else {
    if (!place_of_block(a, 1, 2 * parts, p)) return;
    if (p.part >= parts) dkv_tile<T, DP, KW, WAVES, VALUES, PARTS>(a, p, lds[0]);
    else dkv_tile<T, DP, KW, WAVES, KEYS, PARTS>(a, p, lds[0]);
  }
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attend_dkv_join(Attend a) {
  constexpr int DT = DP / 32;
  const int role = blockIdx.y / (4 * DT) ? VALUES : KEYS, wave = blockIdx.y / DT % 4, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 1, 1, p)) return;
  const int parts = Slice(RowTiles(a, p, 4, DkvTiles<T, DP, DP / 16>::RT).tiles, a.parts_k, 0).parts;
  if (parts == 1) return;
  const F16x acc = add_parts<KEY_PART>(a, key_slot(a, p, DP == 64 ? BOTH : role), parts, wave,
                                       (DP == 64 && role == VALUES ? DT : 0) + block, [](int) { return 1.0f; });
  if (threadIdx.x >= 64) return;
  const int key0 = p.tile * 128 + wave * 32;
  if (role == KEYS) finish_dkv<T, DP, 1, KEYS>(a, p, key0, 32 * block, &acc, nullptr);
  else finish_dkv<T, DP, 1, VALUES>(a, p, key0, 32 * block, nullptr, &acc);
}

// ---- launches -------------------------------------------------------------------------------------------------------

// Keys a tile of the keys' gradients: 128; 32, a wave each, where sequences are short and heads up to 64, since most of a
// workgroup's waves would have no keys there. Backward of 65536 tokens of 8 heads on 2, lengths 1 to twice the mean, alone
// and together: mean 16 113 and 157 us, 32 105 and 125, 64 115 and 123, 96 120 and 146 (all of 96: 107 and 111; all of 128:
// 121 and 114). Heads of 128 gain nothing from tiles of 64 keys (mean 32 445 us for 434, 64 413 for 363).
int key_waves(int dim, int seqs, int tk) { return dim <= 64 && tk <= 96LL * seqs ? 1 : 4; }

// The lists in the order of the sequences: bit 0 the query tiles, bit 1 the key tiles. 131072 tokens of 8 heads on 2, by
// sequence and singly: heads of 64, mean length 100, forward 97 and 102 us, dq 136 and 141, dkv 183 and 135; 700, 194 and 206,
// 265 and 272, 389 and 353; 1500, 297 and 308, 388 and 405, 654 and 574; heads of 128, 700, 358 and 394, 470 and 498, 929
// and 1038; 1500, 544 and 618, 711 and 768, 1540 and 1617. 65536 tokens, mean 2048, heads of 64: forward 220 and 196, all of
// the backward 800 and 605; of 128, 401 and 372, 1559 and 1470. A wave alone has no neighbours: the shorter listing.
int by_sequence(int dim, int seqs, int tq, int tk) {
  const bool queries = (tq > tk ? tq : tk) <= (long long)LONG * seqs;
  const bool keys = key_waves(dim, seqs, tk) == 1 || (dim > 64 && queries);
  return (queries ? 1 : 0) | (keys ? 2 : 0);
}

// Few tiles leave compute units idle while each walks over all keys (rows) alone. Their loops are then split among as many
// workgroups as fill the GPU twice, but with LEAST tiles a part, and not where a sequence of twice the mean length has less
// than four parts: the join takes 4 us. Whole and split, us: 64 queries of 16 heads on 4 of 128 over 100000 keys, forward 2530
// and 123; one sequence of 4096, 1 head of 64, forward 71 and 26, with its backward 246 and 91; 8 of 1000, 8 on 2, 169 and
// 111; one of 3000, 16 on 4 of 128, 460 and 358. Below the limit, one sequence of 500, 4 on 2: 81 and 98.
constexpr int FILL = 512;
int parts_of(long long blocks, long long others, int tile, int seqs) {
  const long long most = 2 * others / ((long long)(seqs > 0 ? seqs : 1) * LEAST * tile), fill = FILL / (blocks > 0 ? blocks : 1);
  return most < 4 || fill < 2 ? 1 : (int)(fill < most ? fill : most);
}
int query_parts(int kv_heads, int seqs, int tq, int tk, int group) {
  return parts_of(order_queries(seqs, tq, group) * kv_heads, tk, TILE, seqs);
}
int key_parts(int kv_heads, int dim, int seqs, int tq, int tk, int group) {
  const int kw = key_waves(dim, seqs, tk);
  return kw < 4 ? 1 : parts_of(order_keys(seqs, tk, kw) * kv_heads * (dim <= 64 ? 1 : 2), (long long)tq * group,
                               dim <= 64 ? 64 : 128, seqs);
}
size_t attend_work_bytes(int dim, int seqs, int tq, int tk, int group) {
  return sizeof(int) * (ORDER_HEAD + 2 * (size_t)(order_queries(seqs, tq, group) +
                                                  order_keys(seqs, tk, key_waves(dim, seqs, tk))));
}
size_t attend_scratch_bytes(int kv_heads, int dim, int seqs, int tq, int tk, int group, bool vjp) {
  const size_t pq = query_parts(kv_heads, seqs, tq, tk, group), pk = vjp ? key_parts(kv_heads, dim, seqs, tq, tk, group) : 1;
  const size_t q = pq == 1 ? 0 : pq * order_queries(seqs, tq, group) * kv_heads * (dim <= 64 ? RowsPart<64>::SIZE : RowsPart<128>::SIZE);
  const size_t k = pk == 1 ? 0 : pk * order_keys(seqs, tk, 4) * kv_heads * (dim <= 64 ? 1 : 2) * Part<KEY_PART>::SIZE;
  return sizeof(float) * (q > k ? q : k);
}

template <typename T, int DP>
int attend(hipStream_t st, const Attend& a) {
  const long long tiles = order_queries(a.seqs, a.tq, a.group);
  if (a.parts_q == 1) {
    k_attend<T, DP, false><<<blocks_of(a, tiles, 1), 256, 0, st>>>(a);
  } else {
    k_attend<T, DP, true><<<blocks_of(a, tiles, a.parts_q), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_join<T, DP><<<dim3(blocks_of(a, tiles, 1), 4 * (DP / 32)), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}
template <typename T, int DP>
int attend_dq(hipStream_t st, const Attend& a) {
  const long long tiles = order_queries(a.seqs, a.tq, a.group);
  if (a.parts_q == 1) {
    k_attend_dq<T, DP, false><<<blocks_of(a, tiles, 1), 256, 0, st>>>(a);
  } else {
    k_attend_dq<T, DP, true><<<blocks_of(a, tiles, a.parts_q), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_dq_join<T, DP><<<dim3(blocks_of(a, tiles, 1), 4 * (DP / 32)), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}
template <typename T, int DP>
int attend_vjp(hipStream_t st, const Attend& a) {
  if (a.tq) {
    const int e = attend_dq<T, DP>(st, a);
    if (e) return e;
  }
  if (!a.tk) return 0;
  const long long tiles = order_keys(a.seqs, a.tk, a.key_waves);
  constexpr int ROLES = DP == 64 ? 1 : 2, THREADS = DP == 64 ? 256 : 512;
  if (a.parts_k > 1) {
    k_attend_dkv<T, DP, 4, DP / 16, true><<<blocks_of(a, tiles, ROLES * a.parts_k), THREADS, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_dkv_join<T, DP><<<dim3(blocks_of(a, tiles, 1), 8 * (DP / 32)), 256, 0, st>>>(a);
  } else if (a.key_waves == 4) {
    k_attend_dkv<T, DP, 4, DP / 16, false><<<blocks_of(a, tiles, ROLES), THREADS, 0, st>>>(a);
  } else if constexpr (DP == 64) {
    k_attend_dkv<T, 64, 1, 1, false><<<(unsigned)((tiles * a.kv_heads + 3) / 4), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}

int launch_attend(hipStream_t st, int type, const Attend& a) {
  k_attend_order<<<1, 1024, 0, st>>>(a.seqs, a.tq, a.tk, a.group, a.key_waves, a.by_sequence, a.starts_q, a.starts_k,
                                  (int*)a.order);
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
bool attention_takes(int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk) {
  return (type == pol::BF16 || type == pol::F16) && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && dim >= 8 &&
         dim <= 128 && dim % 8 == 0 && pol::attention_sizes(heads, kv_heads, seqs, tq, tk);
}
}  // namespace

extern "C" {

int dk_attention(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                 long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v,
                 long long v_t, long long v_h, const int* starts_q, const int* starts_k, float scale, void* out,
                 float* lse, void* work, void* scratch) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || !starts_q || !starts_k || !work ||
      (tq && (!q || !out)) || (tk && (!k || !v)) ||
      (!scratch && dk_attention_scratch_bytes(heads, kv_heads, dim, seqs, tq, tk, 0)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.key_waves = pol::key_waves(dim, seqs, tk);
  a.by_sequence = pol::by_sequence(dim, seqs, tq, tk);
  a.parts_q = pol::query_parts(kv_heads, seqs, tq, tk, a.group), a.scratch = (float*)scratch;
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.out = out, a.lse = lse, a.order = (const int*)work;
  return pol::launch_attend(st, type, a);
}

int dk_attention_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk,
                     const void* q, long long q_t, long long q_h, const void* k, long long k_t, long long k_h,
                     const void* v, long long v_t, long long v_h, const int* starts_q, const int* starts_k,
                     float scale, const void* out, const float* lse, const void* work, const void* dout,
                     long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv,
                     void* scratch) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || !starts_q || !starts_k || !work ||
      (tq && (!q || !out || !lse || !dout || !delta || !dq)) || (tk && (!k || !v || !dk || !dv)) ||
      (!scratch && dk_attention_scratch_bytes(heads, kv_heads, dim, seqs, tq, tk, 1)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.key_waves = pol::key_waves(dim, seqs, tk);
  a.by_sequence = pol::by_sequence(dim, seqs, tq, tk);
  a.parts_q = pol::query_parts(kv_heads, seqs, tq, tk, a.group), a.scratch = (float*)scratch;
  a.parts_k = pol::key_parts(kv_heads, dim, seqs, tq, tk, a.group);
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.order = (const int*)work;
  a.out = const_cast<void*>(out), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.do_t = do_t, a.do_h = do_h, a.delta = delta, a.dq = dq, a.dk = dk, a.dv = dv;
  return pol::launch_attend_vjp(st, type, a);
}

long long dk_attention_work_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || seqs < 0 || tq < 0 || tk < 0) return 0;
  return (long long)pol::attend_work_bytes(dim, seqs, tq, tk, heads / kv_heads);
}

long long dk_attention_scratch_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk, int vjp) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || seqs < 0 || tq < 0 || tk < 0) return 0;
  return (long long)pol::attend_scratch_bytes(kv_heads, dim, seqs, tq, tk, heads / kv_heads, vjp != 0);
}

}  // extern "C"
