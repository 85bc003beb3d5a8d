// Causal attention over packed sequences with shared key/value heads: forward and backward.
//
//   S = scale Q K^T, key j <= i' = i + (keys - queries), P = softmax(S), O = P V
//   with a window (WIN): only keys j > i' - window, and the first `sinks` ones
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
//
// With a window a tile's loop is short, and what a workgroup waits for before it counts: its place in the lists, its rows, its
// first tile. The same 256 episodes with a window of 128 and 4 sinks: forward 156 us (of which 120 are left at a window of 16: 0.41
// GB, 3.4 TB/s), dq 231, dkv 306 and 84 for the sinks' far rows; matrix instructions take 14 to 16 % of the SIMDs' cycles, vector
// instructions 69 % in the forward and 34 % in dkv, which waits for its tiles with eight waves a compute unit. The two
// recordings with a window of 1000 and 16 sinks, heads of 128: 145, 174, 401 and 56.
#include "../../include/nablaengine_memory.h"
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
                                                       int window, int sinks, const int* starts_q, const int* starts_k,
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
  auto near = [&](long long cost, long long most) { return (int)(window && most < cost ? most : cost); };
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
            if (t << bits[1] >= sinks) cost = near(cost, ((long long)window + (1 << bits[1])) * group);
          } else {  // the keys that the tile's last row sees
            const int last = ((t + 1) * QROWS < rows ? (t + 1) * QROWS : rows) - 1;
            cost = near(last / group + mk - mq + 1, (long long)window + sinks + QROWS / group);
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
  if (a.grouped >> which & 1) {
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

// The rows' side: a wave's 32 query rows of a workgroup's 128
template <bool WIN>
struct Rows {
  int pos, head, limit, all_see, any_sees, tiles;
  bool valid;
  // WIN: the workgroup's keys are the `front` sinks before its first row's window and all from that window on, `skip` keys
  // further: their places are counted without the keys between, so that a few sinks fill no tile of their own. A row sees the
  // places up to hi, from lo on or before `sinks`.
  int front, skip, hi, lo;
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
    front = skip = 0;
    if (WIN) {
      const int from = p.tile * QROWS / a.group + off - a.window + 1;
      skip = from > a.sinks ? from - a.sinks : 0;
      front = skip ? a.sinks : 0;
    }
    tiles = last < 0 ? 0 : (last - skip) / TILE + 1;
    hi = limit - skip;
    const int own = WIN ? hi - a.window + 1 : 0;
    lo = WIN && own < a.sinks ? a.sinks : own;
  }
  __device__ __forceinline__ int last_place() const { return any_sees - skip; }
  // of the 32 keys from a place on, up to last_place(): whether any of the wave's rows sees one; whether some row's last key, or
  // its window's first, lies among them
  __device__ __forceinline__ bool sees(const Attend& a, int place) const {
    return !WIN || place < a.sinks || place + 31 > all_see - skip - a.window;
  }
  __device__ __forceinline__ bool ends(int place) const { return place + 31 > all_see - skip; }
  __device__ __forceinline__ bool begins(const Attend& a, int place) const {
    return WIN && place <= any_sees - skip - a.window && place + 31 >= a.sinks;
  }
  // f(j) for register j of a C of those keys where this lane's row does not see it; each border takes one comparison
  template <typename F>
  __device__ __forceinline__ void hidden(const Attend& a, int place, int h, F f) const {
    if (ends(place)) {
      const int last = hi - place - 4 * h;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j % 4 + 8 * (j / 4) > last) f(j);
    }
    if (begins(a, place)) {
      const int from = place + 4 * h - a.sinks;
      const unsigned most = (unsigned)(lo - a.sinks);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if ((unsigned)(from + j % 4 + 8 * (j / 4)) < most) f(j);
    }
  }
};

// The keys' side of the forward and of the queries' gradient: tiles of TILE keys and their values, one tile ahead.
template <int DP, typename T, bool WIN>
struct Keys {
  static constexpr int CH = DP / 8, STEP = 256 / CH, N = TILE / STEP;  // chunks a row; rows a turn of the workgroup
  const T *k, *v;  // this thread's chunk of the tile's first rows
  long long k_t, v_t;
  int row, at, left;  // this thread's row; its wave's place in LDS; keys from the tile's first on
  bool in_row;
  int sunk, skip;  // WIN: sinks from the tile's first key on, and how much further the others lie
  __device__ __forceinline__ Keys(const Attend& a, const Place& p, const Rows<WIN>& r, int first) {  // from tile `first` on
    row = threadIdx.x / CH;
    const int c = threadIdx.x % CH ^ swizzle<DP>(row);  // LDS is filled in order: the swizzle is the source's
    in_row = 8 * c < a.dim;
    k_t = a.k_t, v_t = a.v_t;
    skip = WIN ? r.skip : 0, sunk = WIN ? r.front - first * TILE : 0;
    k = (const T*)a.k + (long long)(p.k0 + skip + first * TILE) * k_t + (long long)p.kv * a.k_h + row * k_t + 8 * c;
    v = (const T*)a.v + (long long)(p.k0 + skip + first * TILE) * v_t + (long long)p.kv * a.v_h + row * v_t + 8 * c;
    at = threadIdx.x / 64 * 64 * 8;
    left = p.nk - skip - first * TILE;
  }
  __device__ __forceinline__ void next(T* ks, T* vs) {
    if (WIN && sunk > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool valid = in_row && row + i * STEP < left;
        const long long back = row + i * STEP < sunk ? skip : 0;
        to_lds(k + (i * STEP - back) * k_t, valid, ks + i * 2048 + at);
        to_lds(v + (i * STEP - back) * v_t, valid, vs + i * 2048 + at);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool valid = in_row && row + i * STEP < left;
        to_lds(k + i * STEP * k_t, valid, ks + i * 2048 + at);
        to_lds(v + i * STEP * v_t, valid, vs + i * 2048 + at);
      }
    }
    k += TILE * k_t;
    v += TILE * v_t;
    left -= TILE;
    sunk -= TILE;
  }
};

// one row of a wave's 32, for all its lanes
struct Sight {
  long long token, head;
  int limit;
  template <bool WIN>
  __device__ __forceinline__ Sight(const Attend& a, const Place& p, const Rows<WIN>& r, int n) {
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
template <typename T, int DP, int N, bool WIN>
__device__ __forceinline__ void finish_rows(const Attend& a, const Place& p, const Rows<WIN>& r, int d0, const F16x* acc, float m,
                                            float sum) {
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const float c = a.scale * LOG2E;
  const long long token = p.q0 + r.pos;
  if (a.lse && r.valid && h == 0 && d0 == 0)
    a.lse[(long long)r.head * a.tq + token] = r.limit < 0 ? INFINITY : m * c + (log2f(sum) - Range<T>::LIFT);
  const unsigned bad = bad_columns(r.valid && not_finite<N>(acc) != 0.0f);
  store_rows<N>(r.valid && !(bad >> n & 1) ? (T*)a.out + (token * a.heads + r.head) * dim : nullptr, d0, dim, h, acc,
                r.limit < 0 ? 0.0f : 1.0f / sum);
  if (WIN && a.rest)
    store_rests<N>(r.valid ? (T*)a.rest + (token * a.heads + r.head) * dim : nullptr, d0, dim, h, acc,
                   r.limit < 0 || (bad >> n & 1) ? 0.0f : 1.0f / sum);
  for (unsigned left = bad; left; left &= left - 1) {
    const Sight one(a, p, r, __builtin_ctz(left));
    const Row<DP> qr((const T*)a.q + one.token * a.q_t + one.head * a.q_h, dim);
    Row<DP> o = {};
    float top = -INFINITY, total = 0.0f;
    for (int j = 0; j <= one.limit && total == total; ++j) {
      if (WIN && window_hides(a, j, one.limit)) {
        j = one.limit - a.window;
        continue;
      }
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

template <typename T, int DP, bool SPLIT, bool WIN>
__global__ __launch_bounds__(256, 2) void k_attend(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[2][TILE * DP];
  __shared__ __align__(16) T vs[2][TILE * DP];
  Place p;
  if (!place_of_block(a, 0, SPLIT ? a.parts_q : 1, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const Rows<WIN> r(a, p, uniform(threadIdx.x / 64));
  const Slice my(r.tiles, SPLIT ? a.parts_q : 1, SPLIT ? p.part : 0);
  const int first = SPLIT ? my.first : 0, end = SPLIT ? my.end : r.tiles;
  if (SPLIT && p.part >= my.parts) return;
  Keys<DP, T, WIN> keys(a, p, r, first);
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
    if (key0 > r.last_place()) continue;
    const bool first_half = r.sees(a, key0), second = key0 + 32 <= r.last_place() && r.sees(a, key0 + 32);
    if (WIN && !first_half && !second) continue;
    F16x s[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 ? !second : WIN && !first_half) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = -INFINITY;
        continue;
      }
#pragma unroll
      for (int x = 0; x < KS; ++x) s[i] = mfma(read_rows<DP>(kt, 32 * i, x, n, h), q[x], s[i]);
      r.hidden(a, key0 + 32 * i, h, [&](int j) { s[i][j] = -INFINITY; });
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
      if (WIN && x < 2 && !first_half) continue;
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
  finish_rows<T, DP, DT, WIN>(a, p, r, 0, acc, m, sum);
}

template <typename T, int DP, bool WIN>
__global__ __launch_bounds__(256) void k_attend_join(Attend a) {
  constexpr int DT = DP / 32, N = DP / 2 + 2;
  const int wave = blockIdx.y / DT, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 0, 1, p)) return;
  const Rows<WIN> r(a, p, wave);
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
  if (threadIdx.x < 64) finish_rows<T, DP, 1, WIN>(a, p, r, 32 * block, &acc, m, sum);
}

// ---- backward: the queries' gradient --------------------------------------------------------------------------------

// The forward's walk with the stored log-sum: P and dP a tile from two products over the same keys, dS rounded to 16 bits for
// the third. Both gradients from one kernel would need atomics on dq, whose order changes results from run to run, or a
// buffer of float32 a key tile: dq has a kernel of its own, at two products of seven computed again.

template <typename T, int DP, int N, bool WIN>
__device__ __forceinline__ void finish_dq(const Attend& a, const Place& p, const Rows<WIN>& r, int d0, const F16x* acc, float lse,
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
      if (WIN && window_hides(a, j, one.limit)) {
        j = one.limit - a.window;
        continue;
      }
      const Row<DP> kr((const T*)a.k + (p.k0 + j) * a.k_t + p.kv * a.k_h, dim);
      const float dp = gr.dot(Row<DP>((const T*)a.v + (p.k0 + j) * a.v_t + p.kv * a.v_h, dim));
      o.add(exp2_fast(qr.dot(kr) * c - lse1) * (dp - delta1), kr);
    }
    o.store((T*)a.dq + (one.token * a.heads + one.head) * dim, d0, d0 + 32 * N < dim ? d0 + 32 * N : dim, a.scale);
  }
}

template <typename T, int DP, bool SPLIT, bool WIN>
__global__ __launch_bounds__(256, 2) void k_attend_dq(Attend a) {
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __align__(16) T ks[2][TILE * DP];
  __shared__ __align__(16) T vs[2][TILE * DP];
  Place p;
  if (!place_of_block(a, 0, SPLIT ? a.parts_q : 1, p)) return;
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim;
  const Rows<WIN> r(a, p, uniform(threadIdx.x / 64));
  const Slice my(r.tiles, SPLIT ? a.parts_q : 1, SPLIT ? p.part : 0);
  const int first = SPLIT ? my.first : 0, end = SPLIT ? my.end : r.tiles;
  if (SPLIT && p.part >= my.parts) return;
  Keys<DP, T, WIN> keys(a, p, r, first);
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
    r.hidden(a, key0 + 32 * i, h, [&](int j) { s[j] = -INFINITY, dp[j] = 0.0f; });
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = exp2_fast(fmaf(s[j], c, -lse));
  };
  // delta = dout . out from the stored output, whose rounding is felt where few keys share a row: rows whose keys all
  // lie in their first tile take it from that tile's products instead, sum P dP in float32, below
  float delta = 0.0f;
  const bool few = r.last_place() < TILE;
  if (!few) {
    V8<T> o[KS];
    load_rows<DP>(r.valid ? (const T*)a.out + (token * a.heads + r.head) * dim : nullptr, dim, h, o);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)o[s][e] * (float)g[s][e];
    if (WIN && a.rest) {  // a narrow window: few keys share every row
      load_rows<DP>(r.valid ? (const T*)a.rest + (token * a.heads + r.head) * dim : nullptr, dim, h, o);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)o[s][e] * (float)g[s][e];
    }
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
      for (int i = 0; 32 * i <= r.last_place(); ++i) {
        F16x s, dp;
        products(kt, vt, 0, i, s, dp);
#pragma unroll
        for (int j = 0; j < 16; ++j) delta += s[j] * dp[j];
      }
      delta = add_halves(delta);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (key0 + 32 * i > r.last_place()) break;
      if (WIN && !r.sees(a, key0 + 32 * i)) continue;
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
  finish_dq<T, DP, DT, WIN>(a, p, r, 0, acc, lse, delta);
}

template <typename T, int DP, bool WIN>
__global__ __launch_bounds__(256) void k_attend_dq_join(Attend a) {
  constexpr int DT = DP / 32;
  const int wave = blockIdx.y / DT, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 0, 1, p)) return;
  const Rows<WIN> r(a, p, wave);
  const int parts = Slice(r.tiles, a.parts_q, 0).parts;
  if (parts == 1) return;
  const F16x acc =
      add_parts<DP / 2 + 2>(a, (size_t)p.at * a.parts_q, parts, wave, block, [](int) { return 1.0f; });
  const long long at = (long long)r.head * a.tq + p.q0 + r.pos;
  if (threadIdx.x < 64)
    finish_dq<T, DP, 1, WIN>(a, p, r, 32 * block, &acc, r.valid ? a.lse[at] : INFINITY, r.valid ? a.delta[at] : 0.0f);
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
constexpr size_t far_slot(int dp) { return 2 * 32 * (size_t)dp; }  // floats of 32 keys' dk and dv
// Heads of 128: dk and dv together take 128 registers a lane, with the keys and values more than two waves a SIMD have.
// One workgroup takes dk and another dv (a fourth more products, the scores twice): 1150 us at sequences of 8192 and 2800
// tokens of 16 heads on 4 against 1480 us with both in one and part of the operands in LDS or scratch, and 1230 us with one
// wave a SIMD. Eight waves share a tile of 128 rows, 995 us: twice the products a byte read. Their waves run their products
// at a higher priority than another's exponentials, 955 us; at heads of 64, where those are the longer part, that gains
// nothing (forward 249 us to 260). The wait for the next tile's load stands between the first products and the column
// operands here; the eight waves fill a CU's LDS, so that no other workgroup covers it.
enum Role { BOTH, KEYS, VALUES };
// A window's sinks are seen by all rows of their sequence, other keys by those of one window: their tiles would take many times as
// long, most of their waves idle, and end last (two sequences of 8192 and 2752 tokens, window 1000, 16 sinks: 1121 us, now 401 and
// 56). The rows
// behind the window of a sequence's first key are taken from those tiles and walked over by workgroups of their own, a part of
// far_tokens tokens each for 32 sinks, all of whose waves share the rows; their sums in float32 go to slots that the key tile's
// workgroup adds before it rounds. A part's slot follows from where its sequence lies: a sequence of n queries from q0 and m keys
// from k0 on has at most one part more than multiples of far_tokens in (q0, q0 + n], and as it has m >= far_least keys there is a
// multiple of that in (k0, k0 + m].
struct Far {
  int parts, base, from;  // its parts (0: none), the first one's slot, their first token
  __device__ __forceinline__ Far(const Attend& a, const Place& p) {
    const int off = p.nk - p.nq, behind = a.window > off ? a.window - off : 0;
    const bool some = a.far_tokens && p.nk >= a.far_least && p.nq > behind;
    from = behind;
    parts = some ? (p.nq - behind - 1) / a.far_tokens + 1 : 0;
    base = some ? p.q0 / a.far_tokens + p.k0 / a.far_least : 0;
  }
  template <int DP>
  __device__ __forceinline__ float* slot(const Attend& a, const Place& p, int part, int chunk) const {
    return a.far + (((size_t)(base + part) * a.far_chunks + chunk) * a.kv_heads + p.kv) * far_slot(DP);
  }
};
// the sinks that a key tile's own walk reaches behind their window
__device__ __forceinline__ int near_sinks(const Attend& a, const Place& p) { return Far(a, p).parts ? 0 : a.sinks; }

enum Mode { ALL, WINDOWED, FAR };  // which of the rows a key tile walks over
template <int MODE>
struct RowTiles {  // the rows that see a key tile, in tiles of RT rows or a little less
  int used, first, tiles;
  int rows;  // their end
  __device__ __forceinline__ RowTiles(const Attend& a, const Place& p, int kw, int rt) {
    used = a.group <= rt ? rt / a.group * a.group : rt;
    rows = p.nq * a.group;
    if (MODE == FAR) {
      const long long from = Far(a, p).from + (long long)p.part * a.far_tokens, end = from + a.far_tokens;
      first = (int)from * a.group;
      if (end < p.nq) rows = (int)end * a.group;
      tiles = rows > first ? (rows - 1 - first) / used + 1 : 0;
      return;
    }
    if (MODE == WINDOWED && p.tile * 32 * kw >= near_sinks(a, p)) {  // no sinks: the first token behind the last key's window
      const int keys = (p.tile + 1) * 32 * kw < p.nk ? (p.tile + 1) * 32 * kw : p.nk;
      const long long end = (long long)keys - 1 + a.window - (p.nk - p.nq);
      rows = end < p.nq ? (end > 0 ? (int)end : 0) * a.group : rows;
    }
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
template <typename T, int DP, int N, int ROLE, bool WIN>
__device__ __forceinline__ void finish_dkv(const Attend& a, const Place& p, int key0, int d0, F16x* dk, F16x* dv) {
  const int l = threadIdx.x % 64, n = l % 32, h = l / 32, dim = a.dim, group = a.group;
  if (WIN && key0 < a.sinks && key0 < p.nk) {
    const Far far(a, p);
#pragma unroll 2
    for (int i = 0; i < far.parts; ++i) {
      const float* from = far.slot<DP>(a, p, i, key0 / 32) + l;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if (ROLE == (which ? KEYS : VALUES)) continue;
        F16x* acc = which ? dv : dk;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[t][j] += from[64 * (16 * (which * (DP / 32) + d0 / 32 + t) + j)];
      }
    }
  }
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
      if (WIN && window_hides(a, one, r / group + off)) continue;
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
template <typename T, int DP, int KW, int WAVES, int ROLE, bool PARTS, int MODE>
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
  const int off = p.nk - p.nq;
  const int key0 = p.tile * 32 * KW + 32 * kw, key = key0 + n;
  const bool valid = key < p.nk;
  const float c = a.scale * LOG2E;

  // Row tiles start at whole tokens (but for groups above RT, whose rows' places are computed anew for each tile), so
  // that a thread's rows keep their distance from the tile's first token: RT or a little less rows are used of each.
  const RowTiles<MODE> all(a, p, KW, RT);
  const int sinks = MODE == WINDOWED ? near_sinks(a, p) : a.sinks;
  // the first row whose window lies behind this lane's key; none for a sink (FAR: for a key that is none)
  const int behind = (key < sinks) == (MODE == FAR) ? key + a.window : 0x7fffffff;
  const int rows = all.rows, used = all.used, first = all.first, back = used / group;  // back: tokens of a tile
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
      if (MODE == WINDOWED && low - a.window >= key0 + 31 && key0 >= sinks) continue;
      if (MODE == FAR && most - a.window < key0) continue;
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
      // some row's last key lies before some of the wave's, or its window behind it
      const bool ends = MODE != FAR && low < key0 + 31;
      const bool begins = MODE == FAR ? low - a.window < key0 + 31 || key0 + 31 >= sinks
                                      : MODE == WINDOWED && key0 <= most - a.window && key0 + 31 >= sinks;
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
        if (ends || begins) {
          const I4 li = *(const I4*)(places_of[turn] + at) + (token + off);
          if (ends)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key > li[e]) s[4 * j + e] = dp[4 * j + e] = 0.0f;
          if (begins)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (MODE == FAR ? li[e] < behind : li[e] >= behind) s[4 * j + e] = dp[4 * j + e] = 0.0f;
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
  if (MODE == FAR) {
    float* to = Far(a, p).slot<DP>(a, p, p.part, p.tile) + l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (ROLE != VALUES) to[64 * (16 * d + j)] = dk[d][j];
        if (ROLE != KEYS) to[64 * (16 * (DT + d) + j)] = dv[d][j];
      }
    return;
  }
  if (PARTS && my.parts > 1) {
    const Part<KEY_PART> mine(a, key_slot(a, p, ROLE) + p.part % a.parts_k, w);
    if (ROLE != VALUES) mine.put(0, dk, DT);
    if (ROLE != KEYS) mine.put(ROLE == BOTH ? DT : 0, dv, DT);
    return;
  }
  finish_dkv<T, DP, DT, ROLE, MODE == WINDOWED>(a, p, key0, 0, dk, dv);
}

template <typename T, int DP, int KW, int WAVES, bool PARTS, bool WIN>
__global__ __launch_bounds__(WAVES == 8 ? 512 : 256) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_attend_dkv(Attend a) {
  __shared__ DkvTiles<T, DP, WAVES> lds[WAVES == 1 ? 4 : 1];
  const int parts = PARTS ? a.parts_k : 1;
  Place p;
  if constexpr (WAVES == 1) {  // each wave a tile of its own
    const int w = uniform(threadIdx.x / 64);
    if (place(a, 1, blockIdx.x * 4 + w, p)) dkv_tile<T, DP, KW, WAVES, BOTH, false, WIN ? WINDOWED : ALL>(a, p, lds[w]);
  } else if constexpr (DP == 64) {
    if (place_of_block(a, 1, parts, p)) dkv_tile<T, DP, KW, WAVES, BOTH, PARTS, WIN ? WINDOWED : ALL>(a, p, lds[0]);
  } else {
    if (!place_of_block(a, 1, 2 * parts, p)) return;
    if (p.part >= parts) dkv_tile<T, DP, KW, WAVES, VALUES, PARTS, WIN ? WINDOWED : ALL>(a, p, lds[0]);
    else dkv_tile<T, DP, KW, WAVES, KEYS, PARTS, WIN ? WINDOWED : ALL>(a, p, lds[0]);
  }
}

// the far rows' parts; WAVES waves, as many as a row tile has subtiles
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_attend_far(Attend a) {
  __shared__ DkvTiles<T, DP, WAVES> lds;
  constexpr int ROLES = DP == 64 ? 1 : 2;
  int b = blockIdx.x;
  const int role = b % ROLES;
  b /= ROLES;
  Place p;
  p.kv = b % a.kv_heads;
  b /= a.kv_heads;
  p.tile = b % a.far_chunks;
  const int slot = b / a.far_chunks, l = threadIdx.x % 64;
  auto in = [](int x, int most) { return x < 0 ? 0 : x > most ? most : x; };
  auto base = [&](int s) {
    return s == 0 ? 0 : in(a.starts_q[s], a.tq) / a.far_tokens + in(a.starts_k[s], a.tk) / a.far_least;
  };
  int s = 0;  // the last sequence whose slots begin at or before this one: 64 at once, one of s .. s + n - 1
  for (int n = a.seqs; n > 1;) {
    const int step = (n - 1) / 64 + 1, at = l * step;
    const int c = __popcll(__ballot(at < n && base(s + (at < n ? at : 0)) <= slot)), skip = c > 0 ? (c - 1) * step : 0;
    s += skip;
    n = n - skip < step ? n - skip : step;
  }
  s = uniform(s);
  sequence(a.starts_q, s, a.seqs, a.tq, p.q0, p.nq);
  sequence(a.starts_k, s, a.seqs, a.tk, p.k0, p.nk);
  p.q0 = uniform(p.q0), p.nq = uniform(p.nq), p.k0 = uniform(p.k0), p.nk = uniform(p.nk);
  const Far far(a, p);
  p.part = slot - far.base;
  if (p.part < 0 || p.part >= far.parts || p.tile * 32 >= p.nk) return;
  if constexpr (DP == 64) {
    dkv_tile<T, DP, 1, WAVES, BOTH, false, FAR>(a, p, lds);
  } else {
    if (role) dkv_tile<T, DP, 1, WAVES, VALUES, false, FAR>(a, p, lds);
    else dkv_tile<T, DP, 1, WAVES, KEYS, false, FAR>(a, p, lds);
  }
}

template <typename T, int DP, bool WIN>
__global__ __launch_bounds__(256) void k_attend_dkv_join(Attend a) {
  constexpr int DT = DP / 32;
  const int role = blockIdx.y / (4 * DT) ? VALUES : KEYS, wave = blockIdx.y / DT % 4, block = blockIdx.y % DT;
  Place p;
  if (!place_of_block(a, 1, 1, p)) return;
  const int parts = Slice(RowTiles<WIN ? WINDOWED : ALL>(a, p, 4, DkvTiles<T, DP, DP / 16>::RT).tiles, a.parts_k, 0).parts;
  if (parts == 1) return;
  F16x acc = add_parts<KEY_PART>(a, key_slot(a, p, DP == 64 ? BOTH : role), parts, wave,
                                       (DP == 64 && role == VALUES ? DT : 0) + block, [](int) { return 1.0f; });
  if (threadIdx.x >= 64) return;
  const int key0 = p.tile * 128 + wave * 32;
  if (role == KEYS) finish_dkv<T, DP, 1, KEYS, WIN>(a, p, key0, 32 * block, &acc, nullptr);
  else finish_dkv<T, DP, 1, VALUES, WIN>(a, p, key0, 32 * block, nullptr, &acc);
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
int by_sequence(int dim, int seqs, int tq, int tk, int window) {
  const bool queries = (tq > tk ? tq : tk) <= (long long)LONG * seqs;
  if (window) return queries ? 3 : 0;  // its tiles cost alike
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
// The other side's tokens, of which a window leaves each row (key) no more than itself.
long long others_of(int tokens, int seqs, int window, int more) {
  const long long most = ((long long)window + more) * (seqs > 0 ? seqs : 1);
  return window && most < tokens ? most : tokens;
}
int query_parts(int kv_heads, int seqs, int tq, int tk, int group, int window, int sinks) {
  return parts_of(order_queries(seqs, tq, group) * kv_heads, others_of(tk, seqs, window, sinks), TILE, seqs);
}
int key_parts(int kv_heads, int dim, int seqs, int tq, int tk, int group, int window) {
  const int kw = key_waves(dim, seqs, tk);
  return kw < 4 ? 1 : parts_of(order_keys(seqs, tk, kw) * kv_heads * (dim <= 64 ? 1 : 2), others_of(tq, seqs, window, 128) * group,
                               dim <= 64 ? 64 : 128, seqs);
}
size_t attend_work_bytes(int dim, int seqs, int tq, int tk, int group) {
  return sizeof(int) * (ORDER_HEAD + 2 * (size_t)(order_queries(seqs, tq, group) +
                                                  order_keys(seqs, tk, key_waves(dim, seqs, tk))));
}
// Where the sinks' far rows are walked over apart: where there are sinks, at most four tiles of 32, and a sequence may be longer
// than a window and half a part; not where their slots would take more than 1 GB. Parts of 512 tokens: 50 us for 34, of two
// sequences of 8192 tokens. Forward and backward with 128 sinks, with 129 as they are, and with five tiles apart: 256 sequences of up
// to 1000, window 128, 817, 746 and 847 us; 8192 and 2752 tokens, window 1000, 761, 1150 and 822; four of 16384, window 512, 643, 2647
// and 643: past the limit long sequences pay for all their rows.
constexpr int FAR_TOKENS = 256;
struct FarPlan { int tokens, least, chunks; long long slots; };
FarPlan far_plan(int kv_heads, int dim, int tq, int tk, int window, int sinks) {
  FarPlan r = {0, window + 1 > 64 ? window + 1 : 64, (sinks + 31) / 32, 0};
  if (window < 1 || sinks < 1 || sinks > 128 || tk <= window + FAR_TOKENS / 2) return r;
  r.slots = (long long)tq / FAR_TOKENS + tk / r.least + 1;
  if (r.slots * r.chunks * kv_heads * far_slot(dim <= 64 ? 64 : 128) <= 1LL << 28) r.tokens = FAR_TOKENS;
  return r;
}
size_t attend_parts_floats(int kv_heads, int dim, int seqs, int tq, int tk, int group, int window, int sinks, bool vjp) {
  const size_t pq = query_parts(kv_heads, seqs, tq, tk, group, window, sinks);
  const size_t pk = vjp ? key_parts(kv_heads, dim, seqs, tq, tk, group, window) : 1;
  const size_t q = pq == 1 ? 0 : pq * order_queries(seqs, tq, group) * kv_heads * (dim <= 64 ? RowsPart<64>::SIZE : RowsPart<128>::SIZE);
  const size_t k = pk == 1 ? 0 : pk * order_keys(seqs, tk, 4) * kv_heads * (dim <= 64 ? 1 : 2) * Part<KEY_PART>::SIZE;
  return q > k ? q : k;
}
size_t attend_scratch_bytes(int kv_heads, int dim, int seqs, int tq, int tk, int group, int window, int sinks, bool vjp) {
  const FarPlan far = far_plan(kv_heads, dim, tq, tk, window, sinks);
  const size_t parts = attend_parts_floats(kv_heads, dim, seqs, tq, tk, group, window, sinks, vjp);
  const size_t slots = vjp && far.tokens ? (size_t)far.slots * far.chunks * kv_heads : 0;
  return sizeof(float) * (parts + slots * far_slot(dim <= 64 ? 64 : 128));
}

template <typename T, int DP, bool WIN>
int attend(hipStream_t st, const Attend& a) {
  const long long tiles = order_queries(a.seqs, a.tq, a.group);
  if (a.parts_q == 1) {
    k_attend<T, DP, false, WIN><<<blocks_of(a, tiles, 1), 256, 0, st>>>(a);
  } else {
    k_attend<T, DP, true, WIN><<<blocks_of(a, tiles, a.parts_q), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_join<T, DP, WIN><<<dim3(blocks_of(a, tiles, 1), 4 * (DP / 32)), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}
template <typename T, int DP, bool WIN>
int attend_dq(hipStream_t st, const Attend& a) {
  const long long tiles = order_queries(a.seqs, a.tq, a.group);
  if (a.parts_q == 1) {
    k_attend_dq<T, DP, false, WIN><<<blocks_of(a, tiles, 1), 256, 0, st>>>(a);
  } else {
    k_attend_dq<T, DP, true, WIN><<<blocks_of(a, tiles, a.parts_q), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_dq_join<T, DP, WIN><<<dim3(blocks_of(a, tiles, 1), 4 * (DP / 32)), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}
template <typename T, int DP, bool WIN>
int attend_vjp(hipStream_t st, const Attend& a) {
  if (a.tq) {
    const int e = attend_dq<T, DP, WIN>(st, a);
    if (e) return e;
  }
  if (!a.tk) return 0;
  if (WIN && a.far_tokens) {
    constexpr int WAVES = DP / 32;
    const FarPlan far = far_plan(a.kv_heads, a.dim, a.tq, a.tk, a.window, a.sinks);
    k_attend_far<T, DP, WAVES><<<(unsigned)(far.slots * far.chunks * a.kv_heads * (DP == 64 ? 1 : 2)), 64 * WAVES, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  const long long tiles = order_keys(a.seqs, a.tk, a.key_waves);
  constexpr int ROLES = DP == 64 ? 1 : 2, THREADS = DP == 64 ? 256 : 512;
  if (a.parts_k > 1) {
    k_attend_dkv<T, DP, 4, DP / 16, true, WIN><<<blocks_of(a, tiles, ROLES * a.parts_k), THREADS, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    k_attend_dkv_join<T, DP, WIN><<<dim3(blocks_of(a, tiles, 1), 8 * (DP / 32)), 256, 0, st>>>(a);
  } else if (a.key_waves == 4) {
    k_attend_dkv<T, DP, 4, DP / 16, false, WIN><<<blocks_of(a, tiles, ROLES), THREADS, 0, st>>>(a);
  } else if constexpr (DP == 64) {
    k_attend_dkv<T, 64, 1, 1, false, WIN><<<(unsigned)((tiles * a.kv_heads + 3) / 4), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}

template <bool WIN>
int launch_attend(hipStream_t st, int type, const Attend& a) {
  k_attend_order<<<1, 1024, 0, st>>>(a.seqs, a.tq, a.tk, a.group, a.key_waves, a.by_sequence, WIN ? a.window : 0,
                                  WIN && !a.far_tokens ? a.sinks : 0, a.starts_q, a.starts_k, (int*)a.order);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.tq) return (int)e;
  if (type == BF16) return a.dim <= 64 ? attend<__bf16, 64, WIN>(st, a) : attend<__bf16, 128, WIN>(st, a);
  return a.dim <= 64 ? attend<_Float16, 64, WIN>(st, a) : attend<_Float16, 128, WIN>(st, a);
}
template <bool WIN>
int launch_attend_vjp(hipStream_t st, int type, const Attend& a) {
  if (type == BF16) return a.dim <= 64 ? attend_vjp<__bf16, 64, WIN>(st, a) : attend_vjp<__bf16, 128, WIN>(st, a);
  return a.dim <= 64 ? attend_vjp<_Float16, 64, WIN>(st, a) : attend_vjp<_Float16, 128, WIN>(st, a);
}

}  // namespace pol

namespace {
bool attention_takes(int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk) {
  return (type == pol::BF16 || type == pol::F16) && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && dim >= 8 &&
         dim <= 128 && dim % 8 == 0 && pol::attention_sizes(heads, kv_heads, seqs, tq, tk);
}
}  // namespace

// A window as long as the keys hides nothing: the kernels without one. Else its length, with the sinks within the keys.
namespace {
int window_of(int window, int tk) { return window < tk ? window : 0; }
int sinks_of(int sinks, int tk) { return sinks < tk ? sinks : tk; }
}  // namespace

extern "C" {

int dk_attention_window(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                        long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v, long long v_t,
                        long long v_h, const int* starts_q, const int* starts_k, float scale, int window, int sinks, void* out,
                        void* rest, float* lse, void* work, void* scratch) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || window < 0 || sinks < 0 || !starts_q ||
      !starts_k || !work || (tq && (!q || !out)) || (tk && (!k || !v)) ||
      (!scratch && dk_attention_window_scratch_bytes(heads, kv_heads, dim, seqs, tq, tk, window, sinks, 0)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.window = window_of(window, tk), a.sinks = sinks_of(sinks, tk), a.rest = rest;
  a.far_tokens = pol::far_plan(kv_heads, dim, tq, tk, a.window, a.sinks).tokens;
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.key_waves = pol::key_waves(dim, seqs, tk);
  a.by_sequence = pol::by_sequence(dim, seqs, tq, tk, a.window), a.grouped = a.window ? 3 : a.by_sequence;
  a.parts_q = pol::query_parts(kv_heads, seqs, tq, tk, a.group, a.window, a.sinks), a.scratch = (float*)scratch;
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.out = out, a.lse = lse, a.order = (const int*)work;
  return a.window ? pol::launch_attend<true>(st, type, a) : pol::launch_attend<false>(st, type, a);
}

int dk_attention_window_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                            long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v, long long v_t,
                            long long v_h, const int* starts_q, const int* starts_k, float scale, int window, int sinks,
                            const void* out, const void* rest, const float* lse, const void* work, const void* dout,
                            long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv, void* scratch) {
  if (!attention_takes(type, heads, kv_heads, dim, seqs, tq, tk) || !(scale > 0.0f) || window < 0 || sinks < 0 || !starts_q ||
      !starts_k || !work || (tq && (!q || !out || !lse || !dout || !delta || !dq)) || (tk && (!k || !v || !dk || !dv)) ||
      (!scratch && dk_attention_window_scratch_bytes(heads, kv_heads, dim, seqs, tq, tk, window, sinks, 1)))
    return (int)hipErrorInvalidValue;
  pol::Attend a = {};
  a.window = window_of(window, tk), a.sinks = sinks_of(sinks, tk), a.rest = const_cast<void*>(rest);
  const pol::FarPlan far = pol::far_plan(kv_heads, dim, tq, tk, a.window, a.sinks);
  a.far_tokens = far.tokens, a.far_least = far.least, a.far_chunks = far.chunks;
  if (scratch)  // the slots behind the parts
    a.far = (float*)scratch + pol::attend_parts_floats(kv_heads, dim, seqs, tq, tk, heads / kv_heads, a.window, a.sinks, true);
  a.q = q, a.k = k, a.v = v;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim, a.seqs = seqs, a.tq = tq, a.tk = tk;
  a.key_waves = pol::key_waves(dim, seqs, tk);
  a.by_sequence = pol::by_sequence(dim, seqs, tq, tk, a.window), a.grouped = a.window ? 3 : a.by_sequence;
  a.parts_q = pol::query_parts(kv_heads, seqs, tq, tk, a.group, a.window, a.sinks), a.scratch = (float*)scratch;
  a.parts_k = pol::key_parts(kv_heads, dim, seqs, tq, tk, a.group, a.window);
  a.starts_q = starts_q, a.starts_k = starts_k, a.scale = scale, a.order = (const int*)work;
  a.out = const_cast<void*>(out), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.do_t = do_t, a.do_h = do_h, a.delta = delta, a.dq = dq, a.dk = dk, a.dv = dv;
  return a.window ? pol::launch_attend_vjp<true>(st, type, a) : pol::launch_attend_vjp<false>(st, type, a);
}

long long dk_attention_window_scratch_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk, int window, int sinks, int vjp) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || seqs < 0 || tq < 0 || tk < 0 || window < 0 || sinks < 0) return 0;
  return (long long)pol::attend_scratch_bytes(kv_heads, dim, seqs, tq, tk, heads / kv_heads, window_of(window, tk),
                                              sinks_of(sinks, tk), vjp != 0);
}

int dk_attention(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                 long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v,
                 long long v_t, long long v_h, const int* starts_q, const int* starts_k, float scale, void* out,
                 float* lse, void* work, void* scratch) {
  return dk_attention_window(st, type, heads, kv_heads, dim, seqs, tq, tk, q, q_t, q_h, k, k_t, k_h, v, v_t, v_h, starts_q, starts_k,
                             scale, 0, 0, out, nullptr, lse, work, scratch);
}

int dk_attention_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk,
                     const void* q, long long q_t, long long q_h, const void* k, long long k_t, long long k_h,
                     const void* v, long long v_t, long long v_h, const int* starts_q, const int* starts_k,
                     float scale, const void* out, const float* lse, const void* work, const void* dout,
                     long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv,
                     void* scratch) {
  return dk_attention_window_vjp(st, type, heads, kv_heads, dim, seqs, tq, tk, q, q_t, q_h, k, k_t, k_h, v, v_t, v_h, starts_q,
                                 starts_k, scale, 0, 0, out, nullptr, lse, work, dout, do_t, do_h, delta, dq, dk, dv, scratch);
}

long long dk_attention_work_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || seqs < 0 || tq < 0 || tk < 0) return 0;
  return (long long)pol::attend_work_bytes(dim, seqs, tq, tk, heads / kv_heads);
}

long long dk_attention_scratch_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk, int vjp) {
  return dk_attention_window_scratch_bytes(heads, kv_heads, dim, seqs, tq, tk, 0, 0, vjp);
}

}  // extern "C"
