// A gated linear recurrence over packed sequences, forward and backward, and its single-token form.
//
//   a = 1 / (1 + exp(-gate)),  h_t = a_t h_{t-1} + (1 - a_t) x_t  a channel, from each sequence's carried state
//   g_t = dh_t + a_{t+1} g_{t+1},  dx = (1 - a) g,  dgate = g (h_{t-1} - x) a (1 - a),  dinitial = a g of the first token
//
// Steps compose: a stretch of tokens takes the state s that enters it to P s + B. A state lasts for as many steps as its gates
// say, a million with one of 14, and what steps are off by must not add up over them: 1 - a has its own places, but a has not,
// and a product of many, or many steps by it, is off by 2^-24 a token. So 1 - P is a sum of its own, from which P is taken
// where it is the larger (map_of, join), wherever a state leaves a stretch, a chunk or a call; inside a stretch the product
// does. 65536 tokens from a state and with inputs of 1: every state 1 within 30 2^-24 at any gate (products throughout: 3.0e-3
// off at a gate of 12; of chunks: 104 2^-24), and over 2^25 tokens within 23; the state's decay alone within 1.4e-6 of itself
// from gates of 8 on. The packed tokens are cut into chunks, whatever sequences they hold, so that work is even over ragged
// lengths; a sequence's first token cuts the chain (a choice, not a product with 0: what is not finite stays in its sequence).
// A workgroup takes a chunk and 64 V channels: each of its waves reads TOK tokens at once into registers, a lane V channels of
// each, finds its stretch's P and B, gets the state that enters it from the stretches before (LDS) and from the chunks before
// (memory), and walks over its tokens once more. Sums and states are float32 throughout; each output is rounded once.
//
// The chunks' P and B come from a kernel of their own, which reads only the tokens after a chunk's last sequence start (none
// where the next chunk starts a sequence), and a third kernel carries states over the chunks: two reads of x and gate
// where sequences are long, one where they are short. The backward does the same from the other end; it takes the forward's
// carried states, so the states between are computed from x and gate again and none is stored.
//
// Memory bounds it, and where sequences are short one read after another: where they start, then their tokens. Measured,
// bfloat16, of the 5.0 to 5.2 TB/s of a large copy: two sequences of 65536 tokens together, 1024 channels, forward 73 us (5.5
// TB/s of x, gate and h, some still in the cache), the chunks' P and B 65 (4.1 TB/s), backward 160 (4.2 TB/s) and 70; 4096
// sequences of up to 32 tokens, 512 channels, 63 and 26, 123 and 25; the states over the chunks 13 each time. 1 - P as a sum of
// its own costs 3 % of a forward and backward (243 and 355 us a call without, 251 and 365 with). Without it: chunks of 128
// tokens, two workgroups of eight waves a compute unit, forward 73 and 81 us for 64 and 71, backward 134 and 186 for 119 and
// 157; stretches of 16 tokens in the backward 127 and 168. One token a world: 16384 worlds of 1024 channels 35 us, 6.7 TB/s.
#include <cfloat>

#include "../../include/nablaengine_memory.h"
#include "policy_device.h"
#include "policy_sizes.h"

namespace pol {

struct Scan {
  const void *x, *gate;
  long long x_t, g_t;  // elements from token to token
  int tokens, channels, seqs, chunks, groups;
  const int* starts;
  const float* initial;  // (seqs, channels), or NULL: zeros
  void* h;
  float* last;   // (seqs, channels)
  float* carry;  // (chunks, channels): the state that enters each chunk
  float* parts;  // (chunks, 2, channels): the map (packed), DROPS where the chunk drops what enters it, and B
  // the backward's
  const void* dh;  // or NULL: zeros
  long long d_t;
  const float* dlast;  // or NULL: zeros
  void *dx, *dgate;
  float *dinitial, *back;  // back (chunks, channels): what the next chunk's first token hands to a chunk's last
};

// V neighbouring elements
template <typename T, int V> struct Few { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ Few<T, V> load_few(const T* p) {
  Few<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
// A state's value in T. float16: of the float32 state, which the compiler would otherwise join with the sum before it in one
// instruction that rounds the exact sum, now and then to the other neighbour.
template <typename T>
__device__ __forceinline__ T rounded(float f) {
  if constexpr (std::is_same<T, _Float16>::value) asm("" : "+v"(f));
  return (T)f;
}
template <typename T, int V>
__device__ __forceinline__ void store_few(T* p, const float* f) {
  Few<T, V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = rounded<T>(f[e]);
  __builtin_memcpy(p, &r, sizeof(r));
}

// What tokens do to the state that enters them, P s + B, with what it takes for states that last long: P and Q = 1 - P are sums
// of their own, each with its own last places. Up to a Q of 0.5, P is taken from it, and what its rounding leaves is added.
struct Map { float p, rest; };
__device__ __forceinline__ Map map_of(float p, float q) {
  const float p1 = 1.0f - q;
  return q <= 0.5f ? Map{p1, 1.0f - p1 - q} : Map{p, 0.0f};
}
// an infinite state is one whatever the rest's sign
__device__ __forceinline__ float mapped(const Map& m, float b, float s) {
  return fmaf(m.p, s, fmaf(m.rest, __builtin_amdgcn_fmed3f(s, -FLT_MAX, FLT_MAX), b));
}
// p and q of what (p1, q1) makes of what they are already
__device__ __forceinline__ void join(float& p, float& q, float p1, float q1) {
  q = fmaf(q1, p, q);
  p = q <= 0.5f ? 1.0f - q : p * p1;  // the product's factors are off by 2^-25 each
}
// a token alone
__device__ __forceinline__ float stepped(float keep, float take, float x, float s) { return mapped(map_of(keep, take), take * x, s); }
// a map in one float: Q, or P with its sign changed
__device__ __forceinline__ float packed(float p, float q) { return q <= 0.5f ? q : -p; }
__device__ __forceinline__ Map unpacked(float m, float& p, float& q) {
  const bool far = (int)__float_as_uint(m) < 0;
  p = far ? -m : 1.0f - m;
  const float left = 1.0f - p;
  q = far ? left : m;
  return {p, far ? 0.0f : left - m};
}
__device__ __forceinline__ Map unpacked(float m) {
  float p, q;
  return unpacked(m, p, q);
}
constexpr float DROPS = 2.0f;  // in a map's place: nothing of what enters leaves; unpacked, a P of -1

__device__ __forceinline__ int scan_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Where sequences start inside a chunk: at[i] is the sequence whose first token is the chunk's token i (the last of those
// that start there; `seqs` where the tokens behind the last sequence begin), -1 where none is; i up to CHUNK, the next
// chunk's first token. Returns the sequence that holds the chunk's first token. Every thread of the workgroup calls it. The
// offsets are searched by all threads at once: one read where lengths are even enough, two more up to NT^2 sequences.
template <int CHUNK, int NT>
__device__ __forceinline__ int find_starts(const Scan& a, int t0, int* at) {
  auto value = [&](int s) {
    const int x = s == 0 ? 0 : a.starts[s];
    return x < 0 ? 0 : x > a.tokens ? a.tokens : x;
  };
  const int tid = threadIdx.x;
  for (int i = tid; i <= CHUNK; i += NT) at[i] = -1;
  // where the chunk's first token would lie if all sequences were as long: mostly the starts are among the NT around
  const long long guess = (long long)(a.seqs + 1) * t0 / a.tokens - NT / 2, most = (long long)a.seqs + 1 - NT;
  int lo = guess < 0 || most < 0 ? 0 : (int)(guess < most ? guess : most), n = a.seqs + 1 - lo < NT ? a.seqs + 1 - lo : NT;
  int v = tid < n ? value(lo + tid) : 0;
  int c = __syncthreads_count(tid < n && v <= t0);
  if ((c == 0 && lo > 0) || (c == n && lo + n <= a.seqs)) {  // they are not: all are searched
    lo = 0, n = a.seqs + 1;  // the last start at or before t0 is one of lo .. lo + n - 1
    while (n > NT) {
      const int step = (n - 1) / NT + 1;
      const long long idx = (long long)tid * step;
      c = __syncthreads_count(idx < n && value(lo + (int)idx) <= t0);
      const int skip = c > 0 ? (c - 1) * step : 0;
      n = n - skip < step ? n - skip : step;
      lo += skip;
    }
    v = tid < n ? value(lo + tid) : 0;
    c = __syncthreads_count(tid < n && v <= t0);
  }
  const int base = lo + (c > 0 ? c : 1) - 1;
  bool mine = tid < n;
  for (int s = lo + tid, next = lo + n;;) {  // until a start lies behind the chunk
    if (mine && v >= t0 && v - t0 <= CHUNK) atomicMax(&at[v - t0], s);
    if (!__syncthreads_and(!mine || v - t0 <= CHUNK) || next > a.seqs) break;
    s = next + tid;
    mine = tid <= a.seqs - next;
    v = mine ? value(s) : 0;
    next = next <= a.seqs - NT ? next + NT : a.seqs + 1;
  }
  __syncthreads();
  return base;
}

// A wave's stretch of TOK tokens
template <int TOK>
struct Stretch {
  int t0, there, live;  // its first token; of its tokens, those that there are, and those that a sequence holds
  int seq;              // the sequence of its first token
  int mine;             // lane i: the sequence that starts at token i, or -1
  unsigned cuts;        // bit i: a sequence starts at token i (bit TOK: at the one after)
  __device__ __forceinline__ Stretch(const Scan& a, const int* at, int base, int chunk0, int w) {
    const int l = threadIdx.x % 64;
    t0 = chunk0 + w * TOK;
    there = a.tokens - t0 < 0 ? 0 : a.tokens - t0 < TOK ? a.tokens - t0 : TOK;
    int s = base;
    for (int i = l; i <= w * TOK; i += 64) s = at[i] > s ? at[i] : s;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_xor(s, d);
      s = o > s ? o : s;
    }
    seq = scan_uniform(s);
    mine = l <= TOK ? at[w * TOK + l] : -1;
    cuts = (unsigned)__ballot(mine >= 0);
    const unsigned end = (unsigned)__ballot(mine == a.seqs);
    live = seq == a.seqs ? 0 : end ? __builtin_ctz(end) : TOK;
    live = live < there ? live : there;
    if (t0 + TOK >= a.tokens && there < TOK) cuts |= 1u << there;  // the tokens' end is one
    else if (t0 + TOK == a.tokens) cuts |= 1u << TOK;
  }
  __device__ __forceinline__ int sequence_at(int i) const { return __builtin_amdgcn_readlane(mine, i); }
};

// chunk and channels of a workgroup; neighbours in the grid share the chunk's tokens
template <int V>
struct Lane {
  int c;        // this lane's first channel
  bool counts;  // whether it has any of its own
  __device__ __forceinline__ Lane(const Scan& a, int group) {
    const int at = (group * 64 + threadIdx.x % 64) * V;
    counts = at < a.channels;
    c = at + V <= a.channels ? at : a.channels - V;  // a lane past the end repeats the last one's channels
  }
};

// the maps of the waves' stretches: (W, 64 V) each, and whether a stretch drops what enters it. WHOLE: with what P's rounding
// leaves, for states that go on past the chunk.
template <int W, int V, bool WHOLE = true>
struct Joined {
  float p[W][64][V], b[W][64][V], rest[WHOLE ? W : 1][64][V];
  int drops[W];
  __device__ __forceinline__ void put(int w, int l, int e, const Map& m, float to) {
    p[w][l][e] = m.p, b[w][l][e] = to;
    if (WHOLE) rest[w][l][e] = m.rest;
  }
  __device__ __forceinline__ Map at(int w, int l, int e) const { return {p[w][l][e], rest[w][l][e]}; }
};

// the state after stretches from .. to - 1 (or, from the end, from .. to + 1 downwards) from the one that enters them
template <int W, int V, bool WHOLE>
__device__ __forceinline__ void through(const Joined<W, V, WHOLE>& j, int w, float* s) {
  const int l = threadIdx.x % 64;
  const bool none = j.drops[w];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float b = j.b[w][l][e];
    s[e] = none ? b : WHOLE ? mapped(j.at(w, l, e), b, s[e]) : fmaf(j.p[w][l][e], s[e], b);
  }
}

// sequence s's row of a (seqs, channels) table, zeros where there is none
template <int V>
__device__ __forceinline__ Few<float, V> state_of(const Scan& a, const float* table, int s, int c) {
  Few<float, V> r = {};
  if (table && s >= 0 && s < a.seqs) r = load_few<float, V>(table + (long long)s * a.channels + (unsigned)c);
  return r;
}

template <typename T, int V, int TOK>
__device__ __forceinline__ void load_tokens(const void* from, long long stride, const Scan& a, int t0, int c, Few<T, V>* r) {
#pragma unroll
  for (int i = 0; i < TOK; ++i) {  // tokens past the end: the last one again
    const int t = t0 + i < a.tokens ? t0 + i : a.tokens - 1;
    r[i] = load_few<T, V>((const T*)from + t * stride + (unsigned)c);  // the row is the wave's, the channel the lane's
  }
}

// A forward walk over tokens from .. to - 1 of a stretch: step(i, keep, take x) for each, start(i) before where a sequence starts.
template <typename T, int V, int TOK, typename Start, typename Step>
__device__ __forceinline__ void walk(const Stretch<TOK>& st, const Few<T, V>* f, Start start, Step step) {
  if (st.live == TOK && !(st.cuts & ((1u << TOK) - 1))) {  // most stretches of long sequences
#pragma unroll
    for (int i = 0; i < TOK; ++i) step(i);
  } else {
#pragma unroll
    for (int i = 0; i < TOK; ++i)
      if (i < st.live) {
        if (st.cuts >> i & 1) start(i);
        step(i);
      }
  }
}

// ---- the chunks' P and B --------------------------------------------------------------------------------------------

// what a chunk does to the state that enters it, for all chunks but the last
template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(64 * W) void k_scan_parts(Scan a) {
  constexpr int CHUNK = W * TOK, NT = 64 * W;
  __shared__ int at[CHUNK + 1];
  __shared__ Joined<W, V> joined;
  const int chunk = blockIdx.x / a.groups, w = scan_uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  const int base = find_starts<CHUNK, NT>(a, chunk * CHUNK, at);
  const Lane<V> lane(a, blockIdx.x % a.groups);
  float* out = a.parts + (long long)chunk * 2 * a.channels + lane.c;
  if (at[CHUNK] >= 0) {  // the next chunk takes nothing over
    if (w == 0 && lane.counts)
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = DROPS, out[a.channels + e] = 0.0f;
    return;
  }
  const Stretch<TOK> st(a, at, base, chunk * CHUNK, w);
  // the last start in the chunk: stretches before its own do not matter
  int from = -1;
  for (int i = l; i < CHUNK; i += 64) from = at[i] >= 0 ? i : from;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_xor(from, d);
    from = o > from ? o : from;
  }
  from = scan_uniform(from);
  float p[V], q[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
  if ((w + 1) * TOK > from) {
    Few<T, V> f[TOK], x[TOK];
    load_tokens<T, V, TOK>(a.gate, a.g_t, a, st.t0, lane.c, f);
    load_tokens<T, V, TOK>(a.x, a.x_t, a, st.t0, lane.c, x);
    Few<float, V> s = {};
    walk<T, V, TOK>(st, f, [&](int i) {
                      s = state_of<V>(a, a.initial, st.sequence_at(i), lane.c);
#pragma unroll
                      for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
                    },
                    [&](int i) {
#pragma unroll
                      for (int e = 0; e < V; ++e) {
                        float keep, take;
                        gates<T>((float)f[i].v[e], keep, take);
                        q[e] = fmaf(take, p[e], q[e]);
                        p[e] *= keep;
                        b[e] = fmaf(keep, b[e], take * (float)x[i].v[e]);
                      }
                    });
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = mapped(map_of(p[e], q[e]), b[e], s.v[e]);  // from the last start's state, or none
  }
#pragma unroll
  for (int e = 0; e < V; ++e) joined.put(w, l, e, map_of(p[e], q[e]), b[e]);
  if (l == 0) joined.drops[w] = (st.cuts & ((1u << TOK) - 1)) != 0;
  __syncthreads();
  if (w || !lane.counts) return;
  bool none = false;
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
  for (int o = 0; o < W; ++o) {
    through(joined, o, b);
    none |= joined.drops[o] != 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Map m = joined.at(o, l, e);
      join(p[e], q[e], m.p, 1.0f - m.p - m.rest);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = none ? DROPS : packed(p[e], q[e]), out[a.channels + e] = b[e];
}

// the same from the other end: what a chunk hands to the token before its first, from what the token after its last hands to
// it; for all chunks but the first
template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(64 * W) void k_scan_back_parts(Scan a) {
  constexpr int CHUNK = W * TOK, NT = 64 * W;
  __shared__ int at[CHUNK + 1];
  __shared__ Joined<W, V> joined;
  const int chunk = blockIdx.x / a.groups + 1, w = scan_uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  const int base = find_starts<CHUNK, NT>(a, chunk * CHUNK, at);
  const Lane<V> lane(a, blockIdx.x % a.groups);
  float* out = a.parts + (long long)chunk * 2 * a.channels + lane.c;
  if (at[0] >= 0) {
    if (w == 0 && lane.counts)
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = DROPS, out[a.channels + e] = 0.0f;
    return;
  }
  const Stretch<TOK> st(a, at, base, chunk * CHUNK, w);
  int to = CHUNK + 1;  // the first start: stretches behind it do not matter
  for (int i = l; i <= CHUNK; i += 64) to = at[i] >= 0 && i < to ? i : to;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_xor(to, d);
    to = o < to ? o : to;
  }
  to = scan_uniform(to);
  float p[V], q[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
  if (w * TOK < to && st.live > 0) {
    Few<T, V> f[TOK], d[TOK];
    load_tokens<T, V, TOK>(a.gate, a.g_t, a, st.t0, lane.c, f);
    if (a.dh) load_tokens<T, V, TOK>(a.dh, a.d_t, a, st.t0, lane.c, d);
    else
#pragma unroll
      for (int i = 0; i < TOK; ++i) d[i] = Few<T, V>{};
    const unsigned later = st.cuts >> 1;
    // tokens 0 .. end - 1, of the first token's sequence, lead to the token before
    const int end = later ? __builtin_ctz(later) + 1 : TOK;
    const auto last = state_of<V>(a, a.dlast, later ? st.seq : -1, lane.c);
#pragma unroll
    for (int i = TOK - 1; i >= 0; --i)
      if (i < end)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float keep, take;
          gates<T>((float)f[i].v[e], keep, take);
          q[e] = fmaf(take, p[e], q[e]);
          p[e] *= keep;
          b[e] = keep * (b[e] + (float)d[i].v[e]);
        }
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = mapped(map_of(p[e], q[e]), b[e], last.v[e]);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) joined.put(w, l, e, map_of(p[e], q[e]), b[e]);
  if (l == 0) joined.drops[w] = (st.cuts >> 1) != 0;
  __syncthreads();
  if (w || !lane.counts) return;
  bool none = false;
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
  for (int o = W - 1; o >= 0; --o) {
    through(joined, o, b);
    none |= joined.drops[o] != 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Map m = joined.at(o, l, e);
      join(p[e], q[e], m.p, 1.0f - m.p - m.rest);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = none ? DROPS : packed(p[e], q[e]), out[a.channels + e] = b[e];
}

// ---- the states that enter the chunks -------------------------------------------------------------------------------

// 8 channels a workgroup and 128 runs of chunks: each run's own P and B, those joined over the runs by doubling, then each
// run once more from the state that enters it. BACK: the chunks from the last to the first. Bound by one read after another: 1340
// chunks of 512 channels 12.5 us; 11 before 1 - P was a sum of its own, the same with 16 channels and 64 runs.
template <bool BACK>
__global__ __launch_bounds__(1024) void k_scan_carry(Scan a, int c0) {
  constexpr int CH = 8, RUNS = 1024 / CH;
  __shared__ float ps[2][RUNS][CH], qs[2][RUNS][CH], bs[2][RUNS][CH];
  const int l = threadIdx.x % CH, c = c0 + blockIdx.x * CH + l, run = threadIdx.x / CH;
  const bool in = c < a.channels;
  const int n = a.chunks - 1, each = (n + RUNS - 1) / RUNS;  // the maps between neighbouring chunks, in the order of the walk
  const int first = run * each < n ? run * each : n, end = first + each < n ? first + each : n;
  auto at = [&](int i) { return a.parts + (long long)(BACK ? a.chunks - 1 - i : i) * 2 * a.channels + (in ? c : 0); };
  constexpr int KEPT = 16;  // maps that stay in registers for the second walk: up to 2048 chunks
  Map mk[KEPT];
  float bk[KEPT], p = 1.0f, q = 0.0f, b = 0.0f;
  bool none = false;
  const bool kept = each <= KEPT;
  // a map's P is below 0 where it drops what enters
  auto from = [&](const Map& m, float bi, float s) { return m.p < 0.0f ? bi : mapped(m, bi, s); };
  auto step = [&](float mi, float bi) {
    float p1, q1;
    const Map m = unpacked(mi, p1, q1);
    b = from(m, bi, b);
    none |= m.p < 0.0f;
    join(p, q, p1, q1);
    return m;
  };
  if (kept) {
    float in[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const bool there = first + i < end;
      in[i] = there ? at(first + i)[0] : 0.0f, bk[i] = there ? at(first + i)[a.channels] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (i < each) mk[i] = step(in[i], bk[i]);
  } else {
#pragma unroll 8
    for (int i = first; i < end; ++i) step(at(i)[0], at(i)[a.channels]);
  }
  int side = 0;
  if (none) p = -1.0f;
  ps[0][run][l] = p, qs[0][run][l] = q, bs[0][run][l] = b;
#pragma unroll
  for (int d = 1; d < RUNS; d *= 2, side ^= 1) {
    __syncthreads();
    if (run >= d && !(p < 0.0f)) {
      const float p0 = ps[side][run - d][l];
      b = mapped(map_of(p, q), b, bs[side][run - d][l]);
      const float p1 = p, q1 = q;
      p = p0, q = qs[side][run - d][l];
      join(p, q, p1, q1);
      if (p0 < 0.0f) p = p0;
    }
    ps[side ^ 1][run][l] = p, qs[side ^ 1][run][l] = q, bs[side ^ 1][run][l] = b;
  }
  __syncthreads();
  float s = run ? bs[side][run - 1][l] : 0.0f;  // nothing enters the first chunk
  float* out = BACK ? a.back : a.carry;
  if (run == 0 && in) out[(long long)(BACK ? a.chunks - 1 : 0) * a.channels + c] = 0.0f;
  auto put = [&](int i, const Map& m, float bi) {
    s = from(m, bi, s);
    if (in) out[(long long)(BACK ? a.chunks - 2 - i : i + 1) * a.channels + c] = s;
  };
  if (kept) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (first + i < end) put(first + i, mk[i], bk[i]);
  } else {
#pragma unroll 8
    for (int i = first; i < end; ++i) put(i, unpacked(at(i)[0]), at(i)[a.channels]);
  }
}

// ---- the states and the gradients -----------------------------------------------------------------------------------

// sequences without tokens, by the workgroups behind the chunks': what enters leaves as it is
__device__ __forceinline__ void empty_sequences(const Scan& a, const float* from, float* to) {
  const int extra = gridDim.x - a.chunks * a.groups, block = blockIdx.x - a.chunks * a.groups;
  const int waves = blockDim.x / 64, w = scan_uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  auto value = [&](int s) {
    const int x = s == 0 ? 0 : a.starts[s];
    return x < 0 ? 0 : x > a.tokens ? a.tokens : x;
  };
  for (long long s0 = ((long long)block * waves + w) * 64; s0 < a.seqs; s0 += (long long)extra * waves * 64) {
    const int s = (int)s0 + l;
    unsigned long long some = __ballot(s0 + l < a.seqs && value(s) >= value(s + 1));
    for (; some; some &= some - 1) {
      const long long row = (s0 + __builtin_ctzll(some)) * a.channels;
      for (int c = l; c < a.channels; c += 64) to[row + c] = from ? from[row + c] : 0.0f;
    }
  }
}

template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(64 * W) void k_scan(Scan a) {
  constexpr int CHUNK = W * TOK, NT = 64 * W;
  __shared__ int at[CHUNK + 1];
  __shared__ Joined<W, V> joined;
  if ((int)blockIdx.x >= a.chunks * a.groups) return empty_sequences(a, a.initial, a.last);
  // from the last chunk on: what the kernel of the chunks' P and B read last is still in the cache
  const int chunk = a.chunks - 1 - blockIdx.x / a.groups, w = scan_uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  const Lane<V> lane(a, blockIdx.x % a.groups);
  Few<T, V> f[TOK], x[TOK];
  load_tokens<T, V, TOK>(a.gate, a.g_t, a, chunk * CHUNK + w * TOK, lane.c, f);
  load_tokens<T, V, TOK>(a.x, a.x_t, a, chunk * CHUNK + w * TOK, lane.c, x);
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = chunk ? a.carry[(long long)chunk * a.channels + lane.c + e] : 0.0f;
  const int base = find_starts<CHUNK, NT>(a, chunk * CHUNK, at);
  const Stretch<TOK> st(a, at, base, chunk * CHUNK, w);
  const unsigned inside = st.cuts & ((1u << TOK) - 1);
  const int first = inside ? __builtin_ctz(inside) : 0;
  // on its way beside the tokens; further starts in the stretch read theirs when they come
  const auto first_state = state_of<V>(a, a.initial, inside ? st.sequence_at(first) : -1, lane.c);
  auto start = [&](int i, float* to) {
    auto s = first_state;
    if (i != first) s = state_of<V>(a, a.initial, st.sequence_at(i), lane.c);
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = s.v[e];
  };
  // What leads to each token from the state that enters its sequence in this stretch: P s + B, P as the gates' product, whose TOK
  // roundings at most end there; at a sequence's end, whose state goes on to other calls, the whole map.
  float to_p[TOK][V], to_b[TOK][V], p[V], q[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
#pragma unroll
  for (int i = 0; i < TOK; ++i) {  // tokens past the last sequence's end too: nothing takes what they lead to
    if (st.cuts >> i & 1)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (i) to_p[i - 1][e] = packed(p[e], q[e]);
        p[e] = 1.0f, q[e] = b[e] = 0.0f;
      }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float keep, take;
      gates<T>((float)f[i].v[e], keep, take);
      q[e] = fmaf(take, p[e], q[e]);
      p[e] *= keep;
      b[e] = fmaf(keep, b[e], take * (float)x[i].v[e]);
      to_p[i][e] = p[e], to_b[i][e] = b[e];
    }
  }
  float s0[V] = {};  // the last start's state
  if (inside) start(31 - __builtin_clz(inside), s0);
  Map whole[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    whole[e] = map_of(p[e], q[e]);
    joined.put(w, l, e, whole[e], mapped(whole[e], b[e], s0[e]));
  }
  if (l == 0) joined.drops[w] = inside != 0;
  __syncthreads();
  for (int o = 0; o < w; ++o) through(joined, o, s);
  if (!lane.counts) return;
  auto put = [&](int i, const float* f) { store_few<T, V>((T*)a.h + (long long)(st.t0 + i) * a.channels + (unsigned)lane.c, f); };
  int seq = st.seq;
  walk<T, V, TOK>(st, f,
                  [&](int i) {
                    start(i, s);
                    seq = st.sequence_at(i);
                  },
                  [&](int i) {
                    float h[V];
                    if (st.cuts >> (i + 1) & 1) {
                      float* last = a.last + (long long)seq * a.channels + (unsigned)lane.c;
#pragma unroll
                      for (int e = 0; e < V; ++e)
                        last[e] = h[e] = mapped(i + 1 == TOK ? whole[e] : unpacked(to_p[i][e]), to_b[i][e], s[e]);
                    } else {
#pragma unroll
                      for (int e = 0; e < V; ++e) h[e] = fmaf(to_p[i][e], s[e], to_b[i][e]);
                    }
                    put(i, h);
                  });
  const float none[V] = {};
#pragma unroll
  for (int i = 0; i < TOK; ++i)
    if (i >= st.live && i < st.there) put(i, none);
}

template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(64 * W, 4) void k_scan_vjp(Scan a) {
  constexpr int CHUNK = W * TOK, NT = 64 * W;
  __shared__ int at[CHUNK + 1];
  __shared__ Joined<W, V, false> ahead;  // to the gates' gradients alone
  __shared__ Joined<W, V> behind;
  if ((int)blockIdx.x >= a.chunks * a.groups) {
    if (a.dinitial) empty_sequences(a, a.dlast, a.dinitial);
    return;
  }
  const int chunk = a.chunks - 1 - blockIdx.x / a.groups, w = scan_uniform(threadIdx.x / 64), l = threadIdx.x % 64;
  const Lane<V> lane(a, blockIdx.x % a.groups);
  Few<T, V> f[TOK], x[TOK], d[TOK];
  load_tokens<T, V, TOK>(a.gate, a.g_t, a, chunk * CHUNK + w * TOK, lane.c, f);
  load_tokens<T, V, TOK>(a.x, a.x_t, a, chunk * CHUNK + w * TOK, lane.c, x);
  if (a.dh) load_tokens<T, V, TOK>(a.dh, a.d_t, a, chunk * CHUNK + w * TOK, lane.c, d);
  else
#pragma unroll
    for (int i = 0; i < TOK; ++i) d[i] = Few<T, V>{};
  float s[V], r[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s[e] = chunk ? a.carry[(long long)chunk * a.channels + lane.c + e] : 0.0f;
    r[e] = chunk < a.chunks - 1 ? a.back[(long long)chunk * a.channels + lane.c + e] : 0.0f;
  }
  const int base = find_starts<CHUNK, NT>(a, chunk * CHUNK, at);
  const Stretch<TOK> st(a, at, base, chunk * CHUNK, w);
  const unsigned inside = st.cuts & ((1u << TOK) - 1), later = st.cuts & ~1u;
  const int first = inside ? __builtin_ctz(inside) : 0, final = later ? 31 - __builtin_clz(later) : TOK + 1;
  // the sequence of the token before cut i (i > 0)
  auto before = [&](int i) {
    const unsigned starts = inside & ((1u << i) - 1);
    return starts ? st.sequence_at(31 - __builtin_clz(starts)) : st.seq;
  };
  const auto first_state = state_of<V>(a, a.initial, inside ? st.sequence_at(first) : -1, lane.c);
  const auto final_d = state_of<V>(a, a.dlast, later ? before(final) : -1, lane.c);
  auto start = [&](int i, float* to) {
    auto s = first_state;
    if (i != first) s = state_of<V>(a, a.initial, st.sequence_at(i), lane.c);
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = s.v[e];
  };
  auto end = [&](int i) {  // the token before cut i
    auto s = final_d;
    if (i != final) s = state_of<V>(a, a.dlast, before(i), lane.c);
    return s;
  };
  // Both ways' P and B in one walk: the other way's B is the sum of the cotangents, each times the product of the gates up to its
  // token, up to the first sequence's end. Gates are computed anew in each of the three walks: kept, they take the registers of
  // other waves (94 a lane for 70; 4096 short sequences 127 us for 119, long ones the same).
  float p[V], q[V], b[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = c[e] = 0.0f;
  const int led = later ? __builtin_ctz(later) : TOK;  // tokens that lead to the stretch's first without an end between
  auto led_d = final_d;
  if (led != final) led_d = state_of<V>(a, a.dlast, later ? st.seq : -1, lane.c);
  auto put_behind = [&] {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Map m = map_of(p[e], q[e]);
      behind.put(w, l, e, m, mapped(m, c[e], led_d.v[e]));
    }
  };
  walk<T, V, TOK>(st, f,
                  [&](int i) {
                    if (i == led) put_behind();
#pragma unroll
                    for (int e = 0; e < V; ++e) p[e] = 1.0f, q[e] = b[e] = 0.0f;
                  },
                  [&](int i) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                      float keep, take;
                      gates<T>((float)f[i].v[e], keep, take);
                      q[e] = fmaf(take, p[e], q[e]);
                      p[e] *= keep;
                      b[e] = fmaf(keep, b[e], take * (float)x[i].v[e]);
                      c[e] = fmaf(p[e], (float)d[i].v[e], c[e]);
                    }
                  });
  const bool plain = st.live == TOK && !st.cuts;
  auto walk_back = [&](auto ends, auto step) {  // from the last token on
    if (plain) {
#pragma unroll
      for (int i = TOK - 1; i >= 0; --i) step(i, std::false_type());
    } else {
#pragma unroll
      for (int i = TOK - 1; i >= 0; --i)
        if (i < st.live) {
          if (st.cuts >> (i + 1) & 1) ends(i + 1);
          step(i, std::true_type());
        }
    }
  };
  if (led >= st.live) put_behind();  // no sequence has started behind those
  float s0[V] = {};  // the last start's state
  if (inside) start(31 - __builtin_clz(inside), s0);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    ahead.put(w, l, e, {p[e], 0.0f}, fmaf(p[e], s0[e], b[e]));
  }
  if (l == 0) ahead.drops[w] = inside != 0, behind.drops[w] = later != 0;
  __syncthreads();
  for (int o = 0; o < w; ++o) through(ahead, o, s);
  for (int o = W - 1; o > w; --o) through(behind, o, r);
  if (!lane.counts) return;
  float off[TOK][V];  // how far the state before each token is from its x
  walk<T, V, TOK>(st, f, [&](int i) { start(i, s); },
                  [&](int i) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                      float keep, take;
                      gates<T>((float)f[i].v[e], keep, take);
                      off[i][e] = s[e] - (float)x[i].v[e];
                      s[e] = fmaf(keep, s[e], take * (float)x[i].v[e]);
                    }
                  });
  auto put = [&](void* to, int i, const float* f) {
    if (to) store_few<T, V>((T*)to + (long long)(st.t0 + i) * a.channels + (unsigned)lane.c, f);
  };
  walk_back([&](int i) {
              const auto s = end(i);
#pragma unroll
              for (int e = 0; e < V; ++e) r[e] = s.v[e];
            },
            [&](int i, auto cut) {  // cut: a sequence may start here, whose dinitial goes on to other calls
              float dx[V], dg[V];
#pragma unroll
              for (int e = 0; e < V; ++e) {
                float k, take;
                gates<T>((float)f[i].v[e], k, take);
                const float g = r[e] + (float)d[i].v[e];
                dx[e] = take * g;
                r[e] = cut ? stepped(k, take, 0.0f, g) : k * g;
                dg[e] = dx[e] * k * off[i][e];
              }
              put(a.dx, i, dx);
              put(a.dgate, i, dg);
              if ((st.cuts >> i & 1) && a.dinitial) {
                float* to = a.dinitial + (long long)st.sequence_at(i) * a.channels + (unsigned)lane.c;
#pragma unroll
                for (int e = 0; e < V; ++e) to[e] = r[e];
              }
            });
  const float none[V] = {};
#pragma unroll
  for (int i = 0; i < TOK; ++i)
    if (i >= st.live && i < st.there) put(a.dx, i, none), put(a.dgate, i, none);
}

// ---- one token a world ----------------------------------------------------------------------------------------------

struct Tick {
  const void *x, *gate;
  long long x_w, g_w, s_w;  // elements from world to world
  const float* state;
  long long worlds;
  int channels;
  void* h;
  float* next;
};

// Bytes bound it; a thread takes 16 bytes of x at a time, the last vector of a row ending with it, so that it holds elements of
// the one before again. Where the next states overwrite the states another thread may have written those already: there a row's
// last elements are taken singly, each by one thread.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(Tick a) {
  constexpr int E = Vec<T>::E;
  const int n = a.channels, nv = n / E + (n % E != 0);
  const long long all = a.worlds * nv;
  for (long long v = (long long)blockIdx.x * 256 + threadIdx.x; v < all; v += (long long)gridDim.x * 256) {
    const long long row = all >> 32 ? v / nv : (unsigned)v / (unsigned)nv;
    const int i = (int)(v - row * nv) * E, c = n >= E && i > n - E && a.next != a.state ? n - E : i;
    const T *x = (const T*)a.x + row * a.x_w + c, *g = (const T*)a.gate + row * a.g_w + c;
    const float* s = a.state + row * a.s_w + c;
    T* h = (T*)a.h + row * n + c;
    float* to = a.next + row * n + c;
    auto one = [](float f, float x, float s) {
      float keep, take;
      gates<T>(f, keep, take);
      return stepped(keep, take, x, s);
    };
    if (c <= n - E) {
      float xf[E], gf[E], sf[E];
      load_floats<E>(xf, x);
      load_floats<E>(gf, g);
      load_floats<E>(sf, s);
      Vec<T> o;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sf[e] = one(gf[e], xf[e], sf[e]);
        o.v[e] = rounded<T>(sf[e]);
      }
      store16(h, o);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        Vec<float> q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q.v[j] = sf[e + j];
        store16(to + e, q);
      }
    } else {
      for (int e = 0; e < n - c; ++e) {
        const float y = one((float)g[e], (float)x[e], s[e]);
        h[e] = rounded<T>(y);
        to[e] = y;
      }
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------

int scan_lanes(int type, int channels) { return type == F32 || channels < 2 ? 1 : 2; }  // channels a lane
int scan_groups(int type, int channels) {
  const int n = 64 * scan_lanes(type, channels);
  return channels / n + (channels % n != 0);
}
int scan_chunks(int tokens) { return tokens / SCAN_CHUNK + (tokens % SCAN_CHUNK != 0); }

template <typename F>
int scan_by_type(int type, int channels, F f) {
  switch (type * 2 + (scan_lanes(type, channels) == 2)) {
    case F32 * 2: return f(float(), std::integral_constant<int, 1>());
    case BF16 * 2: return f(__bf16(), std::integral_constant<int, 1>());
    case BF16 * 2 + 1: return f(__bf16(), std::integral_constant<int, 2>());
    case F16 * 2: return f(_Float16(), std::integral_constant<int, 1>());
    case F16 * 2 + 1: return f(_Float16(), std::integral_constant<int, 2>());
  }
  return (int)hipErrorInvalidValue;
}
unsigned scan_blocks(const Scan& a) {  // the chunks', and those that look for empty sequences
  const int extra = (a.seqs + 511) / 512;
  return (unsigned)(a.chunks * a.groups + (extra < 256 ? extra : 256));
}

// 8 channels a workgroup, in as many launches as keep the work-items of each below 2^32: one up to 2^24 channels
template <bool BACK>
int launch_carry(hipStream_t st, const Scan& a) {
  constexpr int MOST = 1 << 24;
  for (int c0 = 0; c0 < a.channels; c0 += MOST) {
    const int n = a.channels - c0 < MOST ? a.channels - c0 : MOST;
    k_scan_carry<BACK><<<(unsigned)((n + 7) / 8), 1024, 0, st>>>(a, c0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

int launch_scan(hipStream_t st, int type, const Scan& a) {
  return scan_by_type(type, a.channels, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = SCAN_CHUNK / SCAN_TOKENS;
    if (a.chunks > 1) {
      k_scan_parts<T, V, W, SCAN_TOKENS><<<(unsigned)((a.chunks - 1) * a.groups), 64 * W, 0, st>>>(a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
      const int rc = launch_carry<false>(st, a);
      if (rc) return rc;
    }
    const unsigned blocks = scan_blocks(a);
    if (blocks) k_scan<T, V, W, SCAN_TOKENS><<<blocks, 64 * W, 0, st>>>(a);
    return (int)hipGetLastError();
  });
}
int launch_scan_vjp(hipStream_t st, int type, const Scan& a) {
  return scan_by_type(type, a.channels, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = SCAN_CHUNK / SCAN_TOKENS;
    if (a.chunks > 1) {
      k_scan_back_parts<T, V, W, SCAN_TOKENS><<<(unsigned)((a.chunks - 1) * a.groups), 64 * W, 0, st>>>(a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
      const int rc = launch_carry<true>(st, a);
      if (rc) return rc;
    }
    const unsigned blocks = scan_blocks(a);
    if (blocks) k_scan_vjp<T, V, SCAN_CHUNK / SCAN_TOKENS_VJP, SCAN_TOKENS_VJP><<<blocks, 64 * SCAN_CHUNK / SCAN_TOKENS_VJP, 0, st>>>(a);
    return (int)hipGetLastError();
  });
}

bool scan_takes(int type, int tokens, int channels, int seqs) {
  return type >= 0 && type <= 2 && scan_sizes(tokens, channels, seqs);
}

}  // namespace pol

extern "C" {

int dk_recurrence(hipStream_t st, int type, int tokens, int channels, int seqs, const void* x, long long x_t, const void* gate,
                  long long gate_t, const int* starts, const float* initial, void* h, float* last, float* carry, void* work) {
  if (!pol::scan_takes(type, tokens, channels, seqs) || !starts || (seqs && !last) ||
      (tokens && (!x || !gate || !h || !carry || !work)))
    return (int)hipErrorInvalidValue;
  pol::Scan a = {};
  a.x = x, a.gate = gate, a.x_t = x_t, a.g_t = gate_t, a.tokens = tokens, a.channels = channels, a.seqs = seqs;
  a.chunks = pol::scan_chunks(tokens), a.groups = pol::scan_groups(type, channels), a.starts = starts, a.initial = initial;
  a.h = h, a.last = last, a.carry = carry, a.parts = (float*)work;
  return pol::launch_scan(st, type, a);
}

int dk_recurrence_vjp(hipStream_t st, int type, int tokens, int channels, int seqs, const void* x, long long x_t,
                      const void* gate, long long gate_t, const int* starts, const float* initial, const float* carry,
                      const void* dh, long long dh_t, const float* dlast, void* dx, void* dgate, float* dinitial, void* work) {
  if (!pol::scan_takes(type, tokens, channels, seqs) || !starts || (tokens && (!x || !gate || !carry || !work)))
    return (int)hipErrorInvalidValue;
  pol::Scan a = {};
  a.x = x, a.gate = gate, a.x_t = x_t, a.g_t = gate_t, a.tokens = tokens, a.channels = channels, a.seqs = seqs;
  a.chunks = pol::scan_chunks(tokens), a.groups = pol::scan_groups(type, channels), a.starts = starts, a.initial = initial;
  a.carry = const_cast<float*>(carry), a.dh = dh, a.d_t = dh_t, a.dlast = dlast, a.dx = dx, a.dgate = dgate;
  a.dinitial = dinitial, a.parts = (float*)work, a.back = a.parts + (long long)a.chunks * 2 * channels;
  return pol::launch_scan_vjp(st, type, a);
}

long long dk_recurrence_carry_bytes(int tokens, int channels) {
  return tokens > 0 && channels > 0 ? 4LL * pol::scan_chunks(tokens) * channels : 0;
}
long long dk_recurrence_work_bytes(int tokens, int channels, int vjp) {
  return dk_recurrence_carry_bytes(tokens, channels) * (vjp ? 3 : 2);
}

int dk_recurrence_step(hipStream_t st, int type, long long worlds, int channels, const void* x, long long x_w, const void* gate,
                       long long gate_w, const float* state, long long state_w, void* h, float* next) {
  if (type < 0 || type > 2 || worlds < 0 || channels < 1) return (int)hipErrorInvalidValue;
  if (worlds == 0) return 0;
  if (!x || !gate || !state || !h || !next) return (int)hipErrorInvalidValue;
  // the next states lie over the states row by row, or beside them
  const bool rows = worlds == 1 || state_w == channels;
  if (next == state ? !rows : rows && next < state + worlds * channels && state < next + worlds * channels)
    return (int)hipErrorInvalidValue;
  pol::Tick a = {};
  a.x = x, a.gate = gate, a.x_w = x_w, a.g_w = gate_w, a.state = state, a.s_w = state_w;
  a.worlds = worlds, a.channels = channels, a.h = h, a.next = next;
  const int e = type == pol::F32 ? 4 : 8;
  const long long need = (worlds * (channels / e + (channels % e != 0)) + 255) / 256, most = 16384;
  const unsigned blocks = (unsigned)(need < most ? need : most);
  if (type == pol::F32) pol::k_scan_step<float><<<blocks, 256, 0, st>>>(a);
  else if (type == pol::BF16) pol::k_scan_step<__bf16><<<blocks, 256, 0, st>>>(a);
  else pol::k_scan_step<_Float16><<<blocks, 256, 0, st>>>(a);
  return (int)hipGetLastError();
}

}  // extern "C"
