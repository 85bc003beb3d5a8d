// Attention of one new query a world over a history that lies in pages of a shared pool, with or without a window, and the
// writing of new keys and values into the pages.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the tokens j that the world's newest one sees: all, or the `window` last ones and
//       the `sinks` first ones; zeros where a world has no tokens, NaN where a page that holds one of them is not in the pool
//
// Memory bounds it: each key and value in sight is read once, for all the query heads that share it. As in the form over whole
// caches, a workgroup takes one world, one key/value head and one stretch of the tokens in sight, counted without the hidden
// ones; a key's 16-byte chunks lie across LPR lanes, scores come from two-element dot products, each group of LPR lanes keeps its
// own running maximum, sum and output in float32, and the groups are joined at the end. A turn reads the next one's keys and
// values ahead, and the page numbers of the turn after that, so that no read waits for another.
//
// Measured: 4096 worlds with up to 512 tokens in pages of 16, 8 heads on 2 of 64, 0.81 GB in 178 to 190 us (4.3 to 4.6 TB/s, of the
// 5.0 to 5.2 of a large copy); 4 worlds with up to 131072 tokens in pages of 64, 16 heads on 4 of 128, 0.9 GB in 178 us (5.1 TB/s)
// and 5.5 for the join; one world with a window of 256 and 4 sinks 6 us, a launch and four reads one after another. The append of
// a token each to 4096 worlds 5 us, to one 2.3.
#include "../../include/nablaengine_memory.h"
#include "policy_step.h"

namespace pol {

struct Paged {
  const void *q, *k, *v;
  long long q_w, q_h, k_p, k_t, k_h, v_p, v_t, v_h;  // elements from world to world, page to page, token to token, head to head
  int worlds, heads, kv_heads, group, dim;
  int count, shift, capacity;  // the pool's pages, log2 of a page's tokens, the tokens that a world's pages can hold
  const int* pages;            // (worlds, ..), pages_w apart
  long long pages_w;
  const int* lengths;
  int window, sinks;  // window 0: none
  float scale;
  void* out;  // (worlds, heads, dim)
  int stretches, stretch, units;
  float* part;  // (stretches, worlds, heads, dim + 2): output sums, running maximum, sum
};

template <typename T, int LPR, int GC, int W>
__global__ __launch_bounds__(256) void k_paged(Paged a) {
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
  // the tokens in sight: `sunk` first ones, then those from `skip` further on
  const int hidden = a.window && length > a.window ? length - a.window : 0, sunk = a.sinks < hidden ? a.sinks : hidden;
  const int skip = hidden - sunk, seen = length - skip;
  const long long from = (long long)stretch * a.stretch, to = from + a.stretch;
  const int begin = from < seen ? (int)from : seen, end = to < seen ? (int)to : seen;
  const bool in_row = d0 < a.dim;
  const int* table = a.pages + (long long)world * a.pages_w;
  const T* kp = (const T*)a.k + (long long)kv * a.k_h + d0;
  const T* vp = (const T*)a.v + (long long)kv * a.v_h + d0;
  const int mask = (1 << a.shift) - 1;
  int ahead = begin + w % W * BATCH + rg;  // of the turn whose page numbers are read next
  int page[UNROLL], slot[UNROLL];          // those of the turn whose keys are read next; slot -1: no token
  Vec<T> kn[UNROLL], vn[UNROLL];           // one turn ahead
  auto number = [&] {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = ahead + u * RPW, key = i < sunk ? i : i + skip;
      const bool in = i < end;
      page[u] = in ? table[key >> a.shift] : 0;
      slot[u] = in ? key & mask : -1;
    }
    ahead += W * BATCH;
  };
  auto read = [&] {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const bool known = (unsigned)page[u] < (unsigned)a.count;
      Vec<T> none = {};
      if (!known && slot[u] >= 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) none.v[e] = (T)NAN;
      const bool in = in_row && known && slot[u] >= 0;
      kn[u] = in ? load16(kp + page[u] * a.k_p + slot[u] * a.k_t) : none;
      vn[u] = in ? load16(vp + page[u] * a.v_p + slot[u] * a.v_t) : none;
    }
  };
  number();
  Vec<T> q[GC];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    q[g] = Vec<T>{};
    if (in_row && g0 + g < a.group)
      q[g] = load16((const T*)a.q + (long long)world * a.q_w + (long long)(kv * a.group + g0 + g) * a.q_h + d0);
  }
  read();
  number();
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
    number();
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

// ---- new tokens -----------------------------------------------------------------------------------------------------

struct Append {
  const unsigned short *k, *v;  // (tokens, kv_heads, dim) of 16 bits
  unsigned short *kp, *vp;      // (count, page, kv_heads, dim)
  long long k_t, k_h, v_t, v_h, kp_p, kp_t, kp_h, vp_p, vp_t, vp_h;
  int worlds, tokens, kv_heads, dim, count, shift, most;  // most: entries of a world's row of pages
  const int *starts, *pages, *lengths;                     // starts NULL: one token a world
  long long pages_w;
};

// A thread takes 16 bytes of every gridDim.y-th token of a world. Bytes bound it; the smallest call is a launch.
__global__ __launch_bounds__(256) void k_cache_append(Append a) {
  const int chunks = a.dim / 8, each = a.kv_heads * chunks;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int world = (int)(id / each), c = (int)(id - (long long)world * each), head = c / chunks, d = c % chunks * 8;
  if (world >= a.worlds) return;
  auto start = [&](int w) {
    const int x = !a.starts ? w : w == 0 ? 0 : a.starts[w];
    return x < 0 ? 0 : x > a.tokens ? a.tokens : x;
  };
  const int first = start(world), end = start(world + 1);
  const long long length = a.lengths[world];
  for (int t = first + (int)blockIdx.y; t < end; t += (int)gridDim.y) {
    const long long at = length + (t - first);
    if (at < 0 || at >> a.shift >= a.most) continue;  // no place for it
    const int page = a.pages[world * a.pages_w + (at >> a.shift)];
    if ((unsigned)page >= (unsigned)a.count) continue;
    const long long slot = at & ((1 << a.shift) - 1);
    store16(a.kp + page * a.kp_p + slot * a.kp_t + head * a.kp_h + d, load16(a.k + t * a.k_t + head * a.k_h + d));
    store16(a.vp + page * a.vp_p + slot * a.vp_t + head * a.vp_h + d, load16(a.v + t * a.v_t + head * a.v_h + d));
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------

int most_seen(int capacity, int window, int sinks) {
  return window && (long long)window + sinks < capacity ? window + sinks : capacity;
}
size_t paged_work_bytes(int worlds, int heads, int kv_heads, int dim, int seen) {
  if (worlds <= 0) return 0;
  const int n = step_stretches(worlds, kv_heads, heads / kv_heads, seen);
  return n == 1 ? 0 : sizeof(float) * (size_t)n * worlds * heads * (dim + 2);
}

template <typename T, int LPR, int GC>
void paged_units(hipStream_t st, const Paged& a) {
  if (a.stretches == 1 && a.units >= ALONE) k_paged<T, LPR, GC, 1><<<(a.units + 3) / 4, 256, 0, st>>>(a);
  else k_paged<T, LPR, GC, 4><<<a.units, 256, 0, st>>>(a);
}
template <typename T, int LPR>
int paged(hipStream_t st, Paged a) {
  const int gc = step_heads_a_group(a.group);
  const long long units = (long long)a.worlds * a.kv_heads * ((a.group + gc - 1) / gc) * a.stretches;
  if (units >= 1LL << 24 || (long long)a.worlds * a.heads >= 1 << 24) return (int)hipErrorInvalidValue;
  a.units = (int)units;
  switch (gc) {
    case 1: paged_units<T, LPR, 1>(st, a); break;
    case 2: paged_units<T, LPR, 2>(st, a); break;
    case 4: paged_units<T, LPR, 4>(st, a); break;
    default: paged_units<T, LPR, 8>(st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.stretches == 1) return (int)e;
  k_step_join<T, LPR><<<(unsigned)(a.worlds * a.heads), 1024, 0, st>>>(a);
  return (int)hipGetLastError();
}
int launch_paged(hipStream_t st, int type, Paged a) {
  const int seen = most_seen(a.capacity, a.window, a.sinks);
  a.stretches = step_stretches(a.worlds, a.kv_heads, a.group, seen);
  a.stretch = (seen + a.stretches - 1) / a.stretches;
  if (type == BF16) return a.dim <= 64 ? paged<__bf16, 8>(st, a) : paged<__bf16, 16>(st, a);
  return a.dim <= 64 ? paged<_Float16, 8>(st, a) : paged<_Float16, 16>(st, a);
}

// log2 of a page's tokens, or -1: not a power of two
int page_shift(int page) { return page >= 1 && !(page & (page - 1)) ? __builtin_ctz(page) : -1; }
bool cache_takes(int type, int worlds, int kv_heads, int dim, int count, int page, int most) {
  return (type == BF16 || type == F16) && worlds >= 0 && kv_heads >= 1 && dim >= 8 && dim <= 128 && dim % 8 == 0 && count >= 0 &&
         page_shift(page) >= 0 && most >= 0 && (long long)most * page < 1 << 30;
}

}  // namespace pol

extern "C" {

int dk_attention_paged(hipStream_t st, int type, int worlds, int heads, int kv_heads, int dim, int count, int page, int most,
                       const void* q, long long q_w, long long q_h, const void* k, long long k_p, long long k_t, long long k_h,
                       const void* v, long long v_p, long long v_t, long long v_h, const int* pages, long long pages_w,
                       const int* lengths, int window, int sinks, float scale, void* out, void* work) {
  if (!pol::cache_takes(type, worlds, kv_heads, dim, count, page, most) || heads < 1 || heads % kv_heads || window < 0 || sinks < 0 ||
      !(scale > 0.0f))
    return (int)hipErrorInvalidValue;
  if (worlds == 0) return 0;
  if (!q || !lengths || !out || (most && !pages) || (count && (!k || !v)) ||
      (!work && dk_attention_paged_work_bytes(worlds, heads, kv_heads, dim, page, most, window, sinks)))
    return (int)hipErrorInvalidValue;
  pol::Paged a = {};
  a.q = q, a.k = k, a.v = v, a.q_w = q_w, a.q_h = q_h;
  a.k_p = k_p, a.k_t = k_t, a.k_h = k_h, a.v_p = v_p, a.v_t = v_t, a.v_h = v_h;
  a.worlds = worlds, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim;
  a.count = count, a.shift = pol::page_shift(page), a.capacity = most * page, a.pages = pages, a.pages_w = pages_w;
  a.lengths = lengths, a.window = window, a.sinks = sinks, a.scale = scale, a.out = out, a.part = (float*)work;
  return pol::launch_paged(st, type, a);
}

long long dk_attention_paged_work_bytes(int worlds, int heads, int kv_heads, int dim, int page, int most, int window, int sinks) {
  if (worlds < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || page < 1 || most < 0 ||
      (long long)most * page >= 1 << 30 || window < 0 || sinks < 0)
    return 0;
  return (long long)pol::paged_work_bytes(worlds, heads, kv_heads, dim, pol::most_seen(most * page, window, sinks));
}

int dk_cache_append(hipStream_t st, int type, int worlds, int tokens, int kv_heads, int dim, int count, int page, int most,
                    const void* k, long long k_t, long long k_h, const void* v, long long v_t, long long v_h, const int* starts,
                    void* k_pages, long long kp_p, long long kp_t, long long kp_h, void* v_pages, long long vp_p, long long vp_t,
                    long long vp_h, const int* pages, long long pages_w, const int* lengths) {
  if (!pol::cache_takes(type, worlds, kv_heads, dim, count, page, most) || tokens < 0 || (!starts && tokens != worlds))
    return (int)hipErrorInvalidValue;
  const long long threads = (long long)worlds * kv_heads * (dim / 8);
  if (tokens == 0 || worlds == 0 || count == 0 || most == 0) return 0;
  // a world's tokens among as many workgroups as fill the GPU, 4 tokens each at least
  const long long blocks = (threads + 255) / 256, each = (tokens + worlds - 1LL) / worlds;
  long long split = 1;
  while (split < 32768 && split * 4 < each && split * blocks < 2048) split *= 2;
  if (blocks * split >= 1 << 23) return (int)hipErrorInvalidValue;
  if (!k || !v || !k_pages || !v_pages || !pages || !lengths) return (int)hipErrorInvalidValue;
  pol::Append a = {};
  a.k = (const unsigned short*)k, a.v = (const unsigned short*)v, a.kp = (unsigned short*)k_pages, a.vp = (unsigned short*)v_pages;
  a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.kp_p = kp_p, a.kp_t = kp_t, a.kp_h = kp_h, a.vp_p = vp_p, a.vp_t = vp_t, a.vp_h = vp_h;
  a.worlds = worlds, a.tokens = tokens, a.kv_heads = kv_heads, a.dim = dim, a.count = count, a.shift = pol::page_shift(page);
  a.most = most, a.starts = starts, a.pages = pages, a.pages_w = pages_w, a.lengths = lengths;
  pol::k_cache_append<<<dim3((unsigned)blocks, (unsigned)split), 256, 0, st>>>(a);
  return (int)hipGetLastError();
}

}  // extern "C"
