// What the attention kernels share: the arguments, the packed sequences, the matrix instructions and the LDS tiles.
//
// Layouts. The matrix instruction v_mfma_f32_32x32x16 takes A (32 x 16) and B (16 x 32), lane l holding row (column)
// l % 32 and the eight products k = 8 (l / 32) + 0..7, and gives C (32 x 32) with lane l holding column l % 32 and its
// register r row r % 4 + 8 (r / 4) + 4 (l / 32). Every product here is arranged so that one product's C is the next
// one's B as it stands: scores are computed transposed, S^T = K Q^T, so that a lane holds 16 keys of ONE query. Its
// softmax needs no exchange but one with lane l ^ 32, a rescaling is a product with the lane's own number, and the 16
// probabilities, packed to 16 bits, are the B operand of O^T = V^T P^T for two instructions, whose k then runs over the
// keys in the order 4 h + {0..3}, 8 + 4 h + {0..3} (h = l / 32). The A operand follows the same order: it is read from
// the row-major LDS tile with ds_read_b64_tr_b16, which gives each lane four consecutive rows of its column.
#pragma once
#include "policy_device.h"
#include "policy_sizes.h"

namespace pol {

typedef float F16x __attribute__((ext_vector_type(16)));
typedef short S4 __attribute__((ext_vector_type(4)));
template <typename T> struct Frag { typedef T V8 __attribute__((ext_vector_type(8))); };
template <typename T> using V8 = typename Frag<T>::V8;

__device__ __forceinline__ F16x mfma(V8<__bf16> a, V8<__bf16> b, F16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ F16x mfma(V8<_Float16> a, V8<_Float16> b, F16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr float LOG2E = 1.4426950408889634f;
// log2: by how much the subtracted maximum may lag behind the true one, and what probabilities are lifted by before they are
// rounded. float16 holds 2^-24 to 2^16: lifted by 2^11 those down to 2^-36 of the largest stay, so that the many small ones of
// a long history are not lost beside a large one (up to 2^24 keys they then miss less than half a rounding of the result).
// The backward's probabilities are those of the whole row, 1 at most: they can be lifted further.
template <typename T> struct Range { static constexpr float SLACK = 8.0f, LIFT = 0.0f, LIFT_BACK = 0.0f; };
template <> struct Range<_Float16> { static constexpr float SLACK = 4.0f, LIFT = 11.0f, LIFT_BACK = 14.0f; };
constexpr int TILE = 64;    // keys of an LDS tile of the forward and the queries' gradient

struct Attend {
  const void *q, *k, *v;
  long long q_t, q_h, k_t, k_h, v_t, v_h;  // elements from token to token, and from head to head
  int heads, kv_heads, group, dim, seqs, tq, tk;
  int by_sequence, grouped;  // bit `list`: its order, and whether its neighbours go to one XCD, see below
  int key_waves;  // 32 keys each: a tile of the keys' gradients (1 or 4)
  int parts_q, parts_k;  // workgroups (of a role) among which a query tile's keys, a key tile's rows are split
  const int *starts_q, *starts_k;
  float scale;
  float* scratch;  // their sums, one slot each
  void* out;   // (tq, heads, dim)
  float* lse;  // (heads, tq): log2 of the row's sum of exponentials, +inf for a row without keys; NULL: not kept
  const int* order;
  // the backward's
  const void* dout;
  long long do_t, do_h;
  float* delta;  // (heads, tq): the row's dout . out
  void *dq, *dk, *dv;
  // a window (WIN kernels): key j of a row whose last key is i is seen if j > i - window or j < sinks
  int window, sinks;
  void* rest;  // (tq, heads, dim): what the outputs' rounding took off, for delta; NULL: not kept
  // the sinks' gradients from rows whose window has passed them: parts of far_tokens tokens, 0: with the others
  int far_tokens, far_least, far_chunks;
  float* far;
};

// whether the window hides key j from a row whose last key is i
__device__ __forceinline__ bool window_hides(const Attend& a, int j, int i) { return j <= i - a.window && j >= a.sinks; }

// The order: two lists of tiles, (sequence, tile of it): the query tiles (QROWS rows of a key/value head's queries, row =
// token * group + head of the group) and the key tiles (32 * key_waves keys). A list is heaviest first, by the tiles of
// the other side that each one reads: over all tiles, or over sequences, each one's tiles one after another (by_sequence).
// Workgroups go to the XCDs in turn, and each XCD has an L2 cache of its own: in the second case WINDOW neighbours of the
// list go to one XCD, so that a sequence's tiles find what they share in one cache; in the first a list's neighbours are
// tiles of different sequences and heads anyway. With a window a list's neighbours always go to one XCD (two sequences of
// 8192, window 1000, heads of 128: forward 115 -> 107 us, dq 143 -> 135). order_queries() and order_keys() are the lists'
// lengths at most.
constexpr int WINDOW = 64, XCDS = 8;
constexpr int LONG = 1792;  // tokens a sequence, in the mean: above it single tiles are ordered
constexpr int ORDER_HEAD = 16;  // ints before the lists: their lengths

// A tile's loop over `tiles` tiles of the other side, split among `parts` workgroups (at least LEAST each): this one's.
constexpr int LEAST = 4;
struct Slice {
  int first, end, parts;  // parts: those that have any, and one where none has
  __host__ __device__ __forceinline__ Slice(int tiles, int most, int part) {
    const int split = (tiles + most - 1) / most, each = split > LEAST ? split : LEAST;
    first = part * each < tiles ? part * each : tiles;
    end = first + each < tiles ? first + each : tiles;
    parts = tiles > each ? (tiles + each - 1) / each : 1;
  }
};

// Sequence s of the packed tokens [0, total): its first token and length, kept inside the tokens whatever `starts`
// holds. Sequence `seqs` is what lies past the last one: its queries have no keys and its keys no queries.
__device__ __forceinline__ void sequence(const int* starts, int s, int seqs, int total, int& first, int& length) {
  auto in = [&](int x) { return x < 0 ? 0 : x > total ? total : x; };
  first = s == 0 ? 0 : in(starts[s]);
  const int end = s == seqs ? total : in(starts[s + 1]);
  length = end > first ? end - first : 0;
}

// An LDS tile of TILE rows of DP elements in 16-byte chunks. Chunk c of row r lies at chunk c ^ swizzle(r), so that
// both reads are free of bank conflicts: 16 rows of one chunk (A operands, 16 bytes a lane) and 4 rows of 4 chunks
// (transposed reads, 8 bytes a lane, 32 lanes at a time). A row of 64 elements is half of the 64 banks, one of 128 all.
template <int DP>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (DP == 64) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
  else return (r & 3) << 2 | ((r >> 2) & 3);
}
template <int DP>
__device__ __forceinline__ int chunk_at(int r, int c) { return r * DP + ((c ^ swizzle<DP>(r)) << 3); }

// rows of A (row n of the 32 from r0, products 16 s + 8 h ..)
template <int DP, typename T>
__device__ __forceinline__ V8<T> read_rows(const T* tile, int r0, int s, int n, int h) {
  return *(const V8<T>*)(tile + chunk_at<DP>(r0 + n, 2 * s + h));
}
// columns 32 t + l % 32 as rows of A, products over the tile's rows r0 + 4 h + {0..3}, r0 + 8 + 4 h + {0..3}
template <int DP, typename T>
__device__ __forceinline__ V8<T> read_columns(const T* tile, int r0, int t, int l) {
  typedef __attribute__((address_space(3))) S4 L4;
  const int r = r0 + 4 * (l >> 5) + ((l & 15) >> 2), d = 32 * t + (l & 16) + 4 * (l & 3);
  const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4*)(tile + chunk_at<DP>(r, d >> 3) + (d & 7)));
  const S4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4*)(tile + chunk_at<DP>(r + 8, d >> 3) + (d & 7)));
  typedef short S8 __attribute__((ext_vector_type(8)));
  const S8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(V8<T>, both);
}
// registers 8 s .. 8 s + 7 of a C, packed: products k of B
template <typename T>
__device__ __forceinline__ V8<T> pack(const F16x& c, int s) {
  typedef float F8 __attribute__((ext_vector_type(8)));
  const F8 f = s ? __builtin_shufflevector(c, c, 8, 9, 10, 11, 12, 13, 14, 15) : __builtin_shufflevector(c, c, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_convertvector(f, V8<T>);
}

// Score gradients on their way to 16 bits. bfloat16 has the range of float32. float16 has not: over a long history, or where
// the loss is a mean, they are far below its smallest step of 2^-24, and where the loss is scaled they pass its 2^16. Each
// column (a query's, a key's) has a factor, a power of two: the first gradients that are not 0 are brought to 2^7, and later
// ones that pass 2^15 lower the factor, and with it the sums so far. The sums are divided by it at the end. Forward and backward
// in float16 without and with it, a call alone: 4096 sequences of up to 32 tokens, 8 heads on 2 of 64, 219 and 225 us; 256 of up to 1000
// 1079 and 1130; 8192 and 2752 tokens, 16 on 4 of 128, 1912 and 1973.
template <typename T> struct Lift {
  template <int N>
  __device__ __forceinline__ void scale(F16x&, F16x*) {}
  template <int N>
  __device__ __forceinline__ void unscale(F16x*, float) const {}
};
template <> struct Lift<_Float16> {
  float f = 0.0f;  // 0: none yet
  template <int N>
  __device__ __forceinline__ void scale(F16x& ds, F16x* acc) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(ds[j]));
    auto other = [&](float t) { return f == 0.0f ? t > 0.0f : t * f > 32768.0f; };
    if (__any(other(top))) {
      top = max_halves(top);
      if (other(top)) {
        const int e = 261 - (int)(__float_as_uint(top) >> 23);  // of 2^7 / top, between 2^-100 and 2^100
        const float f1 = __uint_as_float((unsigned)(e < 27 ? 27 : e > 227 ? 227 : e) << 23), less = f == 0.0f ? 1.0f : f1 / f;
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[d][j] *= less;
        f = f1;
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) ds[j] *= f;
  }
  // the sums of products with the scaled gradients, without the factor and times `more`
  template <int N>
  __device__ __forceinline__ void unscale(F16x* acc, float more) const {
    const float g = f == 0.0f ? 1.0f : more / f;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[d][j] *= g;
  }
};

// Infinities and NaN under the mask. A masked probability is 0, but 0 times an infinity in a row that the mask hides is
// NaN: such sums are not what the mask asks for. The kernels do not look for them; they look at their results, and compute
// a row (a key) whose sums are not finite once more, over what it sees alone, one product after another in float32. That
// takes long, and nothing where all is finite.
// 0, or NaN where a register is not finite
template <int N>
__device__ __forceinline__ float not_finite(const F16x* acc) {
  float t = 0.0f;
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) t = fmaf(acc[d][j], 0.0f, t);
  return t;
}
// columns for which `bad` holds in either half of the wave
__device__ __forceinline__ unsigned bad_columns(bool bad) {
  const unsigned long long b = __ballot(bad);
  return (unsigned)b | (unsigned)(b >> 32);
}
// a row's elements l and l + 64 of up to DP
template <int DP>
struct Row {
  float x[DP / 64];
  Row() = default;
  template <typename T>
  __device__ __forceinline__ Row(const T* p, int dim) {
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
      const int d = threadIdx.x % 64 + 64 * i;
      x[i] = d < dim ? (float)p[d] : 0.0f;
    }
  }
  __device__ __forceinline__ float dot(const Row& o) const {
    float s = x[0] * o.x[0];
#pragma unroll
    for (int i = 1; i < DP / 64; ++i) s += x[i] * o.x[i];
    return sum_lanes<64>(s);
  }
  __device__ __forceinline__ void add(float f, const Row& o) {
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) x[i] += f * o.x[i];
  }
  __device__ __forceinline__ bool all_nan(int dim) const {  // nothing more changes it
    bool nan = true;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) nan &= (int)threadIdx.x % 64 + 64 * i >= dim || x[i] != x[i];
    return __all(nan);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p, int from, int to, float f) const {  // elements from .. to - 1
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
      const int d = threadIdx.x % 64 + 64 * i;
      if (d >= from && d < to) p[d] = (T)(x[i] * f);
    }
  }
};

// 2^x in one instruction: results below 2^-126 become 0, which a sum of exponentials up to 1 does not notice
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A tile on its way from memory to LDS without passing registers: each lane gives the address of its 16 bytes, which
// land lane after lane; a lane without any gives that of zeros. All of a wave's are there after loads_done().
__device__ __align__(16) const unsigned no_row[4] = {0, 0, 0, 0};
template <typename T>
__device__ __forceinline__ void to_lds(const T* from, bool valid, T* wave_at) {
  typedef __attribute__((address_space(1))) const void* G;
  typedef __attribute__((address_space(3))) void* L;
  const T* p = valid ? from : (const T*)no_row;
  __builtin_amdgcn_global_load_lds((G)p, (L)wave_at, 16, 0, 0);
}
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// The compiler moves nothing across: LDS reads that a phase issues ahead of the next one's use stay ahead. Left to
// itself it puts each read just before its product, and waits for every one.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

template <typename T>
__device__ __forceinline__ V8<T> zero8() { return V8<T>{}; }

template <typename T>
__device__ __forceinline__ V8<T> load8(const T* p) {
  V8<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}

// 32 rows' B operands straight from memory: lane's row p (NULL: none), products 16 s + 8 h ..
template <int DP, typename T>
__device__ __forceinline__ void load_rows(const T* p, int dim, int h, V8<T>* f) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * h;
    f[s] = p && d < dim ? load8(p + d) : zero8<T>();
  }
}

// A C of columns = rows of a result (transposed result), d = d0 + 32 t + register's row, to p (NULL: none), times f
template <int N, typename T>
__device__ __forceinline__ void store_rows(T* p, int d0, int dim, int h, const F16x* acc, float f) {
  if (!p) return;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = d0 + 32 * t + 8 * j + 4 * h;
      if (d < dim) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)(acc[t][4 * j + e] * f);
        __builtin_memcpy(p + d, &o, 8);
      }
    }
}

// what store_rows' rounding takes off, rounded in its turn
template <int N, typename T>
__device__ __forceinline__ void store_rests(T* p, int d0, int dim, int h, const F16x* acc, float f) {
  if (!p) return;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = d0 + 32 * t + 8 * j + 4 * h;
      if (d < dim) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[t][4 * j + e] * f;
          o[e] = f == 0.0f ? (T)0.0f : (T)(x - (float)(T)x);
        }
        __builtin_memcpy(p + d, &o, 8);
      }
    }
}

}  // namespace pol
