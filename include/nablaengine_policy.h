/* C ABI of the policy operators in libnablaengine_g1.so: what a policy trained through the control step is built from
 * and trained with (no counterpart in the reference, which stops at the step's gradients). The conventions are
 * nablaengine_g1.h's: every entry launches on the given stream, allocates nothing, waits for nothing, throws nothing
 * and returns 0 or a hipError_t (hipErrorInvalidValue before any launch for arguments it does not take). Element types
 * are 0 float32, 1 bfloat16, 2 float16; strides count elements; pointers need the element type's alignment only.
 * Everything is summed in float32 or float64 and rounded once to the output's type; no atomics touch a result, which
 * is bitwise the same on every run. No output overlaps an input or another output, but where an entry says so. */
#ifndef NABLAENGINE_POLICY_H
#define NABLAENGINE_POLICY_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* Layer norm of `rows` rows of n elements (x_row apart): y = (x - mean) / sqrt(var + eps) * w + b, y rows contiguous.
 * w, b: n elements of type w_type (0, or the type of x), each NULL for ones / zeros. stats: (2, rows) float32, mean
 * and reciprocal standard deviation for the backward, or NULL. */
int dk_layer_norm(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, int w_type,
                  const void* w, const void* b, float eps, void* y, float* stats);
/* Its VJP from the same x, w and the stats: dy rows dy_row apart; dx (rows contiguous), dw, db (type w_type), each NULL
 * where not wanted. work: dk_layer_norm_work_bytes(rows, n, type) bytes, NULL allowed without dw and db. No rows give
 * zero dw, db. */
int dk_layer_norm_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* dy,
                      long long dy_row, int w_type, const void* w, const float* stats, void* dx, void* dw, void* db,
                      void* work);
long long dk_layer_norm_work_bytes(long long rows, int n, int type);

/* The global norm of `count` gradients, norm[0] = sqrt(sum of all squares), and their clipping: out[i] = g[i] *
 * min(1, limit / (norm + 1e-6)). g, n, type (and out, out_type) are HOST arrays of device addresses, element counts
 * and types, read before the call returns; out[i] is g[i] itself or does not overlap any g; out_type[i] is type[i] or
 * 0. out NULL: the norm alone. A norm that is not finite makes the factor 0 (inf) or NaN. work:
 * dk_clip_work_bytes(count) bytes. */
int dk_clip(hipStream_t st, int count, const void* const* g, const long long* n, const int* type, void* const* out,
            const int* out_type, float limit, float* norm, void* work);
long long dk_clip_work_bytes(int count);

/* Causal attention over packed sequences. q (tq, heads, dim), k, v (tk, kv_heads, dim) in type 1 or 2, rows of dim
 * elements contiguous, q_t / q_h (...) elements from token to token and from head to head; heads a multiple of
 * kv_heads, query head i reading key/value head i / (heads / kv_heads); dim a multiple of 8, at most 128; tq * (heads /
 * kv_heads) and tk below 2^30, and (tq * (heads / kv_heads) / 128 + seqs) * kv_heads and (tk / 32 + seqs) * kv_heads a little
 * below 2^22 (a launch's work-items). starts_q, starts_k: seqs + 1 int32 on the device, 0 first: sequence s has the tokens
 * starts[s] .. starts[s + 1] - 1. Query i of a sequence of nq queries and nk keys sees its keys 0 .. i + nk - nq; one
 * that sees none gives zeros, as do tokens past the last sequence. out (tq, heads, dim) contiguous; lse (heads, tq)
 * float32 for the backward, or NULL; work: dk_attention_work_bytes bytes, which the backward reads again; scratch:
 * dk_attention_scratch_bytes bytes (vjp 0), or NULL when 0. scale > 0.
 * Offsets outside the tokens are moved inside them; they never make the call read or write out of bounds. */
int dk_attention(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                 long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v,
                 long long v_t, long long v_h, const int* starts_q, const int* starts_k, float scale, void* out,
                 float* lse, void* work, void* scratch);
/* Its VJP, from the forward's arguments, out, lse and work: dout (strides do_t, do_h) -> dq (tq, heads, dim), dk, dv
 * (tk, kv_heads, dim), contiguous. delta: (heads, tq) float32 scratch; scratch:
 * dk_attention_scratch_bytes bytes (vjp 1), or NULL when 0. */
int dk_attention_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk,
                     const void* q, long long q_t, long long q_h, const void* k, long long k_t, long long k_h,
                     const void* v, long long v_t, long long v_h, const int* starts_q, const int* starts_k,
                     float scale, const void* out, const float* lse, const void* work, const void* dout,
                     long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv,
                     void* scratch);
long long dk_attention_work_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk);
long long dk_attention_scratch_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk, int vjp);

/* Attention of one query a world over that world's cache: q (worlds, heads, dim), k, v (worlds, capacity, kv_heads,
 * dim) with elements from world to world (_w), token to token (_t) and head to head (_h); lengths: worlds int32 on the
 * device, the first lengths[w] tokens of world w count (below 0 is 0, above capacity is capacity; the others are never
 * read). out (worlds, heads, dim) contiguous, zeros for a world without tokens. work: dk_attention_step_work_bytes
 * bytes, or NULL when 0. */
int dk_attention_step(hipStream_t st, int type, int worlds, int heads, int kv_heads, int dim, int capacity,
                      const void* q, long long q_w, long long q_h, const void* k, long long k_w, long long k_t,
                      long long k_h, const void* v, long long v_w, long long v_t, long long v_h, const int* lengths,
                      float scale, void* out, void* work);
long long dk_attention_step_work_bytes(int worlds, int heads, int kv_heads, int dim, int capacity);

#ifdef __cplusplus
}
#endif
#endif
