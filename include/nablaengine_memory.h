/* C ABI of the operators of policies with a longer memory in libnablaengine_g1.so (no counterpart in the reference): a gated
 * linear recurrence, the gated residual between two blocks' norms, single-token attention over paged
 * histories, and attention over packed sequences with a window. The conventions are nablaengine_policy.h's. */
#ifndef NABLAENGINE_MEMORY_H
#define NABLAENGINE_MEMORY_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* The recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a = 1 / (1 + exp(-gate)), of each channel over packed sequences. x, gate:
 * (tokens, channels), x_t and gate_t elements from token to token; starts: seqs + 1 int32 on the device, 0 first: sequence s has
 * the tokens starts[s] .. starts[s + 1] - 1, not falling (offsets outside the tokens are moved inside them). initial: (seqs,
 * channels) float32, the states before the first tokens, or NULL for zeros. h (tokens, channels) contiguous, zeros behind the
 * last sequence; last (seqs, channels) float32, the states after the last tokens (of a sequence without tokens: its initial one).
 * carry: dk_recurrence_carry_bytes bytes, which the backward reads again; work: dk_recurrence_work_bytes bytes (vjp 0); both
 * NULL when 0. channels >= 1; a launch's work-items bound (tokens / 64) (channels / 64) by a little below 2^23. */
int dk_recurrence(hipStream_t st, int type, int tokens, int channels, int seqs, const void* x, long long x_t, const void* gate,
                  long long gate_t, const int* starts, const float* initial, void* h, float* last, float* carry, void* work);
/* Its VJP, from the forward's arguments and carry: dh (type, dh_t elements from token to token) and dlast (seqs, channels)
 * float32, each NULL for zeros -> dx, dgate (tokens, channels) contiguous, dinitial (seqs, channels) float32, each NULL where not
 * wanted. work: dk_recurrence_work_bytes bytes (vjp 1). */
int dk_recurrence_vjp(hipStream_t st, int type, int tokens, int channels, int seqs, const void* x, long long x_t,
                      const void* gate, long long gate_t, const int* starts, const float* initial, const float* carry,
                      const void* dh, long long dh_t, const float* dlast, void* dx, void* dgate, float* dinitial, void* work);
long long dk_recurrence_carry_bytes(int tokens, int channels);
long long dk_recurrence_work_bytes(int tokens, int channels, int vjp);
/* One token of every world: next = a state + (1 - a) x, float32, and h, its value in `type`; x, gate, state: (worlds, channels),
 * x_w, gate_w, state_w elements from world to world; h, next contiguous. next may be state where
 * that is contiguous, and lies apart from it otherwise. */
int dk_recurrence_step(hipStream_t st, int type, long long worlds, int channels, const void* x, long long x_w, const void* gate,
                       long long gate_w, const float* state, long long state_w, void* h, float* next);

/* The gated residual of `rows` rows of n elements: y = x + scale sg rms(u) w, z = rms(y) next_w (of the y that is not rounded),
 * rms(v) = v / sqrt(mean v^2 + eps), sg = 1 / (1 + exp(-gate)). Rows of x, u, gate (NULL: sg = 1) x_row, u_row, gate_row
 * elements apart, y and z contiguous; w, next_w, scale: n elements of type w_type (0, or the type of x), each NULL for ones.
 * stats: (2, rows) float32, both norms' factors for the backward, or NULL. */
int dk_gated_residual(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* u,
                      long long u_row, const void* gate, long long gate_row, int w_type, const void* w, const void* next_w,
                      const void* scale, float eps, void* y, void* z, float* stats);
/* Its VJP from the same inputs and the stats: rows of dy and dz (each NULL: zeros) dy_row and dz_row apart -> dx, du, dgate (rows
 * contiguous), dw, dnext_w, dscale (type w_type), each NULL where not wanted. work: dk_gated_residual_work_bytes bytes, NULL
 * allowed without dw, dnext_w and dscale. No rows give zero dw, dnext_w, dscale. */
int dk_gated_residual_vjp(hipStream_t st, long long rows, int n, int type, const void* x, long long x_row, const void* u,
                          long long u_row, const void* gate, long long gate_row, int w_type, const void* w, const void* next_w,
                          const void* scale, const float* stats, const void* dy, long long dy_row, const void* dz,
                          long long dz_row, void* dx, void* du, void* dgate, void* dw, void* dnext_w, void* dscale, void* work);
long long dk_gated_residual_work_bytes(long long rows, int n, int type);

/* Attention of one query a world over its history in pages: q (worlds, heads, dim); k, v: pools of `count` pages (count, page,
 * kv_heads, dim) with elements from page to page (_p), token to token (_t) and head to head (_h), page a power of two; pages:
 * (worlds, most) int32 on the device, rows pages_w apart: token j of world w is token j % page of page pages[w][j / page];
 * lengths: worlds int32 on the device, the world's tokens, its newest one's query being q (below 0 is 0, above most * page that).
 * window > 0: the query sees the window last tokens and the sinks first ones (0: all); what it does not see is not read, nor are
 * the entries of its pages. out (worlds, heads, dim) contiguous, zeros for a world without tokens, NaN for one that has a page
 * in sight whose number is none of the pool's. most * page < 2^30, worlds * heads < 2^24. work: dk_attention_paged_work_bytes
 * bytes, or NULL when 0. */
int dk_attention_paged(hipStream_t st, int type, int worlds, int heads, int kv_heads, int dim, int count, int page, int most,
                       const void* q, long long q_w, long long q_h, const void* k, long long k_p, long long k_t, long long k_h,
                       const void* v, long long v_p, long long v_t, long long v_h, const int* pages, long long pages_w,
                       const int* lengths, int window, int sinks, float scale, void* out, void* work);
long long dk_attention_paged_work_bytes(int worlds, int heads, int kv_heads, int dim, int page, int most, int window, int sinks);
/* New keys and values into the pages: k, v (tokens, kv_heads, dim), packed by starts (worlds + 1 int32 on the device, 0 first, not
 * falling), or one a world where starts is NULL (tokens = worlds). The i-th of world w becomes its token lengths[w] + i. One
 * that has no place, below 0, past `most` pages or on a page that is not in the pool, is dropped. */
int dk_cache_append(hipStream_t st, int type, int worlds, int tokens, int kv_heads, int dim, int count, int page, int most,
                    const void* k, long long k_t, long long k_h, const void* v, long long v_t, long long v_h, const int* starts,
                    void* k_pages, long long kp_p, long long kp_t, long long kp_h, void* v_pages, long long vp_p, long long vp_t,
                    long long vp_h, const int* pages, long long pages_w, const int* lengths);

/* dk_attention and its VJP with a window: of the keys that the causal mask leaves a query, it sees the `window` last ones and the
 * `sinks` first ones of its sequence (window 0, or as long as tk: all). rest: (tq, heads, dim) in the outputs' type, contiguous:
 * what their rounding took off, which the backward adds where it is given one; worth its bytes for windows of few keys, whose
 * outputs' rounding is felt in the gradients. NULL: none. work: dk_attention_work_bytes bytes. */
int dk_attention_window(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                        long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v, long long v_t,
                        long long v_h, const int* starts_q, const int* starts_k, float scale, int window, int sinks, void* out,
                        void* rest, float* lse, void* work, void* scratch);
int dk_attention_window_vjp(hipStream_t st, int type, int heads, int kv_heads, int dim, int seqs, int tq, int tk, const void* q,
                            long long q_t, long long q_h, const void* k, long long k_t, long long k_h, const void* v, long long v_t,
                            long long v_h, const int* starts_q, const int* starts_k, float scale, int window, int sinks,
                            const void* out, const void* rest, const float* lse, const void* work, const void* dout,
                            long long do_t, long long do_h, float* delta, void* dq, void* dk, void* dv, void* scratch);
long long dk_attention_window_scratch_bytes(int heads, int kv_heads, int dim, int seqs, int tq, int tk, int window, int sinks, int vjp);

#ifdef __cplusplus
}
#endif
#endif
