// The attention's and the recurrence's sizes, for their kernels and for the checks of whoever calls them (no device code).
#pragma once

namespace pol {

constexpr int QROWS = 128;  // query rows a workgroup: 32 a wave

// The most tiles that the packed sequences can have: QROWS rows of a key/value head's queries, 32 * key_waves keys.
constexpr long long order_queries(int seqs, int tq, int group) { return (long long)tq * group / QROWS + seqs + 1; }
constexpr long long order_keys(int seqs, int tk, int key_waves) { return (long long)tk / (32 * key_waves) + seqs + 1; }

// whether the kernels' indices and their grids hold these sizes
constexpr bool attention_sizes(int heads, int kv_heads, int seqs, int tq, int tk) {
  const int group = heads / kv_heads;
  const long long most = (1LL << 22) - 1024;  // workgroups of 256 or 512 work-items a launch
  return seqs >= 0 && tq >= 0 && tk >= 0 && tk < 1 << 30 && (long long)tq * group < 1 << 30 &&
         order_queries(seqs, tq, group) * kv_heads <= most && order_keys(seqs, tk, 1) * kv_heads <= most;
}

// Windows of so few keys (sinks among them) that the rounding of the outputs is felt in the gradients: what it took off is kept
// for the backward, as for rows of no more keys without a window.
constexpr int NARROW = 64;

constexpr int SCAN_TOKENS = 16, SCAN_TOKENS_VJP = 8, SCAN_CHUNK = 64;  // the recurrence's tokens a wave (of its backward) and a workgroup

// whether the recurrence's indices and grids hold these sizes: workgroups of 512 work-items, one a chunk and 64 channels at least
constexpr bool scan_sizes(int tokens, int channels, int seqs) {
  return tokens >= 0 && tokens < 0x7fffffff - 2 * SCAN_CHUNK && channels >= 1 && channels < 1 << 30 && seqs >= 0 &&
         seqs < 1 << 30 && ((long long)tokens / SCAN_CHUNK + 1) * ((long long)channels / 64 + 1) <= (1LL << 23) - 1024;
}

}  // namespace pol
