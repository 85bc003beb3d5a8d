// The attention's sizes, for its kernels and for the checks of whoever calls them (no device code).
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

}  // namespace pol
