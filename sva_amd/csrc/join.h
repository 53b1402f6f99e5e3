// Joining the key ranges of split attention: each workgroup of a split call
// leaves, per query item and range, a reference m that its scores q . K do not
// pass by much, the sum z of the weights 2^((score - m) sl) and the weighted
// sums of V, in fp32.  References are kept before the scale: differences of
// close scores are then exact, whatever their size.  A z below 0 says that its
// weights and sums were taken 2^-60 times (V near the largest number).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sva {

struct JoinParams {
  const float* sums;   // [n_seq * H * Q, splits, D]
  const float* stats;  // [n_seq * H * Q, splits, 2]: m, z; a range in which the item sees no key: z and sums of 0
  float sl;            // score_scale(scaling)
  int splits, H, G, Q, D;
  const int64_t* q_lens;     // packed tokens: sequence b's are rows q_offsets[b] + t, t < q_lens[b], of q_rows;
  const int64_t* q_offsets;  // NULL: Q tokens of every sequence
  int64_t q_rows;
  const int64_t* lens;  // keys: seq_keys
  const int64_t* offs;
  int64_t N, rows;
  int tile_rows;  // query rows that one workgroup takes
  int chunk;      // keys of a range
  bool causal;
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

// Bytes of the sums and stats of `items` items, the stats' first.
inline size_t join_bytes(int64_t items, int64_t splits, int64_t D) {
  return sizeof(float) * (size_t)(items * splits) * (size_t)(D + 2) + 256;
}
inline int64_t join_stats_floats(int64_t items, int64_t splits) { return (items * splits * 2 + 3) / 4 * 4; }

int launch_join(const JoinParams& p, int64_t n_seq, hipStream_t stream);

constexpr float kShifted = 0x1p-60f;

// What turns a score q . K (of -q, where the scale is below 0) into a base-2
// exponent.  (A scale of 0: the smallest normal number gives the same weights,
// and -inf times it stays -inf.)
__host__ __device__ inline float score_scale(float scaling) {
  const float sl = (scaling < 0.0f ? -scaling : scaling) * 1.44269504088896340736f;
  return sl > 1.17549435e-38f ? sl : (sl <= 1.17549435e-38f ? 1.17549435e-38f : sl);
}

// Tokens of packed sequence b and the row of its first, inside [0, q_rows).
__device__ inline int seq_tokens(const int64_t* q_lens, const int64_t* q_offsets, int64_t q_rows, int Q, int b,
                                 int64_t& first) {
  first = 0;
  if (!q_lens) return Q;
  first = q_offsets[b];
  if (first < 0 || first >= q_rows) return 0;
  int64_t n = q_lens[b];
  n = n < q_rows - first ? n : q_rows - first;
  n = n < Q ? n : Q;
  return n > 0 ? (int)n : 0;
}

// Keys of sequence b and the cache row of its first, inside [0, rows) and no
// more than N.
__device__ inline int64_t seq_keys(const int64_t* lens, const int64_t* offs, int64_t N, int64_t rows, int b,
                                   int64_t& off) {
  off = offs ? offs[b] : 0;
  if (off < 0 || off >= rows) return 0;
  int64_t n = lens ? lens[b] : N;
  n = n < N ? n : N;
  n = n < rows - off ? n : rows - off;
  return n > 0 ? n : 0;
}

// The end of the keys that some row of tile rt sees, of q_len tokens x grp
// heads over len keys, and the ranges of `chunk` keys up to it (at least 1).
// A tile of one range writes its outputs itself; the others are joined.
__device__ inline int64_t tile_keys(int rt, int tile_rows, int q_len, int grp, int64_t len, bool causal) {
  if (!causal) return len;
  const int64_t rows = (int64_t)q_len * grp, end = (int64_t)(rt + 1) * tile_rows;
  const int64_t last_token = ((end < rows ? end : rows) - 1) / grp;
  const int64_t keys = last_token + len - q_len + 1;
  return keys < 0 ? 0 : (keys < len ? keys : len);
}
__device__ inline int tile_ranges(int64_t keys, int64_t chunk) {
  return keys <= chunk ? 1 : (int)((keys + chunk - 1) / chunk);
}

}  // namespace sva
