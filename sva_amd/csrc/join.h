// Joining the key ranges of split attention: each workgroup of a split call
// leaves, per query item and range, the maximum m of its scores (in base 2),
// the sum z of 2^(score - m) and the weighted sums of V, in fp32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sva {

struct JoinParams {
  const float* part;  // [n_seq * H * Q, splits, D + 2]: m, z, sums; z = 0: no key in the range, the sums are not read
  int splits, H, Q, D;
  const int64_t* q_lens;     // packed tokens: sequence b's are rows q_offsets[b] + t, t < q_lens[b], of q_rows;
  const int64_t* q_offsets;  // NULL: Q tokens of every sequence
  int64_t q_rows;
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

int launch_join(const JoinParams& p, int64_t n_seq, hipStream_t stream);

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

}  // namespace sva
