// Dense attention of whole prompts (sva_prompt_attention): argument checks,
// the choice of tile and of key ranges, launches.  The kernel: prompt.cuh.
#include <algorithm>

#include "prompt_launch.h"

using namespace sva;

namespace {

constexpr int BM = 128;  // query rows of a workgroup

int64_t row_tiles(int64_t H, int64_t G, int64_t Q) { return (H / G * Q + BM - 1) / BM; }

// Keys per workgroup: all of them, or ranges of at least 256.  The row tiles
// of whole prompts are of every length, and dispatch evens them out: they are
// split only where they do not fill the card once.  Tokens over a cache that
// is much longer make row tiles of one length: about five workgroups for each
// of the two places of a CU (head_dim above 128, and fp32 above 64, have one
// place, and so ten workgroups for it), so that a last round of them is a small part;
// fewer where there are many rows, whose sums go through memory once for each
// range.  (9 x 64 bf16: 8192 whole tokens 120 us in one range, 145 with a
// second behind key 4736; 512 tokens each over 8 x 32768 keys 530 us in two
// ranges, 437 in six, 462 in nine, 520 in 16; a token each of 32 sequences of
// up to 131072 keys 376 us in eight, 289 in 28, 318 in 64; 12 x 64 fp32, 1001
// tokens 77 us in one, 46 in three, 51 in four.)
int64_t chunk_keys(int64_t n_seq, int64_t H, int64_t G, int64_t Q, int64_t n_keys) {
  const int64_t tiles = n_seq * G * row_tiles(H, G, Q), cus = sva::device_cu_count();
  const int64_t places = n_seq * H * Q > 8192 ? 7 * cus : 10 * cus;
  const int64_t want = 2 * Q > n_keys ? (cus + tiles - 1) / tiles : (places + tiles / 2) / tiles;
  const int64_t ranges = std::max<int64_t>(1, std::min<int64_t>(64, want));
  return std::max<int64_t>(256, ((n_keys + ranges - 1) / ranges + 63) / 64 * 64);
}

// (few rows: their second terms cost nothing there; from 17 rows on they would
// need columns of their own, prompt.cuh)
template <int DT>
int launch_type(const PromptParams& p, bool vec, hipStream_t stream) {
  if constexpr (DT != F32) {
    if ((int64_t)p.H / p.G * p.Q <= kFewRows) return launch_prompt_few(p, DT, vec, stream);
  }
  return launch_prompt<DT, 0>(p, vec, stream);
}

}  // namespace

extern "C" size_t sva_prompt_attention_workspace_bytes(int64_t n_seq, int64_t H, int64_t G, int64_t Q, int64_t D,
                                                       int64_t n_keys) {
  if (n_seq <= 0 || H <= 0 || G <= 0 || Q <= 0 || D <= 0 || n_keys <= 0 || H % G != 0) return 0;
  const int64_t chunk = chunk_keys(n_seq, H, G, Q, n_keys);
  const int64_t splits = (n_keys + chunk - 1) / chunk;
  return splits == 1 ? 256 : join_bytes(n_seq * H * Q, splits, D);
}

extern "C" int sva_prompt_attention(const void* q, int dtype, int64_t q_seq_stride, int64_t q_head_stride,
                                    int64_t q_tok_stride, const int64_t* q_offsets, const int64_t* q_lens,
                                    int64_t q_rows, const void* keys, const void* values, int64_t kv_head_stride,
                                    int64_t kv_row_stride, int64_t kv_rows, const int64_t* seq_offsets,
                                    const int64_t* seq_lens, int64_t n_keys, int64_t n_seq, int64_t H, int64_t G,
                                    int64_t Q, int64_t D, float scaling, const void* mask, int mask_type,
                                    int64_t mask_seq_stride, int64_t mask_tok_stride, void* out, int out_dtype,
                                    int64_t out_seq_stride, int64_t out_head_stride, int64_t out_tok_stride,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(q && keys && values && out, "sva_prompt_attention: null pointer");
  SVA_REQUIRE((seq_offsets == nullptr) == (seq_lens == nullptr) && (q_offsets == nullptr) == (q_lens == nullptr),
              "sva_prompt_attention: offsets and lengths go together");
  SVA_REQUIRE(seq_offsets || n_seq == 1, "sva_prompt_attention: several sequences need offsets and lengths");
  SVA_REQUIRE(n_seq > 0 && H > 0 && G > 0 && Q > 0 && n_keys > 0 && kv_rows > 0 && H % G == 0 &&
                  (!q_lens || q_rows > 0),
              "sva_prompt_attention: bad sizes");
  SVA_REQUIRE(D > 0 && D <= 256, "sva_prompt_attention: head_dim %lld out of range (at most 256)", (long long)D);
  SVA_REQUIRE(dtype >= 0 && dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, "sva_prompt_attention: bad dtype");
  SVA_REQUIRE((mask == nullptr) == (mask_type == SVA_MASK_NONE) && mask_type >= 0 && mask_type <= 4,
              "sva_prompt_attention: bad mask type");
  SVA_REQUIRE(!mask || !q_lens, "sva_prompt_attention: packed tokens take no mask");
  SVA_REQUIRE(n_keys < (1ll << 31) - 1024 && n_seq < (1ll << 31) && H < (1ll << 20) && Q < (1ll << 31) &&
                  H * Q < (1ll << 31) && n_seq * H < (1ll << 31) && n_seq * H * Q < (1ll << 31),
              "sva_prompt_attention: too many items or keys");
  SVA_REQUIRE(kv_row_stride >= 0 && kv_row_stride < (1ll << 23), "sva_prompt_attention: row stride out of range");
  const size_t need = sva_prompt_attention_workspace_bytes(n_seq, H, G, Q, D, n_keys);
  SVA_REQUIRE(workspace != nullptr && workspace_bytes >= need, "sva_prompt_attention: workspace of %zu bytes required",
              need);
  const int64_t word = dtype == F32 ? 4 : 8;  // elements of 16 bytes
  PromptParams p;
  p.q = q;
  p.q_bs = q_seq_stride;
  p.q_hs = q_head_stride;
  p.q_ts = q_tok_stride;
  p.q_offsets = q_offsets;
  p.q_lens = q_lens;
  p.q_rows = q_rows;
  p.keys = keys;
  p.values = values;
  p.kv_hs = kv_head_stride;
  p.kv_rs = kv_row_stride;
  p.kv_rows = kv_rows;
  p.offs = seq_offsets;
  p.lens = seq_lens;
  p.N = n_keys;
  p.n_seq = (int)n_seq;
  p.H = (int)H;
  p.G = (int)G;
  p.Q = (int)Q;
  p.D = (int)D;
  p.row_tiles = (int)row_tiles(H, G, Q);
  p.chunk = (int)chunk_keys(n_seq, H, G, Q, n_keys);
  p.splits = (int)((n_keys + p.chunk - 1) / p.chunk);
  const bool vec = (D == 64 || D == 128 || D == 256) && (((uintptr_t)q | (uintptr_t)keys | (uintptr_t)values) & 15u) == 0 &&
                   q_seq_stride % word == 0 && q_head_stride % word == 0 && q_tok_stride % word == 0 &&
                   kv_head_stride % word == 0 && kv_row_stride % word == 0;
  p.scaling = scaling;
  p.mask = mask;
  p.mask_type = mask_type;
  p.mask_bs = mask_seq_stride;
  p.mask_ts = mask_tok_stride;
  p.stats = (float*)workspace;
  p.sums = p.stats + join_stats_floats(n_seq * H * Q, p.splits);
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_vec = D % 4 == 0 && ((uintptr_t)out & 15u) == 0 && out_seq_stride % 4 == 0 && out_head_stride % 4 == 0 &&
              out_tok_stride % 4 == 0;
  p.o_bs = out_seq_stride;
  p.o_hs = out_head_stride;
  p.o_ts = out_tok_stride;
  SVA_REQUIRE((int64_t)p.G * p.row_tiles * p.splits * n_seq < (1ll << 31), "sva_prompt_attention: too many items");
  int rc;
  if (dtype == F32) rc = launch_type<F32>(p, vec, (hipStream_t)stream);
  else if (dtype == BF16) rc = launch_type<BF16>(p, vec, (hipStream_t)stream);
  else rc = launch_type<F16>(p, vec, (hipStream_t)stream);
  if (rc != SVA_OK || p.splits == 1) return rc;
  JoinParams j;
  j.sums = p.sums;
  j.stats = p.stats;
  j.sl = score_scale(scaling);
  j.splits = p.splits;
  j.H = p.H;
  j.G = p.G;
  j.lens = seq_lens;
  j.offs = seq_offsets;
  j.N = n_keys;
  j.rows = kv_rows;
  j.tile_rows = BM;
  j.chunk = p.chunk;
  j.causal = mask == nullptr;
  j.Q = p.Q;
  j.D = p.D;
  j.q_lens = q_lens;
  j.q_offsets = q_offsets;
  j.q_rows = q_rows;
  j.out = out;
  j.out_dtype = out_dtype;
  j.o_bs = out_seq_stride;
  j.o_hs = out_head_stride;
  j.o_ts = out_tok_stride;
  return sva::launch_join(j, n_seq, (hipStream_t)stream);
}
