// Attention of a few tokens over every row of a KV cache held in 4 bits.
//
// out[h, t] = sum_n p[n] V[n] / sum_n p[n], p[n] = exp(s (q[h, t] . K[n]) - m)
// over the rows n <= len - Q + t of the sequence, in one pass over the cache
// with a running maximum m.  What it has to read is 17 / 32 bytes per element
// of K and V; a tile's rows serve every query row (token, head of the KV
// group) of the workgroup, so the matrix products take 16 query rows at a
// time: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16.
//  * K codes become bf16 in registers (exact: a code times a power of two).
//    A lane holds D / 4 consecutive elements of one key, the operand's
//    elements in an order of their own that the query operand shares.
//  * The query is split into NT bf16 terms (bf16: 1, fp16: 2, fp32: 3, all
//    its bits), the weights into 2 (16 bits): the products keep about fp32's
//    accuracy while the cache, not the matrix cores, sets the time (one term of
//    the weights would save 8 % at head_dim 64).
//  * S^T leaves a lane with 8 scores of one query row, which are its share of
//    the P^T operand: weights never cross lanes.  V goes through LDS, each
//    wave its own 32 rows, and comes back transposed (ds_read_b64_tr_b16).
//  * V near the type's largest meets weights of 2^-60 (the reference lies 60
//    above the maximum from the first such block on): its sums stay finite.
//  * A block that reads as NaN is kept out of V (0 * NaN would reach rows that
//    may not see it) and marks the query rows that may.
// Workgroups split the keys (partials joined by a second kernel), a
// workgroup's four waves take its 32-key tiles in turn, two tiles ahead in
// registers.  What bounds it: one token over 1M keys, 9 x 64, 48 us of this
// kernel, 4.4 TB/s (a large copy moves 4.9), the vector units half busy; 24
// sequences, 32 x 128, 150 us, 3.7 TB/s, sequences of different lengths.
#include <algorithm>

#include "cache4.h"
#include "capi_internal.h"
#include "join.h"

using namespace sva;

namespace {

constexpr int AW = 4;       // waves per workgroup
constexpr int TK = 32;      // keys per tile
constexpr int TR = 16;      // query rows per workgroup

struct Attend4Params {
  const void* q;
  int q_dtype;
  int64_t q_bs, q_hs, q_ts;
  const uint8_t* data;
  const uint8_t* scales;
  int64_t rows;
  const int64_t* offs;
  const int64_t* lens;
  int64_t N;
  int H, G, Q, D, row_tiles, splits;
  int chunk;    // keys per workgroup, a multiple of AW * TK
  float scaling;
  float* sums;   // join.h
  float* stats;
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

// NB: 32-element blocks of a row that the tiles are laid out for, a lane
// holding words qd * NB .. of 8 codes each; PAD: only p.D / 32 of them are
// there.  NT: bf16 terms of the query.
template <int NB, bool PAD, int NT>
__global__ void __launch_bounds__(AW * WAVE, NB <= 2 ? 4 : (NB == 4 ? 3 : 1)) cache4_attention_kernel(Attend4Params p) {
  constexpr int D = 32 * NB;
  constexpr int VS = 2 * D + 32;  // V row pitch in LDS: 4 rows x 32 bytes of a transposed read meet no bank twice
  constexpr int PS = D + 3;       // a query row's m, z, NaN blocks and sums of one wave
  constexpr int SB = NB > 4 ? NB / 4 : 1;  // scale blocks a lane's words lie in
  constexpr int LDS = AW * (TK * VS > TR * PS * 4 ? TK * VS : TR * PS * 4);
  constexpr float kMost = 65536.0f;  // a lane's weights of a tile may sum to
  // scales of V from 2^64 on: sums of smaller V (weights of 2^18 a row and tile) and, with weights of 2^-60 of that,
  // of any V stay below 2^110 over 2^24 tiles, and all waves and ranges together below fp32's largest number
  constexpr uint32_t kLarge = (127u + 64u) << 23;
  __shared__ __align__(16) unsigned char lds[LDS];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int m16 = lane & 15, qd = lane >> 4;
  const int split = (int)blockIdx.x;
  const int y = (int)blockIdx.y;
  const int rt = y % p.row_tiles, g = y / p.row_tiles % p.G, b = y / (p.row_tiles * p.G);
  const int grp = p.H / p.G;
  int64_t off;
  const int len = (int)seq_keys(p.lens, p.offs, p.N, p.rows, b, off);
  const int ranges = tile_ranges(len, p.chunk);
  if (split >= ranges) return;
  const int k0 = split * p.chunk, k1 = k0 + min(p.chunk, len - k0);
  const int blocks = PAD ? p.D / kCache4Block : NB;
  const int dim = PAD ? p.D : D;

  // this lane's query row, as the products' second operand
  const int r = rt * TR + m16;
  const int tok = r / grp, head = g * grp + r % grp;
  const bool live = r < grp * p.Q;
  bf16x8 bq[NT][NB];
  {
    const int64_t qb = (int64_t)b * p.q_bs + (int64_t)head * p.q_hs + (int64_t)tok * p.q_ts;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = (qd * NB + j) * 8 + i;
        float x = live && d < dim ? load_elem(p.q, qb + d, p.q_dtype) : 0.0f;
        const bool finite = (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const __bf16 h = (__bf16)x;
          bq[n][j][i] = p.scaling < 0.0f ? -h : h;
          x = finite ? x - (float)h : 0.0f;
        }
      }
    }
  }
  const int lim = live ? min(k1 - 1, len - p.Q + tok) : -1;     // the last key this query row may see here
  const int full = min(k1, len - p.Q + rt * TR / grp + 1);      // keys below are seen by every row
  const float sl = score_scale(p.scaling);
  float top = -3.40282347e38f, z = 0.0f;  // weights are 2^((score - top) sl - above)
  float above = 0.0f, most_sum = kMost;
  uint32_t nan_blocks = 0u;
  f32x4 o[2 * NB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int64_t row0 = (int64_t)g * p.rows + off;
  unsigned char* vl = lds + w * TK * VS;
  struct Tile {
    uint32_t kc[2][NB], vc[2][NB];
    uint32_t ks[2][SB], vs[2][SB];  // scale bytes, moved to a float's exponent
  };
  // a tile's codes and scales: key base + 16 t + m16 (past the end: the last key's, weight 0), words qd * NB ..
  auto fetch = [&](int base, Tile& x) {
    const uint8_t* data = p.data + (row0 + base) * dim;
    const uint8_t* scales = p.scales + (row0 + base) * (2 * blocks);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t at = (uint32_t)min(16 * t + m16, k1 - 1 - base);
      const uint8_t* kp = data + (at * (uint32_t)dim + (uint32_t)(qd * NB * 4));
      const uint8_t* vp = kp + dim / 2;
      const uint8_t* sp = scales + at * (uint32_t)(2 * blocks);
      if constexpr (!PAD && NB == 2) {
        const uint32_t u = *(const uint32_t*)sp;  // K K V V
        x.ks[t][0] = (u >> (qd < 2 ? 0 : 8) & 255u) << 23;
        x.vs[t][0] = (u >> (qd < 2 ? 16 : 24) & 255u) << 23;
        const uint2 a = *(const uint2*)kp, c = *(const uint2*)vp;
        x.kc[t][0] = a.x, x.kc[t][1] = a.y, x.vc[t][0] = c.x, x.vc[t][1] = c.y;
      } else if constexpr (!PAD && NB == 4) {
        const uint2 u = *(const uint2*)sp;
        x.ks[t][0] = (u.x >> (8 * qd) & 255u) << 23;
        x.vs[t][0] = (u.y >> (8 * qd) & 255u) << 23;
        const u32x4 a = *(const u32x4*)kp, c = *(const u32x4*)vp;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.kc[t][j] = a[j], x.vc[t][j] = c[j];
      } else {
#pragma unroll
        for (int s = 0; s < SB; ++s) {
          const int blk = NB >= 4 ? qd * SB + s : qd * NB / 4;
          const bool there = blk < blocks;
          x.ks[t][s] = (there ? (uint32_t)sp[blk] : 127u) << 23;
          x.vs[t][s] = (there ? (uint32_t)sp[blocks + blk] : 127u) << 23;
#pragma unroll
          for (int j = 0; j < NB / SB; ++j) {
            x.kc[t][NB / SB * s + j] = there ? ((const uint32_t*)kp)[NB / SB * s + j] : 0u;
            x.vc[t][NB / SB * s + j] = there ? ((const uint32_t*)vp)[NB / SB * s + j] : 0u;
          }
        }
      }
    }
  };
  auto use = [&](int base, const Tile& x) {
    // scores: rows = keys 16 t + .., columns = query rows
    f32x4 s[2];
    bool bad = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const bf16x8 a = cache4_unpack8_bf16(x.kc[t][j], __uint_as_float(x.ks[t][NB > 4 ? j / 4 : 0]));
#pragma unroll
        for (int n = 0; n < NT; ++n) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, bq[n][j], s[t], 0, 0, 0);
      }
      // V rows into LDS
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const uint32_t sc = x.vs[t][NB > 4 ? j / 4 : 0];
        const bool nan = sc == 0x7F800000u;
        bad = bad || sc >= kLarge;
        const bf16x8 v = cache4_unpack8_bf16(nan ? 0u : x.vc[t][j], __uint_as_float(nan ? 0x3F800000u : sc));
        *(bf16x8*)(vl + (16 * t + m16) * VS + (qd * NB + j) * 16) = v;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // this lane's 8 keys are base + 16 t + 4 qd + i
    if (base + TK > full) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = base + 16 * t + 4 * qd + i <= lim ? s[t][i] : -INFINITY;
    }
    if (__ballot(bad) != 0ull) {  // some V block of the tile is large, or reads as NaN
      bool large = false;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < SB; ++n) large = large || (x.vs[t][n] >= kLarge && x.vs[t][n] != 0x7F800000u);
      if (above == 0.0f && __any(large)) {
        above = 60.0f, most_sum = kMost * kShifted;
        z *= kShifted;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[i] *= kShifted;
      }
      // which NaN blocks may this query row see?
      for (int i = 0; i < 8; ++i) {
        const int key = base + 16 * (i / 4) + 4 * qd + i % 4;
        if (key > lim) continue;
        const uint8_t* sp = p.scales + ((row0 + key) * 2 + 1) * blocks;
        for (int n = 0; n < blocks; ++n)
          if (sp[n] == kCache4Nan) nan_blocks |= 1u << n;
      }
    }
    bf16x8 pw[2];
    // (the reference comes off before the scale, exactly: rounded after it, as fma(s, sl, -m) would take it, it is off
    // by more than the weights' range from scores of 2^30 on)
    auto weigh = [&]() {
      float zs = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4] - top, sl, -above));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4 + 1] - top, sl, -above));
        bf16x2 h;
        h[0] = (__bf16)e0, h[1] = (__bf16)e1;
        pw[0][i] = h[0], pw[0][i + 1] = h[1];
        pw[1][i] = (__bf16)(e0 - (float)h[0]), pw[1][i + 1] = (__bf16)(e1 - (float)h[1]);
        zs += e0 + e1;
      }
      return zs;
    };
    // the reference moves where the weights sum to more than kMost (the first tile always: it starts below every
    // score): the sum is needed anyway, so an ordinary tile looks for no maximum
    float zs = weigh();
    if (__any(zs > most_sum)) {
      float most = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, s[i / 4][i % 4]);
      most = fmaxf(most, __shfl_xor(most, 16, WAVE));
      most = fmaxf(most, __shfl_xor(most, 32, WAVE));
      const float corr = __builtin_amdgcn_exp2f((top - most) * sl);
      top = most;
      z *= corr;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[i] *= corr;
      zs = weigh();
    }
    z += zs;
    // sums: rows = elements 16 i + .., columns = query rows
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      union {
        s16x4 half[2];
        bf16x8 v;
      } a;
      unsigned char* at = vl + (4 * qd + m16 / 4) * VS + (16 * i + m16 % 4 * 4) * 2;
      a.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
      a.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 16 * VS));
#pragma unroll
      for (int n = 0; n < 2; ++n) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, pw[n], o[i], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  // two tiles ahead, in registers: enough bytes under way to hide the memory's latency
  constexpr int STEP = AW * TK;
  Tile a, c;
  int base = k0 + w * TK;
  if (base < k1) fetch(base, a);
  if (base + STEP < k1) fetch(base + STEP, c);
  for (; base < k1; base += 2 * STEP) {
    use(base, a);
    if (base + 2 * STEP < k1) fetch(base + 2 * STEP, a);
    if (base + STEP < k1) {
      use(base + STEP, c);
      if (base + 3 * STEP < k1) fetch(base + 3 * STEP, c);
    }
  }
  // the waves' parts: [wave][query row][m, z (join.h), NaN blocks, sums]
  z += __shfl_xor(z, 16, WAVE);
  z += __shfl_xor(z, 32, WAVE);
  nan_blocks |= (uint32_t)__shfl_xor((int)nan_blocks, 16, WAVE);
  nan_blocks |= (uint32_t)__shfl_xor((int)nan_blocks, 32, WAVE);
  __syncthreads();
  float* mine = (float*)lds + (w * TR + m16) * PS;
  if (qd == 0) mine[0] = top, mine[1] = above == 0.0f ? z : -z, mine[2] = __uint_as_float(nan_blocks);
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[3 + 16 * i + 4 * qd + k] = o[i][k];
  }
  __syncthreads();
  const int here = min(TR, grp * p.Q - rt * TR);
  for (int e = (int)threadIdx.x; e < here * D; e += AW * WAVE) {
    const int row = e / D, d = e % D;
    const int gr = rt * TR + row;
    if (d >= dim) continue;
    const float* f = (const float*)lds + row * PS;
    float M = f[0], Z = 0.0f, a = 0.0f;
    uint32_t nb = 0u;
    bool shifted = false;
#pragma unroll
    for (int v = 0; v < AW; ++v) {
      M = fmaxf(M, f[v * TR * PS]);
      shifted = shifted || f[v * TR * PS + 1] < 0.0f;
      nb |= __float_as_uint(f[v * TR * PS + 2]);
    }
#pragma unroll
    for (int v = 0; v < AW; ++v) {
      const float zv = f[v * TR * PS + 1];
      float c = __builtin_amdgcn_exp2f((f[v * TR * PS] - M) * sl);
      if (shifted && !(zv < 0.0f)) c *= kShifted;
      Z += fabsf(zv) * c;
      a += f[v * TR * PS + 3 + d] * c;
    }
    if (nb >> (d / kCache4Block) & 1u) a = NAN;
    const int t = gr / grp, h = g * grp + gr % grp;
    if (ranges == 1) {
      const int64_t at = (int64_t)b * p.o_bs + (int64_t)h * p.o_hs + (int64_t)t * p.o_ts + d;
      store_elem(p.out, at, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
    } else {
      const int64_t at = (((int64_t)b * p.H + h) * p.Q + t) * p.splits + split;
      p.sums[at * p.D + d] = a;
      if (d == 0) p.stats[2 * at] = M, p.stats[2 * at + 1] = shifted ? -Z : Z;
    }
  }
}

// Keys per workgroup: enough workgroups to fill the card, four times as many
// where sequences may differ in length (the last to end is then a small part
// of the call); ranges of at least 256 keys and at most 384 of them (each
// costs a row of partial sums).
int64_t chunk_keys(int64_t n_seq, int64_t groups, int64_t n_keys) {
  const int64_t want = std::min<int64_t>(384, std::max<int64_t>(1, (n_seq > 1 ? 4096 : 1024) / groups));
  const int64_t unit = AW * TK;
  return std::max<int64_t>(2 * unit, ((n_keys + want - 1) / want + unit - 1) / unit * unit);
}

int64_t row_tiles(int64_t H, int64_t G, int64_t Q) { return (H / G * Q + TR - 1) / TR; }

template <int NB, bool PAD>
int launch(const Attend4Params& p, dim3 grid, hipStream_t stream) {
  if (p.q_dtype == BF16)
    hipLaunchKernelGGL((cache4_attention_kernel<NB, PAD, 1>), grid, dim3(AW * WAVE), 0, stream, p);
  else if (p.q_dtype == F16)
    hipLaunchKernelGGL((cache4_attention_kernel<NB, PAD, 2>), grid, dim3(AW * WAVE), 0, stream, p);
  else
    hipLaunchKernelGGL((cache4_attention_kernel<NB, PAD, 3>), grid, dim3(AW * WAVE), 0, stream, p);
  SVA_CHECK_LAUNCH("cache4_attention_kernel");
  return SVA_OK;
}

}  // namespace

extern "C" size_t sva_cache4_attention_workspace_bytes(int64_t n_seq, int64_t H, int64_t G, int64_t Q, int64_t D,
                                                       int64_t n_keys) {
  if (n_seq <= 0 || H <= 0 || G <= 0 || Q <= 0 || D <= 0 || n_keys <= 0 || H % G != 0) return 0;
  const int64_t chunk = chunk_keys(n_seq, n_seq * G * row_tiles(H, G, Q), n_keys);
  const int64_t splits = (n_keys + chunk - 1) / chunk;
  return splits == 1 ? 256 : join_bytes(n_seq * H * Q, splits, D);
}

extern "C" int sva_cache4_attention(const void* q, int q_dtype, int64_t q_seq_stride, int64_t q_head_stride,
                                    int64_t q_tok_stride, const uint8_t* data, const uint8_t* scales, int64_t rows,
                                    const int64_t* seq_offsets, const int64_t* seq_lens, int64_t n_keys, int64_t n_seq,
                                    int64_t H, int64_t G, int64_t Q, int64_t D, float scaling, void* out,
                                    int out_dtype, int64_t out_seq_stride, int64_t out_head_stride,
                                    int64_t out_tok_stride, void* workspace, size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(q && data && scales && out, "sva_cache4_attention: null pointer");
  SVA_REQUIRE((seq_offsets == nullptr) == (seq_lens == nullptr),
              "sva_cache4_attention: offsets and lengths go together");
  SVA_REQUIRE(seq_offsets || n_seq == 1, "sva_cache4_attention: several sequences need offsets and lengths");
  SVA_REQUIRE(n_seq > 0 && H > 0 && G > 0 && Q > 0 && n_keys > 0 && rows > 0 && H % G == 0,
              "sva_cache4_attention: bad sizes");
  SVA_REQUIRE(D > 0 && D <= 256 && D % kCache4Block == 0,
              "sva_cache4_attention: head_dim %lld is not a multiple of 32 up to 256", (long long)D);
  SVA_REQUIRE(q_dtype >= 0 && q_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, "sva_cache4_attention: bad dtype");
  SVA_REQUIRE(((uintptr_t)data & 15u) == 0, "sva_cache4_attention: data is not 16-byte aligned");
  SVA_REQUIRE(n_seq < (1ll << 31) && H < (1ll << 31) && Q < (1ll << 31) && n_seq * H < (1ll << 31) &&
                  n_seq * H * Q < (1ll << 31) && n_keys < (1ll << 31) - 1024,
              "sva_cache4_attention: too many items or keys");
  const int64_t tiles = row_tiles(H, G, Q);
  SVA_UNSUPPORTED(n_seq * G * tiles <= 65535, "sva_cache4_attention: %lld tokens of %lld sequences in one call",
                  (long long)Q, (long long)n_seq);
  const size_t need = sva_cache4_attention_workspace_bytes(n_seq, H, G, Q, D, n_keys);
  SVA_REQUIRE(workspace != nullptr && workspace_bytes >= need, "sva_cache4_attention: workspace of %zu bytes required",
              need);
  Attend4Params p;
  p.q = q;
  p.q_dtype = q_dtype;
  p.q_bs = q_seq_stride;
  p.q_hs = q_head_stride;
  p.q_ts = q_tok_stride;
  p.data = data;
  p.scales = scales;
  p.rows = rows;
  p.offs = seq_offsets;
  p.lens = seq_lens;
  p.N = n_keys;
  p.H = (int)H;
  p.G = (int)G;
  p.Q = (int)Q;
  p.D = (int)D;
  p.row_tiles = (int)tiles;
  p.chunk = (int)chunk_keys(n_seq, n_seq * G * tiles, n_keys);
  p.splits = (int)((n_keys + p.chunk - 1) / p.chunk);
  p.scaling = scaling;
  p.stats = (float*)workspace;
  p.sums = p.stats + join_stats_floats(n_seq * H * Q, p.splits);
  p.out = out;
  p.out_dtype = out_dtype;
  p.o_bs = out_seq_stride;
  p.o_hs = out_head_stride;
  p.o_ts = out_tok_stride;
  const dim3 grid((unsigned)p.splits, (unsigned)(n_seq * G * tiles));
  int rc;
  if (D == 32) rc = launch<1, false>(p, grid, (hipStream_t)stream);
  else if (D == 64) rc = launch<2, false>(p, grid, (hipStream_t)stream);
  else if (D == 128) rc = launch<4, false>(p, grid, (hipStream_t)stream);
  else if (D == 256) rc = launch<8, false>(p, grid, (hipStream_t)stream);
  else if (D < 128) rc = launch<4, true>(p, grid, (hipStream_t)stream);
  else rc = launch<8, true>(p, grid, (hipStream_t)stream);
  if (rc != SVA_OK || p.splits == 1) return rc;
  JoinParams j;
  j.sums = p.sums;
  j.stats = p.stats;
  j.sl = score_scale(scaling);
  j.splits = p.splits;
  j.H = p.H;
  j.G = p.G;
  j.Q = p.Q;
  j.D = p.D;
  j.q_lens = j.q_offsets = nullptr;
  j.q_rows = 0;
  j.lens = seq_lens;
  j.offs = seq_offsets;
  j.N = n_keys;
  j.rows = rows;
  j.tile_rows = TR;
  j.chunk = p.chunk;
  j.causal = false;
  j.out = out;
  j.out_dtype = out_dtype;
  j.o_bs = out_seq_stride;
  j.o_hs = out_head_stride;
  j.o_ts = out_tok_stride;
  return sva::launch_join(j, n_seq, (hipStream_t)stream);
}
