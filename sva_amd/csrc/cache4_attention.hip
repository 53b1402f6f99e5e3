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
//    accuracy while the cache, not the matrix cores, sets the time.
//  * S^T leaves a lane with 8 scores of one query row, which are its share of
//    the P^T operand: weights never cross lanes.  V goes through LDS, each
//    wave its own 32 rows, and comes back transposed (ds_read_b64_tr_b16).
//  * A block that reads as NaN is kept out of V (0 * NaN would reach rows that
//    may not see it) and marks the query rows that may.
// Workgroups split the keys (partials joined by a second kernel), a
// workgroup's four waves take its 32-key tiles in turn.
#include <algorithm>

#include "cache4.h"
#include "capi_internal.h"

using namespace sva;

namespace {

constexpr int AW = 4;       // waves per workgroup
constexpr int TK = 32;      // keys per tile
constexpr int TR = 16;      // query rows per workgroup
constexpr int CMB = 256;    // threads per combine workgroup
constexpr float kLog2e = 1.44269504088896340736f;

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
  int64_t chunk;  // keys per workgroup, a multiple of AW * TK
  float scaling;
  float* part;  // [items, splits, D + 2]: m (base 2), z, sums
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

// Sequence b's keys: its first row and length, kept inside the cache.
SVA_DEV int64_t seq_range(const Attend4Params& p, int b, int64_t& off) {
  off = p.offs ? p.offs[b] : 0;
  const int64_t len = min(min(p.lens ? p.lens[b] : p.N, p.N), p.rows - off);
  return off < 0 ? 0 : max(len, (int64_t)0);
}

// NB: 32-element blocks of a row the tiles are laid out for (p.D / 32 of them
// are there); a lane holds words qd * NB .. of 8 codes.
template <int NB, int NT>
__global__ void __launch_bounds__(AW * WAVE) cache4_attention_kernel(Attend4Params p) {
  constexpr int D = 32 * NB;
  constexpr int VS = 2 * D + 32;  // V row pitch in LDS: 4 rows x 32 bytes of a transposed read meet no bank twice
  constexpr int PS = D + 3;       // a query row's m, z, NaN blocks and sums of one wave
  constexpr int SB = NB > 4 ? NB / 4 : 1;  // scale blocks a lane's words lie in
  constexpr int LDS = AW * (TK * VS > TR * PS * 4 ? TK * VS : TR * PS * 4);
  __shared__ __align__(16) unsigned char lds[LDS];
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
  const int m16 = lane & 15, qd = lane >> 4;
  const int split = (int)blockIdx.x;
  const int y = (int)blockIdx.y;
  const int rt = y % p.row_tiles, g = y / p.row_tiles % p.G, b = y / (p.row_tiles * p.G);
  const int grp = p.H / p.G;
  int64_t off;
  const int64_t len = seq_range(p, b, off);
  const int64_t k0 = split * p.chunk, k1 = min(len, k0 + p.chunk);
  if (k0 >= len && split > 0) return;  // nothing here (the first workgroup of a row writes an empty sequence's zeros)
  const int blocks = p.D / kCache4Block;

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
        float x = live && d < p.D ? load_elem(p.q, qb + d, p.q_dtype) : 0.0f;
        const bool finite = (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const __bf16 h = (__bf16)x;
          bq[n][j][i] = h;
          x = finite ? x - (float)h : 0.0f;
        }
      }
    }
  }
  const int64_t last = live ? min(k1 - 1, len - p.Q + tok) : -1;  // the last key this query row may see here
  const float sl = p.scaling * kLog2e;
  float m = -INFINITY, z = 0.0f;
  uint32_t nan_blocks = 0u;
  f32x4 o[2 * NB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int64_t row0 = (int64_t)g * p.rows + off;
  unsigned char* vl = lds + w * TK * VS;
  uint32_t kc[2][NB], vc[2][NB], ksc[2][SB], vsc[2][SB];
  // a tile's codes and scales: key base + 16 t + m16 (past the end: the last key's, weight 0), words qd * NB ..
  auto fetch = [&](int64_t base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t half = (row0 + min(base + 16 * t + m16, k1 - 1)) * 2;
      const uint8_t* kp = p.data + half * (p.D / 2) + qd * NB * 4;
      const uint8_t* vp = kp + p.D / 2;
      const uint8_t* sp = p.scales + half * blocks;
#pragma unroll
      for (int s = 0; s < SB; ++s) {
        const int blk = NB >= 4 ? qd * SB + s : qd * NB / 4;
        const bool there = blk < blocks;
        ksc[t][s] = there ? sp[blk] : 127u;
        vsc[t][s] = there ? sp[blocks + blk] : 127u;
        if constexpr (NB >= 4) {
          const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
          const uint4 a = there ? *(const uint4*)(kp + 16 * s) : zero;
          const uint4 c = there ? *(const uint4*)(vp + 16 * s) : zero;
          kc[t][4 * s] = a.x, kc[t][4 * s + 1] = a.y, kc[t][4 * s + 2] = a.z, kc[t][4 * s + 3] = a.w;
          vc[t][4 * s] = c.x, vc[t][4 * s + 1] = c.y, vc[t][4 * s + 2] = c.z, vc[t][4 * s + 3] = c.w;
        } else {
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            kc[t][j] = ((const uint32_t*)kp)[j];
            vc[t][j] = ((const uint32_t*)vp)[j];
          }
        }
      }
    }
  };
  int64_t base = k0 + w * TK;
  if (base < k1) fetch(base);
  for (; base < k1; base += AW * TK) {
    // scores: rows = keys 16 t + .., columns = query rows
    f32x4 s[2];
    bool bad = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const bf16x8 a = cache4_unpack8_bf16(kc[t][j], cache4_scale(ksc[t][NB > 4 ? j / 4 : 0]));
#pragma unroll
        for (int n = 0; n < NT; ++n) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, bq[n][j], s[t], 0, 0, 0);
      }
      // V rows into LDS
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const uint32_t sc = vsc[t][NB > 4 ? j / 4 : 0];
        const bool nan = sc == (uint32_t)kCache4Nan;
        bad = bad || nan;
        const bf16x8 v = cache4_unpack8_bf16(nan ? 0u : vc[t][j], cache4_scale(nan ? 127u : sc));
        *(bf16x8*)(vl + (16 * t + m16) * VS + (qd * NB + j) * 16) = v;
      }
    }
    if (base + AW * TK < k1) fetch(base + AW * TK);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // running maximum and weights of this lane's 8 keys: base + 16 t + 4 qd + i
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = base + 16 * t + 4 * qd + i <= last;
        s[t][i] = ok ? s[t][i] * sl : -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, WAVE));
    top = fmaxf(top, __shfl_xor(top, 32, WAVE));
    const float mn = fmaxf(m, top);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float corr = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    z *= corr;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) o[i] *= corr;
    bf16x8 ph, pl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - ref);
      z += e;
      const __bf16 h = (__bf16)e;
      ph[i] = h;
      pl[i] = (__bf16)(e - (float)h);
    }
    if (__ballot(bad) != 0ull) {  // some V block of the tile reads as NaN: which of them may this query row see?
      for (int i = 0; i < 8; ++i) {
        const int64_t key = base + 16 * (i / 4) + 4 * qd + i % 4;
        if (key > last) continue;
        const uint8_t* sp = p.scales + ((row0 + key) * 2 + 1) * blocks;
        for (int n = 0; n < blocks; ++n)
          if (sp[n] == kCache4Nan) nan_blocks |= 1u << n;
      }
    }
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
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, ph, o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, pl, o[i], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the waves' parts: [wave][query row][m, z, NaN blocks, sums]
  z += __shfl_xor(z, 16, WAVE);
  z += __shfl_xor(z, 32, WAVE);
  nan_blocks |= (uint32_t)__shfl_xor((int)nan_blocks, 16, WAVE);
  nan_blocks |= (uint32_t)__shfl_xor((int)nan_blocks, 32, WAVE);
  __syncthreads();
  float* mine = (float*)lds + (w * TR + m16) * PS;
  if (qd == 0) mine[0] = m, mine[1] = z, mine[2] = __uint_as_float(nan_blocks);
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[3 + 16 * i + 4 * qd + k] = o[i][k];
  }
  __syncthreads();
  for (int e = (int)threadIdx.x; e < TR * D; e += AW * WAVE) {
    const int row = e / D, d = e % D;
    const int gr = rt * TR + row;
    if (gr >= grp * p.Q || d >= p.D) continue;
    const float* f = (const float*)lds + row * PS;
    float M = -INFINITY, Z = 0.0f, a = 0.0f;
    uint32_t nb = 0u;
#pragma unroll
    for (int v = 0; v < AW; ++v) {
      M = fmaxf(M, f[v * TR * PS]);
      nb |= __float_as_uint(f[v * TR * PS + 2]);
    }
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int v = 0; v < AW; ++v) {
      const float mv = f[v * TR * PS];
      const float c = mv == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mv - ref);  // (no key: the sums are 0, or NaN)
      Z += f[v * TR * PS + 1] * c;
      a += f[v * TR * PS + 3 + d] * c;
    }
    if (nb >> (d / kCache4Block) & 1u) a = NAN;
    const int t = gr / grp, h = g * grp + gr % grp;
    if (p.splits == 1) {
      const int64_t at = (int64_t)b * p.o_bs + (int64_t)h * p.o_hs + (int64_t)t * p.o_ts + d;
      store_elem(p.out, at, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
    } else {
      float* dst = p.part + ((((int64_t)b * p.H + h) * p.Q + t) * p.splits + split) * (p.D + 2);
      dst[2 + d] = a;
      if (d == 0) dst[0] = M, dst[1] = Z;
    }
  }
}

// Joins an item's key ranges: 32 elements of it a workgroup, eight ranges at
// a time.
__global__ void __launch_bounds__(CMB) cache4_combine_kernel(Attend4Params p) {
  __shared__ float red[CMB];
  __shared__ float wave[2][CMB / WAVE];
  const int item = (int)blockIdx.x, d = (int)blockIdx.y * 32 + (int)threadIdx.x % 32, lane8 = (int)threadIdx.x / 32;
  const int t = item % p.Q, h = item / p.Q % p.H, b = item / (p.Q * p.H);
  int64_t off;
  const int64_t len = seq_range(p, b, off);
  const int n = (int)((len + p.chunk - 1) / p.chunk);
  const float* src = p.part + (int64_t)item * p.splits * (p.D + 2);
  float M = -INFINITY;
  for (int s = (int)threadIdx.x; s < n; s += CMB) M = fmaxf(M, src[(int64_t)s * (p.D + 2)]);
  M = wave_max(M);
  if (lane_id() == 0) wave[0][threadIdx.x / WAVE] = M;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < CMB / WAVE; ++v) M = fmaxf(M, wave[0][v]);
  const float ref = M == -INFINITY ? 0.0f : M;
  float Z = 0.0f, a = 0.0f;
  for (int s = lane8; s < n; s += CMB / 32) {
    const float* f = src + (int64_t)s * (p.D + 2);
    const float mv = f[0];
    const float c = mv == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mv - ref);
    Z += f[1] * c;
    a += f[2 + d] * c;
  }
  red[threadIdx.x] = a;
  __syncthreads();
  a = 0.0f;
  if (threadIdx.x < 32)
    for (int v = 0; v < CMB / 32; ++v) a += red[32 * v + threadIdx.x];
  __syncthreads();
  red[threadIdx.x] = Z;
  __syncthreads();
  if (threadIdx.x < 32) {
    Z = 0.0f;
    for (int v = 0; v < CMB / 32; ++v) Z += red[32 * v];
    const int64_t at = (int64_t)b * p.o_bs + (int64_t)h * p.o_hs + (int64_t)t * p.o_ts + d;
    store_elem(p.out, at, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
  }
}

// Keys per workgroup: enough workgroups to fill the card, ranges of at least
// 256 keys and at most 256 of them (each costs a row of partial sums).
int64_t chunk_keys(int64_t groups, int64_t n_keys) {
  const int64_t want = std::min<int64_t>(256, std::max<int64_t>(1, 1024 / groups));
  const int64_t unit = AW * TK;
  return std::max<int64_t>(2 * unit, ((n_keys + want - 1) / want + unit - 1) / unit * unit);
}

int64_t row_tiles(int64_t H, int64_t G, int64_t Q) { return (H / G * Q + TR - 1) / TR; }

template <int NB>
int launch(const Attend4Params& p, dim3 grid, hipStream_t stream) {
  if (p.q_dtype == BF16)
    hipLaunchKernelGGL((cache4_attention_kernel<NB, 1>), grid, dim3(AW * WAVE), 0, stream, p);
  else if (p.q_dtype == F16)
    hipLaunchKernelGGL((cache4_attention_kernel<NB, 2>), grid, dim3(AW * WAVE), 0, stream, p);
  else
    hipLaunchKernelGGL((cache4_attention_kernel<NB, 3>), grid, dim3(AW * WAVE), 0, stream, p);
  SVA_CHECK_LAUNCH("cache4_attention_kernel");
  return SVA_OK;
}

}  // namespace

extern "C" size_t sva_cache4_attention_workspace_bytes(int64_t n_seq, int64_t H, int64_t G, int64_t Q, int64_t D,
                                                       int64_t n_keys) {
  if (n_seq <= 0 || H <= 0 || G <= 0 || Q <= 0 || D <= 0 || n_keys <= 0 || H % G != 0) return 0;
  const int64_t chunk = chunk_keys(n_seq * G * row_tiles(H, G, Q), n_keys);
  const int64_t splits = (n_keys + chunk - 1) / chunk;
  return splits == 1 ? 256 : sizeof(float) * (size_t)(n_seq * H * Q) * (size_t)splits * (size_t)(D + 2) + 256;
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
                  n_seq * H * Q < (1ll << 31) && n_keys < (1ll << 40),
              "sva_cache4_attention: too many items");
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
  p.chunk = chunk_keys(n_seq * G * tiles, n_keys);
  p.splits = (int)((n_keys + p.chunk - 1) / p.chunk);
  p.scaling = scaling;
  p.part = (float*)workspace;
  p.out = out;
  p.out_dtype = out_dtype;
  p.o_bs = out_seq_stride;
  p.o_hs = out_head_stride;
  p.o_ts = out_tok_stride;
  const dim3 grid((unsigned)p.splits, (unsigned)(n_seq * G * tiles));
  int rc;
  if (D <= 32) rc = launch<1>(p, grid, (hipStream_t)stream);
  else if (D <= 64) rc = launch<2>(p, grid, (hipStream_t)stream);
  else if (D <= 128) rc = launch<4>(p, grid, (hipStream_t)stream);
  else rc = launch<8>(p, grid, (hipStream_t)stream);
  if (rc != SVA_OK || p.splits == 1) return rc;
  hipLaunchKernelGGL(cache4_combine_kernel, dim3((unsigned)(n_seq * H * Q), (unsigned)(D / 32)), dim3(CMB), 0,
                     (hipStream_t)stream, p);
  SVA_CHECK_LAUNCH("cache4_combine_kernel");
  return SVA_OK;
}
