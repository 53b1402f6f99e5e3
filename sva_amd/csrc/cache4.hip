// The KV cache in 4 bits: writing rows, reading them back, and the exact
// verifier over them (the attention over all of them: cache4_attention.hip).
//
// Format (cache4.h): per 32 consecutive elements of a row a power-of-two
// scale 2^e, e = floor(log2(largest magnitude)) - 2, and per element the sign
// and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 in units of it (ties to the
// even code, saturating at 6): 17 bits where bf16 takes 64, for 4 elements.
// gfx950 converts between this and fp32 / bf16 in one instruction per two
// elements, and every step is exact but the one rounding, so the result does
// not depend on how the work is laid out.
#include "cache4.h"
#include "capi_internal.h"

using namespace sva;

namespace {

constexpr int WB = 256;

struct Cache4Rows {
  const void* keys;  // written to by the read
  const void* values;
  int64_t seq_stride, head_stride, row_stride;  // elements
  const int64_t* first_rows;                    // [n_seq] cache row of each sequence's row 0, or NULL:
  int64_t first_row;                            // that of the one sequence
  uint8_t* data;
  uint8_t* scales;
  int64_t rows;     // of the cache
  int64_t n_rows;   // of each sequence
  int G, D;
  bool vec;  // rows are whole aligned 16-byte words
};

// Elements [e, e + 8) of a row.
template <int DT>
SVA_DEV void load8(const void* base, int64_t e, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (DT == F32) {
      const float4 a = ((const float4*)((const float*)base + e))[0], b = ((const float4*)((const float*)base + e))[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 a = *(const uint4*)((const uint16_t*)base + e);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = elem_from_bits(u[k] & 0xFFFFu, DT);
        x[2 * k + 1] = elem_from_bits(u[k] >> 16, DT);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = load_elem(base, e + k, DT);
}

// One thread per 8 elements; the 4 threads of a block share its largest
// magnitude by quad permutes.  Reads 16 (fp32: 32) and writes 4 consecutive
// bytes per thread, and a scale byte per block: bound by memory (131072 rows
// of 8 x 128 bf16: written and read back 306 us, 4.4 TB/s, where a large copy
// moves 4.9; a decode step's rows are 2.5 us, a launch).
template <int DT>
__global__ void __launch_bounds__(WB) cache4_write_kernel(Cache4Rows p) {
  const uint32_t per_row = (uint32_t)p.D / 8;  // threads of a K or V row
  const uint32_t c = blockIdx.x * WB + threadIdx.x;
  if (c >= (uint32_t)p.n_rows * 2 * per_row) return;  // a multiple of 4: quads are whole blocks
  const int chunk = (int)(c % per_row);
  const int64_t t = c / per_row >> 1;
  const int kv = (int)(c / per_row & 1);
  const int g = (int)blockIdx.y % p.G, b = (int)blockIdx.y / p.G;
  const int64_t row = (p.first_rows ? p.first_rows[b] : p.first_row) + t;
  if (row < 0 || row >= p.rows) return;  // outside the cache: nothing is written (the same for a whole quad)
  float x[8];
  load8<DT>(kv ? p.values : p.keys, b * p.seq_stride + g * p.head_stride + t * p.row_stride + 8 * chunk, p.vec, x);
  uint32_t top = 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
  const uint32_t e = top >> 23;  // 255: an infinity or a NaN among the 32
  const uint32_t byte = e == 255u ? (uint32_t)kCache4Nan : (e < 3u ? 1u : e - 2u);
  uint32_t w = 0u;
  if (e != 255u) {
    const float s = cache4_scale(byte);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  }
  const int64_t half = (g * p.rows + row) * 2 + kv;
  *(uint32_t*)(p.data + half * (p.D / 2) + 4 * chunk) = w;
  if ((chunk & 3) == 0) p.scales[half * (p.D / kCache4Block) + chunk / 4] = (uint8_t)byte;
}

template <int DT>
__global__ void __launch_bounds__(WB) cache4_read_kernel(Cache4Rows p) {
  const uint32_t per_row = (uint32_t)p.D / 8;
  const uint32_t c = blockIdx.x * WB + threadIdx.x;
  if (c >= (uint32_t)p.n_rows * 2 * per_row) return;
  const int chunk = (int)(c % per_row);
  const int64_t t = c / per_row >> 1;
  const int kv = (int)(c / per_row & 1);
  const int g = (int)blockIdx.y % p.G, b = (int)blockIdx.y / p.G;
  const int64_t row = (p.first_rows ? p.first_rows[b] : p.first_row) + t;
  if (row < 0 || row >= p.rows) return;
  const int64_t half = (g * p.rows + row) * 2 + kv;
  const uint32_t w = *(const uint32_t*)(p.data + half * (p.D / 2) + 4 * chunk);
  const uint32_t byte = p.scales[half * (p.D / kCache4Block) + chunk / 4];
  float x[8];
  cache4_unpack8(w, cache4_scale(byte), x);
  void* base = const_cast<void*>(kv ? p.values : p.keys);
  const int64_t o = b * p.seq_stride + g * p.head_stride + t * p.row_stride + 8 * chunk;
  if (p.vec) {
    if constexpr (DT == F32) {
      ((float4*)((float*)base + o))[0] = make_float4(x[0], x[1], x[2], x[3]);
      ((float4*)((float*)base + o))[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint16_t h[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) store_elem(h, k, DT, x[k]);
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = (uint32_t)h[2 * k] | (uint32_t)h[2 * k + 1] << 16;
      *(uint4*)((uint16_t*)base + o) = make_uint4(u[0], u[1], u[2], u[3]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) store_elem(base, o + k, DT, x[k]);
}

// ---------------------------------------------------------------------------
// The verifier over chosen rows: one workgroup of WPI waves per query item.
// LPR lanes (D / 8 rounded up to a power of two) hold 8 elements each of the
// query, of a row's K and V and of the sums, so a row is one 4-byte load per
// lane and half, and a wave takes 64 / LPR rows a round, U rounds in flight.
// Each row slot keeps an online softmax of its own (32-bit); slots merge by
// cross-lane sums, waves through LDS.  (From the first V block with a scale of
// 2^64 on a wave's weights and sums are 2^-60 of themselves: sums of any V stay
// finite.)  A chosen row is two lines of the
// cache wherever it is, so what bounds a decode step's few hundred rows is
// the latency of list, row and merge, not bandwidth (9 heads x 512 rows of 1M:
// 8.4 us; 72 items x 2048 rows 19.1 us with 16 waves an item, 23.5 with 8; two,
// four or eight rounds in flight are alike).
struct Verify4Params {
  const void* q;
  int q_dtype;
  int64_t q_bs, q_hs, q_ts;
  const uint8_t* data;
  const uint8_t* scales;
  int64_t rows;
  const int64_t* offs;
  const int64_t* lens;
  int64_t N;
  const int32_t* fin_idx;
  const int32_t* fin_count;
  int H, G, Q, D, B;
  float scaling;
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

template <int LPR, int WPI>
__global__ void __launch_bounds__(WPI * WAVE) cache4_verify_kernel(Verify4Params p) {
  constexpr int RPW = WAVE / LPR;  // rows a wave takes a round
  constexpr int U = 4;             // rounds in flight
  constexpr uint32_t kLarge = 127 + 64;  // a scale byte
  __shared__ float part[WPI][LPR * 8 + 3];  // a wave's m, z, scale of weights, sums
  const int64_t item = blockIdx.x;
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
  const int slot = lane / LPR, c = lane % LPR;
  const bool live = 8 * c < p.D;
  const int t = (int)(item % p.Q);
  const int h = (int)((item / p.Q) % p.H);
  const int b = (int)(item / ((int64_t)p.Q * p.H));
  const int g = h / (p.H / p.G);
  const int64_t off = p.offs ? p.offs[b] : 0;
  int64_t len = min(p.lens ? p.lens[b] : p.N, p.rows - off);
  if (off < 0) len = 0;
  const int count = max(0, min(p.fin_count[item], p.B));
  const int32_t* list = p.fin_idx + item * p.B;
  float q[8];
  {
    const int64_t qb = (int64_t)b * p.q_bs + (int64_t)h * p.q_hs + (int64_t)t * p.q_ts + 8 * c;
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = live ? load_elem(p.q, qb + k, p.q_dtype) : 0.0f;
  }
  const int NB = p.D / kCache4Block;
  const int64_t row0 = (int64_t)g * p.rows + off;
  float m = -INFINITY, z = 0.0f, down = 1.0f, acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
  for (int r0 = w * RPW * U; r0 < count; r0 += WPI * RPW * U) {
    uint32_t kc[U], vc[U], ks[U], vs[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = r0 + u * RPW + slot;
      const int x = e < count ? list[e] : -1;
      ok[u] = x >= 0 && (int64_t)x < len;
      kc[u] = vc[u] = 0u;
      ks[u] = vs[u] = 127u;
      if (ok[u] && live) {
        const int64_t half = (row0 + x) * 2;
        kc[u] = *(const uint32_t*)(p.data + half * (p.D / 2) + 4 * c);
        vc[u] = *(const uint32_t*)(p.data + (half + 1) * (p.D / 2) + 4 * c);
        ks[u] = p.scales[half * NB + c / 4];
        vs[u] = p.scales[(half + 1) * NB + c / 4];
      }
    }
    float sc[U], mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[8], d = 0.0f;
      cache4_unpack8(kc[u], cache4_scale(ks[u]), k);
#pragma unroll
      for (int i = 0; i < 8; ++i) d = __builtin_fmaf(k[i], q[i], d);
#pragma unroll
      for (int s = 1; s < LPR; s <<= 1) d += __shfl_xor(d, s, WAVE);
      sc[u] = ok[u] ? d * p.scaling : -INFINITY;
      mn = fmaxf(mn, sc[u]);
    }
    bool large = false;
#pragma unroll
    for (int u = 0; u < U; ++u) large = large || (vs[u] >= kLarge && vs[u] != (uint32_t)kCache4Nan);
    if (down == 1.0f && __any(large)) {
      down = 0x1p-60f;
      z *= down;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= down;
    }
    // no row yet: the sums stay 0.  A NaN score leaves the maximum alone and makes its own weight NaN.
    const float corr = mn == -INFINITY ? 1.0f : __expf(m - mn);
    z *= corr;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= corr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wt = ok[u] ? __expf(sc[u] - (mn == -INFINITY ? 0.0f : mn)) * down : 0.0f;
      float v[8];
      cache4_unpack8(vc[u], cache4_scale(vs[u]), v);
      z += wt;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(wt, v[i], acc[i]);
    }
    m = mn;
  }
  // the wave's row slots, then the waves
  float M = m;
#pragma unroll
  for (int s = LPR; s < WAVE; s <<= 1) M = fmaxf(M, __shfl_xor(M, s, WAVE));
  const float f = m == -INFINITY ? (z != z ? z : 0.0f) : __expf(m - M);  // z is NaN where every score was
  float Z = z * f;
#pragma unroll
  for (int s = LPR; s < WAVE; s <<= 1) Z += __shfl_xor(Z, s, WAVE);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a = acc[i] * f;
#pragma unroll
    for (int s = LPR; s < WAVE; s <<= 1) a += __shfl_xor(a, s, WAVE);
    if (slot == 0) part[w][3 + 8 * c + i] = a;
  }
  if (lane == 0) part[w][0] = M, part[w][1] = Z, part[w][2] = down;
  __syncthreads();
  for (int d = (int)threadIdx.x; d < p.D; d += WPI * WAVE) {
    float Mi = -INFINITY, least = 1.0f;
#pragma unroll
    for (int v = 0; v < WPI; ++v) Mi = fmaxf(Mi, part[v][0]), least = fminf(least, part[v][2]);
    float Zi = 0.0f, a = 0.0f;
#pragma unroll
    for (int v = 0; v < WPI; ++v) {
      const float mv = part[v][0];
      const float even = part[v][2] == least ? 1.0f : least;
      const float fv = mv == -INFINITY ? 1.0f : __expf(mv - Mi) * even;  // (no rows: its sums are 0, or NaN)
      Zi += part[v][1] * fv;
      a += part[v][3 + d] * fv;
    }
    const int64_t o = (int64_t)b * p.o_bs + (int64_t)h * p.o_hs + (int64_t)t * p.o_ts + d;
    store_elem(p.out, o, p.out_dtype, Zi == 0.0f ? 0.0f : a / Zi);
  }
}

template <int LPR>
int launch_verify(const Verify4Params& p, int64_t items, hipStream_t stream) {
  hipLaunchKernelGGL((cache4_verify_kernel<LPR, 16>), dim3((unsigned)items), dim3(16 * WAVE), 0, stream, p);
  SVA_CHECK_LAUNCH("cache4_verify_kernel");
  return SVA_OK;
}

int check_rows(const char* name, const void* keys, const void* values, int dtype, int64_t n_seq, int64_t n_rows,
               int64_t G, int64_t D, const int64_t* first_rows, const uint8_t* data, const uint8_t* scales,
               int64_t rows) {
  SVA_REQUIRE(keys && values && data && scales, "%s: null pointer", name);
  SVA_REQUIRE(first_rows || n_seq == 1, "%s: several sequences need their first rows", name);
  SVA_REQUIRE(n_seq > 0 && n_rows > 0 && G > 0 && rows > 0, "%s: bad sizes", name);
  SVA_REQUIRE(dtype >= 0 && dtype <= 2, "%s: bad dtype", name);
  SVA_REQUIRE(D > 0 && D <= 256 && D % kCache4Block == 0, "%s: head_dim %lld is not a multiple of 32 up to 256", name,
              (long long)D);
  SVA_REQUIRE(((uintptr_t)data & 15u) == 0, "%s: data is not 16-byte aligned", name);
  SVA_REQUIRE(n_seq * G <= 65535 && n_rows <= (1ll << 31) / D, "%s: too many rows in one call", name);
  return SVA_OK;
}

Cache4Rows rows_params(const void* keys, const void* values, int dtype, int64_t seq_stride, int64_t head_stride,
                       int64_t row_stride, int64_t n_rows, int64_t G, int64_t D, const int64_t* first_rows,
                       int64_t first_row, uint8_t* data, uint8_t* scales, int64_t rows) {
  const int64_t word = dtype == F32 ? 4 : 8;  // elements of 16 bytes
  Cache4Rows p;
  p.keys = keys;
  p.values = values;
  p.seq_stride = seq_stride;
  p.head_stride = head_stride;
  p.row_stride = row_stride;
  p.first_rows = first_rows;
  p.first_row = first_row;
  p.data = data;
  p.scales = scales;
  p.rows = rows;
  p.n_rows = n_rows;
  p.G = (int)G;
  p.D = (int)D;
  p.vec = (((uintptr_t)keys | (uintptr_t)values) & 15u) == 0 && seq_stride % word == 0 && head_stride % word == 0 &&
          row_stride % word == 0;
  return p;
}

}  // namespace

extern "C" int sva_cache4_write(const void* keys, const void* values, int kv_dtype, int64_t kv_seq_stride,
                                int64_t kv_head_stride, int64_t kv_row_stride, int64_t n_seq, int64_t n_rows,
                                int64_t G, int64_t D, const int64_t* first_rows, int64_t first_row,
                                uint8_t* data, uint8_t* scales, int64_t rows, void* stream) {
  sva::clear_error();
  if (const int rc = check_rows("sva_cache4_write", keys, values, kv_dtype, n_seq, n_rows, G, D, first_rows, data,
                                scales, rows))
    return rc;
  const Cache4Rows p = rows_params(keys, values, kv_dtype, kv_seq_stride, kv_head_stride, kv_row_stride, n_rows, G, D,
                                   first_rows, first_row, data, scales, rows);
  const dim3 grid((unsigned)((n_rows * 2 * (D / 8) + WB - 1) / WB), (unsigned)(n_seq * G));
  auto* fn = kv_dtype == F32 ? cache4_write_kernel<F32>
                             : (kv_dtype == BF16 ? cache4_write_kernel<BF16> : cache4_write_kernel<F16>);
  hipLaunchKernelGGL(fn, grid, dim3(WB), 0, (hipStream_t)stream, p);
  SVA_CHECK_LAUNCH("cache4_write_kernel");
  return SVA_OK;
}

extern "C" int sva_cache4_read(const uint8_t* data, const uint8_t* scales, int64_t rows, const int64_t* first_rows,
                               int64_t first_row, int64_t n_seq, int64_t n_rows, int64_t G, int64_t D, void* keys, void* values,
                               int kv_dtype, int64_t kv_seq_stride, int64_t kv_head_stride, int64_t kv_row_stride,
                               void* stream) {
  sva::clear_error();
  if (const int rc = check_rows("sva_cache4_read", keys, values, kv_dtype, n_seq, n_rows, G, D, first_rows, data,
                                scales, rows))
    return rc;
  const Cache4Rows p = rows_params(keys, values, kv_dtype, kv_seq_stride, kv_head_stride, kv_row_stride, n_rows, G, D,
                                   first_rows, first_row, const_cast<uint8_t*>(data), const_cast<uint8_t*>(scales), rows);
  const dim3 grid((unsigned)((n_rows * 2 * (D / 8) + WB - 1) / WB), (unsigned)(n_seq * G));
  auto* fn = kv_dtype == F32 ? cache4_read_kernel<F32>
                             : (kv_dtype == BF16 ? cache4_read_kernel<BF16> : cache4_read_kernel<F16>);
  hipLaunchKernelGGL(fn, grid, dim3(WB), 0, (hipStream_t)stream, p);
  SVA_CHECK_LAUNCH("cache4_read_kernel");
  return SVA_OK;
}

extern "C" int sva_cache4_verify(const void* q, int q_dtype, int64_t q_seq_stride, int64_t q_head_stride,
                                 int64_t q_tok_stride, const uint8_t* data, const uint8_t* scales, int64_t rows,
                                 const int64_t* seq_offsets, const int64_t* seq_lens, int64_t n_keys,
                                 const int32_t* fin_idx, const int32_t* fin_count, int64_t n_seq, int64_t H, int64_t G,
                                 int64_t Q, int64_t D, int64_t B, float scaling, void* out, int out_dtype,
                                 int64_t out_seq_stride, int64_t out_head_stride, int64_t out_tok_stride,
                                 void* stream) {
  sva::clear_error();
  SVA_REQUIRE(q && data && scales && fin_idx && fin_count && out, "sva_cache4_verify: null pointer");
  SVA_REQUIRE((seq_offsets == nullptr) == (seq_lens == nullptr), "sva_cache4_verify: offsets and lengths go together");
  SVA_REQUIRE(seq_offsets || n_seq == 1, "sva_cache4_verify: several sequences need offsets and lengths");
  SVA_REQUIRE(n_seq > 0 && H > 0 && G > 0 && Q > 0 && B > 0 && n_keys > 0 && rows > 0 && H % G == 0,
              "sva_cache4_verify: bad sizes");
  SVA_REQUIRE(D > 0 && D <= 256 && D % kCache4Block == 0,
              "sva_cache4_verify: head_dim %lld is not a multiple of 32 up to 256", (long long)D);
  SVA_REQUIRE(q_dtype >= 0 && q_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, "sva_cache4_verify: bad dtype");
  SVA_REQUIRE(((uintptr_t)data & 15u) == 0, "sva_cache4_verify: data is not 16-byte aligned");
  SVA_REQUIRE(n_seq < (1ll << 31) && H < (1ll << 31) && Q < (1ll << 31) && n_seq * H < (1ll << 31) &&
                  n_seq * H * Q < (1ll << 31) && B < (1ll << 30),
              "sva_cache4_verify: too many items");
  Verify4Params p;
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
  p.fin_idx = fin_idx;
  p.fin_count = fin_count;
  p.H = (int)H;
  p.G = (int)G;
  p.Q = (int)Q;
  p.D = (int)D;
  p.B = (int)B;
  p.scaling = scaling;
  p.out = out;
  p.out_dtype = out_dtype;
  p.o_bs = out_seq_stride;
  p.o_hs = out_head_stride;
  p.o_ts = out_tok_stride;
  const int64_t items = n_seq * H * Q;
  if (D <= 32) return launch_verify<4>(p, items, (hipStream_t)stream);
  if (D <= 64) return launch_verify<8>(p, items, (hipStream_t)stream);
  if (D <= 128) return launch_verify<16>(p, items, (hipStream_t)stream);
  return launch_verify<32>(p, items, (hipStream_t)stream);
}
