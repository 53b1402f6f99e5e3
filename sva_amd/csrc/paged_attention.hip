// Attention of a few tokens over a KV cache in pages (pages.h).
//
// out[h, t] = sum_n p[n] V[n] / sum_n p[n], p[n] = exp(s (q[h, t] . K[n]) - m)
// over the rows n <= len - Q + t of the sequence that are read, in one pass over
// its pages with a running reference m.  Each wave takes 32-key tiles on its
// own, K and V of the next ones under way in registers; the query rows (token,
// head of the KV group) of a workgroup are 16 at a time, so that a tile serves
// all of them: S^T = K Q^T and O^T = V^T P^T on 16x16 matrix instructions.
//  * 16 aligned keys lie in one page: a tile is two halves whose addresses are
//    scalars.  Page numbers come 64 at a time, one a lane, 32 tiles ahead.
//  * S^T leaves a lane with scores of one query row that are its share of the
//    P^T operand: weights never cross lanes.  16-bit V goes through LDS, each
//    wave its own rows, and comes back transposed (ds_read_b64_tr_b16); fp32 V
//    is loaded as its operand wants it, 16 elements of 4 keys a load.
//  * 16-bit weights are split into two terms of V's type: the products keep
//    about 16 bits of the weights while memory sets the time.
//  * The reference moves only where a lane's weights of a tile sum to more
//    than 2^16 (fp16: 2^15, and weights of 2^8 at a new reference keep small
//    ones normal); it comes off before the scale, exactly, whatever the
//    scores' size.
//  * What a masked key's V holds meets a weight of 0, which a NaN survives: a
//    query row whose sums are not finite, or larger than the ranges' sums
//    together can hold, is done again key by key over the keys it sees.
// Workgroups split the keys (partials joined by a second kernel, join.h).
// Bound by the read of K and V: 32 sequences of 4K to 131K rows, 9 x 64 bf16, 296
// us (5.6 TB/s); 24 of 1K to 42K, 32 x 128, 386 us (5.5 TB/s); one of 1000 rows
// by the chain of its steps, 9 us and 4 for the join.
#include <algorithm>

#include "cache4.h"
#include "capi_internal.h"
#include "join.h"
#include "pages.h"

using namespace sva;

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int AW = 4;   // waves per workgroup
constexpr int TK = 32;  // keys per tile
constexpr int TR = 16;  // query rows per workgroup
constexpr int STEP = AW * TK;

struct PagedParams {
  const void* q;
  int64_t q_bs, q_hs, q_ts;
  bool q_vec;  // a query row is whole aligned 16-byte words
  Pages c;
  const int64_t* lens;
  int64_t N;  // rows of a sequence behind this are not read
  int n_seq, H, G, Q, D, row_tiles, splits;
  int chunk;  // keys per workgroup, a multiple of STEP
  float scaling;
  float* sums;  // join.h
  float* stats;
  void* out;
  int out_dtype;
  int64_t o_bs, o_hs, o_ts;
};

template <int DT>
struct PagedType {
  static constexpr int ES = DT == F32 ? 4 : 2;
  using elem = typename std::conditional<DT == BF16, __bf16, _Float16>::type;
  using frag = typename std::conditional<DT == BF16, bf16x8, f16x8>::type;
  // weights are 2^kBelow at a new reference; in a range's sums too, whoever takes them
  static constexpr float kBelow = DT == F16 ? 8.0f : 0.0f;
  // waves per SIMD that the registers are kept to (four for the narrowest send 20 registers through scratch memory: 32
  // sequences of up to 131072 keys, 9 x 64 bf16, 416 us against 297)
  static constexpr int waves(int dp) { return dp * ES <= 128 ? 3 : (dp * ES <= 256 ? 2 : 1); }
};

template <int DT>
SVA_DEV f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  union {
    u32x4 u;
    bf16x8 h;
    f16x8 f;
  } x, y;
  x.u = a, y.u = b;
  if constexpr (DT == BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.h, y.h, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.f, y.f, c, 0, 0, 0);
}

// One query row again over keys [k0, end), key by key, by one wave: lanes take
// 64 keys' scores, then the row's elements.  Weights are those of the tiles, as
// other ranges' sums join these.  Finite V whose sums are too large: once more,
// weights and sums 2^-60 of themselves.
template <int DT, int DP>
SVA_DEV void attend_again(const PagedParams& p, int64_t qa, int b, int g, int k0, int end, float sl, float (&acc)[DP / 64],
                          float& m, float& z) {
  const int lane = lane_id();
  const int64_t v_off = (int64_t)p.G * p.D << p.c.bits;  // elements between a page's K and V
  auto row_at = [&](int page, int key) {
    return (const unsigned char*)p.c.pool + (int64_t)page * p.c.page_bytes +
           (((int64_t)g << p.c.bits) + (key & ((1 << p.c.bits) - 1))) * p.D * PagedType<DT>::ES;
  };
  float down = 1.0f;
  for (;;) {
    m = -INFINITY, z = 0.0f;
    bool finite[DP / 64];
#pragma unroll
    for (int k = 0; k < DP / 64; ++k) acc[k] = 0.0f, finite[k] = true;
    for (int n0 = k0; n0 < end; n0 += WAVE) {
      const int key = n0 + lane;
      const int page = key < end ? page_of(p.c, b, key >> p.c.bits) : -1;
      float sc = -INFINITY;
      if (page >= 0) {
        sc = 0.0f;
        const unsigned char* k = row_at(page, key);
        for (int d = 0; d < p.D; ++d) sc = __builtin_fmaf(load_elem(p.q, qa + d, DT), load_elem(k, d, DT), sc);
        sc = p.scaling < 0.0f ? -sc : sc;
      }
      const float mn = fmaxf(m, wave_max(sc));
      const float corr = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * sl);
      const float below = __builtin_fmaf(sc - (mn == -INFINITY ? 0.0f : mn), sl, PagedType<DT>::kBelow);
      const float e = page >= 0 ? __builtin_amdgcn_exp2f(below) * down : 0.0f;
      m = mn;
      z = z * corr + wave_sum(e);
#pragma unroll
      for (int k = 0; k < DP / 64; ++k) acc[k] *= corr;
      for (int j = 0; j < min(WAVE, end - n0); ++j) {
        const int pj = __builtin_amdgcn_readlane(page, j);
        if (pj < 0) continue;
        const float ej = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(e), j));
        const unsigned char* v = row_at(pj, n0 + j);
#pragma unroll
        for (int k = 0; k < DP / 64; ++k) {
          const int d = lane + 64 * k;
          if (d < p.D) {
            const float x = load_elem(v, v_off + d, DT);
            finite[k] = finite[k] && fabsf(x) <= 3.40282347e38f;
            acc[k] = __builtin_fmaf(ej, x, acc[k]);
          }
        }
      }
    }
    bool large = false;
#pragma unroll
    for (int k = 0; k < DP / 64; ++k) large = large || (finite[k] && z == z && !(fabsf(acc[k]) <= 0x1p110f));
    if (down != 1.0f || !__any(large)) break;
    down = kShifted;
  }
  if (down != 1.0f) z = -z;
}

// DP: elements of a row that the tiles are laid out for; PAD: only p.D of them
// are there.
template <int DT, int DP, bool PAD>
__global__ void __launch_bounds__(AW * WAVE, PagedType<DT>::waves(DP)) paged_attention_kernel(PagedParams p) {
  using Type = PagedType<DT>;
  constexpr bool WIDE = DT == F32;  // 32-bit elements
  constexpr int ES = Type::ES;
  constexpr int EC = 16 / ES;              // elements of a 16-byte chunk
  constexpr int NC = DP / (4 * EC);        // chunks of half a tile's K (or V) per lane
  constexpr int NO = DP / 16;              // 16-element blocks of the sums
  constexpr int VS = 2 * DP + 32;          // V row pitch in LDS: 4 rows x 32 bytes of a transposed read meet no bank twice
  constexpr int PS = DP + 3;               // a query row's m, z and sums of one wave
  constexpr int VB = WIDE ? 0 : AW * TK * VS, PB = AW * TR * PS * 4;
  constexpr float kMost = DT == F16 ? 32768.0f : 65536.0f;  // a lane's weights of a tile may sum to
  constexpr float kBelow = Type::kBelow;
  constexpr float kLarge = 0x1p110f;                        // all ranges' sums of less stay finite together
  __shared__ __align__(16) unsigned char lds[VB > PB ? VB : PB];
  __shared__ uint32_t odd_rows;
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int m16 = lane & 15, qd = lane >> 4;
  // (the row tiles over the same keys are eight workgroups apart: on one XCD, whose L2 they share)
  const uint32_t id = blockIdx.x, unit = id / (uint32_t)(kXcds * p.row_tiles) * kXcds + id % kXcds;
  const int rt = (int)(id / kXcds % (uint32_t)p.row_tiles);
  const int split = (int)(unit % (uint32_t)p.splits);
  const int g = (int)(unit / (uint32_t)p.splits % (uint32_t)p.G), b = (int)(unit / (uint32_t)p.splits / (uint32_t)p.G);
  if (b >= p.n_seq) return;
  const int grp = p.H / p.G;
  int64_t off;
  const int len = (int)seq_keys(p.lens, nullptr, p.N, p.N, b, off);
  const int ranges = tile_ranges(len, p.chunk);
  if (split >= ranges) return;
  const int k0 = split * p.chunk, k1 = k0 + min(p.chunk, len - k0);
  // rows that the first token sees: of the length itself, also where not all of it is read
  const int64_t seen = min(max(p.lens[b], (int64_t)0), (int64_t)1 << 40) - p.Q + 1;
  auto seen_by = [&](int t) { return (int)max(min(seen + t, (int64_t)k1), (int64_t)0); };  // of keys below k1
  const int dim = PAD ? p.D : DP;
  const uint32_t rowb = (uint32_t)dim * ES;

  // Table entries of this wave's tiles, 64 halves at a time: lane l has half
  // l % 2 of its tile 32 * group + l / 2 (past the end: the last key's).
  const int first = k0 + w * TK;
  auto entries = [&](int group) {
    const int64_t key = (int64_t)first + (int64_t)(32 * group + lane / 2) * STEP + 16 * (lane & 1);
    const int at = (int)(key < k1 ? key : k1 - 1) >> p.c.bits;
    return k1 > k0 ? page_of(p.c, b, at) : -1;
  };
  int ids = entries(0), ids_next = entries(1);

  // this lane's query row, as the products' second operand
  const int r = rt * TR + m16;
  const int tok = r / grp, head = g * grp + r % grp;
  const bool live = r < grp * p.Q;
  u32x4 bq[NC];
  {
    const int64_t qb = (int64_t)b * p.q_bs + (int64_t)(live ? head : 0) * p.q_hs + (int64_t)(live ? tok : 0) * p.q_ts;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int d = (4 * j + qd) * EC;
      const bool there = live && (!PAD || d < dim);
      u32x4 x = {0u, 0u, 0u, 0u};
      if (there) {
        if (p.q_vec) {
          x = *(const u32x4*)((const unsigned char*)p.q + (qb + d) * ES);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (WIDE) x[i] = load_elem_bits(p.q, qb + d + i, DT);
            else x[i] = load_elem_bits(p.q, qb + d + 2 * i, DT) | load_elem_bits(p.q, qb + d + 2 * i + 1, DT) << 16;
          }
        }
        if (p.scaling < 0.0f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] ^= WIDE ? 0x80000000u : 0x80008000u;
        }
      }
      bq[j] = x;
    }
  }
  const int lim = live ? seen_by(tok) - 1 : -1;  // the last key this query row may see here
  const int full = seen_by(rt * TR / grp);       // keys below are seen by every row
  const float sl = score_scale(p.scaling);
  float top = -3.40282347e38f, z = 0.0f;  // weights are 2^((score - top) sl + kBelow)
  f32x4 o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  unsigned char* vl = lds + w * TK * VS;
  const uint32_t head_off = ((uint32_t)g << p.c.bits) * rowb, v_off = ((uint32_t)p.G << p.c.bits) * rowb;
  struct Tile {
    u32x4 k[2][NC], v[2][NC];
    int there;  // bit t: half t has a page
  };
  // tile number `step` of this wave: keys first + step * STEP + ..
  auto fetch = [&](int step, Tile& x) {
    if ((step & 31) == 0 && step != 0) {
      ids = ids_next;
      ids_next = entries(step / 32 + 1);
    }
    const int base = first + step * STEP;
    x.there = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int id = __builtin_amdgcn_readlane(ids, 2 * (step & 31) + t);
      x.there |= id >= 0 ? 1 << t : 0;
      const int key = min(base + 16 * t, k1 - 1);  // (a half behind the end: the last key, weight 0)
      const int most = k1 - 1 - key;
      const unsigned char* kp = p.c.pool + (int64_t)(id < 0 ? 0 : id) * p.c.page_bytes + head_off +
                                (uint32_t)(key & ((1 << p.c.bits) - 1)) * rowb;
      const unsigned char* vp = kp + v_off;
      const uint32_t row = (uint32_t)min(m16, most) * rowb;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const uint32_t c = (uint32_t)(4 * j + qd) * 16u;
        const bool in = !PAD || c < rowb;
        x.k[t][j] = *(const u32x4*)(kp + row + (in ? c : 0u));
        if constexpr (!WIDE) {
          x.v[t][j] = *(const u32x4*)(vp + row + (in ? c : 0u));
          if (PAD && !in) x.v[t][j] = u32x4{0u, 0u, 0u, 0u};
        }
        if (PAD && !in) x.k[t][j] = u32x4{0u, 0u, 0u, 0u};
      }
      if constexpr (WIDE) {  // [key 4 qd + i][64-element block]: elements 4 m16 ..
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < DP / 64; ++n) {
            const uint32_t c = (uint32_t)(16 * n + m16) * 16u;
            const bool in = !PAD || c < rowb;
            u32x4 a = *(const u32x4*)(vp + (uint32_t)min(4 * qd + i, most) * rowb + (in ? c : 0u));
            if (PAD && !in) a = u32x4{0u, 0u, 0u, 0u};
            x.v[t][i * (DP / 64) + n] = a;
          }
      }
    }
  };
  auto use = [&](int step, const Tile& x) {
    const int base = first + step * STEP;
    // scores: rows = keys 16 t + .., columns = query rows
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if constexpr (WIDE) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[t][j][i]), __uint_as_float(bq[j][i]), s[t], 0,
                                                        0, 0);
        } else {
          s[t] = mfma16<DT>(x.k[t][j], bq[j], s[t]);
          *(u32x4*)(vl + (16 * t + m16) * VS + (4 * j + qd) * 16) = x.v[t][j];
        }
      }
    }
    if constexpr (!WIDE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // this lane's 8 keys are base + 16 t + 4 qd + i
    if (base + TK > full || x.there != 3) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][i] = base + 16 * t + 4 * qd + i <= lim && (x.there >> t & 1) ? s[t][i] : -INFINITY;
    }
    float e[8];
    auto weigh = [&]() {
      float zs = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4] - top, sl, kBelow));
        zs += e[i];
      }
      return zs;
    };
    float zs = weigh();
    if (__any(zs > kMost)) {
      float most = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, s[i / 4][i % 4]);
      most = fmaxf(most, __shfl_xor(most, 16, WAVE));
      most = fmaxf(most, __shfl_xor(most, 32, WAVE));
      const float corr = __builtin_amdgcn_exp2f((top - most) * sl);
      top = most;
      z *= corr;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= corr;
      zs = weigh();
    }
    z += zs;
    if constexpr (WIDE) {
      // sums: o[4 n + c], row m: element 64 n + 4 m + c
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < DP / 64; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              o[4 * n + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[t][i * (DP / 64) + n][c]),
                                                                  e[4 * t + i], o[4 * n + c], 0, 0, 0);
    } else {
      typename Type::frag pw[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const typename Type::elem h = (typename Type::elem)e[i];
        pw[0][i] = h;
        pw[1][i] = (typename Type::elem)(e[i] - (float)h);
      }
      // sums: rows = elements 16 i + .., columns = query rows
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        union {
          s16x4 half[2];
          u32x4 v;
        } a;
        unsigned char* at = vl + (4 * qd + m16 / 4) * VS + (16 * i + m16 % 4 * 4) * 2;
        a.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        a.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 16 * VS));
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          union {
            typename Type::frag f;
            u32x4 u;
          } pn;
          pn.f = pw[n];
          o[i] = mfma16<DT>(a.v, pn.u, o[i]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };
  const int steps = first < k1 ? (k1 - first + STEP - 1) / STEP : 0;
  if constexpr (DP * ES >= 1024) {  // (a second tile does not fit the registers)
    Tile a;
    for (int step = 0; step < steps; ++step) {
      fetch(step, a);
      use(step, a);
    }
  } else {  // two tiles in registers: one is used, the other under way
    Tile a, c;
    if (steps > 0) fetch(0, a);
    if (steps > 1) fetch(1, c);
    for (int step = 0; step < steps; step += 2) {
      use(step, a);
      if (step + 2 < steps) fetch(step + 2, a);
      if (step + 1 < steps) {
        use(step + 1, c);
        if (step + 3 < steps) fetch(step + 3, c);
      }
    }
  }
  // the waves' parts: [wave][query row][m, z (join.h), sums]
  z += __shfl_xor(z, 16, WAVE);
  z += __shfl_xor(z, 32, WAVE);
  if (threadIdx.x == 0) odd_rows = 0u;
  __syncthreads();
  float* mine = (float*)lds + (w * TR + m16) * PS;
  if (qd == 0) mine[0] = top, mine[1] = z;
#pragma unroll
  for (int i = 0; i < NO; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[2 + (WIDE ? 64 * (i / 4) + 16 * qd + 4 * k + i % 4 : 16 * i + 4 * qd + k)] = o[i][k];
  }
  __syncthreads();
  const int here = min(TR, grp * p.Q - rt * TR);
  const bool partial = ranges > 1;
  auto put = [&](int row, int d, float a, float m, float zz) {
    const int gr = rt * TR + row;
    const int t = gr / grp, h = g * grp + gr % grp;
    if (!partial) {
      const int64_t at = (int64_t)b * p.o_bs + (int64_t)h * p.o_hs + (int64_t)t * p.o_ts + d;
      store_elem(p.out, at, p.out_dtype, zz == 0.0f ? 0.0f : a / fabsf(zz));
    } else {
      const int64_t at = (((int64_t)b * p.H + h) * p.Q + t) * p.splits + split;
      p.sums[at * p.D + d] = a;
      if (d == 0) p.stats[2 * at] = m, p.stats[2 * at + 1] = zz;
    }
  };
  for (int n = (int)threadIdx.x; n < here * DP; n += AW * WAVE) {
    const int row = n / DP, d = n % DP;
    if (PAD && d >= dim) continue;
    const float* f = (const float*)lds + row * PS;
    float M = f[0], Z = 0.0f, x = 0.0f;
#pragma unroll
    for (int v = 1; v < AW; ++v) M = fmaxf(M, f[v * TR * PS]);
#pragma unroll
    for (int v = 0; v < AW; ++v) {
      const float share = __builtin_amdgcn_exp2f((f[v * TR * PS] - M) * sl);
      Z += f[v * TR * PS + 1] * share;
      x += f[v * TR * PS + 2 + d] * share;
    }
    if (!(fabsf(x) <= (partial ? kLarge : 3.40282347e38f)) || !(Z <= 3.40282347e38f)) {
      atomicOr(&odd_rows, 1u << row);
      continue;
    }
    put(row, d, x, M, Z);
  }
  __syncthreads();
  for (uint32_t left = odd_rows, i = 0; left != 0u; left &= left - 1, ++i) {
    if ((int)(i % AW) != w) continue;
    const int row = __builtin_ctz(left), gr = rt * TR + row;
    const int t = gr / grp, h = g * grp + gr % grp;
    float acc[DP / 64], m, zz;
    attend_again<DT, DP>(p, (int64_t)b * p.q_bs + (int64_t)h * p.q_hs + (int64_t)t * p.q_ts, b, g, k0,
                         seen_by(t), sl, acc, m, zz);
#pragma unroll
    for (int k = 0; k < DP / 64; ++k)
      if (lane + 64 * k < p.D) put(row, lane + 64 * k, acc[k], m, zz);
  }
}

// Keys per workgroup.  A CU holds three workgroups of rows of up to 256 bytes
// (K and V), two of 512, one of more.
//  * A range of 128 KB is one workgroup's business, whatever follows: a CU takes
//    50 GB/s, and a second launch 3 us (500 keys of 9 x 64: 7.4 us in one range,
//    9.2 in two; 1000 10.8 in one, 9.2 in four).
//  * One sequence: one round of the places of the CUs where that makes ranges of
//    up to 1024 keys, else two (100000 keys of 9 x 64 fp32: 42 us in 471
//    workgroups on 512 places, 53 in 294, 48 in 783).
//  * Sequences that may differ in length: eight times the card's workgroups (the
//    last to end is then a small part of the call: 32 sequences of up to 131072
//    keys 297 us, 330 with a quarter as many), but ranges of 1024 keys where those
//    fill it already (16 x 8192 keys of 16 x 128: 40 us, 48 with 384).
// At most 384 ranges (each costs a row of partial sums), of at least 256 keys.
int64_t chunk_keys(int64_t n_seq, int64_t groups, int64_t row_bytes, int64_t n_keys) {
  if (n_keys * row_bytes <= 131072) return (n_keys + STEP - 1) / STEP * STEP;
  const int64_t places = row_bytes <= 256 ? 768 : (row_bytes <= 512 ? 512 : 256), work = n_keys * groups;
  const int64_t most = n_seq > 1 ? 8192 : (work <= 1024 * places ? places : 2 * places);
  const int64_t want = std::min<int64_t>(384, std::max<int64_t>(1, most / groups));
  const int64_t least = n_seq > 1 ? std::min<int64_t>(8 * STEP, work / (row_bytes <= 256 ? 768 : 256)) : 0;
  return (std::max<int64_t>(std::max<int64_t>(least, 2 * STEP), (n_keys + want - 1) / want) + STEP - 1) / STEP * STEP;
}

int64_t row_tiles(int64_t H, int64_t G, int64_t Q) { return (H / G * Q + TR - 1) / TR; }

template <int DT>
int launch(const PagedParams& p, dim3 grid, hipStream_t stream) {
  const dim3 block(AW * WAVE);
  if (p.D == 64) hipLaunchKernelGGL((paged_attention_kernel<DT, 64, false>), grid, block, 0, stream, p);
  else if (p.D == 128) hipLaunchKernelGGL((paged_attention_kernel<DT, 128, false>), grid, block, 0, stream, p);
  else if (p.D == 256) hipLaunchKernelGGL((paged_attention_kernel<DT, 256, false>), grid, block, 0, stream, p);
  else if (p.D < 64) hipLaunchKernelGGL((paged_attention_kernel<DT, 64, true>), grid, block, 0, stream, p);
  else if (p.D < 128) hipLaunchKernelGGL((paged_attention_kernel<DT, 128, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((paged_attention_kernel<DT, 256, true>), grid, block, 0, stream, p);
  SVA_CHECK_LAUNCH("paged_attention_kernel");
  return SVA_OK;
}

}  // namespace

extern "C" size_t sva_paged_attention_workspace_bytes(int64_t n_seq, int64_t H, int64_t G, int64_t Q, int64_t D,
                                                      int dtype, int64_t n_keys) {
  if (n_seq <= 0 || H <= 0 || G <= 0 || Q <= 0 || D <= 0 || n_keys <= 0 || H % G != 0) return 0;
  const int64_t chunk = chunk_keys(n_seq, n_seq * G * row_tiles(H, G, Q), 2 * D * (dtype == F32 ? 4 : 2), n_keys);
  const int64_t splits = (n_keys + chunk - 1) / chunk;
  return splits == 1 ? 0 : join_bytes(n_seq * H * Q, splits, D);
}

extern "C" int sva_paged_attention(const void* q, int dtype, int64_t q_seq_stride, int64_t q_head_stride,
                                   int64_t q_tok_stride, const void* pool, int64_t n_pages, int64_t page_stride,
                                   int64_t page_rows, const int32_t* tables, int64_t table_stride, int64_t max_pages,
                                   const int64_t* seq_lens, int64_t n_keys, int64_t n_seq, int64_t H, int64_t G,
                                   int64_t Q, int64_t D, float scaling, void* out, int out_dtype,
                                   int64_t out_seq_stride, int64_t out_head_stride, int64_t out_tok_stride,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(q && pool && tables && seq_lens && out, "sva_paged_attention: null pointer");
  SVA_REQUIRE(n_seq > 0 && H > 0 && G > 0 && Q > 0 && n_keys > 0 && n_pages > 0 && max_pages > 0 && H % G == 0,
              "sva_paged_attention: bad sizes");
  SVA_REQUIRE(D > 0 && D <= 256 && D % 8 == 0, "sva_paged_attention: head_dim %lld is not a multiple of 8 up to 256",
              (long long)D);
  SVA_REQUIRE(page_rows_ok(page_rows), "sva_paged_attention: %lld rows a page are no power of two from 16 to 1024",
              (long long)page_rows);
  SVA_REQUIRE(dtype >= 0 && dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, "sva_paged_attention: bad dtype");
  const int64_t es = dtype == F32 ? 4 : 2;
  SVA_REQUIRE(((uintptr_t)pool & 15u) == 0 && page_stride * es % 16 == 0 && page_stride >= 2 * G * page_rows * D,
              "sva_paged_attention: pages are not 16-byte aligned blocks of 2 x G x rows x head_dim elements");
  SVA_REQUIRE(2 * G * page_rows * D * es < (1ll << 31), "sva_paged_attention: pages of 2 GiB and more");
  SVA_REQUIRE(n_pages < (1ll << 31) && max_pages < (1ll << 31), "sva_paged_attention: too many pages");
  const int64_t keys = std::min(n_keys, max_pages * page_rows);
  SVA_REQUIRE(n_seq < (1ll << 31) && H < (1ll << 31) && Q < (1ll << 31) && n_seq * H < (1ll << 31) &&
                  n_seq * H * Q < (1ll << 31) && keys < (1ll << 31) - 1024,
              "sva_paged_attention: too many items or keys");
  const int64_t tiles = row_tiles(H, G, Q);
  const size_t need = sva_paged_attention_workspace_bytes(n_seq, H, G, Q, D, dtype, keys);
  SVA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "sva_paged_attention: workspace of %zu bytes required",
              need);
  PagedParams p;
  p.q = q;
  p.q_bs = q_seq_stride;
  p.q_hs = q_head_stride;
  p.q_ts = q_tok_stride;
  p.q_vec = ((uintptr_t)q & 15u) == 0 && q_seq_stride * es % 16 == 0 && q_head_stride * es % 16 == 0 &&
            q_tok_stride * es % 16 == 0;
  p.c.pool = (unsigned char*)const_cast<void*>(pool);
  p.c.page_bytes = page_stride * es;
  p.c.pages = n_pages;
  p.c.tables = tables;
  p.c.table_stride = table_stride;
  p.c.max_pages = (int)max_pages;
  p.c.bits = page_bits(page_rows);
  p.lens = seq_lens;
  p.N = keys;
  p.n_seq = (int)n_seq;
  p.H = (int)H;
  p.G = (int)G;
  p.Q = (int)Q;
  p.D = (int)D;
  p.row_tiles = (int)tiles;
  p.chunk = (int)chunk_keys(n_seq, n_seq * G * tiles, 2 * D * es, keys);
  p.splits = (int)((keys + p.chunk - 1) / p.chunk);
  p.scaling = scaling;
  p.stats = (float*)workspace;
  p.sums = p.stats + join_stats_floats(n_seq * H * Q, p.splits);
  p.out = out;
  p.out_dtype = out_dtype;
  p.o_bs = out_seq_stride;
  p.o_hs = out_head_stride;
  p.o_ts = out_tok_stride;
  const int64_t units = n_seq * G * p.splits, blocks = (units + kXcds - 1) / kXcds * kXcds * tiles;
  SVA_UNSUPPORTED(blocks < (1ll << 31), "sva_paged_attention: %lld tokens of %lld sequences in one call", (long long)Q,
                  (long long)n_seq);
  const dim3 grid((unsigned)blocks);
  int rc;
  if (dtype == F32) rc = launch<F32>(p, grid, (hipStream_t)stream);
  else if (dtype == BF16) rc = launch<BF16>(p, grid, (hipStream_t)stream);
  else rc = launch<F16>(p, grid, (hipStream_t)stream);
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
  j.offs = nullptr;
  j.N = j.rows = keys;
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
