// Dense attention of whole prompts: the kernel.
//
// out[r] = sum_n p[n] V[n] / sum_n p[n], p[n] = 2^(s (q[r] . K[n]) - m), over
// the keys row r may see, in one pass over the keys with a running reference
// m.  The query rows of a KV head are (token, head of its group) pairs,
// token-major, so one K / V tile serves every head of the group.  Four waves
// of 32 query rows each share tiles of BN keys in LDS (two buffers of K and
// of V: the next tiles arrive, straight from memory, while these are used).
//  * S^T = K Q^T (rows: keys) leaves each lane with half of the tile's scores
//    of one query row, and exactly the elements of P^T that the second
//    product O^T = V^T P^T wants from it: weights stay in registers, a row's
//    maximum takes one exchange between the wave's halves.
//  * The reference m is a maximum of the row's first keys and only moves when
//    a lane's weights of a tile sum to more than 2^16 (fp16: 2^15): the tile's
//    maximum is then taken, the sums rescaled and the weights done again.  The
//    sum is needed anyway, so an ordinary tile looks for no maximum.  (fp16
//    weights are 2^8 at a new reference, to keep small ones normal.)
//  * Weights are rounded to the type of V for the product (bf16: at most 2^-8
//    of each, of random sign, as V's own rounding); m, the sum of weights and
//    the sums are fp32.  (A second term for the rest would cost 8192 tokens of
//    9 x 64 161 us against 120, 8 x 512 over 32768 keys 591 against 431, and
//    prompts of 32 x 128, out of registers, four times.)  fp32 inputs use the
//    fp32 matrix instructions throughout.
//  * At most 16 query rows a KV head (decode tokens): memory sets the time, and
//    half of the product's 32 columns are free.  They take each weight's second
//    term, its rest after rounding: the outputs keep about 16 bits of the
//    weights (bf16 difference from fp32 attention 2.5e-3 -> 6e-5).  Two waves
//    take a tile's 32-key halves, joined in LDS.  32 sequences of up to 131072
//    keys, 9 x 64: 302 us, as one wave with one term; 24 of up to 42K, 32 x 128:
//    384 (417).
//  * Three tiles are in work at once: while tile t is weighed on the vector
//    units, tile t + 1's scores and tile t - 1's sums are on the matrix units.
// What bounds it: at 9 x 64, 32768 bf16 tokens (1.33 ms, 930 TFLOP/s; a
// library product of 16384 reaches 1372 here) the matrix units are busy two
// fifths of the time and the vector units half, an exponential and four
// other instructions a score; at 32 x 128, 8192 tokens 557 us, 986 TFLOP/s.
// Two waves a SIMD do not fill what one leaves; three (without tiles in
// work at once) gave 870, eight waves in one workgroup 840, a meeting of the
// waves every second tile 913.  Whole prompts of a few thousand tokens wait
// for their longest row tile (8192 tokens: 576 workgroups, 120 us).
//  * A masked key's V meets a weight of 0, which a NaN or an infinity
//    survives: a wave whose sums are not finite does its rows again, key by
//    key, over the keys they may see alone (some hundred times the time).  So
//    does one with a score past 2^26, where a reference in fp32 is no longer
//    within a few units of it, and one with larger sums than the ranges'
//    together can hold.
#pragma once
// (loads to LDS name m0 among what they change)
#pragma clang diagnostic ignored "-Winline-asm"
#include "cache4.h"
#include "join.h"

namespace sva {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct PromptParams {
  const void* q;
  int64_t q_bs, q_hs, q_ts;
  const int64_t* q_offsets;
  const int64_t* q_lens;
  int64_t q_rows;
  const void* keys;
  const void* values;
  int64_t kv_hs, kv_rs, kv_rows;
  const int64_t* offs;
  const int64_t* lens;
  int64_t N;
  int n_seq, H, G, Q, D, row_tiles, splits;
  int chunk;     // keys per workgroup, a multiple of 64
  float scaling;
  const void* mask;
  int mask_type;
  int64_t mask_bs, mask_ts;
  float* sums;   // join.h
  float* stats;
  void* out;
  int out_dtype;
  bool out_vec;  // four elements of an output row are one aligned store
  int64_t o_bs, o_hs, o_ts;
};

// Where 16-byte chunk ch of row r of a tile lies in LDS: ch ^ k_chunk(r) (K:
// the rows of one column, 16 at a time, meet no bank twice) and ch ^
// v_chunk(r) (V: nor do the four 64-byte row pieces of half a wave's
// transposed read).  CPR: chunks of a row, 8 of them half of the banks.
template <int CPR>
SVA_DEV int k_chunk(int r) {
  return CPR == 8 ? (r & 7) ^ (r >> 3 & 1) : r & 15;
}
template <int CPR>
SVA_DEV int v_chunk(int r) {
  return CPR == 8 ? 2 * (r & 3) : (4 * (r & 3)) ^ (r & 2);
}

template <int DT>
struct PromptType {
  using type = typename std::conditional<DT == BF16, __bf16, _Float16>::type;
  typedef type pair __attribute__((ext_vector_type(2)));
  // z + e[0] + e[1]: the sum of the weights as the second product takes them
  static SVA_DEV float sum2(pair e, float z) {
    const pair one = {(type)1.0f, (type)1.0f};
    if constexpr (DT == BF16) return __builtin_amdgcn_fdot2_f32_bf16(e, one, z, false);
    else return __builtin_amdgcn_fdot2(e, one, z, false);
  }
  static constexpr int ES = DT == F32 ? 4 : 2;
  static constexpr int BN = DT == F32 ? 32 : 64;
  // waves per SIMD that the registers are kept to
  static constexpr int waves(int dp) { return dp > 128 || (DT == F32 && dp > 64) ? 1 : 2; }
};

// Which of the four keys at mask element i (of its row) a mask allows, bit by
// bit, in one load of any alignment.
SVA_DEV uint32_t prompt_mask_allows4(const void* row, int64_t i, int mtype) {
  if (mtype == MASK_BOOL) {
    uint32_t u;
    __builtin_memcpy(&u, (const uint8_t*)row + i, 4);
    return (u & 0xFFu ? 1u : 0u) | (u & 0xFF00u ? 2u : 0u) | (u & 0xFF0000u ? 4u : 0u) | (u >> 24 ? 8u : 0u);
  }
  uint32_t bits = 0u;
  if (mtype == MASK_F32) {
    float x[4];
    __builtin_memcpy(x, (const float*)row + i, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) bits |= x[k] > -1e4f ? 1u << k : 0u;
  } else {
    uint16_t x[4];
    __builtin_memcpy(x, (const uint16_t*)row + i, 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) bits |= elem_from_bits(x[k], mtype == MASK_BF16 ? BF16 : F16) > -1e4f ? 1u << k : 0u;
  }
  return bits;
}

SVA_DEV bool prompt_mask_allows(const void* mask, int64_t i, int mtype) {
  return mtype == MASK_BOOL ? ((const uint8_t*)mask)[i] != 0 : mask_allows(mask, i, mtype);
}

// How a call's rows are read and masked: whole aligned rows of DP elements
// under the causal rule, the same under a mask, anything else.  PROMPT_FEW
// added: 16-bit calls of at most 16 query rows a KV head, two-term weights.
enum PromptMode : int { PROMPT_CAUSAL = 0, PROMPT_MASK = 1, PROMPT_ANY = 2, PROMPT_FEW = 4 };
constexpr int kFewRows = 16;

template <int DT, int DP, int MODE>
__global__ void __launch_bounds__(256, PromptType<DT>::waves(DP)) prompt_kernel(PromptParams p) {
  constexpr int FORM = MODE % PROMPT_FEW;
  constexpr bool VEC = FORM != PROMPT_ANY, FEW = MODE >= PROMPT_FEW;
  const bool MASK = FORM == PROMPT_MASK || (FORM == PROMPT_ANY && p.mask != nullptr);
  constexpr int ES = PromptType<DT>::ES, BN = PromptType<DT>::BN;
  constexpr int KT = FEW ? 1 : BN / 32;  // 32-key blocks of a tile that a wave takes
  constexpr int CPR = DP * ES / 16;      // 16-byte chunks of a row
  constexpr int CH = BN * CPR / 256;     // chunks per thread
  constexpr int EC = 16 / ES;            // elements of a chunk
  constexpr int BM = 4 * 32;             // query rows of a workgroup
  constexpr int TB = BN * DP * ES;       // bytes of a K or V tile
  constexpr int NO = DP / 32;            // 32-element blocks of the sums
  constexpr float kMost = DT == F16 ? 32768.0f : 65536.0f;  // a lane's weights of a tile may sum to
  constexpr float kBelow = DT == F16 ? 8.0f : 0.0f;         // how far below the maximum a new reference lies
  constexpr float kNoKey = -3.40282347e38f;                 // the reference of a row that has seen no key
  constexpr float kLarge = 0x1p110f;                        // 64 ranges' sums of less stay finite together
  constexpr float kFar = 67108864.0f;                       // references past 2^26: done again
  using Elem = PromptType<DT>;
  using pair = typename Elem::pair;
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = (int)threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int l32 = lane & 31, hf = lane >> 5, m16 = lane & 15;

  // KV heads fastest (8 of them: one XCD's L2 each), then the row tiles, the longest first
  int64_t id = blockIdx.x;
  const int g = (int)(id % p.G);
  id /= p.G;
  const int rt = p.row_tiles - 1 - (int)(id % p.row_tiles);
  id /= p.row_tiles;
  const int split = (int)(id % p.splits);
  const int b = (int)(id / p.splits);
  const int grp = p.H / p.G;
  int64_t q_first;
  const int q_len = seq_tokens(p.q_lens, p.q_offsets, p.q_rows, p.Q, b, q_first);
  const int rows = q_len * grp;
  if (rt * BM >= rows) return;
  int64_t off;
  const int len = (int)seq_keys(p.lens, p.offs, p.N, p.kv_rows, b, off);
  const int shift = len - q_len;  // token t sees keys n <= t + shift
  const int keys = (int)tile_keys(rt, BM, q_len, grp, len, !MASK);
  const int ranges = tile_ranges(keys, p.chunk);
  if (split >= ranges) return;
  const bool partial = ranges > 1;  // joined by a second kernel
  const int kbeg = split * p.chunk;
  const int kend = kbeg + min(p.chunk, max(keys - kbeg, 0));

  // this wave's rows, one per lane and half
  const int wrow = FEW ? 0 : rt * BM + w * 32;
  const int wend = min(rows, wrow + 32);
  const bool busy = FEW ? w < BN / 32 : wrow < rows;
  const int kt0 = FEW ? w : 0;  // this wave's first block of a tile
  const int wfull = min(len, wrow / grp + shift + 1);  // keys below are seen by every row of the wave
  const int64_t kvb = (int64_t)g * p.kv_hs + off * p.kv_rs;  // element offset of key 0
  auto q_at = [&](int r, int64_t bs, int64_t hs, int64_t ts) {
    const int tok = r / grp, head = g * grp + r % grp;
    return (p.q_lens ? (q_first + tok) * ts : (int64_t)b * bs + (int64_t)tok * ts) + (int64_t)head * hs;
  };
  using frag = typename std::conditional<DT == BF16, bf16x8, typename std::conditional<DT == F16, f16x8, f32x4>::type>::type;
  struct frag_pair {
    frag v[2];
    SVA_DEV frag& operator[](int i) { return v[i]; }
    SVA_DEV const frag& operator[](int i) const { return v[i]; }
  };
  using weights = typename std::conditional<DT == F32, f32x16, frag_pair>::type;  // of 32 keys
  constexpr int NF = DT == F32 ? DP / 8 : DP / 16;  // fragments of a row per lane
  constexpr int FE = DT == F32 ? 4 : 8;             // elements of one: d = 2 FE f + FE hf + i
  const bool second = FEW && l32 >= kFewRows;  // this lane's weights are the second terms of its row's
  const int row = wrow + (FEW ? l32 % kFewRows : l32);
  const bool live = row < rows;
  const int lim = live ? (MASK ? kend - 1 : min(kend - 1, row / grp + shift)) : -1;  // the last key of the row
  const unsigned char* mrow = nullptr;                                                 // its mask row
  if (MASK) {
    const int64_t at = (int64_t)b * p.mask_bs + (int64_t)(live ? row / grp : 0) * p.mask_ts;
    mrow = (const unsigned char*)p.mask + at * (p.mask_type == MASK_F32 ? 4 : (p.mask_type == MASK_BOOL ? 1 : 2));
  }
  frag bq[NF];
  {
    const int64_t at = q_at(live ? row : 0, p.q_bs, p.q_hs, p.q_ts);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int d = 2 * FE * f + FE * hf;
      if (VEC) {
        union {
          u32x4 u;
          frag v;
        } x;
        x.u = *(const u32x4*)((const unsigned char*)p.q + (at + d) * ES);
        bq[f] = live ? x.v : frag{};
      } else {
#pragma unroll
        for (int i = 0; i < FE; ++i) {
          const float x = live && d + i < p.D ? load_elem(p.q, at + d + i, DT) : 0.0f;
          if constexpr (DT == BF16) bq[f][i] = (__bf16)x;
          else if constexpr (DT == F16) bq[f][i] = (_Float16)x;
          else bq[f][i] = x;
        }
      }
      if (p.scaling < 0.0f) bq[f] = -bq[f];
    }
  }
  const float sl = score_scale(p.scaling);

  f32x16 o[NO];
  float top = kNoKey, mref = kNoKey, z = 0.0f;  // the reference before the scale and after it
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[i][k] = 0.0f;

  // Tiles go to LDS as the loads return (whole aligned rows: 16 bytes a lane,
  // a wave's 64 one after another; otherwise element by element through
  // registers).  Slot i of a tile holds chunk i % CPR ^ swizzle(row) of row
  // i / CPR: a lane's source lies a 32-bit byte offset from the tile's first
  // row (checked by the host), the same for every tile but the last.
  const uint32_t rowb = (uint32_t)p.kv_rs * ES;
  auto swizzle = [&](int r, bool v) { return v ? (ES == 2 ? v_chunk<CPR>(r) : 0) : k_chunk<CPR>(r); };
  uint32_t from[2][CH];
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = tid + 256 * c;
      from[v][c] = i / CPR * rowb + (i % CPR ^ swizzle(i / CPR, v)) * 16;
    }
  auto load = [&](int v, int n0, unsigned char* buf) {
    const unsigned char* tile =
        (const unsigned char*)(v ? p.values : p.keys) + (kvb + (int64_t)n0 * p.kv_rs) * ES;
    const int most = len - 1 - n0;  // rows past the end: the last key
    if constexpr (VEC) {
      const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)buf + w * 1024;
      const bool last = most < BN - 1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t o = from[v][c];
        if (last) {
          const int r = (tid + 256 * c) / CPR;
          if (r > most) o -= (uint32_t)(r - most) * rowb;
        }
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :
                     : "v"(o), "s"(tile), "s"(at + c * 4096)
                     : "memory", "m0");
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int i = tid + 256 * c;
        const int r = i / CPR, ch = i % CPR ^ swizzle(r, v);
        const uint32_t o = min(r, most) * rowb + ch * 16;
        union {
          u32x4 u;
          uint16_t h[8];
          uint32_t w[4];
        } a;
#pragma unroll
        for (int k = 0; k < EC; ++k) {
          const bool in = ch * EC + k < p.D;
          if constexpr (ES == 4) a.w[k] = in ? *(const uint32_t*)(tile + o + 4 * k) : 0u;
          else a.h[k] = in ? *(const uint16_t*)(tile + o + 2 * k) : (uint16_t)0;
        }
        *(u32x4*)(buf + i * 16) = a.u;
      }
    }
  };
  // every load of this wave is in LDS, then every wave's
  auto arrive = [&]() {
    if constexpr (VEC) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  // the steps of a tile: scores, masking, weights, sums
  auto scores = [&](const unsigned char* kb, f32x16 (&s)[KT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int k = 0; k < 16; ++k) s[kt][k] = 0.0f;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const frag a = *(const frag*)(kb + ((32 * (kt0 + kt) + l32) * CPR + ((2 * f + hf) ^ k_chunk<CPR>(l32))) * 16);
        if constexpr (DT == BF16) {
          s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, bq[f], s[kt], 0, 0, 0);
        } else if constexpr (DT == F16) {
          s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, bq[f], s[kt], 0, 0, 0);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], bq[f][i], s[kt], 0, 0, 0);
        }
      }
    }
  };
  // a lane's score k of block kt0 + kt is its key 8 (k / 4) + 4 hf + k % 4
  auto hide = [&](int n0, f32x16 (&s)[KT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int key = n0 + 32 * (kt0 + kt) + 2 * k + 4 * hf;
        uint32_t seen = 15u;
        if (MASK) {
          seen = 0u;
          if (key + 3 <= lim) {
            seen = prompt_mask_allows4(mrow, key, p.mask_type);
          } else {
            for (int j = 0; j < 4; ++j)
              if (key + j <= lim && prompt_mask_allows(mrow, key + j, p.mask_type)) seen |= 1u << j;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[kt][k + j] = key + j <= lim && (seen >> j & 1u) ? s[kt][k + j] : -INFINITY;
      }
  };
  auto weigh = [&](const f32x16 (&s)[KT], weights (&pw)[KT]) {
    float zs = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      if constexpr (DT == F32) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          pw[kt][k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][k], sl, -mref));
          zs += pw[kt][k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][k], sl, -mref));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][k + 1], sl, -mref));
          pair e;
          e[0] = (typename Elem::type)e0, e[1] = (typename Elem::type)e1;
          if constexpr (FEW) {
            pair r;
            r[0] = (typename Elem::type)(e0 - (float)e[0]), r[1] = (typename Elem::type)(e1 - (float)e[1]);
            e = second ? r : e;
          }
          pw[kt][k / 8][k % 8] = e[0], pw[kt][k / 8][k % 8 + 1] = e[1];
          zs = Elem::sum2(e, zs);
        }
      }
    }
    return zs;
  };
  // where a tile's weights sum to more than kMost (the first one's with a key
  // always: the reference starts below every score), the reference moves to
  // its maximum
  auto settle = [&](float zs, const f32x16 (&s)[KT], weights (&pw)[KT]) {
    if (__any(zs > kMost)) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int k = 0; k < 16; ++k) top = fmaxf(top, s[kt][k]);
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      const float mn = fmaxf(mref, top * sl - kBelow);
      const float corr = __builtin_amdgcn_exp2f(mref - mn);
      mref = mn;
      z *= corr;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= corr;
      zs = weigh(s, pw);
    }
    z += zs;
  };
  auto sums = [&](const unsigned char* vb, const weights (&pw)[KT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      if constexpr (DT == F32) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float* vrow = (const float*)(vb + (32 * (kt0 + kt) + 8 * (k / 4) + 4 * hf + k % 4) * CPR * 16);
#pragma unroll
          for (int i = 0; i < NO; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(vrow[32 * i + l32], pw[kt][k], o[i], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
#pragma unroll
          for (int i = 0; i < NO; ++i) {
            union {
              s16x4 half[2];
              frag v;
            } a;
            const int row = 32 * (kt0 + kt) + 16 * st + 4 * hf + m16 / 4;
            const int ch = (4 * i + 2 * (lane >> 4 & 1) + (m16 & 3) / 2) ^ v_chunk<CPR>(m16 / 4);
            const unsigned char* at = vb + (row * CPR + ch) * 16 + (m16 & 1) * 8;
            a.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            a.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(at + 8 * CPR * 16));
            if constexpr (DT == BF16) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, pw[kt][st], o[i], 0, 0, 0);
            else o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, pw[kt][st], o[i], 0, 0, 0);
          }
        }
      }
    }
  };

  // Tile t's scores are taken while tile t - 1 is weighed and tile t - 2's
  // sums are added: the matrix and the vector instructions of one step do not
  // wait for one another.  K is a tile ahead of that, V two behind it.
  unsigned char* const kbuf = lds;
  unsigned char* const vbuf = lds + 2 * TB;
  const int nt = (kend - kbeg + BN - 1) / BN;
  if (nt > 0) {
    f32x16 s[KT], s2[KT];
    weights pw[KT], pw2[KT];
    auto step = [&](int t, f32x16 (&sc)[KT], f32x16 (&sn)[KT], weights (&pc)[KT], weights (&pp)[KT], bool first) {
      // weigh tile t (scores sc) into pc, add tile t - 1 (weights pp), score tile t + 1 into sn
      const int n0 = kbeg + t * BN;
      if (t + 2 < nt) load(0, n0 + 2 * BN, kbuf + (t & 1) * TB);
      load(1, n0, vbuf + (t & 1) * TB);
      if (busy) {
        if (MASK || n0 + BN > wfull) hide(n0, sc);
        scores(kbuf + ((t + 1) & 1) * TB, sn);  // (behind the last tile: not used)
        if (!first) sums(vbuf + ((t + 1) & 1) * TB, pp);
        const float zs = weigh(sc, pc);
        if constexpr (DP == 128 && ES == 2) {  // a matrix instruction, then the vector instructions of its time
#pragma unroll
          for (int i = 0; i < 2 * KT * NF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
          }
        }
        settle(zs, sc, pc);
      }
      arrive();
    };
    load(0, kbeg, kbuf);
    if (nt > 1) load(0, kbeg + BN, kbuf + TB);
    arrive();
    if (busy) scores(kbuf, s);
    __syncthreads();  // (tile 2 takes tile 0's place)
    step(0, s, s2, pw, pw2, true);
    int t = 1;
    for (; t + 1 < nt; t += 2) {
      step(t, s2, s, pw2, pw, false);
      step(t + 1, s, s2, pw, pw2, false);
    }
    if (t < nt) {
      step(t, s2, s, pw2, pw, false);
      if (busy) sums(vbuf + (t & 1) * TB, pw2);
    } else if (busy) {
      sums(vbuf + ((t - 1) & 1) * TB, pw);
    }
  }
  if (!FEW && !busy) return;

  // the two halves of the wave hold a row's keys
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(z), __float_as_uint(z), false, false);
    z = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  const bool far = top != kNoKey && fabsf(mref) > kFar;
  // what brings weights relative to m, rounded, to `top`, which is not
  float even = top == kNoKey ? 1.0f : __builtin_amdgcn_exp2f(-__builtin_fmaf(top, sl, -mref));
  if constexpr (FEW) {  // both terms, then both waves: wave 0 goes on with all of it
    z += __shfl_xor(z, kFewRows, WAVE);
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[i][k] += __shfl_xor(o[i][k], kFewRows, WAVE);
    float* part = (float*)lds + lane;  // [m, z, sums][lane], in the tiles' place
    __syncthreads();
    if (w == 1) {
      part[0] = top, part[WAVE] = far ? NAN : z * even;
#pragma unroll
      for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) part[(2 + 16 * i + k) * WAVE] = far ? NAN : o[i][k] * even;
    }
    __syncthreads();
    if (w != 0) return;
    const float m1 = part[0], mn = fmaxf(top, m1);
    const float f0 = __builtin_amdgcn_exp2f((top - mn) * sl) * even, f1 = __builtin_amdgcn_exp2f((m1 - mn) * sl);
    top = mn;
    even = 1.0f;
    z = z * f0 + part[WAVE] * f1;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[i][k] = o[i][k] * f0 + part[(2 + 16 * i + k) * WAVE] * f1;
  }
  const float most = partial ? kLarge : 3.40282347e38f;
  // (fma(s, sl, -m) is exact before its rounding, m is not: it is off by up to 2 at 2^26, by 128 at 2^31)
  bool odd = far;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) odd = odd || !(fabsf(o[i][k]) <= most);
  auto part_at = [&](int r) {
    const int tok = r / grp, head = g * grp + r % grp;
    return (((int64_t)b * p.H + head) * p.Q + tok) * p.splits + split;
  };
  if (__any(odd)) {
    // again, key by key: lanes take 64 keys' scores, then the row's elements
    for (int r = wrow; r < wend; ++r) {
      const int end = MASK ? kend : min(kend, r / grp + shift + 1);
      const int64_t qa = q_at(r, p.q_bs, p.q_hs, p.q_ts);
      // (finite V with larger sums: once more, weights and sums 2^-60 of themselves)
      float m, zz, down = 1.0f, acc[DP / 64];
      for (;;) {
        m = -INFINITY, zz = 0.0f;
        bool finite[DP / 64];
#pragma unroll
        for (int k = 0; k < DP / 64; ++k) acc[k] = 0.0f, finite[k] = true;
        for (int n0 = kbeg; n0 < end; n0 += WAVE) {
          const int key = n0 + lane;
          bool ok = key < end;
          if (MASK)
            ok = ok && prompt_mask_allows(p.mask, (int64_t)b * p.mask_bs + (int64_t)(r / grp) * p.mask_ts + key,
                                          p.mask_type);
          float sc = -INFINITY;
          if (ok) {
            sc = 0.0f;
            const int64_t ka = kvb + (int64_t)key * p.kv_rs;
            for (int d = 0; d < p.D; ++d)
              sc = __builtin_fmaf(load_elem(p.q, qa + d, DT), load_elem(p.keys, ka + d, DT), sc);
            sc = p.scaling < 0.0f ? -sc : sc;
          }
          const float mn = fmaxf(m, wave_max(sc));
          const float corr = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * sl);
          const float e = ok ? __builtin_amdgcn_exp2f((sc - (mn == -INFINITY ? 0.0f : mn)) * sl) * down : 0.0f;
          m = mn;
          zz = zz * corr + wave_sum(e);
#pragma unroll
          for (int k = 0; k < DP / 64; ++k) acc[k] *= corr;
          const uint64_t seen = __ballot(ok);
          for (int j = 0; j < min(WAVE, end - n0); ++j) {
            if (!(seen >> j & 1ull)) continue;
            const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(e), j));
            const int64_t va = kvb + (int64_t)(n0 + j) * p.kv_rs;
#pragma unroll
            for (int k = 0; k < DP / 64; ++k) {
              const int d = lane + 64 * k;
              if (d < p.D) {
                const float v = load_elem(p.values, va + d, DT);
                finite[k] = finite[k] && fabsf(v) <= 3.40282347e38f;
                acc[k] = __builtin_fmaf(pj, v, acc[k]);
              }
            }
          }
        }
        bool large = false;
#pragma unroll
        for (int k = 0; k < DP / 64; ++k) large = large || (finite[k] && zz == zz && !(fabsf(acc[k]) <= kLarge));
        if (down != 1.0f || !__any(large)) break;
        down = kShifted;
      }
#pragma unroll
      for (int k = 0; k < DP / 64; ++k) {
        const int d = lane + 64 * k;
        if (d >= p.D) continue;
        if (partial)
          p.sums[part_at(r) * p.D + d] = acc[k];
        else
          store_elem(p.out, q_at(r, p.o_bs, p.o_hs, p.o_ts) + d, p.out_dtype, zz == 0.0f ? 0.0f : acc[k] / zz);
      }
      if (partial && lane == 0) p.stats[2 * part_at(r)] = m, p.stats[2 * part_at(r) + 1] = down == 1.0f ? zz : -zz;
    }
    return;
  }
  if (!live || second) return;
  // four consecutive elements at a time
  void* dst = partial ? (void*)p.sums : p.out;
  const int type = partial ? (int)F32 : p.out_dtype;
  const int64_t at = partial ? part_at(row) * p.D : q_at(row, p.o_bs, p.o_hs, p.o_ts);
  const float f = partial ? even : (z == 0.0f ? 0.0f : 1.0f / z);
  if (partial && hf == 0) p.stats[2 * part_at(row)] = top, p.stats[2 * part_at(row) + 1] = z * even;
  const bool whole = partial ? p.D % 4 == 0 : p.out_vec;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      const int d = 32 * i + 2 * k + 4 * hf;
      if (d >= p.D) continue;
      const float x[4] = {o[i][k] * f, o[i][k + 1] * f, o[i][k + 2] * f, o[i][k + 3] * f};
      if (whole) {
        if (type == F32) {
          *(f32x4*)((float*)dst + at + d) = f32x4{x[0], x[1], x[2], x[3]};
        } else {
          uint16_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) store_elem(h, j, type, x[j]);
          *(uint2*)((uint16_t*)dst + at + d) =
              make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < p.D) store_elem(dst, at + d + j, type, x[j]);
      }
    }
}

}  // namespace sva
