// The next token of every row of logits, from a given random number.
//
// Weights w = exp((x - M) / T), M the largest logit.  Of the tokens in the
// order of falling logits (ties: the lower token first) those are kept that
// are among the first top_k, have less than top_p of the sum of these before
// them, and weigh at least min_p; the answer is the first token, by number, up
// to which the kept weights sum to more than u of their sum.  T <= 0: the
// largest logit.  A NaN counts as -inf; infinity counts as the largest number.
//
// A token is a whole number, so weights are taken in 64 bits: exp2 from a table
// of 256 and a cubic (2e-13), rounded to fixed point: 46 bits behind the point,
// above 65536 tokens 62 less the bits of their number, so that half a step of at
// most 2^-47 of the largest is lost, 2^-46 with 131072 tokens, 2^-43 with 2^20.
// Sums of fixed-point weights are exact, whatever their order: LDS atomics change
// no result.
//
// A row is one workgroup's, which reads it twice, the first time from memory:
//  * for M and each thread's largest; where a cut is asked for, for a histogram
//    over 2048 bins of x too, of counts or fp32 weights: it names the bin in
//    which the cut falls.  (top_k of a few: the bin that top_k of the threads'
//    largest reach bounds the cut, no histogram is needed);
//  * for the exact weights above that bin (and of the whole row, for top_p),
//    summed by shares of 2048 elements (short rows: 512), and the bin's elements,
//    which are sorted in LDS: exact weights decide the cut.
// The share in which the answer lies is gone over again.  What the histogram
// cannot decide (a bin of more elements than are sorted, logits or a temperature
// at the ends of their range) is done over again with exact weights throughout,
// bins narrowed by the bits of x (256 constant rows of fp16: 0.6 to 1.1 ms).
// Long bf16 rows have few values for their tokens: draw_values counts them, and
// takes weights once for a value, not for a token.
// What is masked, or no token of a last step, weighs 0 in all of this.
// What bounds it (256 rows of 131072 bf16 logits, 67 MB): the read for greedy
// rows, 17 us; the 64-bit operations of the weights, 28 us a pass, in rows
// without a cut (42); for top_p (45) the two passes, 16 us each, bin numbers
// and LDS as long as the read, and between and behind them a dozen short steps.
// fp16 and fp32, top_p: the histogram's exponentials and LDS atomics, 25 us, and
// a pass of weights (fp16 79 to 82 at T = 0.7 to 1.3, of 128256 tokens 78 to 82).
// One row of 49152 fp32 logits, top_k 50, top_p 0.95: 14 us, two passes of one CU
// over 192 KB and a dozen short steps between barriers.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

using namespace sva;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int SB = 512;         // threads: two waves a SIMD, whose registers hold several weights in work
constexpr int SW = SB / WAVE;
constexpr int E = 8;            // consecutive elements of a thread
constexpr int STEP = WAVE * E;  // elements that a wave takes at a time, 2^turns times one after another: a share
constexpr int STEP_BITS = 9;
static_assert(STEP == 1 << STEP_BITS, "");
constexpr int TURNS = 2;        // rows of more than kSpread elements; 0: all waves have something of a short row
constexpr int kSpread = 16384;
constexpr int LIGHT = 6, HEAVY = 2;  // steps under way of passes that do little, or much, with them
constexpr int BINS = 2048;
constexpr int CAP = 2048;       // elements of a bin that are sorted
constexpr int PT = BINS / SB;    // bins, or elements of a list, of a thread
static_assert(CAP == BINS, "");
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int SHARES = (int)(kMaxVocab >> (STEP_BITS + TURNS)) + SW;
static_assert(SHARES <= 2 * SB, "");
constexpr int MANY = 8192;       // tokens that are listed
constexpr u64 kRaw = 0x4330000000000000ull;  // the bits of 2^52
constexpr int kFew = 256;       // top_k that the threads' largest bound

// bf16 has few values, each its own bin, in falling order: 64 binades of either
// sign from 2^-55 to 510, 0 and what is smaller, and what is at most -510.  (32
// binades, from 2^-23, leave out an element of one row in two hundred.)
constexpr int VALUES = 16384;
constexpr int VALUE0 = (127 - 55) << 7;  // the bits of 2^-55
constexpr int PV = VALUES / SB;          // bins of a thread
constexpr int VROWS = VALUES / WAVE;
constexpr int ZERO = VALUES / 2 - 1;     // -0: the next
static_assert(PV == 32 && 2 * VROWS <= SHARES, "");
constexpr float kLow = -510.0f;

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int vocab;
  const float* uniforms;
  const float* temperature;  // NULL: the scalar
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int64_t top_k1;
  int64_t* out;
  int point;       // bits behind the fixed point
  int vocab_bits;  // 2^vocab_bits tokens at least
};

struct SampleLds {
  double table[256];  // 2^(j / 256 + point)
  union {
    struct {
      u64 hist[BINS];
      uint32_t count[BINS];
      u64 list[2][CAP];
      uint32_t many[MANY];
    };
    uint32_t counts[VALUES];  // draw_values
    u64 weights[VALUES];
  };
  u64 sums[SHARES];   // the kept weights of a share
  u64 ties[SHARES];
  u64 scan[2 * SW];
  u64 word[8];
  float top[SW];
  uint32_t n[3];
};

// A NaN is no token's, and infinity the largest number.
SVA_DEV float number(float x) { return x == x ? fminf(x, 3.40282347e38f) : -INFINITY; }

// x moved N lanes up within its DPP row (0 moves in).
template <int N>
SVA_DEV u64 row_shr_u64(u64 x) {
  return (u64)row_shr0<N>((uint32_t)x) | (u64)row_shr0<N>((uint32_t)(x >> 32)) << 32;
}
SVA_DEV u64 readlane_u64(u64 x, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane) << 32;
}
// Inclusive sum over the wave (all lanes active).
SVA_DEV u64 wave_upto_u64(u64 v) {
  v += row_shr_u64<1>(v);
  v += row_shr_u64<2>(v);
  v += row_shr_u64<4>(v);
  v += row_shr_u64<8>(v);
  const u64 a = readlane_u64(v, 15), b = a + readlane_u64(v, 31), c = b + readlane_u64(v, 47);
  const int row = lane_id() >> 4;
  return v + (row == 0 ? 0ull : (row == 1 ? a : (row == 2 ? b : c)));
}
SVA_DEV u64 wave_sum_u64(u64 v) { return readlane_u64(wave_upto_u64(v), WAVE - 1); }

// Inclusive sum over the workgroup's threads in order; `total` of all.
SVA_DEV u64 upto_u64(u64 v, SampleLds& s, u64& total) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
  v = wave_upto_u64(v);
  __syncthreads();
  if (lane == WAVE - 1) s.scan[w] = v;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < SW; ++k) {
    before += k < w ? s.scan[k] : 0ull;
    total += s.scan[k];
  }
  return v + before;
}
// Both summed over the workgroup.
SVA_DEV void sum_both(u64& a, u64& b, SampleLds& s) {
  const u64 x = wave_sum_u64(a), y = wave_sum_u64(b);
  __syncthreads();
  if (lane_id() == 0) s.scan[(int)threadIdx.x / WAVE] = x, s.scan[SW + (int)threadIdx.x / WAVE] = y;
  __syncthreads();
  a = b = 0;
#pragma unroll
  for (int k = 0; k < SW; ++k) a += s.scan[k], b += s.scan[SW + k];
}

// Eight elements as they lie in memory.
template <int DT>
struct Raw {
  u32x4 w[DT == F32 ? 2 : 1];
  SVA_DEV float operator[](int k) const {
    if constexpr (DT == F32) return __uint_as_float(w[k / 4][k % 4]);
    else return elem_from_bits(bits(k), DT);
  }
  SVA_DEV uint32_t bits(int k) const { return k & 1 ? w[0][k / 2] >> 16 : w[0][k / 2] & 0xFFFFu; }  // of 16-bit elements
};

template <int DT>
struct Row {
  static constexpr int ES = DT == F32 ? 4 : 2;
  const unsigned char* p;  // a whole 16-byte word: element `skip` of it is the row's first
  int skip, vocab, steps, turns;
  float M;                 // the largest logit
  float ref, per;          // where the bins begin, and bins for a logit's difference of 1
  double rate, off;        // x rate + off: 256ths of a binade below M
  float T, least;          // logits below the least weigh nothing
  float min_p;
  u64 least_w;             // min_p of the largest weight
  const double* table;

  // elements at + k of the aligned window; what lies outside the row is -inf
  SVA_DEV Raw<DT> load(int at) const {
    Raw<DT> r;
    if (at >= skip && at + E <= skip + vocab) {
      const u32x4* q = (const u32x4*)(p + (int64_t)at * ES);
      r.w[0] = q[0];
      if constexpr (DT == F32) r.w[1] = q[1];
    } else {
      const uint32_t none = DT == F32 ? 0xFF800000u : (DT == BF16 ? 0xFF80u : 0xFC00u);
      if (at >= skip + vocab) {
#pragma unroll
        for (int k = 0; k < 4 * (int)(sizeof(r.w) / sizeof(r.w[0])); ++k) r.w[k / 4][k % 4] = DT == F32 ? none : none << 16 | none;
        return r;
      }
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const bool in = at + k >= skip && at + k < skip + vocab;
        const uint32_t b = in ? load_elem_bits(p, at + k, DT) : none;
        if constexpr (DT == F32) r.w[k / 4][k % 4] = b;
        else r.w[0][k / 2] = k & 1 ? r.w[0][k / 2] | b << 16 : b;
      }
    }
    return r;
  }
  // the largest logit is known (and the table).  Its weight is not a whole 2^point: `off` is rounded, and M = 50 at T =
  // 0.2 weighs 2^46 - 1.  What is kept by min_p = 1 weighs as much as it does.
  SVA_DEV void begin(float largest) {
    M = largest;
    off = -(double)M * rate;
    least = M - 55.4f * T;  // 2^-80
    least_w = min_p > 0.0f && plain() ? share_of_largest(weight(M)) : 0ull;
  }
  SVA_DEV u64 share_of_largest(u64 w) const { return (u64)__builtin_ceil((double)min_p * (double)w); }
  SVA_DEV bool plain() const { return T >= 1e-30f && __builtin_fabs(off) <= 268435456.0; }
  SVA_DEV bool has(int token) const { return (uint32_t)token < (uint32_t)vocab; }
  // this thread's elements of a step, in the window
  SVA_DEV int place(int step) const {
    const int tid = (int)threadIdx.x, turn = step & ((1 << turns) - 1);
    return ((((step >> turns) * SW + tid / WAVE) << turns) + turn) * STEP + tid % WAVE * E;
  }
  SVA_DEV int shares() const { return (steps >> turns) * SW; }
  SVA_DEV int share_of(int token) const { return (token + skip) >> (STEP_BITS + turns); }
  // f(step, the first one's token, elements), A steps under way (one turn of
  // the loop takes A: registers that are loaded into do not move)
  template <int A, typename F>
  SVA_DEV void each(F f) const {
    Raw<DT> r[A];
#pragma unroll
    for (int j = 0; j < A; ++j)
      if (j < steps) r[j] = load(place(j));
    for (int base = 0; base < steps; base += A) {
#pragma unroll
      for (int j = 0; j < A; ++j) {
        const int step = base + j;
        if (step < steps) {
          const Raw<DT> x = r[j];
          if (step + A < steps) r[j] = load(place(step + A));
          f(step, place(step) - skip, x);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  SVA_DEV float at(int token) const { return load_elem(p, (int64_t)token + skip, DT); }
  SVA_DEV float below(float x) const { return (ref - x) * per; }
  // 2^(t / 256) in fixed point, with kRaw added
  SVA_DEV u64 raw(double t) const {
    const double y = t + 6755399441055744.0;  // the integer in the low bits
    const int n = (int)__double_as_longlong(y);
    const double r = t - (y - 6755399441055744.0);
    constexpr double c = 0.69314718055994530942 / 256.0;
    double e = __builtin_fma(r, c * c * c / 6.0, c * c / 2.0);
    e = __builtin_fma(r, e, c);
    e = __builtin_fma(r, e, 1.0);
    union {
      double d;
      uint32_t w[2];
    } two;
    two.d = table[n & 255];
    two.w[1] += (uint32_t)(n & ~255) << 12;
    return (u64)__double_as_longlong(__builtin_fma(e, two.d, 4503599627370496.0));
  }
  // exp((x - M) / T) so.  x rate + off is off by 2^-53 of off, the same for all;
  // a NaN counts as the least.  (One of eight 64-bit operations less than from
  // x - M, and these take twice as long as others here.)
  SVA_DEV u64 raw_weight(float x) const { return raw(__builtin_fma((double)fmaxf(x, least), rate, off)); }
  SVA_DEV u64 weight(float x) const { return raw_weight(x) - kRaw; }
};

// The same for temperatures so far from the logits' size that off is too large,
// or the least logit that counts is M itself.
template <int DT>
struct OddRow : Row<DT> {
  SVA_DEV u64 weight(float x) const {
    return this->raw(__builtin_fmax(((double)x - (double)this->M) * this->rate, -20480.0)) - kRaw;
  }
  SVA_DEV void begin_odd() { this->least_w = this->share_of_largest(weight(this->M)); }
};

template <typename R>
SVA_DEV int bin_of(const R& row, float x) {
  return (int)fmaxf(fminf(row.below(x), (float)(BINS - 1)), 0.0f);
}

// A thread's largest element, and the first step that has it.
struct Largest {
  float x = -INFINITY;
  int step = 0;

  template <typename X>
  SVA_DEV void add(int at, const X& e) {
    float y = e[0];
#pragma unroll
    for (int k = 1; k < E; ++k) y = fmaxf(y, e[k]);  // (a NaN is none)
    step = y > x ? at : step;
    x = fmaxf(x, y);
  }
};
SVA_DEV float block_max(SampleLds& s, float x) {
  x = wave_max(x);
  __syncthreads();
  if (lane_id() == 0) s.top[(int)threadIdx.x / WAVE] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w) x = fmaxf(x, s.top[w]);
  return fminf(x, 3.40282347e38f);
}

// Tokens that a pass lists in s.many: a thread keeps a bit for each of its
// elements of eight steps, then their places come from one scan of the wave's
// counts and one LDS atomic (for every step these took longer than the pass).
struct Marks {
  u64 bits = 0;

  template <typename R>
  SVA_DEV void add(const R& row, SampleLds& s, int step, uint32_t mask) {
    bits |= (u64)mask << (8 * (step & 7));
    if ((step & 7) == 7 || step == row.steps - 1) put(row, s, step & ~7);
  }
  template <typename R>
  SVA_DEV void put(const R& row, SampleLds& s, int step) {
    const uint32_t mine = (uint32_t)__popcll(bits);
    if (__ballot(mine != 0u) == 0ull) return;
    const uint32_t upto = wave_incl_scan(mine);
    uint32_t i = 0;
    if (lane_id() == WAVE - 1) i = atomicAdd(&s.n[2], upto);
    i = (uint32_t)__builtin_amdgcn_readlane((int)i, WAVE - 1) + upto - mine;
    for (; bits != 0ull; bits &= bits - 1, ++i) {
      const int k = __builtin_ctzll(bits);
      if (i < MANY) s.many[i] = (uint32_t)(row.place(step + k / E) + k % E - row.skip);
    }
  }
};

// The list's n elements in falling order, in the histogram's place: into 512
// buckets of their keys' range, then each behind those of its bucket that are
// larger (2 to 4 us for 300 to 1000 elements; a bitonic sort of 1024 took 9).
SVA_DEV const u64* sort_list(SampleLds& s, const u64* list, int n) {
  const int tid = (int)threadIdx.x;
  uint32_t* start = s.count + SB;
  u64* temp = (u64*)s.many;  // (its tokens are in the lists)
  __syncthreads();
  if (n <= 128) {  // (one bucket)
    if (tid < n) {
      const u64 mine = list[tid];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += list[j] > mine ? 1 : 0;
      s.hist[rank] = mine;
    }
    __syncthreads();
    return s.hist;
  }
  s.count[tid] = 0u;
  if (tid == 0) s.word[6] = 0ull, s.word[7] = ~0ull;
  u64 mine[PT], top = 0ull, bottom = ~0ull;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    mine[k] = SB * k + tid < n ? list[SB * k + tid] : 0ull;
    if (SB * k + tid < n) top = max(top, mine[k] >> 32), bottom = min(bottom, mine[k] >> 32);
  }
  __syncthreads();
#pragma unroll
  for (int k = 1; k < WAVE; k <<= 1) top = max(top, __shfl_xor(top, k, WAVE)), bottom = min(bottom, __shfl_xor(bottom, k, WAVE));
  if (lane_id() == 0) atomicMax(&s.word[6], top), atomicMin(&s.word[7], bottom);
  __syncthreads();
  top = s.word[6];
  const uint32_t range = n > 0 ? (uint32_t)(top - s.word[7]) : 0u;
  const int shift = range < SB ? 0 : 32 - __clz((int)range) - 9;
  uint32_t bucket[PT], place[PT];
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    if (SB * k + tid >= n) continue;
    bucket[k] = (uint32_t)(top - (mine[k] >> 32)) >> shift;
    place[k] = atomicAdd(&s.count[bucket[k]], 1u);
  }
  __syncthreads();
  u64 total;
  const u64 count = s.count[tid];
  start[tid] = (uint32_t)(upto_u64(count, s, total) - count);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PT; ++k)
    if (SB * k + tid < n) temp[start[bucket[k]] + place[k]] = mine[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    if (SB * k + tid >= n) continue;
    const uint32_t first = start[bucket[k]], end = first + s.count[bucket[k]];
    uint32_t rank = first;
#pragma unroll 4
    for (uint32_t j = first; j < end; ++j) rank += temp[j] > mine[k] ? 1u : 0u;
    s.hist[rank] = mine[k];
  }
  __syncthreads();
  return s.hist;
}

// What less than `share` of the whole sum comes to: elements with less than
// this before them are kept.
SVA_DEV u64 share_of(double share, u64 total) {
  const double t = __builtin_ceil((double)total * share);
  const u64 want = t >= 1.0 ? (u64)t : 1ull;  // (a NaN: 1)
  return want < total ? want : total;
}

// Of n elements in falling order, with `above` of weight before them: how many
// have less than `share` of `whole` (0: of theirs and `above`) before them; -1
// where the last of these is none of the n.
template <typename R>
SVA_DEV int within_share(const R& row, SampleLds& s, const u64* sorted, int n, u64 above, u64 whole, double share) {
  const int tid = (int)threadIdx.x;
  u64 mine[PT], sum = 0, here;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    mine[k] = PT * tid + k < n ? row.weight(key2f(composite_key(sorted[PT * tid + k]))) : 0ull;
    sum += mine[k];
  }
  u64 before = above + upto_u64(sum, s, here) - sum;
  const u64 want = share_of(share, whole ? whole : above + here);
  if (want <= above || want > above + here) return -1;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    if (PT * tid + k < n && before < want && before + mine[k] >= want) s.word[2] = (u64)(PT * tid + k + 1);
    before += mine[k];
  }
  __syncthreads();
  return (int)s.word[2];
}

// A step's weights v into its share's sum: of the wave together after the last.
struct Share {
  u64 sum = 0;

  template <typename R>
  SVA_DEV void add(const R& row, SampleLds& s, int step, u64 v) {
    sum += v;
    if ((~step & ((1 << row.turns) - 1)) != 0) return;
    sum = wave_sum_u64(sum);
    if (lane_id() == 0) s.sums[(step >> row.turns) * SW + (int)threadIdx.x / WAVE] = sum;
    sum = 0;
  }
};

// The sums of f(x, token) by share (0 for what is no token, at -inf).  No branch
// around an f: eight at once hide one another's latency (131072 weights: 48 us
// where each stood behind its own condition).
template <typename R, typename F>
SVA_DEV void sum_shares(const R& row, SampleLds& s, F f) {
  __syncthreads();
  Share share;
  row.template each<HEAVY>([&](int step, int at, const auto& x) {
    u64 v = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) v += f(x[k], at + k);
    share.add(row, s, step, v);
  });
  __syncthreads();
}

// The first token up to which f(x, token) sums to more than pick(the whole
// sum), from the shares' sums; -1 where that is 0.
template <typename R, typename F, typename P>
SVA_DEV int find(const R& row, SampleLds& s, F f, P pick) {
  const int tid = (int)threadIdx.x, lane = lane_id(), w = tid / WAVE;
  constexpr int PER = (SHARES + SB - 1) / SB;
  const int n = row.shares();
  u64 mine = 0, total;
#pragma unroll
  for (int k = 0; k < PER; ++k) mine += PER * tid + k < n ? s.sums[PER * tid + k] : 0ull;
  u64 before = upto_u64(mine, s, total) - mine;
  if (total == 0ull) return -1;
  const u64 target = pick(total);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (PER * tid + k >= n) continue;
    const u64 v = s.sums[PER * tid + k];
    if (before <= target && before + v > target) s.word[0] = before, s.word[1] = (u64)(PER * tid + k);
    before += v;
  }
  __syncthreads();
  // the share again, a step a wave
  const int at = (((int)s.word[1] << row.turns) + w) * STEP + lane * E;
  const bool mine_too = w >> row.turns == 0;
  u64 g[E], v = 0;
  if (mine_too) {
    const auto x = row.load(at);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      g[k] = f(x[k], at + k - row.skip);
      v += g[k];
    }
  }
  u64 upto = s.word[0] + upto_u64(v, s, total) - v;
  if (mine_too) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      if (upto <= target && upto + g[k] > target) s.word[3] = (u64)(at + k - row.skip);
      upto += g[k];
    }
  }
  __syncthreads();
  return (int)s.word[3];
}

// A cut in the order of falling logits, with exact weights throughout:
// composites of at least the answer are kept.  MASS false: the first `want`
// elements.  MASS true: of the elements of at least `from`, those with less
// than `share` of their sum before them (one at least).
template <bool MASS, typename R>
SVA_DEV u64 exact_cut(const R& row, SampleLds& s, u64 from, u64 want, double share) {
  const int tid = (int)threadIdx.x;
  u64 above = 0;  // counts or weights before the current range:
  int bin = -1;   // elements of this bin whose key's bits from `bits` on are `prefix`
  int bits = 32;
  uint32_t prefix = 0;
  auto inside = [&](float x, uint32_t key, int token) {
    return row.has(token) && composite(key, (uint32_t)token) >= from && (bin < 0 || bin_of(row, x) == bin) &&
           (bits == 32 || key >> bits == prefix);
  };
  for (int level = 0;; ++level) {
    __syncthreads();
    for (int k = tid; k < BINS; k += SB) s.count[k] = 0u, s.hist[k] = 0ull;
    __syncthreads();
    const int next = bits >= 11 ? bits - 11 : 0;
    row.template each<HEAVY>([&](int, int at, const auto& x) {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float v = number(x[k]);
        const uint32_t key = f2key(v);
        if (!inside(v, key, at + k)) continue;
        const int i = level == 0 ? bin_of(row, v) : (int)(key >> next) & ((1 << (bits - next)) - 1);
        atomicAdd(&s.count[i], 1u);
        if (MASS) atomicAdd(&s.hist[i], row.weight(v));
      }
    });
    __syncthreads();
    // falling order: bins of level 0 rise, keys fall
    u64 mine[PT], sum = 0, total;
    int at[PT];
#pragma unroll
    for (int k = 0; k < PT; ++k) {
      at[k] = level == 0 ? PT * tid + k : BINS - 1 - (PT * tid + k);
      mine[k] = MASS ? s.hist[at[k]] : s.count[at[k]];
      sum += mine[k];
    }
    u64 before = above + upto_u64(sum, s, total) - sum;
    if (MASS && level == 0) want = share_of(share, total);
    if (total == 0ull) return from;  // (no weight at all)
    // the range in which the want-th unit lies
#pragma unroll
    for (int k = 0; k < PT; ++k) {
      if (before < want && before + mine[k] >= want) s.word[0] = before, s.word[1] = (u64)at[k];
      before += mine[k];
    }
    __syncthreads();
    above = s.word[0];
    const int hit = (int)s.word[1];
    const uint32_t count = s.count[hit];
    if (level == 0) bin = hit;
    else prefix = (bits == 32 ? 0u : prefix << (bits - next)) | (uint32_t)hit, bits = next;
    if (count <= CAP) {
      __syncthreads();
      if (tid == 0) s.n[0] = 0u;
      __syncthreads();
      row.template each<HEAVY>([&](int, int at, const auto& x) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const float v = number(x[k]);
          const uint32_t key = f2key(v);
          if (inside(v, key, at + k)) s.list[0][atomicAdd(&s.n[0], 1u)] = composite(key, (uint32_t)(at + k));
        }
      });
      __syncthreads();
      const int n = (int)count;
      const u64* sorted = sort_list(s, s.list[0], n);
      sum = 0;
#pragma unroll
      for (int k = 0; k < PT; ++k) {
        const int i = PT * tid + k;
        mine[k] = i >= n ? 0ull : (MASS ? row.weight(key2f(composite_key(sorted[i]))) : 1ull);
        sum += mine[k];
      }
      u64 upto = above + upto_u64(sum, s, total) - sum;
#pragma unroll
      for (int k = 0; k < PT; ++k) {
        if (upto < want && upto + mine[k] >= want) s.word[2] = sorted[PT * tid + k];
        upto += mine[k];
      }
      __syncthreads();
      return s.word[2];
    }
    if (level > 0 && bits == 0) {
      // more ties than are sorted: of equal weights, the lowest tokens
      const u64 each = MASS ? row.weight(key2f(prefix)) : 1ull;
      const u64 n = (want - above + each - 1) / each;  // (each > 0: the range holds the want-th unit)
      const auto tie = [&](float x, int token) {
        return f2key(number(x)) == prefix && row.has(token) && composite(prefix, (uint32_t)token) >= from ? 1ull : 0ull;
      };
      sum_shares(row, s, tie);
      return composite(prefix, (uint32_t)find(row, s, tie, [&](u64) { return n - 1; }));
    }
  }
}

// What is asked of one row.
struct Wish {
  bool few, share;  // cut by top_k, by top_p
  u64 top_k;
  double top_p, u;
};

template <typename R>
SVA_DEV int draw(const R& row, SampleLds& s, const Wish& wish, u64 thr) {
  return find(
      row, s,
      [&](float x, int token) {
        const u64 w = row.weight(number(x));
        return w >= row.least_w && composite(f2key(number(x)), (uint32_t)token) >= thr ? w : 0ull;
      },
      [&](u64 total) {
        const double t = __builtin_floor((double)total * wish.u);
        const u64 v = t >= 0.0 ? (u64)__builtin_fmin(t, 9.0e18) : 0ull;
        return v < total ? v : total - 1;
      });
}

// No cut: every weight.
template <typename R>
SVA_DEV int draw_all(const R& row, SampleLds& s, const Wish& wish) {
  __syncthreads();
  Share share;
  row.template each<HEAVY>([&](int step, int, const auto& x) {
    u64 v = 0, w[E];
#pragma unroll
    for (int k = 0; k < E; ++k) w[k] = row.raw_weight(x[k]);
    if (row.least_w) {
#pragma unroll
      for (int k = 0; k < E; ++k) v += w[k] - kRaw >= row.least_w ? w[k] - kRaw : 0ull;
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) v += w[k];
      v -= E * kRaw;
    }
    share.add(row, s, step, v);
  });
  __syncthreads();
  return draw(row, s, wish, 0ull);
}

template <typename R>
SVA_DEV int exact_draw(const R& row, SampleLds& s, const Wish& wish) {
  u64 thr = 0ull;
  if (wish.few) thr = exact_cut<false>(row, s, thr, wish.top_k, 0.0);
  if (wish.share) thr = exact_cut<true>(row, s, thr, 0ull, wish.top_p);
  sum_shares(row, s, [&](float x, int token) {
    const u64 w = row.weight(number(x));
    return w >= row.least_w && composite(f2key(number(x)), (uint32_t)token) >= thr ? w : 0ull;
  });
  return draw(row, s, wish, thr);
}

// The kept elements of a sorted list into the shares' sums.
template <typename R>
SVA_DEV void add_kept(const R& row, SampleLds& s, const u64* sorted, int n) {
  for (int i = (int)threadIdx.x; i < n; i += SB) {
    const u64 c = sorted[i], w = row.weight(key2f(composite_key(c)));
    if (w >= row.least_w) atomicAdd(&s.sums[row.share_of((int)composite_index(c))], w);
  }
  __syncthreads();
}

// top_k of a few: as many of the threads' largest lie in the first bins up to
// one, so that the cut does too: their elements are listed (-2: too many).
template <typename R>
SVA_DEV int draw_few(const R& row, SampleLds& s, const Wish& wish, float largest) {
  const int tid = (int)threadIdx.x;
  for (int k = tid; k < BINS; k += SB) s.count[k] = 0u;
  for (int k = tid; k < row.shares(); k += SB) s.sums[k] = 0ull;
  if (tid == 0) s.n[2] = 0u, s.word[1] = ~0ull;
  __syncthreads();
  if (largest > -INFINITY) atomicAdd(&s.count[bin_of(row, largest)], 1u);
  __syncthreads();
  u64 mine = 0, total;
#pragma unroll
  for (int k = 0; k < PT; ++k) mine += s.count[PT * tid + k];
  const u64 end = upto_u64(mine, s, total);
  if (end - mine < wish.top_k && end >= wish.top_k) s.word[1] = (u64)(PT * tid + PT - 1);
  __syncthreads();
  if (s.word[1] == ~0ull) return -2;
  const float most = s.word[1] >= BINS - 1 ? INFINITY : (float)((int)s.word[1] + 1);
  if (most == INFINITY) return -2;
  Marks marks;
  row.template each<LIGHT>([&](int step, int, const auto& x) {
    uint32_t mask = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) mask |= row.below(x[k]) < most ? 1u << k : 0u;  // (no NaN, and no -inf)
    marks.add(row, s, step, mask);
  });
  __syncthreads();
  const int n = (int)s.n[2];
  if (n > CAP) return -2;
  for (int i = tid; i < n; i += SB) s.list[0][i] = composite(f2key(number(row.at((int)s.many[i]))), s.many[i]);
  const u64* sorted = sort_list(s, s.list[0], n);
  int kept = (int)wish.top_k;
  if (wish.share) kept = within_share(row, s, sorted, kept, 0ull, 0ull, wish.top_p);
  add_kept(row, s, sorted, kept);
  return draw(row, s, wish, sorted[kept - 1]);
}

// The bins of two elements, 16 bits each.
SVA_DEV uint32_t value_bins(uint32_t two) {
  s16x2 i = __builtin_bit_cast(s16x2, two & 0x7FFF7FFFu) - (short)VALUE0;
  i = __builtin_elementwise_min(__builtin_elementwise_max(i, s16x2{0, 0}), s16x2{VALUES / 2 - 1, VALUES / 2 - 1});
  const u16x2 minus = __builtin_bit_cast(u16x2, two) >> (unsigned short)15;
  return __builtin_bit_cast(uint32_t, i) ^ (__builtin_bit_cast(uint32_t, minus) + (VALUES / 2 - 1) * 0x10001u);
}
SVA_DEV float bin_value(int bin) {
  const bool minus = bin >= VALUES / 2;
  const int i = minus ? bin - VALUES / 2 : VALUES / 2 - 1 - bin;
  return __uint_as_float((uint32_t)((i == 0 ? 0 : i + VALUE0) | (minus ? 0x8000 : 0)) << 16);
}

// Sums of the rows of 64 bins, in order: the row in which they come to `want` of
// the whole sum (VROWS: none), and what is before it.  Every wave gets the same.
template <typename W>
SVA_DEV int row_of(const u64* rows, W want, u64& wanted, u64& before) {
  constexpr int PER = VROWS / WAVE;
  const int lane = lane_id();
  u64 v[PER], sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) sum += v[k] = rows[PER * lane + k];
  const u64 upto = wave_upto_u64(sum);
  wanted = want(readlane_u64(upto, WAVE - 1));
  u64 at = upto - sum, mine = 0;
  int row = -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const bool here = at < wanted && at + v[k] >= wanted;
    row = here ? PER * lane + k : row;
    mine = here ? at : mine;
    at += v[k];
  }
  const u64 found = __ballot(row >= 0);
  if (found == 0ull) return VROWS;
  const int from = __builtin_ctzll(found);
  before = readlane_u64(mine, from);
  return __builtin_amdgcn_readlane(row, from);
}

// bf16, any cut: one pass counts the values.  Counts and exact weights of the
// values are the row's: they name the value at which the cut falls, and how many
// of the tokens that have it are kept.  A second pass takes the weights from a
// table, 0 for what is cut off.  -2: a logit of at least 510, or between 0 and
// 2^-55, or one of at most -510 that weighs something.
template <typename R>
SVA_DEV int draw_values(R& row, SampleLds& s, const Wish& wish) {
  const int tid = (int)threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  constexpr u64 kTie = 1ull << 58;  // (a thread's weights of a share come to 2^51)
  for (int k = tid; k < VALUES / 4; k += SB) ((u32x4*)s.counts)[k] = u32x4{0u, 0u, 0u, 0u};
  if (tid == 0) s.n[0] = 0u, s.n[1] = VALUES, s.n[2] = 0u, s.word[4] = ~0ull;
  __syncthreads();
  u16x2 small = {0xFFFF, 0xFFFF};
  row.template each<LIGHT>([&](int, int, const auto& x) {
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      small = __builtin_elementwise_min(small, __builtin_bit_cast(u16x2, x.w[0][k] & 0x7FFF7FFFu) - (unsigned short)1);
      const uint32_t two = value_bins(x.w[0][k]), lo = two & 0xFFFFu, hi = two >> 16;
      if (lo < VALUES - 1) atomicAdd(&s.counts[lo], 1u);  // (masked logits would meet in one word)
      if (hi < VALUES - 1) atomicAdd(&s.counts[hi], 1u);
    }
  });
  if (min(small[0], small[1]) < VALUE0) s.n[2] = 1u;
  __syncthreads();
  if (tid == 0) s.counts[ZERO] += s.counts[ZERO + 1], s.counts[ZERO + 1] = 0u;  // (-0 equals 0)
  __syncthreads();
  // A wave's bins: every eighth row of 64.  Most are empty: loops over the others
  // are not unrolled (this code runs once, and waits for its instructions).
  const int bin0 = wave * WAVE + lane;
  u64 total = 0, none = 0;
  int first = VALUES;
  uint32_t used = 0;  // bit k: row k * SW + wave
#pragma unroll
  for (int k = PV - 1; k >= 0; --k) {
    const uint32_t n = s.counts[bin0 + SB * k];
    total += n;
    const u64 any = __ballot(n != 0u);
    used |= any ? 1u << k : 0u;
    first = any ? bin0 - lane + SB * k + (int)__builtin_ctzll(any) : first;
  }
  if (lane == 0 && first < VALUES) atomicMin(&s.n[1], (uint32_t)first);
  if (lane < PV) s.ties[lane * SW + wave] = s.ties[VROWS + lane * SW + wave] = 0ull;
  sum_both(total, none, s);
  const int top = (int)s.n[1];
  if (s.n[2] != 0u || top == 0 || top == VALUES) return -2;
  row.begin(bin_value(top));
  if (!row.plain() || (total < (u64)row.vocab && !(row.least >= kLow))) return -2;
  const auto weight = [&](int k) { return row.raw_weight(bin_value(bin0 + SB * k)) - kRaw; };
  const auto rows_upto = [&](int cut) {  // those of this wave
    const int n = cut >= wave ? (cut - wave) / SW + 1 : 0;
    return n >= PV ? used : used & ((1u << n) - 1u);
  };
  int cut = VROWS;     // the last row of which something is kept,
  uint32_t kept = 0;   // and of this lane's bin in it: how many are,
  u64 want, before;
  if (wish.few) {
#pragma unroll 1
    for (uint32_t m = used; m != 0u; m &= m - 1) {
      const int k = __builtin_ctz(m);
      const u64 sum = wave_sum_u64(s.counts[bin0 + SB * k]);
      if (lane == 0) s.ties[k * SW + wave] = sum;
    }
    __syncthreads();
    cut = row_of(s.ties, [&](u64) { return wish.top_k; }, want, before);
    if (cut < VROWS) {
      const uint32_t n = s.counts[cut * WAVE + lane];
      const u64 above = before + wave_upto_u64(n) - n, left = want > above ? want - above : 0ull;
      kept = (u64)n < left ? n : (uint32_t)left;
    }
  }
  if (wish.share) {
    const int last = cut;
#pragma unroll 1
    for (uint32_t m = rows_upto(last); m != 0u; m &= m - 1) {
      const int k = __builtin_ctz(m);
      const u64 sum = wave_sum_u64((k * SW + wave == last ? kept : s.counts[bin0 + SB * k]) * weight(k));
      if (lane == 0) s.ties[VROWS + k * SW + wave] = sum;
    }
    __syncthreads();
    cut = row_of(s.ties + VROWS, [&](u64 all) { return share_of(wish.top_p, all); }, want, before);
    kept = cut == last ? kept : s.counts[cut * WAVE + lane];
    const u64 each = row.raw_weight(bin_value(cut * WAVE + lane)) - kRaw;
    const u64 mass = kept * each, above = before + wave_upto_u64(mass) - mass;
    if (above >= want) {
      kept = 0u;
    } else if (above + mass >= want) {
      const u64 rest = want - above;
      u64 n = (u64)((double)rest / (double)each);  // (at most 2^20: off by one at most)
      if (n * each < rest) ++n;
      if (n * each < rest) ++n;
      if (n > 1 && (n - 1) * each >= rest) --n;
      kept = (uint32_t)n;
    }
  }
  const bool whole = cut < VROWS && kept == s.counts[cut * WAVE + lane];  // all of the bin
  const uint32_t live = rows_upto(cut);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PV; ++k)
    if (!(live >> k & 1u)) s.weights[bin0 + SB * k] = 0ull;
#pragma unroll 1
  for (uint32_t m = live; m != 0u; m &= m - 1) {
    const int k = __builtin_ctz(m), bin = bin0 + SB * k;
    u64 w = weight(k);
    w = w >= row.least_w && bin < VALUES - 1 ? w : 0ull;
    if (k * SW + wave == cut) {
      const bool part = kept != 0u && !whole;
      if (part) s.word[4] = (u64)bin, s.word[5] = kept, s.word[6] = w;
      const u64 some = __ballot(kept != 0u);
      if (lane == 63 - (int)__builtin_clzll(some)) s.n[0] = (uint32_t)bin;
      w = part ? kTie : (kept != 0u ? w : 0ull);
    }
    s.weights[bin] = w;
  }
  __syncthreads();
  if (tid == 0) s.weights[ZERO + 1] = s.weights[ZERO];
  __syncthreads();
  const int part = (int)s.word[4];
  const u64 of_part = s.word[5], w_part = s.word[6];
  u64 here = 0;
  row.template each<LIGHT>([&](int step, int, const auto& x) {
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const uint32_t two = value_bins(x.w[0][k]);
      here += s.weights[two & 0xFFFFu];
      here += s.weights[two >> 16];
    }
    if ((~step & ((1 << row.turns) - 1)) != 0) return;
    const int share = (step >> row.turns) * SW + wave;
    const u64 v = wave_sum_u64(here & (kTie - 1));
    if (lane == 0) s.sums[share] = v;
    if (part >= 0) {
      const u64 same = wave_sum_u64(here / kTie);
      if (lane == 0) s.ties[share] = same;
    }
    here = 0;
  });
  __syncthreads();
  u64 thr = cut < VROWS ? composite(f2key(bin_value((int)s.n[0])), (uint32_t)row.vocab) : 0ull;
  if (part >= 0) {
    // which tokens of that value: the first ones
    const uint32_t key = f2key(bin_value(part));
    const auto tie = [&](float x, int token) { return f2key(x) == key && row.has(token) ? 1ull : 0ull; };
    for (int k = tid; k < row.shares(); k += SB) s.hist[k] = s.sums[k], s.sums[k] = s.ties[k];
    __syncthreads();
    const int end = find(row, s, tie, [&](u64) { return of_part - 1; });
    thr = composite(key, (uint32_t)end);
    const int share = (int)s.word[1];
    for (int k = tid; k < row.shares(); k += SB)
      s.sums[k] = s.hist[k] + w_part * (k < share ? s.ties[k] : (k == share ? of_part - s.word[0] : 0ull));
    __syncthreads();
  }
  const int token = draw(row, s, wish, thr);
  return token < 0 ? -2 : token;
}

// Any cut, by a histogram of counts (top_k) and fp32 weights (top_p), exact
// weights beside it (-1: no token at all, -2: it does not decide, -3: weights
// cannot be taken so, -4: nothing is cut off).  A cut as `near` to the end of its
// bin as the fp32 sums may be off takes the next one in.
//
// The bins begin above the largest of the row's first elements, by as much as
// the rest is not expected to pass (if it does, the pass is done again), so that
// the pass that finds the largest of all is this one (256 rows of 131072: 13 us
// less).
template <typename R>
SVA_DEV int draw_cut(R& row, SampleLds& s, Wish& wish, double slope, int bits, Largest& largest) {
  const int tid = (int)threadIdx.x;
  float top;
  uint32_t weighty = 0;
  {
    Largest some;
#pragma unroll
    for (int k = 0; k < 1 << TURNS; ++k) some.add(0, row.load(row.place(k)));
    top = block_max(s, some.x);
    if (top == -INFINITY) {
      row.template each<LIGHT>([&](int, int, const auto& x) { some.add(0, x); });
      top = block_max(s, some.x);
    }
    row.ref = top + 512.0f / row.per;
    largest = Largest();
  }
  const double unit = __builtin_amdgcn_ldexp(1.0, min(51, 62 - bits));  // of a weight of 1, at ref; 2^bits of them fit
  const float hi_slope = (float)slope, lo_slope = (float)(slope - (double)hi_slope);
  // Differences stop where weights are far below the fixed point (2^-200): -inf times two slopes of opposite sign would
  // be a NaN (what is masked or no token, at T = 0.7 and 0.9, not at 1: 256 rows of 128256 fp16 then took 238 us for 79).
  const float furthest = -200.0f / hi_slope;
  for (bool again = false;; again = true) {
    for (int k = tid; k < BINS; k += SB) s.hist[k] = 0ull, s.count[k] = 0u;
    if (tid < 3) s.n[tid] = 0u;
    if (tid == 0) s.word[4] = s.word[5] = 0ull;
    __syncthreads();
    row.template each<HEAVY>([&](int step, int, const auto& x) {
      if (!again) largest.add(step, x);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float v = number(x[k]);
        const int bin = bin_of(row, v);
        if (wish.few) {
          if (bin < BINS - 1) atomicAdd(&s.count[bin], 1u);
          weighty += (v - top) * hi_slope > -60.0f ? 1u : 0u;
        }
        if (wish.share) {
          const float d = fmaxf(fminf(v - row.ref, 0.0f), furthest);
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi_slope, d * lo_slope));
          const u64 fixed = (u64)__double_as_longlong(__builtin_fma((double)w, unit, 4503599627370496.0)) - kRaw;
          atomicAdd(&s.hist[fixed != 0ull ? bin : tid], fixed);  // (0 anywhere: not all in one word)
        }
      }
    });
    if (again) break;
    if (wish.few) {
      u64 all = weighty, none = 0;
      sum_both(all, none, s);
      if (all <= wish.top_k) {  // (what top_k cuts off weighs nothing)
        wish.few = false;
        if (!wish.share) {
          row.begin(block_max(s, largest.x));
          return row.plain() ? -4 : -3;
        }
      }
    }
    row.begin(block_max(s, largest.x));
    if (row.M == -INFINITY) return -1;
    if (!row.plain()) return -3;
    if (!wish.share || row.M <= row.ref) break;
    row.ref = row.M;
  }
  __syncthreads();
  u64 mass[PT], first = 0, sum = 0;  // weights before this thread's bins, of all
  if (wish.share) {
#pragma unroll
    for (int k = 0; k < PT; ++k) first += mass[k] = s.hist[PT * tid + k];
    first = upto_u64(first, s, sum) - first;
  }
  int last = BINS;  // the bin of the top_k-th
  u64 before_last = 0;
  if (wish.few) {
    u64 count[PT], before = 0, all, weight = first;
#pragma unroll
    for (int k = 0; k < PT; ++k) before += count[k] = s.count[PT * tid + k];
    before = upto_u64(before, s, all) - before;
    if (tid == SB - 1) {  // (the last bin holds the rest: masked logits by the thousand would meet in one word)
      count[PT - 1] = (u64)row.vocab - all;
      s.count[BINS - 1] = (uint32_t)count[PT - 1];
    }
#pragma unroll
    for (int k = 0; k < PT; ++k) {
      if (before < wish.top_k && before + count[k] >= wish.top_k)
        s.word[0] = before, s.word[1] = (u64)(PT * tid + k), s.word[2] = weight;
      before += count[k];
      if (wish.share) weight += mass[k];
    }
    __syncthreads();
    last = (int)s.word[1];
    before_last = s.word[0];
    if (s.count[last] > CAP) return -2;
    if (wish.share)
      sum = s.word[2] + (u64)((double)s.hist[last] * (double)(wish.top_k - before_last) / (double)s.count[last]);
  }
  int lo = last, hi = last;  // bins in which the cut may fall
  if (wish.share) {
    const u64 want = share_of(wish.top_p, sum > 0 ? sum : 1);
    u64 before = first;
#pragma unroll
    for (int k = 0; k < PT; ++k) {
      if (before < want && before + mass[k] >= want) s.word[4] = (u64)(PT * tid + k), s.word[5] = before;
      before += mass[k];
    }
    __syncthreads();
    lo = hi = min((int)s.word[4], last == BINS ? BINS - 1 : last);
    const u64 near = sum >> 14, begin = s.word[5], end = begin + s.hist[lo];
    if (lo > 0 && want < begin + near) --lo;
    if (hi < BINS - 1 && hi < last && want + near > end) ++hi;
  }
  const bool joined = hi == last;  // the bin of the top_k-th is among them
  const int n_last = wish.few ? (int)s.count[last] : 0;
  if (wish.few && s.count[lo] + (hi > lo ? s.count[hi] : 0u) > CAP) return -2;
  __syncthreads();
  // The elements of these bins (list 0) and of the top_k-th's (list 1), and
  // exact weights: `above` them, and of all before the top_k-th's bin, `whole`.
  const bool need_whole = wish.share && !joined;
  const float lo_f = lo == 0 ? -INFINITY : (float)lo, end_f = hi == BINS - 1 ? INFINITY : (float)(hi + 1);
  const float last_f = last == BINS ? INFINITY : (float)last, behind_f = last >= BINS - 1 ? INFINITY : (float)(last + 1);
  const bool by_list = wish.few && wish.top_k <= MANY - CAP;
  if (by_list)
    for (int k = tid; k < row.shares(); k += SB) s.sums[k] = 0ull;
  // (what is no token lies in the last bin)
  const bool last_bin = hi == BINS - 1 || last == BINS - 1;
  const auto in_lists = [&](float b) { return (b >= lo_f && b < end_f) || (b >= last_f && b < behind_f); };
  const auto tokens = [&](int at) {
    uint32_t mask = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) mask |= row.has(at + k) ? 1u << k : 0u;
    return mask;
  };
  __syncthreads();
  u64 above = 0, whole = 0;
  Marks marks;
  if (by_list) {
    // not many in all: listed, and the weights are theirs alone
    row.template each<LIGHT>([&](int step, int at, const auto& x) {
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) mask |= row.below(x[k]) < behind_f ? 1u << k : 0u;
      if (last_bin) mask = tokens(at);
      marks.add(row, s, step, mask);
    });
  } else if (last == BINS && !last_bin) {
    // top_p alone: the whole sum, and what lies above the bins
    Share share;
    row.template each<HEAVY>([&](int step, int, const auto& x) {
      u64 w[E], here = 0, kept = 0;
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float b = row.below(x[k]);  // (a NaN compares with nothing)
        w[k] = row.raw_weight(x[k]);
        whole += w[k];
        mask |= b >= lo_f && b < end_f ? 1u << k : 0u;
        w[k] = b < lo_f ? w[k] - kRaw : 0ull;
        here += w[k];
      }
      whole -= E * kRaw;
      above += kept = here;
      if (row.least_w) {
        kept = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) kept += w[k] >= row.least_w ? w[k] : 0ull;
      }
      marks.add(row, s, step, mask);
      share.add(row, s, step, kept);
    });
  } else {
    Share share;
    row.template each<HEAVY>([&](int step, int at, const auto& x) {
      float v[E], b[E];
      bool weigh = need_whole;
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        v[k] = number(x[k]);
        b[k] = fminf(row.below(v[k]), (float)(BINS - 1));
        weigh = weigh || b[k] < lo_f;
        mask |= in_lists(b[k]) ? 1u << k : 0u;
      }
      u64 kept = 0;
      if (__any(weigh)) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const u64 w = row.weight(v[k]);
          whole += b[k] < last_f ? w : 0ull;
          above += b[k] < lo_f ? w : 0ull;
          kept += b[k] < lo_f && w >= row.least_w ? w : 0ull;
        }
      }
      if (last_bin) mask &= tokens(at);
      marks.add(row, s, step, mask);
      share.add(row, s, step, kept);
    });
  }
  __syncthreads();
  if (s.n[2] > MANY) return -2;
  for (int i = tid, all = (int)s.n[2]; i < all; i += SB) {
    const uint32_t token = s.many[i];
    const float v = number(row.at((int)token)), b = fminf(row.below(v), (float)(BINS - 1));
    const u64 c = composite(f2key(v), token);
    if (b >= lo_f && b < end_f) {
      const uint32_t place = atomicAdd(&s.n[0], 1u);
      if (place < CAP) s.list[0][place] = c;
    } else if (b >= last_f) {
      s.list[1][atomicAdd(&s.n[1], 1u)] = c;
    }
    if (by_list && b < last_f) {
      const u64 w = row.weight(v);
      whole += w;
      if (b < lo_f) {
        above += w;
        if (w >= row.least_w) atomicAdd(&s.sums[row.share_of((int)token)], w);
      }
    }
  }
  sum_both(above, whole, s);
  const int n_list = (int)s.n[0];
  if (n_list > CAP) return -2;
  int n = n_list;
  if (wish.few) {
    const int of_last = (int)(wish.top_k - before_last);
    if (joined) {
      n -= n_last - of_last;
    } else {
      const u64* sorted = sort_list(s, s.list[1], n_last);
      u64 w = 0, all;
      for (int i = tid; i < of_last; i += SB) w += row.weight(key2f(composite_key(sorted[i])));
      upto_u64(w, s, all);
      whole += all;
    }
  }
  const u64* sorted = sort_list(s, s.list[0], n_list);
  if (wish.share) n = within_share(row, s, sorted, n, above, need_whole ? whole : 0ull, wish.top_p);
  if (n < 0) return -2;
  add_kept(row, s, sorted, n);
  return draw(row, s, wish, sorted[n - 1]);
}

template <int DT>
__global__ void __launch_bounds__(SB) sample_kernel(SampleParams p) {
  __shared__ SampleLds s;
  const int tid = (int)threadIdx.x;
  const int64_t b = blockIdx.x;
  OddRow<DT> odd;
  Row<DT>& row = odd;
  const uintptr_t from = (uintptr_t)p.logits + b * p.row_stride * Row<DT>::ES;
  row.p = (const unsigned char*)(from & ~(uintptr_t)15);
  row.skip = (int)(from & 15) / Row<DT>::ES;
  row.vocab = p.vocab;
  row.turns = p.vocab > kSpread ? TURNS : 0;
  const int group = SB * E << row.turns;
  row.steps = ((p.vocab + row.skip + group - 1) / group) << row.turns;
  row.table = s.table;
  float T = p.temperature ? p.temperature[b] : p.temperature1;
  T = T > 1e30f ? 1e30f : T;  // (all of them weigh the same)
  const int64_t k = p.top_k ? p.top_k[b] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p1;
  const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p1, 1.0f);
  Wish wish;
  wish.u = p.uniforms[b];
  wish.few = k > 0 && k < p.vocab;
  wish.top_k = (u64)k;
  wish.share = !(top_p >= 1.0f);
  wish.top_p = top_p;

  row.T = T;
  const double slope = 1.44269504088896340736 / (double)T;
  row.rate = 256.0 * slope;
  row.per = 64.0f / fmaxf(T, 0.25f);
  row.min_p = fmaxf(min_p, 0.0f);
  if (tid < 256) s.table[tid] = exp2((double)tid / 256.0 + (double)p.point);
  const bool random = !(T <= 0.0f) && k != 1;
  const bool cut = random && (wish.few || wish.share), few = cut && wish.few && wish.top_k <= kFew;

  Largest largest;
  int token = -2;
  // (T under 4.3e-39 puts 1 / (T ln 2) past fp32, in which draw_cut counts what weighs something; none so cold is plain)
  if (!cut || few || !(T >= 1e-30f)) {
    row.template each<LIGHT>([&](int step, int, const auto& x) { largest.add(step, x); });
    row.begin(block_max(s, largest.x));
    row.ref = row.M;
    if (!random || row.M == -INFINITY) token = -1;
    else if (!row.plain()) token = -3;
    else if (few) token = draw_few(row, s, wish, fminf(largest.x, 3.40282347e38f));
    else token = draw_all(row, s, wish);
  }
  if constexpr (DT == BF16) {
    // (64 rows of 20000, top_p 0.9: 22 us, 27 by the histogram; 8 of 4000: its steps between the passes alone take
    // as long as what they save)
    if (token == -2 && p.vocab > kSpread) token = draw_values(row, s, wish);
  }
  if (token == -2) token = draw_cut(row, s, wish, slope, p.vocab_bits, largest);
  if (token == -4) token = draw_all(row, s, wish);
  if (token == -2) token = exact_draw(row, s, wish);
  if (token == -3) {
    odd.begin_odd();
    token = exact_draw(odd, s, wish);
  }
  if (token < 0 && row.M > -INFINITY) {  // the largest, the lowest of equal ones
    __syncthreads();
    if (tid == 0) s.n[1] = 0xFFFFFFFFu;
    __syncthreads();
    if (fminf(largest.x, 3.40282347e38f) == row.M) {
      const int at = row.place(largest.step);
      const Raw<DT> x = row.load(at);
      uint32_t first = 0;
#pragma unroll
      for (int i = E - 1; i >= 0; --i) first = number(x[i]) == row.M ? (uint32_t)(at + i - row.skip) : first;
      atomicMin(&s.n[1], first);
    }
    __syncthreads();
    token = (int)s.n[1];
  }
  if (tid == 0) p.out[b] = token;
}

template <int DT>
int launch(const SampleParams& p, int64_t rows, hipStream_t stream) {
  hipLaunchKernelGGL((sample_kernel<DT>), dim3((unsigned)rows), dim3(SB), 0, stream, p);
  SVA_CHECK_LAUNCH("sample_kernel");
  return SVA_OK;
}

}  // namespace

extern "C" int sva_sample_tokens(const void* logits, int dtype, int64_t row_stride, int64_t n_rows, int64_t vocab,
                                 const float* uniforms, const float* temperature, float temperature1,
                                 const int64_t* top_k, int64_t top_k1, const float* top_p, float top_p1,
                                 const float* min_p, float min_p1, int64_t* tokens, void* stream) {
  sva::clear_error();
  SVA_REQUIRE(logits && uniforms && tokens, "sva_sample_tokens: null pointer");
  SVA_REQUIRE(dtype >= 0 && dtype <= 2, "sva_sample_tokens: bad dtype");
  SVA_REQUIRE(n_rows > 0 && n_rows < (1ll << 31) && vocab > 0 && row_stride >= 0, "sva_sample_tokens: bad sizes");
  SVA_REQUIRE((uintptr_t)logits % (dtype == F32 ? 4 : 2) == 0, "sva_sample_tokens: logits are not aligned");
  SVA_UNSUPPORTED(vocab <= kMaxVocab, "sva_sample_tokens: %lld tokens (at most %lld)", (long long)vocab,
                  (long long)kMaxVocab);
  SampleParams p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = (int)vocab;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature1 = temperature1;
  p.top_k1 = top_k1;
  p.top_p1 = top_p1;
  p.min_p1 = min_p1;
  p.out = tokens;
  int bits = 0;
  while ((1ll << bits) < vocab) ++bits;
  p.point = std::min(46, 62 - bits);
  p.vocab_bits = bits;
  if (dtype == F32) return launch<F32>(p, n_rows, (hipStream_t)stream);
  if (dtype == BF16) return launch<BF16>(p, n_rows, (hipStream_t)stream);
  return launch<F16>(p, n_rows, (hipStream_t)stream);
}
