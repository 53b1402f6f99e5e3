// The next token of every row of logits, from a given random number.
//
// Weights w = exp((x - M) / T), M the largest logit.  Of the tokens in the
// order of falling logits (ties: the lower token first) those are kept that
// are among the first top_k, have less than top_p of the sum of these before
// them, and weigh at least min_p; the answer is the first token, by number, up
// to which the kept weights sum to more than u of their sum.  T <= 0: the
// largest logit.  A NaN counts as -inf; logits of +inf share all of the weight.
//
// A token is a whole number, so weights are taken in 64 bits: exp2 from a table
// of 64 and a polynomial, rounded to fixed point (up to 46 bits behind the
// point; 2^-47 of the largest is lost at most).  Sums of fixed-point weights are
// exact, whatever their order: LDS atomics change no result.
//
// A row is one workgroup's, which reads it a few times (from the caches, after
// the first): for M; for a histogram of counts or weights over 2048 bins of
// x, linear below M; for the elements of the bin in which a cut falls, which
// are sorted in LDS (a bin of too many is narrowed by the bits of x); for the
// weights of the kept tokens by wave, then again by the one wave in whose share
// the answer lies.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

using namespace sva;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int SB = 1024;        // threads
constexpr int SW = SB / WAVE;
constexpr int E = 8;            // consecutive elements of a thread
constexpr int TILE = SB * E;    // elements that the workgroup takes at a time
constexpr int BINS = 2048;
constexpr int CAP = 2048;       // elements of a bin that are sorted
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int MAX_TILES = (int)(kMaxVocab / TILE);
static_assert(MAX_TILES * SW <= BINS, "the waves' sums take the histogram's place");

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
  int point;  // bits behind the fixed point
};

struct SampleLds {
  double table[64];              // 2^(j / 64)
  unsigned long long mass[BINS]; // also the waves' sums of the last pass
  uint32_t count[BINS];
  unsigned long long list[CAP];
  unsigned long long scan[SW];
  unsigned long long word[4];
  float top[SW];
  uint32_t n;
};

// Inclusive sum over the workgroup's threads in order; `total` of all.
SVA_DEV unsigned long long upto_u64(unsigned long long v, SampleLds& s, unsigned long long& total) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
#pragma unroll
  for (int k = 1; k < WAVE; k <<= 1) {
    const unsigned long long x = __shfl_up(v, k, WAVE);
    if (lane >= k) v += x;
  }
  __syncthreads();
  if (lane == WAVE - 1) s.scan[w] = v;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < SW; ++k) {
    before += k < w ? s.scan[k] : 0ull;
    total += s.scan[k];
  }
  return v + before;
}

template <int DT, bool VEC>
struct Row {
  const unsigned char* p;
  int vocab;
  float M;         // the largest logit
  double rate;     // log2(e) / T
  float per;       // bins below M for a logit's difference of 1
  double one;      // 2^point
  const double* table;

  // elements at .. at + 7; those behind the row and NaN are -inf
  SVA_DEV void load(int at, float (&x)[E]) const {
    if (VEC && at + E <= vocab) {
      if constexpr (DT == F32) {
        const float4 a = *(const float4*)(p + (int64_t)at * 4), b = *(const float4*)(p + (int64_t)at * 4 + 16);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
      } else {
        const u32x4 a = *(const u32x4*)(p + (int64_t)at * 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[2 * k] = elem_from_bits(a[k] & 0xFFFFu, DT), x[2 * k + 1] = elem_from_bits(a[k] >> 16, DT);
      }
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = at + k < vocab ? load_elem(p, at + k, DT) : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = x[k] == x[k] ? x[k] : -INFINITY;
  }
  // f(tile, first element, the elements), the next tile's under way
  template <typename F>
  SVA_DEV void each(F f) const {
    const int first = (int)threadIdx.x * E;
    float x[E], y[E];
    load(first, x);
    for (int tile = 0; tile * TILE < vocab; ++tile) {
      const int at = tile * TILE + first;
      if ((tile + 1) * TILE < vocab) load(at + TILE, y);
      f(tile, at, x);
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = y[k];
    }
  }
  // exp((x - M) / T) and its fixed-point number
  SVA_DEV double weight(float x) const {
    const double t = x == M ? 0.0 * rate : ((double)x - (double)M) * rate;
    const double c = __builtin_fmax(t, -128.0);  // (a NaN: -128)
    const double n = __builtin_rint(c * 64.0);
    const double u = (c - n * 0.015625) * 0.69314718055994530942;
    const int i = (int)n;
    double e = __builtin_fma(u, 1.0 / 24.0, 1.0 / 6.0);
    e = __builtin_fma(u, e, 0.5);
    e = __builtin_fma(u, e, 1.0);
    e = __builtin_fma(u, e, 1.0);
    return __builtin_amdgcn_ldexp(e * table[i & 63], i >> 6);
  }
  SVA_DEV unsigned long long fixed(double w) const {
    // (at most 2^46: behind 2^52 the integer stands in the low bits)
    return (unsigned long long)__double_as_longlong(__builtin_fma(w, one, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }
  SVA_DEV int bin(float x) const {
    const float b = x == M ? 0.0f : (M - x) * per;
    return (int)fminf(b, (float)(BINS - 1));
  }
};

// A cut in the order of falling logits: composites of at least `thr` are kept.
// MASS false: the first `want` elements.  MASS true: of the elements of at
// least `from`, those with less than `share` of their sum before them (one at
// least).
template <bool MASS, typename R>
SVA_DEV unsigned long long cut(const R& row, SampleLds& s, unsigned long long from, unsigned long long want, double share) {
  const int tid = (int)threadIdx.x;
  unsigned long long above = 0;  // counts or weights before the current range
  int bin = -1;                  // the current range: elements of this bin whose key's bits from `bits` on are `prefix`
  int bits = 32;
  uint32_t prefix = 0;
  auto inside = [&](float x, uint32_t key, int at) {
    return composite(key, (uint32_t)at) >= from && (bin < 0 || row.bin(x) == bin) &&
           (bits == 32 || key >> bits == prefix);
  };
  for (int level = 0;; ++level) {
    for (int k = tid; k < BINS; k += SB) s.count[k] = 0u, s.mass[k] = 0ull;
    __syncthreads();
    const int next = bits >= 11 ? bits - 11 : 0;
    row.each([&](int, int at, const float (&x)[E]) {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const uint32_t key = f2key(x[k]);
        if (at + k >= row.vocab || !inside(x[k], key, at + k)) continue;
        const int i = level == 0 ? row.bin(x[k]) : (int)(key >> next) & ((1 << (bits - next)) - 1);
        atomicAdd(&s.count[i], 1u);
        if (MASS) atomicAdd(&s.mass[i], row.fixed(row.weight(x[k])));
      }
    });
    __syncthreads();
    // falling order: bins of level 0 rise, keys fall
    unsigned long long mine[2], total;
    int at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      at[k] = level == 0 ? 2 * tid + k : BINS - 1 - (2 * tid + k);
      mine[k] = MASS ? s.mass[at[k]] : s.count[at[k]];
    }
    const unsigned long long end = upto_u64(mine[0] + mine[1], s, total);
    if (MASS && level == 0) {
      const double t = __builtin_ceil((double)total * share);
      want = t >= 1.0 ? (unsigned long long)t : 1ull;  // (a NaN: 1)
      want = want < total ? want : total;
    }
    // the range in which the want-th unit lies
    unsigned long long before = above + end - mine[0] - mine[1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (before < want && before + mine[k] >= want) s.word[0] = before, s.word[1] = (unsigned long long)at[k];
      before += mine[k];
    }
    __syncthreads();
    above = s.word[0];
    const int hit = (int)s.word[1];
    const uint32_t count = s.count[hit];
    __syncthreads();
    if (level == 0) bin = hit;
    else prefix = (bits == 32 ? 0u : prefix << (bits - next)) | (uint32_t)hit, bits = next;
    if (count <= CAP) {
      // sorted: the last one kept
      if (tid == 0) s.n = 0u;
      __syncthreads();
      row.each([&](int, int at, const float (&x)[E]) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const uint32_t key = f2key(x[k]);
          if (at + k < row.vocab && inside(x[k], key, at + k)) s.list[atomicAdd(&s.n, 1u)] = composite(key, (uint32_t)(at + k));
        }
      });
      __syncthreads();
      const int n = (int)s.n, padded = max(2, next_pow2(n));
      for (int k = n + tid; k < padded; k += SB) s.list[k] = 0ull;
      __syncthreads();
      bitonic_sort_u64<SB>((uint64_t*)s.list, padded, true);
      __syncthreads();
      unsigned long long mine[2], total;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * tid + k;
        mine[k] = i >= n ? 0ull : (MASS ? row.fixed(row.weight(key2f(composite_key(s.list[i])))) : 1ull);
      }
      unsigned long long before = above + upto_u64(mine[0] + mine[1], s, total) - mine[0] - mine[1];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (before < want && before + mine[k] >= want) s.word[2] = s.list[2 * tid + k];
        before += mine[k];
      }
      __syncthreads();
      return s.word[2];
    }
    if (level > 0 && bits == 0) {
      // more ties than can be sorted: of equal weights, the lowest tokens
      const float x = key2f(prefix);
      const unsigned long long each = MASS ? row.fixed(row.weight(x)) : 1ull;
      const unsigned long long n = (want - above + each - 1) / each;  // (each > 0: the range holds the want-th unit)
      const int token = locate(row, s, [&](float v, int at) { return f2key(v) == prefix && composite(prefix, (uint32_t)at) >= from ? 1ull : 0ull; },
                               [&](unsigned long long) { return n - 1; });
      return composite(prefix, (uint32_t)token);
    }
  }
}

// The first element up to which f(x, number) sums to more than pick(the whole
// sum); -1 where the sum is 0.
template <typename R, typename F, typename P>
SVA_DEV int locate(const R& row, SampleLds& s, F f, P pick) {
  const int tid = (int)threadIdx.x, lane = lane_id(), w = tid / WAVE;
  unsigned long long* sums = s.mass;  // [tile][wave]
  auto of8 = [&](int at, const float (&x)[E]) {
    unsigned long long v = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) v += at + k < row.vocab ? f(x[k], at + k) : 0ull;
    return v;
  };
  __syncthreads();
  row.each([&](int tile, int at, const float (&x)[E]) {
    unsigned long long v = of8(at, x);
    if (__ballot(v != 0ull) != 0ull) {
#pragma unroll
      for (int k = 1; k < WAVE; k <<= 1) v += __shfl_xor(v, k, WAVE);
    }
    if (lane == 0) sums[tile * SW + w] = v;
  });
  __syncthreads();
  const int n = (row.vocab + TILE - 1) / TILE * SW;
  unsigned long long mine = 0, total;
  constexpr int PER = MAX_TILES * SW / SB;
#pragma unroll
  for (int k = 0; k < PER; ++k) mine += PER * tid + k < n ? sums[PER * tid + k] : 0ull;
  unsigned long long before = upto_u64(mine, s, total) - mine;
  if (total == 0ull) return -1;
  const unsigned long long target = pick(total);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (PER * tid + k >= n) continue;
    const unsigned long long v = sums[PER * tid + k];
    if (before <= target && before + v > target) s.word[0] = before, s.word[1] = (unsigned long long)(PER * tid + k);
    before += v;
  }
  __syncthreads();
  const int at0 = (int)s.word[1];
  if (w == at0 % SW) {
    const int at = at0 / SW * TILE + tid * E;
    float x[E];
    row.load(at, x);
    unsigned long long v = of8(at, x), end = v;
#pragma unroll
    for (int k = 1; k < WAVE; k <<= 1) {
      const unsigned long long y = __shfl_up(end, k, WAVE);
      if (lane >= k) end += y;
    }
    unsigned long long before = s.word[0] + end - v;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const unsigned long long g = at + k < row.vocab ? f(x[k], at + k) : 0ull;
      if (before <= target && before + g > target) s.word[3] = (unsigned long long)(at + k);
      before += g;
    }
  }
  __syncthreads();
  return (int)s.word[3];
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(SB) sample_kernel(SampleParams p) {
  __shared__ SampleLds s;
  const int tid = (int)threadIdx.x;
  const int64_t b = blockIdx.x;
  Row<DT, VEC> row;
  row.p = (const unsigned char*)p.logits + b * p.row_stride * (DT == F32 ? 4 : 2);
  row.vocab = p.vocab;
  row.table = s.table;
  if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
  const float T = p.temperature ? p.temperature[b] : p.temperature1;
  const int64_t k = p.top_k ? p.top_k[b] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p1;
  const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p1, 1.0f);
  const float u = p.uniforms[b];

  float M = -INFINITY;
  row.each([&](int, int, const float (&x)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) M = fmaxf(M, x[i]);
  });
  M = wave_max(M);
  if (lane_id() == 0) s.top[tid / WAVE] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w) M = fmaxf(M, s.top[w]);
  row.M = M;
  if (M == -INFINITY) {  // no token at all
    if (tid == 0) p.out[b] = -1;
    return;
  }
  const auto largest = [&]() {
    return locate(row, s, [&](float x, int) { return x == M ? 1ull : 0ull; }, [](unsigned long long) { return 0ull; });
  };
  int token = -1;
  if (!(T <= 0.0f) && k != 1) {
    row.rate = 1.44269504088896340736 / (double)T;
    row.per = 64.0f / fmaxf(T, 0.25f);
    row.one = __builtin_amdgcn_ldexp(1.0, p.point);
    unsigned long long thr = 0ull;
    if (k > 0 && k < p.vocab) thr = cut<false>(row, s, 0ull, (unsigned long long)k, 0.0);
    if (!(top_p >= 1.0f)) thr = cut<true>(row, s, thr, 0ull, (double)top_p);
    token = locate(
        row, s,
        [&](float x, int at) {
          if (composite(f2key(x), (uint32_t)at) < thr) return 0ull;
          const double w = row.weight(x);
          return w >= (double)min_p ? row.fixed(w) : 0ull;
        },
        [&](unsigned long long total) {
          const double t = __builtin_floor((double)total * (double)u);
          const unsigned long long v = t >= 0.0 ? (unsigned long long)__builtin_fmin(t, 9.0e18) : 0ull;
          return v < total ? v : total - 1;
        });
  }
  if (token < 0) token = largest();
  if (tid == 0) p.out[b] = token;
}

template <int DT>
int launch(const SampleParams& p, int64_t rows, bool vec, hipStream_t stream) {
  if (vec) hipLaunchKernelGGL((sample_kernel<DT, true>), dim3((unsigned)rows), dim3(SB), 0, stream, p);
  else hipLaunchKernelGGL((sample_kernel<DT, false>), dim3((unsigned)rows), dim3(SB), 0, stream, p);
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
  p.point = std::min(46, 63 - bits - 1);
  const int64_t es = dtype == F32 ? 4 : 2;
  const bool vec = ((uintptr_t)logits & 15u) == 0 && row_stride * es % 16 == 0;
  if (dtype == F32) return launch<F32>(p, n_rows, vec, (hipStream_t)stream);
  if (dtype == BF16) return launch<BF16>(p, n_rows, vec, (hipStream_t)stream);
  return launch<F16>(p, n_rows, vec, (hipStream_t)stream);
}
