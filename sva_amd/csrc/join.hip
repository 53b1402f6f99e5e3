// The second kernel of split attention (join.h).  Bound by the way of the sums
// through memory, which other XCDs wrote: 9 items of 328 ranges 6 us, 768 of
// at most 21 14 us, 36864 of six 30 us.
#include "join.h"

#include "capi_internal.h"
#include "common.cuh"

namespace sva {
namespace {

constexpr int JB = 512;  // 32 elements x 16 ranges
constexpr int RB = 256;

struct JoinItem {
  const float* sums;   // [ranges, D]
  const float* stats;  // [ranges, 2]
  int ranges;          // 1: nothing to join
  int64_t at;          // its output
};

SVA_DEV JoinItem join_item(const JoinParams& p, int item) {
  JoinItem x;
  const int t = item % p.Q, h = item / p.Q % p.H, b = item / (p.Q * p.H);
  int64_t first, off;
  const int q_len = seq_tokens(p.q_lens, p.q_offsets, p.q_rows, p.Q, b, first);
  x.ranges = 1;
  if (t >= q_len) return x;
  const int64_t len = seq_keys(p.lens, p.offs, p.N, p.rows, b, off);
  const int grp = p.H / p.G;
  const int rt = (int)(((int64_t)t * grp + h % grp) / p.tile_rows);
  x.ranges = tile_ranges(tile_keys(rt, p.tile_rows, q_len, grp, len, p.causal), p.chunk);
  x.sums = p.sums + (int64_t)item * p.splits * p.D;
  x.stats = p.stats + (int64_t)item * p.splits * 2;
  x.at = (p.q_lens ? (first + t) * p.o_ts : (int64_t)b * p.o_bs + (int64_t)t * p.o_ts) + (int64_t)h * p.o_hs;
  return x;
}

// A range's share of the joined sums: 2^((m - M) sl).  A share of 0 still
// counts: sums that are not finite stay so, as in one range.  (A range without
// a key has sums of 0; one done again whose scores are all NaN has m = -inf
// and z NaN.)
SVA_DEV float join_share(float m, float M, float sl) {
  return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * sl);
}

// Few items of many ranges (decode): a workgroup takes 32 elements of one
// item, 16 ranges at a time, eight rounds of loads in flight: 256 ranges are
// two round trips.
__global__ void __launch_bounds__(JB) join_kernel(JoinParams p) {
  __shared__ float red[2][JB];
  __shared__ float2 top[JB / WAVE];
  const JoinItem x = join_item(p, (int)blockIdx.x);
  const int d = (int)blockIdx.y * 32 + (int)threadIdx.x % 32, part = (int)threadIdx.x / 32;
  if (x.ranges == 1) return;
  constexpr int U = 8, PARTS = JB / 32;
  float M = -INFINITY;
  bool shifted = false;
  for (int s = (int)threadIdx.x; s < x.ranges; s += JB) {
    const float2 st = *(const float2*)(x.stats + 2 * s);
    M = fmaxf(M, st.x);
    shifted = shifted || st.y < 0.0f;
  }
  M = wave_max(M);
  float down = __any(shifted) ? kShifted : 1.0f;  // of ranges that are not
  if (lane_id() == 0) top[threadIdx.x / WAVE] = make_float2(M, down);
  __syncthreads();
#pragma unroll
  for (int v = 0; v < JB / WAVE; ++v) M = fmaxf(M, top[v].x), down = fminf(down, top[v].y);
  float Z = 0.0f, a = 0.0f;
  for (int s0 = part; s0 < x.ranges; s0 += U * PARTS) {
    float2 st[U];
    float sm[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * PARTS;
      st[u] = make_float2(0.0f, 0.0f);
      sm[u] = 0.0f;
      if (s < x.ranges) {
        st[u] = *(const float2*)(x.stats + 2 * s);
        sm[u] = x.sums[(int64_t)s * p.D + min(d, p.D - 1)];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * PARTS >= x.ranges) continue;
      const float c = join_share(st[u].x, M, p.sl) * (st[u].y < 0.0f ? 1.0f : down);
      Z += fabsf(st[u].y) * c;
      a += sm[u] * c;
    }
  }
  red[0][threadIdx.x] = a;
  red[1][threadIdx.x] = Z;
  __syncthreads();
  if (threadIdx.x < 32 && d < p.D) {
    a = Z = 0.0f;
#pragma unroll
    for (int v = 0; v < JB / 32; ++v) {
      a += red[0][32 * v + threadIdx.x];
      Z += red[1][32 * v + threadIdx.x];
    }
    store_elem(p.out, x.at + d, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
  }
}

// Many items of few ranges (prompts): a wave an item, 64 elements and eight
// ranges at a time, with a running maximum: a range's stats and sums are
// loaded together, so an item is two round trips to memory.
__global__ void __launch_bounds__(RB) join_rows_kernel(JoinParams p, int items) {
  const int item = (int)blockIdx.x * (RB / WAVE) + (int)threadIdx.x / WAVE;
  if (item >= items) return;
  const JoinItem x = join_item(p, item);
  if (x.ranges == 1) return;
  constexpr int U = 8;
  for (int d = lane_id(); d < p.D; d += WAVE) {
    float M = -INFINITY, Z = 0.0f, a = 0.0f;
    bool shifted = false;
    for (int s0 = 0; s0 < x.ranges; s0 += U) {
      float2 st[U];
      float sm[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        st[u] = make_float2(-INFINITY, 0.0f);
        sm[u] = 0.0f;
        if (s0 + u < x.ranges) {
          st[u] = *(const float2*)(x.stats + 2 * (s0 + u));
          sm[u] = x.sums[(int64_t)(s0 + u) * p.D + d];
        }
      }
      float top = M;
      bool now = shifted;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, st[u].x), now = now || st[u].y < 0.0f;
      float c = join_share(M, top, p.sl);
      if (now && !shifted) c *= kShifted, shifted = true;
      Z *= c, a *= c, M = top;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u >= x.ranges) continue;
        float f = join_share(st[u].x, M, p.sl);
        if (shifted && !(st[u].y < 0.0f)) f *= kShifted;
        Z += fabsf(st[u].y) * f;
        a += sm[u] * f;
      }
    }
    store_elem(p.out, x.at + d, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
  }
}

}  // namespace

int launch_join(const JoinParams& p, int64_t n_seq, hipStream_t stream) {
  const int64_t items = n_seq * p.H * p.Q;
  if (items <= 1024) {
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)items, (unsigned)((p.D + 31) / 32)), dim3(JB), 0, stream, p);
    SVA_CHECK_LAUNCH("join_kernel");
  } else {
    hipLaunchKernelGGL(join_rows_kernel, dim3((unsigned)((items + RB / WAVE - 1) / (RB / WAVE))), dim3(RB), 0, stream, p,
                       (int)items);
    SVA_CHECK_LAUNCH("join_rows_kernel");
  }
  return SVA_OK;
}

}  // namespace sva
