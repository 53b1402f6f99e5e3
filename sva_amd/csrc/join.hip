// The second kernel of split attention (join.h).
#include "join.h"

#include "capi_internal.h"
#include "common.cuh"

namespace sva {
namespace {

constexpr int JB = 256;  // 32 elements x 8 ranges at a time

__global__ void __launch_bounds__(JB) join_kernel(JoinParams p) {
  __shared__ float red[2][JB];
  __shared__ float top[JB / WAVE];
  const int item = (int)blockIdx.x, d = (int)blockIdx.y * 32 + (int)threadIdx.x % 32, lane8 = (int)threadIdx.x / 32;
  const int t = item % p.Q, h = item / p.Q % p.H, b = item / (p.Q * p.H);
  int64_t first;
  if (t >= seq_tokens(p.q_lens, p.q_offsets, p.q_rows, p.Q, b, first)) return;
  const float* src = p.part + (int64_t)item * p.splits * (p.D + 2);
  float M = -INFINITY;
  for (int s = (int)threadIdx.x; s < p.splits; s += JB) {
    const float* f = src + (int64_t)s * (p.D + 2);
    if (f[1] != 0.0f) M = fmaxf(M, f[0]);
  }
  M = wave_max(M);
  if (lane_id() == 0) top[threadIdx.x / WAVE] = M;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < JB / WAVE; ++v) M = fmaxf(M, top[v]);
  float Z = 0.0f, a = 0.0f;
#pragma unroll 4
  for (int s = lane8; s < p.splits; s += JB / 32) {
    const float* f = src + (int64_t)s * (p.D + 2);
    const float m = f[0], z = f[1];
    if (z != 0.0f) {  // (a NaN counts)
      const float c = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
      Z += z * c;
      if (d < p.D) a += f[2 + d] * c;
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
    const int64_t at = (p.q_lens ? (first + t) * p.o_ts : (int64_t)b * p.o_bs + (int64_t)t * p.o_ts) +
                       (int64_t)h * p.o_hs + d;
    store_elem(p.out, at, p.out_dtype, Z == 0.0f ? 0.0f : a / Z);
  }
}

}  // namespace

int launch_join(const JoinParams& p, int64_t n_seq, hipStream_t stream) {
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)(n_seq * p.H * p.Q), (unsigned)((p.D + 31) / 32)), dim3(JB), 0,
                     stream, p);
  SVA_CHECK_LAUNCH("join_kernel");
  return SVA_OK;
}

}  // namespace sva
