// Launches of prompt_kernel by head_dim and row form.
#pragma once
#include <type_traits>

#include "prompt.cuh"

#include "capi_internal.h"
#include "summon.h"

namespace sva {

// 16-bit calls of at most kFewRows query rows a KV head (prompt_few.hip).
int launch_prompt_few(const PromptParams& p, int dtype, bool vec, hipStream_t stream);

template <int DT, int DP, int MODE>
int launch_prompt_kernel(const PromptParams& p, hipStream_t stream) {
  constexpr int lds = 4 * PromptType<DT>::BN * DP * PromptType<DT>::ES;
  constexpr auto fn = prompt_kernel<DT, DP, MODE>;
  SVA_SET_MAX_LDS_ONCE(fn, sva::kMaxLds, "hipFuncSetAttribute(prompt_kernel)");
  const int64_t blocks = (int64_t)p.G * p.row_tiles * p.splits * p.n_seq;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), lds, stream, p);
  SVA_CHECK_LAUNCH("prompt_kernel");
  return SVA_OK;
}

template <int DT, int MODE>
int launch_prompt_dim(const PromptParams& p, hipStream_t stream) {
  if (p.D <= 64) return launch_prompt_kernel<DT, 64, MODE>(p, stream);
  if (p.D <= 128) return launch_prompt_kernel<DT, 128, MODE>(p, stream);
  return launch_prompt_kernel<DT, 256, MODE>(p, stream);
}

// ROWS: 0 or PROMPT_FEW.
template <int DT, int ROWS>
int launch_prompt(const PromptParams& p, bool vec, hipStream_t stream) {
  if (!vec) return launch_prompt_dim<DT, PROMPT_ANY + ROWS>(p, stream);
  return p.mask ? launch_prompt_dim<DT, PROMPT_MASK + ROWS>(p, stream)
                : launch_prompt_dim<DT, PROMPT_CAUSAL + ROWS>(p, stream);
}

}  // namespace sva
