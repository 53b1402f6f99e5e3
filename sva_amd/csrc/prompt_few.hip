// Dense attention of a few 16-bit query rows over many keys: prompt_kernel
// with weights of two terms (the reason stands there).
#include "prompt_launch.h"

namespace sva {

int launch_prompt_few(const PromptParams& p, int dtype, bool vec, hipStream_t stream) {
  return dtype == BF16 ? launch_prompt<BF16, PROMPT_FEW>(p, vec, stream) : launch_prompt<F16, PROMPT_FEW>(p, vec, stream);
}

}  // namespace sva
