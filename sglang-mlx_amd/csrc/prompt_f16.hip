// Attention of packed prompts, type F16.
#include "prompt_impl.h"

namespace pkv {
template hipError_t launch_prompt<F16>(const PromptParams&, int, hipStream_t);
}  // namespace pkv
