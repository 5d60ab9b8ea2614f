// Attention of packed prompts, type BF16.
#include "prompt_impl.h"

namespace pkv {
template hipError_t launch_prompt<BF16>(const PromptParams&, int, hipStream_t);
}  // namespace pkv
