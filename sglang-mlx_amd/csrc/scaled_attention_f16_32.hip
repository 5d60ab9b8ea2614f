// Attention over caches with a scale per block and head: queries of type F16, blocks of 32 tokens.
#include "scaled_attention_impl.h"

namespace pkv {
template hipError_t launch_scaled_attention<F16, 32>(const ScaledAttentionParams&, int, hipStream_t);
}  // namespace pkv
