// Attention over caches with a scale per block and head: queries of type BF16, blocks of 16 tokens.
#include "scaled_attention_impl.h"

namespace pkv {
template hipError_t launch_scaled_attention<BF16, 16>(const ScaledAttentionParams&, int, hipStream_t);
}  // namespace pkv
