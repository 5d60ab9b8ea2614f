// Attention of new tokens for queries of type BF16 over BF16 caches.
#include "extend_impl.h"

namespace pkv {
template hipError_t launch_extend_typed<BF16, BF16>(const ExtendParams&, int, hipStream_t);
}  // namespace pkv
