// Attention of new tokens for queries of type F16 over FP8 caches.
#include "extend_impl.h"

namespace pkv {
template hipError_t launch_extend_typed<F16, FP8>(const ExtendParams&, int, hipStream_t);
}  // namespace pkv
