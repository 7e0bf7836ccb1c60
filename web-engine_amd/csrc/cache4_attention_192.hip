// cache4_attention.h for head dim 192
#include "cache4_attention.h"

namespace we {
hipError_t cache4_attention_192(const Attn4& a, hipStream_t s) { return launch_dim<3>(a, s); }
}  // namespace we
