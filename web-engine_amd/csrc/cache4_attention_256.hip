// cache4_attention.h for head dim 256
#include "cache4_attention.h"

namespace we {
hipError_t cache4_attention_256(const Attn4& a, hipStream_t s) { return launch_dim<4>(a, s); }
}  // namespace we
