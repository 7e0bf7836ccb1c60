// cache4_attention.h for head dim 64
#include "cache4_attention.h"

namespace we {
hipError_t cache4_attention_64(const Attn4& a, hipStream_t s) { return launch_dim<1>(a, s); }
}  // namespace we
