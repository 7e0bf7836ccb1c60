// cache4_attention.h for head dim 128
#include "cache4_attention.h"

namespace we {
hipError_t cache4_attention_128(const Attn4& a, hipStream_t s) { return launch_dim<2>(a, s); }
}  // namespace we
