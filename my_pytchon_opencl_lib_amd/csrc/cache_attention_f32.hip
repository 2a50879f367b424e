// attention over the 8-bit cache, float32 queries (cache_attention.h)
#include "cache_attention.h"

namespace migemm {

int launch_attention_f32(hipStream_t stream, const AttnArgs &p) {
    return launch_widths<float>(stream, p);
}

}  // namespace migemm
