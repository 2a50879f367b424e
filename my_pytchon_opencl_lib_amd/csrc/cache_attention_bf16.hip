// attention over the 8-bit cache, bfloat16 queries (cache_attention.h)
#include "cache_attention.h"

namespace migemm {

int launch_attention_bf16(hipStream_t stream, const AttnArgs &p) {
    return launch_widths<Bf16>(stream, p);
}

}  // namespace migemm
