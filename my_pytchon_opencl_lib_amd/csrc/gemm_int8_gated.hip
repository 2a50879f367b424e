// Products of 8-bit rows of a gate's activation and the other half (gemm_int8.h).
#include "gemm_int8.h"

namespace migemm {

int launch_product_gated(hipStream_t stream, const Int8Product &p) {
    return product_int8<kGated>(stream, p);
}

int launch_linear_gated(hipStream_t stream, const void *X, int64_t ldx, int cols,
                      const Int8Product &p) {
    return linear_int8<kGated>(stream, X, ldx, cols, p);
}

}  // namespace migemm
