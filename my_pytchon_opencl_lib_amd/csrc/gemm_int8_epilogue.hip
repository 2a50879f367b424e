// Products of 8-bit rows with an activation or a residual (gemm_int8.h).
#include "gemm_int8.h"

namespace migemm {

int launch_product_epilogue(hipStream_t stream, const Int8Product &p) {
    return product_int8<kEpilogue>(stream, p);
}

int launch_linear_epilogue(hipStream_t stream, const void *X, int64_t ldx, int cols,
                      const Int8Product &p) {
    return linear_int8<kEpilogue>(stream, X, ldx, cols, p);
}

}  // namespace migemm
