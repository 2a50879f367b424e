// Products of 8-bit rows without an epilogue of their own, and the choice of the kind
// (gemm_int8.h).
#include "gemm_int8.h"

namespace migemm {

int launch_product_int8(hipStream_t stream, const Int8Product &p) {
    if (p.gated) return launch_product_gated(stream, p);
    if (p.act != MIGEMM_ACT_NONE || p.residual != nullptr)
        return launch_product_epilogue(stream, p);
    return product_int8<kProduct>(stream, p);
}

int launch_linear_int8(hipStream_t stream, const void *X, int64_t ldx, int cols,
                       const Int8Product &p) {
    if (p.gated) return launch_linear_gated(stream, X, ldx, cols, p);
    if (p.act != MIGEMM_ACT_NONE || p.residual != nullptr)
        return launch_linear_epilogue(stream, X, ldx, cols, p);
    return linear_int8<kProduct>(stream, X, ldx, cols, p);
}

}  // namespace migemm
