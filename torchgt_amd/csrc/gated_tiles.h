// Gated projections and linears with an epilogue where the widths are small (gated_tiles.hip) for gated.hip.
#pragma once
#include "common.h"

namespace tgt {

struct NarrowArgs {
    const void* x;          // [N, K], K a multiple of 16 bytes
    const void* W[2];       // [F, K]; the second one only with two
    const void* bias[2];    // [F] or null
    const void* more;       // [N, F]: the residual, or with `grad` the gradient of the result; null: no residual
    void* out[2];           // [N, out_ld]; `grad` with two weights: dg and du
    int64_t N;
    int K, F;
    int out_ld;             // F, or with `grad` F rounded up to 16 bytes: the columns behind F are zeros then
    int act;
    void* padded;           // `grad` with one weight: where to put W[0] with rows of zeros up to out_ld (16-byte aligned), or null
};

// act(x W0^T + b0) * (x W1^T + b1), or with one weight act(x W0^T + b0) + residual; grad: the gradients of what the activation and the other factor
// were taken of
int gated_tiles(const NarrowArgs& a, bool grad, int dtype, hipStream_t st);

}  // namespace tgt
