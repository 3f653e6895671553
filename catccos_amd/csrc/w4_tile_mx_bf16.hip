// Instantiations of w4_tile_kernel.h: bf16 activations, MXFP4 weights.
#include "w4_tile_kernel.h"

namespace cch {

int w4_tile_mx_bf16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    return w4_tile_choose<__bf16, W4_MX, false>(out_kind, rows, w, out, s);
}

}  // namespace cch
