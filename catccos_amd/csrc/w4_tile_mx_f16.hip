// Instantiations of w4_tile_kernel.h: IEEE half activations, MXFP4 weights.
#include "w4_tile_kernel.h"

namespace cch {

int w4_tile_mx_f16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    return w4_tile_choose<_Float16, W4_MX, false>(out_kind, rows, w, out, s);
}

}  // namespace cch
