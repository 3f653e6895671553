// Instantiations of w4_tile_kernel.h: bf16 activations, integer weights.
#include "w4_tile_kernel.h"

namespace cch {

int w4_tile_int4_bf16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    if (kind == W4_I4_G32) return w.zeros ? w4_tile_choose<__bf16, W4_I4_G32, true>(out_kind, rows, w, out, s) : w4_tile_choose<__bf16, W4_I4_G32, false>(out_kind, rows, w, out, s);
    if (kind == W4_I4_G64) return w.zeros ? w4_tile_choose<__bf16, W4_I4_G64, true>(out_kind, rows, w, out, s) : w4_tile_choose<__bf16, W4_I4_G64, false>(out_kind, rows, w, out, s);
    if (kind == W4_I4_G128) return w.zeros ? w4_tile_choose<__bf16, W4_I4_G128, true>(out_kind, rows, w, out, s) : w4_tile_choose<__bf16, W4_I4_G128, false>(out_kind, rows, w, out, s);
    return fail(CCH_EINVAL, "weights of kind %d", kind);
}

}  // namespace cch
