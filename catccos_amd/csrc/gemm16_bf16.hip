// Instantiations of gemm16_kernel.h: bf16.
#include "gemm16_choose.h"

namespace cch {

int gemm16_launch_bf16(const Gemm16 &p, const Plan16 &plan, int layout, int epilogue, hipStream_t stream)
{
    return choose16<Bf16>(p, plan, layout, epilogue, stream);
}

}  // namespace cch
