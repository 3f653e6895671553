// A product of 16-bit operands to the kernel that its plan names.
#pragma once
#include "gemm16_big_kernel.h"
#include "gemm16_stream_kernel.h"

namespace cch {

template <class T, int LAYOUT, int EPI> int shape16(Gemm16 p, const Plan16 &plan, hipStream_t stream)
{
    CCH_REQUIRE((tiles16(p, 128, 128) + 8 * (int64_t)p.groups) * plan.splits < (int64_t)1 << 31, "a product of %d x %d in %d groups has too many tiles", p.m, p.n, p.groups);
    p.splits = plan.splits;
    p.tail = plan.tail;
    if constexpr (LAYOUT != ROWS_TN && (EPI == EPI16_OUT || EPI == EPI16_ACT)) {
        if (plan.kernel == KERNEL16_ROWS) {
            const int rows = rows16(p);
            if (rows == 8) return launch16_stream_rows<T, LAYOUT, EPI, 8>(p, tiles16(p, 8, Stream16<LAYOUT, 8>::TN), stream);
            if (rows == 16) return launch16_stream_rows<T, LAYOUT, EPI, 16>(p, tiles16(p, 16, Stream16<LAYOUT, 16>::TN), stream);
            return launch16_stream_rows<T, LAYOUT, EPI, 32>(p, tiles16(p, 32, Stream16<LAYOUT, 32>::TN), stream);
        }
    }
    if (plan.kernel == KERNEL16_256) return launch16_big<T, LAYOUT, EPI>(p, tiles16(p, 256, 256), stream);
    if (plan.deep) return launch16<T, LAYOUT, EPI, Shape16<2, 2, 2, 2, 4>>(p, tiles16(p, 128, 128), stream);
    return launch16<T, LAYOUT, EPI, Shape16<2, 2, 2, 2, 2>>(p, tiles16(p, 128, 128), stream);
}

template <class T> int choose16(const Gemm16 &p, const Plan16 &plan, int layout, int epilogue, hipStream_t stream)
{
    switch (layout * 4 + epilogue) {
    case ROWS_NK * 4 + EPI16_OUT: return shape16<T, ROWS_NK, EPI16_OUT>(p, plan, stream);
    case ROWS_NN * 4 + EPI16_OUT: return shape16<T, ROWS_NN, EPI16_OUT>(p, plan, stream);
    case ROWS_TN * 4 + EPI16_OUT: return shape16<T, ROWS_TN, EPI16_OUT>(p, plan, stream);
    case ROWS_NK * 4 + EPI16_ACT: return shape16<T, ROWS_NK, EPI16_ACT>(p, plan, stream);
    case ROWS_NN * 4 + EPI16_ACT: return shape16<T, ROWS_NN, EPI16_ACT>(p, plan, stream);
    case ROWS_NK * 4 + EPI16_STATS: return shape16<T, ROWS_NK, EPI16_STATS>(p, plan, stream);
    case ROWS_NK * 4 + EPI16_GRAD: return shape16<T, ROWS_NK, EPI16_GRAD>(p, plan, stream);
    }
    return fail(CCH_EINVAL, "no product of layout %d with epilogue %d", layout, epilogue);
}

}  // namespace cch
