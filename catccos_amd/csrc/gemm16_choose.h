// Which kernel a product of 16-bit operands runs on.
#pragma once
#include "gemm16_big_kernel.h"
#include "gemm16_stream_kernel.h"

namespace cch {

// Tiles that a launch may have: the groups' sizes are on the device.
inline int64_t tiles16(const Gemm16 &p, int tm, int tn)
{
    const int64_t cols = (p.n + tn - 1) / tn;
    if (p.k_grouped) return (int64_t)p.groups * ((p.m + tm - 1) / tm) * cols;
    return (p.group_sizes ? p.m / tm + std::min(p.groups, p.m) : (p.m + tm - 1) / tm) * cols;
}

template <class T, int LAYOUT, int EPI> int shape16(const Gemm16 &p, hipStream_t stream)
{
    using Mid = Shape16<2, 2, 2, 2, 2>;
    int dev = 0, cus = 0;
    CCH_HIP(hipGetDevice(&dev));
    CCH_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    if constexpr (LAYOUT != ROWS_TN && (EPI == EPI16_OUT || EPI == EPI16_ACT)) {
        const int64_t per_group = (p.m + p.groups - 1) / p.groups;
        const bool plain = !p.a_rows && !p.sums && !p.out_rows && !p.scale;
        const int asked = g_kernel16.load();
        if (plain && (asked == KERNEL16_ROWS || (asked < 0 && per_group <= 32))) {
            if (per_group <= 8) return launch16_stream_rows<T, LAYOUT, EPI, 8>(p, tiles16(p, 8, Stream16<LAYOUT, 8>::TN), stream);
            if (per_group <= 16) return launch16_stream_rows<T, LAYOUT, EPI, 16>(p, tiles16(p, 16, Stream16<LAYOUT, 16>::TN), stream);
            return launch16_stream_rows<T, LAYOUT, EPI, 32>(p, tiles16(p, 32, Stream16<LAYOUT, 32>::TN), stream);
        }
    }
    const int64_t big = tiles16(p, 256, 256);
    const int asked = g_kernel16.load();
    CCH_REQUIRE(tiles16(p, 128, 128) < (int64_t)1 << 31, "a product of %d x %d in %d groups has too many tiles", p.m, p.n, p.groups);
    if (!p.a_rows && p.pitch_out < MAX_PITCH16 / 2 && (asked == KERNEL16_256 || (asked < 0 && big >= BIG_TILES16))) return launch16_big<T, LAYOUT, EPI>(p, big, cus, stream);
    return launch16<T, LAYOUT, EPI, Mid>(p, tiles16(p, Mid::TM, Mid::TN), stream);
}

template <class T> int choose16(const Gemm16 &p, int layout, int epilogue, hipStream_t stream)
{
    switch (layout * 4 + epilogue) {
    case ROWS_NK * 4 + EPI16_OUT: return shape16<T, ROWS_NK, EPI16_OUT>(p, stream);
    case ROWS_NN * 4 + EPI16_OUT: return shape16<T, ROWS_NN, EPI16_OUT>(p, stream);
    case ROWS_TN * 4 + EPI16_OUT: return shape16<T, ROWS_TN, EPI16_OUT>(p, stream);
    case ROWS_NK * 4 + EPI16_ACT: return shape16<T, ROWS_NK, EPI16_ACT>(p, stream);
    case ROWS_NN * 4 + EPI16_ACT: return shape16<T, ROWS_NN, EPI16_ACT>(p, stream);
    case ROWS_NK * 4 + EPI16_STATS: return shape16<T, ROWS_NK, EPI16_STATS>(p, stream);
    case ROWS_NK * 4 + EPI16_GRAD: return shape16<T, ROWS_NK, EPI16_GRAD>(p, stream);
    }
    return fail(CCH_EINVAL, "no product of layout %d with epilogue %d", layout, epilogue);
}

}  // namespace cch
