// How the router and the balance loss lay a token's logits over lanes, and the sums and maxima over them.
//
// A token is L neighbouring lanes of V consecutive experts each, 64 / L tokens to a wave.  Experts past the last read as -inf, which nothing selects and whose
// exponential is zero.  A lane's own work grows with V, the steps between lanes, and the lanes that repeat what is done once per token, with L; up to L = 16 such a
// step is a DPP move.  Measured in us (router forward / backward, balance loss forward / backward, bf16, softmax over the experts, 8 routes):
//                   16384 tokens                                       64 tokens
//   64 experts      V 8, L 8    4.6 /  3.8   10.2 /  4.0                3.5 / 3.0    5.1 / 3.4
//                   V 4, L 16   5.5 /  3.8   10.1 /  4.2                3.3 / 2.6    4.2 / 3.3
//   128             V 8, L 16   6.7 /  4.5   14.1 /  5.0                3.6 / 2.9    4.8 / 3.5
//                   V 4, L 32   8.9 /  4.8   14.9 /  5.9                3.8 / 2.7    4.7 / 3.4
//                   V 16, L 8   6.1 /  4.8   14.6 /  5.2                4.4 / 3.5    6.8 / 3.9
//   256             V 16, L 16  9.3 /  6.5   15.4 /  7.0                4.4 / 3.4    6.2 / 3.9
//                   V 8, L 32  11.2 /  6.5   15.8 /  7.5                4.1 / 3.0    5.3 / 3.7
//                   V 32, L 8   9.3 /  8.0   17.1 /  8.9                6.5 / 4.9   10.0 / 5.4
//   512             V 16, L 32 16.0 / 10.9   17.7 / 10.5                5.1 / 3.5    6.8 / 4.1
//                   V 8, L 64  19.0 / 10.9   18.9 / 10.8                4.4 / 3.1   10.6 / 3.8
//   1024            V 16, L 64 28.0 / 16.7   22.8 / 16.0                5.4 / 3.6   11.8 / 4.1
//                   V 32, L 32 25.7 / 20.5   23.1 / 19.2                7.1 / 4.9   12.3 / 5.5
// The first of each is taken: the best or near it where there is work, within a microsecond of the best where launches count.
#pragma once
#include <cmath>

#include "common.h"

namespace cch {

constexpr int ROUTER_MAX_EXPERTS = 1024, ROUTER_MAX_TOPK = 8;
constexpr int64_t ROUTER_MAX_TOKENS = 1 << 30;   // (a workgroup's last token and its step fit 32 bits)

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}

// Over the L lanes of a token; every lane has the result.  (After the steps within 4 lanes the mirrors meet lanes of the other half.)
template <int L, class F>
__device__ __forceinline__ float over_lanes(float x, F f)
{
    static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes of a token");
    x = f(x, dpp_f32<0xB1>(x));    // quad_perm [1,0,3,2]
    x = f(x, dpp_f32<0x4E>(x));    // quad_perm [2,3,0,1]
    x = f(x, dpp_f32<0x141>(x));   // row_half_mirror
    if (L > 8) x = f(x, dpp_f32<0x140>(x));   // row_mirror
    if (L > 16) x = f(x, __shfl_xor(x, 16, 64));
    if (L > 32) x = f(x, __shfl_xor(x, 32, 64));
    return x;
}
template <int L>
__device__ __forceinline__ float lanes_max(float x)
{
    return over_lanes<L>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
__device__ __forceinline__ float lanes_sum(float x)
{
    return over_lanes<L>(x, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }

// This lane's V logits of a row, `experts` long, as they come from memory, so that a row can be on its way while another is worked on.  VEC: rows start and end
// on boundaries of a lane's loads of up to 16 bytes (router forward / backward, balance forward / backward: 16384 x 64 in bf16 4.6 / 3.8, 10.1 / 4.0 us; one element
// at a time 5.2 / 4.7, 11.1 / 6.0; 4096 x 256 4.7 / 3.9, 11.8 / 4.4 against 6.2 / 7.4, 15.0 / 10.3).
template <class T, int V>
struct LanePieces {
    static constexpr int CHUNK = V * (int)sizeof(T) < 16 ? V : 16 / (int)sizeof(T);   // elements of one access
    typedef T Piece __attribute__((ext_vector_type(CHUNK)));
    static bool vec(const void *p, int64_t experts) { return (experts * (int64_t)sizeof(T)) % (CHUNK * (int)sizeof(T)) == 0 && aligned(p, CHUNK * sizeof(T)); }
};
template <class T, int V, bool VEC>
struct LaneRow {
    static constexpr int CHUNK = VEC ? LanePieces<T, V>::CHUNK : 1;
    typedef T Piece __attribute__((ext_vector_type(CHUNK)));
    Piece raw[V / CHUNK];

    __device__ __forceinline__ void load(const T *row, int first, int experts)
    {
#pragma unroll
        for (int c = 0; c < V / CHUNK; c++) {
            raw[c] = Piece{};
            if (first + c * CHUNK < experts) raw[c] = *reinterpret_cast<const Piece *>(row + first + c * CHUNK);
        }
    }
    __device__ __forceinline__ void values(int first, int experts, float (&l)[V]) const
    {
#pragma unroll
        for (int i = 0; i < V; i++) l[i] = first + i / CHUNK * CHUNK < experts ? to_f32(raw[i / CHUNK][i % CHUNK]) : -INFINITY;
    }
    static __device__ __forceinline__ void store(T *row, int first, int experts, const float (&d)[V])
    {
#pragma unroll
        for (int c = 0; c < V / CHUNK; c++)
            if (first + c * CHUNK < experts) {
                Piece p;
#pragma unroll
                for (int i = 0; i < CHUNK; i++) p[i] = (T)d[c * CHUNK + i];
                *reinterpret_cast<Piece *>(row + first + c * CHUNK) = p;
            }
    }
};
template <class T, int V>
__device__ __forceinline__ void load_row(const T *row, int first, int experts, bool vec, float (&l)[V])
{
    if (vec) {
        LaneRow<T, V, true> r;
        r.load(row, first, experts);
        r.values(first, experts, l);
    } else {
        LaneRow<T, V, false> r;
        r.load(row, first, experts);
        r.values(first, experts, l);
    }
}
template <class T, int V>
__device__ __forceinline__ void store_row(T *row, int first, int experts, bool vec, const float (&d)[V])
{
    if (vec) LaneRow<T, V, true>::store(row, first, experts, d);
    else LaneRow<T, V, false>::store(row, first, experts, d);
}

// 1 / x to a unit in the last place, one instruction (an exact division is ten).
__device__ __forceinline__ float reciprocal(float x) { return __builtin_amdgcn_rcpf(x); }

// e^x: the product with log2(e) and that constant are rounded, so that the result is off by up to |x| log2(e) 2^-23 relative and the instruction's unit.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// sigmoid(l) / e^c for c <= 0, c no smaller than l or zero: with c the smaller of 0 and the largest of several logits, their sum is at least 1/2
// however negative all of them are.  `ec` = e^c.
__device__ __forceinline__ float scaled_sigmoid(float l, float c, float ec)
{
    // (where l > 0 c is 0)
    const float t = exp_of(l > 0 ? -l : l - c), over = reciprocal(1.0f + (l > 0 ? t : t * ec));
    return l > 0 ? over : t * over;
}
// sigmoid(l) and 1 - sigmoid(l) from one exponential and one reciprocal.
__device__ __forceinline__ void sigmoid_pair(float l, float &s, float &rest)
{
    const float u = exp_of(-fabsf(l)), r = reciprocal(1.0f + u), ur = u * r;
    s = l > 0 ? r : ur;
    rest = l > 0 ? ur : r;
}
__device__ __forceinline__ float sigmoid(float l) { return reciprocal(1.0f + exp_of(-l)); }
// Logits so far below zero that their sigmoids leave the range are scaled; above this none are.
constexpr float SIGMOID_IN_RANGE = -60.0f;

// The instantiation for this many experts: f(integral_constant V, integral_constant L).
template <int N>
struct Int {
    static constexpr int value = N;
};
template <class F>
int with_lanes(int experts, F f)
{
    if (experts <= 16) return f(Int<2>{}, Int<8>{});
    if (experts <= 32) return f(Int<4>{}, Int<8>{});
    if (experts <= 64) return f(Int<8>{}, Int<8>{});
    if (experts <= 128) return f(Int<8>{}, Int<16>{});
    if (experts <= 256) return f(Int<16>{}, Int<16>{});
    if (experts <= 512) return f(Int<16>{}, Int<32>{});
    return f(Int<16>{}, Int<64>{});
}
template <class F>
int with_logits_type(int dtype, F f)
{
    if (dtype == CCH_DTYPE_F32) return f((float *)nullptr);
    if (dtype == CCH_DTYPE_F16) return f((_Float16 *)nullptr);
    return f((__bf16 *)nullptr);
}
inline bool logits_type_ok(int dtype) { return dtype == CCH_DTYPE_BF16 || dtype == CCH_DTYPE_F16 || dtype == CCH_DTYPE_F32; }

}  // namespace cch
