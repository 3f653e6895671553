// How the router and the balance loss lay a token's logits over lanes, and the sums and maxima over them.
//
// A token is L neighbouring lanes of V consecutive experts each, 64 / L tokens to a wave.  V grows with the number of experts, so that the steps
// between lanes stay few: up to 256 experts they are DPP moves within a row of 16.  Experts past the last read as -inf, which nothing selects
// and whose exponential is zero.
#pragma once
#include <cmath>

#include "common.h"

namespace cch {

constexpr int ROUTER_MAX_EXPERTS = 1024, ROUTER_MAX_TOPK = 8;

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

// This lane's V logits of the row at `row`, `experts` long.  vec: rows start and end on boundaries of a lane's loads.
template <class T, int V>
struct LaneRow {
    static constexpr int CHUNK = V * (int)sizeof(T) < 16 ? V : 16 / (int)sizeof(T);   // elements of one access
    typedef T Piece __attribute__((ext_vector_type(CHUNK)));

    static bool vec(const void *p, int64_t experts) { return (experts * (int64_t)sizeof(T)) % (CHUNK * (int)sizeof(T)) == 0 && aligned(p, CHUNK * sizeof(T)); }

    static __device__ __forceinline__ void load(const T *row, int first, int experts, bool vec, float (&l)[V])
    {
#pragma unroll
        for (int i = 0; i < V; i++) l[i] = -INFINITY;
        if (vec) {
#pragma unroll
            for (int c = 0; c < V; c += CHUNK)
                if (first + c < experts) {
                    const Piece p = *reinterpret_cast<const Piece *>(row + first + c);
#pragma unroll
                    for (int i = 0; i < CHUNK; i++) l[c + i] = to_f32(p[i]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (first + i < experts) l[i] = to_f32(row[first + i]);
        }
    }
    static __device__ __forceinline__ void store(T *row, int first, int experts, bool vec, const float (&d)[V])
    {
        if (vec) {
#pragma unroll
            for (int c = 0; c < V; c += CHUNK)
                if (first + c < experts) {
                    Piece p;
#pragma unroll
                    for (int i = 0; i < CHUNK; i++) p[i] = (T)d[c + i];
                    *reinterpret_cast<Piece *>(row + first + c) = p;
                }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (first + i < experts) row[first + i] = (T)d[i];
        }
    }
};

// sigmoid(l) / e^c for c <= 0, c no smaller than l or zero: with c the smaller of 0 and the largest of several logits, their sum is at least 1/2
// however negative all of them are.  `ec` = e^c.
__device__ __forceinline__ float scaled_sigmoid(float l, float c, float ec)
{
    if (l > 0) return 1.0f / (1.0f + __expf(-l));   // (then c is 0)
    const float t = __expf(l - c);
    return t / (1.0f + t * ec);
}
__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + __expf(-l)); }

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
