// y = x w^T of a few 16-bit rows with 4-bit weights, on matrix instructions, for K a multiple of 32 and pointers on 16-byte boundaries.
//
// A wave takes 16 rows of weights (a tile; NT of them at a time) and 128 of K at a time (a block): every lane has 16 bytes of codes, 32 weights of row
// lane % 16 from K = 32 (lane / 16) on, in one load, and they go from the registers they were loaded to into v_mfma_f32_16x16x32 as its right operand; the left one is
// 16 rows of x (MT times).  No LDS and no barrier until the end: the waves of a workgroup share the tiles and split K, and their sums meet in LDS.
//
// A sum over K may be taken in any order, so the instruction's 32 values of K are whichever lie ready.  A code of 4 bits becomes a 16-bit number with one shift and
// one and-or: 16 + q, the code in the leading bits of 1.xxxx * 2^4.  Masks with two nibbles 16 bits apart give pairs (j, j + 4) of a dword's eight elements, and x is
// put in the same order.  The 16 and the zero point leave by a second instruction with the constant -(16 + z) as its right operand, exactly: in
// fp32 the products of a group sum to what (q - z) gives, and one fused multiply-add per group brings its scale in, which is never rounded into a weight.
// That asks for a group's values to meet in one instruction and no others: with groups of 128 they do; for groups of 32 and 64 the four dwords of the four
// lanes of a row are transposed first (four lane swaps per 32 weights).  MXFP4 with bf16 needs none of it: the conversion instruction applies the power of two, exactly.
//
// Bound: the weights' bytes from HBM, below some 100 rows.  Per weight the vector units spend 1.1 to 1.7 instructions with one tile of x (0.6 for MXFP4), of
// the 3.5 or so that they have time for at the rate of HBM.
#pragma once
#include <algorithm>
#include <type_traits>

#include "w4_decode.h"

namespace cch {

typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));

constexpr int W4_WAVES = 8, W4_THREADS = 64 * W4_WAVES;

template <class T>
struct W4Type;
template <>
struct W4Type<__bf16> {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
    static constexpr uint32_t SIXTEEN = 0x41804180u, MASK = 0x00780078u;   // 16.0 twice, and where a code goes in it
    static constexpr int SHIFT = 3;
    static __device__ __forceinline__ w4_f32x4 mfma(w4_u32x4 a, w4_u32x4 b, w4_f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x) >> 16; }   // of a number that bf16 holds
    template <int BYTE>
    static __device__ __forceinline__ uint32_t fp4(uint32_t q, float scale)
    {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, BYTE));
    }
};
template <>
struct W4Type<_Float16> {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
    static constexpr uint32_t SIXTEEN = 0x4C004C00u, MASK = 0x03C003C0u;
    static constexpr int SHIFT = 6;
    static __device__ __forceinline__ w4_f32x4 mfma(w4_u32x4 a, w4_u32x4 b, w4_f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
    template <int BYTE>
    static __device__ __forceinline__ uint32_t fp4(uint32_t q, float scale)
    {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, BYTE));
    }
};

// a's lanes 32..63 for b's lanes 0..31 / within either half: a's lanes 16..31 for b's 0..15.
__device__ __forceinline__ void w4_swap32(uint32_t &a, uint32_t &b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void w4_swap16(uint32_t &a, uint32_t &b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
// Element (g, i): dword i of lane group g.  Afterwards (i, g).
__device__ __forceinline__ void w4_transpose(w4_u32x4 &v)
{
    uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
    w4_swap32(a, c);
    w4_swap32(b, d);
    w4_swap16(a, b);
    w4_swap16(c, d);
    v = (w4_u32x4){a, b, c, d};
}

template <class T, int KIND>
struct W4Tile {
    typedef W4Type<T> Type;
    static constexpr bool MX = KIND == W4_MX, IN_WEIGHT = MX && std::is_same_v<T, __bf16>;   // the scale is in the weight
    static constexpr int GROUP = KIND == W4_I4_G128 ? 128 : KIND == W4_I4_G64 ? 64 : 32;
    static constexpr int GROUPS = IN_WEIGHT ? 1 : 128 / GROUP, PER = 4 / GROUPS;   // of a block; matrix instructions of a group
    static constexpr bool TRANSPOSED = GROUPS > 1;

    // What one lane has of one tile and one block.
    struct Codes {
        w4_u32x4 q;
        uint32_t scale, zero;
    };

    // Everything by lane: `codes` and `scales` at the tile's row lane % 16.
    static __device__ __forceinline__ Codes load(const W4Matrix &w, const uint8_t *codes, int64_t row, int block)
    {
        const int g = (threadIdx.x & 63) >> 4;
        const int first = block * 128 + g * 32;                          // of this lane's K
        const int group = GROUP == 128 && !IN_WEIGHT ? block : GROUP == 64 ? block * 2 + (g >> 1) : block * 4 + g;
        Codes c;
        c.q = (w4_u32x4){0, 0, 0, 0};
        c.scale = 0;
        c.zero = 8;
        if (first < w.k) c.q = *reinterpret_cast<const w4_u32x4 *>(codes + first / 2);
        if (group * GROUP < w.k) {
            const int64_t at = row * w.row_groups + group;
            if (MX) {
                c.scale = static_cast<const uint8_t *>(w.scales)[at];
            } else {
                c.scale = static_cast<const uint16_t *>(w.scales)[at];
                if (w.zeros) c.zero = w.zeros[at];
            }
        }
        return c;
    }

    // The four right operands of a block, in K's order of `x_of`.
    static __device__ __forceinline__ w4_u32x4 operand(uint32_t q, float scale)
    {
        w4_u32x4 r;
        if (MX) {
            r[0] = Type::template fp4<0>(q, scale);
            r[1] = Type::template fp4<1>(q, scale);
            r[2] = Type::template fp4<2>(q, scale);
            r[3] = Type::template fp4<3>(q, scale);
        } else {
            constexpr int S = Type::SHIFT;
            r[0] = (q << S & Type::MASK) | Type::SIXTEEN;
            r[1] = ((S >= 4 ? q << (S >= 4 ? S - 4 : 0) : q >> (S >= 4 ? 0 : 4 - S)) & Type::MASK) | Type::SIXTEEN;
            r[2] = (q >> (8 - S) & Type::MASK) | Type::SIXTEEN;
            r[3] = (q >> (12 - S) & Type::MASK) | Type::SIXTEEN;
        }
        return r;
    }

    // x's K of matrix instruction i of a block in this lane: eight values from here on.
    static __device__ __forceinline__ int x_at(int i)
    {
        const int g = (threadIdx.x & 63) >> 4;
        return TRANSPOSED ? 32 * i + 8 * g : 32 * g + 8 * i;
    }
    static __device__ __forceinline__ w4_u32x4 x_order(w4_u32x4 v)
    {
        if (MX) return v;
        return (w4_u32x4){__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                          __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
    }

    // A value per lane group (in its lanes) to one per group of the block, in all lanes.
    static __device__ __forceinline__ void spread(uint32_t v, uint32_t (&out)[GROUPS])
    {
        if constexpr (GROUPS == 1) {
            out[0] = v;
        } else {
            uint32_t lo = v, hi = v;
            w4_swap32(lo, hi);
            if constexpr (GROUPS == 2) {
                out[0] = lo;
                out[1] = hi;
            } else {
                out[0] = out[1] = lo;
                out[2] = out[3] = hi;
                w4_swap16(out[0], out[1]);
                w4_swap16(out[2], out[3]);
            }
        }
    }

    template <int MT>
    static __device__ __forceinline__ void multiply(Codes c, const w4_u32x4 (&x)[MT][4], w4_f32x4 (&acc)[MT])
    {
        if constexpr (IN_WEIGHT) {
            const float scale = w4_e8m0(c.scale);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const w4_u32x4 b = operand(c.q[i], scale);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) acc[mt] = Type::mfma(x[mt][i], b, acc[mt]);
            }
        } else {
            if (TRANSPOSED) w4_transpose(c.q);
            float s;
            if (MX) s = w4_e8m0(c.scale);
            else if constexpr (std::is_same_v<T, __bf16>) s = __uint_as_float(c.scale << 16);
            else s = (float)__builtin_bit_cast(_Float16, (uint16_t)c.scale);
            uint32_t scale[GROUPS], zero[GROUPS];
            spread(__float_as_uint(s), scale);
            if (!MX) spread(Type::bits(-16.0f - (float)c.zero) * 0x10001u, zero);
#pragma unroll
            for (int gr = 0; gr < GROUPS; gr++) {
                w4_u32x4 b[PER];
#pragma unroll
                for (int i = 0; i < PER; i++) b[i] = operand(c.q[gr * PER + i], 1.0f);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    w4_f32x4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        if (!MX) d = Type::mfma(x[mt][gr * PER + i], (w4_u32x4){zero[gr], zero[gr], zero[gr], zero[gr]}, d);
                        d = Type::mfma(x[mt][gr * PER + i], b[i], d);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[mt][r] += __uint_as_float(scale[gr]) * d[r];
                }
            }
        }
    }
};

// The wave's sums over its blocks [begin, end) of NT tiles, rows `row[j]` (by lane) of the weights, and MT tiles of x whose rows start at x[mt] (by lane).
template <class T, int KIND, int NT, int MT>
__device__ __forceinline__ void w4_sums(const W4Matrix &w, const int64_t (&row)[NT], const T *const (&x)[MT], int begin, int end, w4_f32x4 (&acc)[NT][MT])
{
    typedef W4Tile<T, KIND> Tile;
    const uint8_t *codes[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        codes[j] = w.codes + row[j] * w.row_bytes;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) acc[j][mt] = (w4_f32x4){0, 0, 0, 0};
    }
    if (begin >= end) return;
    struct Stage {
        typename Tile::Codes c[NT];
        w4_u32x4 x[MT][4];
    };
    auto fetch_x = [&](Stage &s, int block) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = block * 128 + Tile::x_at(i);
                s.x[mt][i] = (w4_u32x4){0, 0, 0, 0};
                if (k < w.k) s.x[mt][i] = *reinterpret_cast<const w4_u32x4 *>(x[mt] + k);
            }
    };
    auto fetch = [&](Stage &s, int block) {
#pragma unroll
        for (int j = 0; j < NT; j++) s.c[j] = Tile::load(w, codes[j], row[j], block);
        if (MT <= 2) fetch_x(s, block);
    };
    auto use = [&](Stage &s, int block) {
        if (MT > 2) fetch_x(s, block);
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) s.x[mt][i] = Tile::x_order(s.x[mt][i]);
#pragma unroll
        for (int j = 0; j < NT; j++) Tile::template multiply<MT>(s.c[j], s.x, acc[j]);
    };
    Stage a, b;
    fetch(a, begin);
    for (int block = begin; block < end; block += 2) {
        fetch(b, min(block + 1, end - 1));
        use(a, block);
        if (block + 1 >= end) break;
        fetch(a, min(block + 2, end - 1));
        use(b, block + 1);
    }
}

// Which matrix, and which rows of x: workgroup column `slot` of the grid takes the slot-th expert that some route names (up to 64 routes: the expert of route
// `slot`, if no earlier one names it).  Returns the number of its routes, their numbers in `list`; 0: nothing to do.
__device__ __forceinline__ int w4_routes(const W4Rows &rows, int slot, int (&list)[W4_LIST], int (&scratch)[1024 + 2], int &expert)
{
    const int lane = threadIdx.x & 63, routes = (int)rows.rows;
    if (routes <= 64) {
        int e = lane < routes ? rows.experts[lane] : -1;
        if (e >= rows.num_experts) e = -1;
        expert = __builtin_amdgcn_readfirstlane(__shfl(e, slot, 64));
        const uint64_t same = __ballot(e == expert);
        if (expert < 0 || __ffsll((unsigned long long)same) - 1 != slot) return 0;
        if (threadIdx.x < 64 && e == expert) list[__builtin_popcountll(same & ((1ull << lane) - 1))] = lane;
        __syncthreads();
        return __builtin_popcountll(same);
    }
    int *count = scratch;
    for (int e = threadIdx.x; e < 1024; e += W4_THREADS) count[e] = 0;
    __syncthreads();
    int mine[W4_LIST / W4_THREADS];
#pragma unroll
    for (int u = 0; u < W4_LIST / W4_THREADS; u++) {
        const int r = u * W4_THREADS + (int)threadIdx.x;
        mine[u] = r < routes ? rows.experts[r] : -1;
        if (mine[u] >= rows.num_experts) mine[u] = -1;
        if (mine[u] >= 0) atomicAdd(&count[mine[u]], 1);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        int seen = 0, found = -1;
        for (int e0 = 0; e0 < rows.num_experts && found < 0; e0 += 64) {
            const bool some = count[e0 + lane] > 0;                // (1024 counters, whatever num_experts is)
            const uint64_t is = __ballot(some);
            const uint64_t at = __ballot(some && seen + __builtin_popcountll(is & ((1ull << lane) - 1)) == slot);
            if (at) found = e0 + __ffsll((unsigned long long)at) - 1;
            seen += __builtin_popcountll(is);
        }
        if (lane == 0) {
            scratch[1024] = found;
            scratch[1025] = 0;
        }
    }
    __syncthreads();
    expert = __builtin_amdgcn_readfirstlane(scratch[1024]);
    if (expert < 0) return 0;
    const int total = __builtin_amdgcn_readfirstlane(count[expert]);
#pragma unroll
    for (int u = 0; u < W4_LIST / W4_THREADS; u++)
        if (mine[u] == expert) list[atomicAdd(&scratch[1025], 1)] = u * W4_THREADS + (int)threadIdx.x;   // (any order: rows do not touch one another)
    __syncthreads();
    return total;
}

// NT tiles of columns (for SwiGLU half of them gate columns, the others the up columns of the same places) times MT tiles of rows.
template <class T, int KIND, int NT, int MT, int OUT, bool GROUPED>
__device__ __forceinline__ void w4_pass(const W4Rows &rows, const W4Matrix &w, int64_t matrix, const int *list, int m0, int total, float *sums, void *out)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t cols = OUT == W4_OUT_SWIGLU ? w.rows / 2 : w.rows;
    constexpr int COLS = OUT == W4_OUT_SWIGLU ? NT / 2 : NT;     // tiles of output columns
    const int64_t n0 = (int64_t)blockIdx.x * (16 * COLS);
    int64_t row[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int64_t n = min(n0 + 16 * (j % COLS) + (lane & 15), cols - 1);
        row[j] = matrix * w.rows + n + (j >= COLS ? cols : 0);
    }
    const T *x[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int at = min(m0 + 16 * mt + (lane & 15), total - 1);
        const int64_t r = GROUPED ? list[at] / rows.x_div : at;
        x[mt] = static_cast<const T *>(rows.x) + r * w.k;
    }
    const int blocks = (w.k + 127) / 128;
    w4_f32x4 acc[NT][MT];
    w4_sums<T, KIND, NT, MT>(w, row, x, blocks * wave / W4_WAVES, blocks * (wave + 1) / W4_WAVES, acc);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) sums[((wave * NT + j) * 4 + r) * 64 + lane] = acc[j][mt][r];
        __syncthreads();
        for (int i = threadIdx.x; i < COLS * 256; i += W4_THREADS) {
            float y[OUT == W4_OUT_SWIGLU ? 2 : 1];
#pragma unroll
            for (int half = 0; half < (OUT == W4_OUT_SWIGLU ? 2 : 1); half++) {
                y[half] = 0.0f;
#pragma unroll
                for (int v = 0; v < W4_WAVES; v++) y[half] += sums[v * NT * 256 + half * COLS * 256 + i];
            }
            const int l = i & 63, m = m0 + 16 * mt + 4 * (l >> 4) + (i >> 6 & 3);
            const int64_t n = n0 + 16 * (i >> 8) + (l & 15);
            if (m >= total || n >= cols) continue;
            const int64_t at = (GROUPED ? list[m] : m) * cols + n;
            if (OUT == W4_OUT_SWIGLU) static_cast<T *>(out)[at] = (T)(y[0] / (1.0f + __expf(-y[0])) * y[1]);
            else if (OUT == W4_OUT_F32) static_cast<float *>(out)[at] = y[0];
            else static_cast<T *>(out)[at] = (T)y[0];
        }
    }
}

template <class T, int KIND, int NT, int MT, int OUT, bool GROUPED>
__global__ __launch_bounds__(W4_THREADS, MT == 1 ? 4 : 2) void w4_tile_kernel(W4Rows rows, W4Matrix w, void *__restrict__ out)
{
    __shared__ float sums[W4_WAVES * NT * 256];
    if constexpr (!GROUPED) {
        const int total = (int)rows.rows;
        for (int m0 = (int)blockIdx.y * (16 * MT); m0 < total; m0 += (int)gridDim.y * (16 * MT)) w4_pass<T, KIND, NT, MT, OUT, false>(rows, w, 0, nullptr, m0, total, sums, out);
    } else {
        __shared__ int list[W4_LIST], scratch[1024 + 2];
        int expert = 0;
        const int total = w4_routes(rows, blockIdx.y, list, scratch, expert);
        for (int m0 = 0; m0 < total;) {
            const int left = total - m0;
            if (MT == 1 || left <= 16) {
                w4_pass<T, KIND, NT, 1, OUT, true>(rows, w, expert, list, m0, total, sums, out);
                m0 += 16;
            } else if (MT == 2 || left <= 32) {
                w4_pass<T, KIND, NT, 2, OUT, true>(rows, w, expert, list, m0, total, sums, out);
                m0 += 32;
            } else {
                w4_pass<T, KIND, NT, MT, OUT, true>(rows, w, expert, list, m0, total, sums, out);
                m0 += 16 * MT;
            }
        }
    }
}

// The launch of one instantiation.
template <class T, int KIND, int NT, int MT, int OUT, bool GROUPED>
int w4_tile_launch(const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    const int64_t cols = OUT == W4_OUT_SWIGLU ? w.rows / 2 : w.rows, per = 16 * (OUT == W4_OUT_SWIGLU ? NT / 2 : NT);
    const int64_t y = GROUPED ? (rows.rows <= 64 ? rows.rows : std::min<int64_t>(rows.num_experts, rows.rows)) : std::min<int64_t>((rows.rows + 16 * MT - 1) / (16 * MT), 65535);
    hipLaunchKernelGGL((w4_tile_kernel<T, KIND, NT, MT, OUT, GROUPED>), dim3((unsigned)((cols + per - 1) / per), (unsigned)y), dim3(W4_THREADS), 0, s, rows, w, out);
    return launch_status("w4_tile_kernel");
}

// The number of columns says how many tiles a workgroup takes: as many as leave all CUs one.
template <class T, int KIND>
int w4_tile_choose(int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    if (out_kind == W4_OUT_PLAIN) {
        const bool two = w.rows >= 16 * 2 * 256;
        if (rows.rows <= 16) return two ? w4_tile_launch<T, KIND, 2, 1, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, 1, 1, W4_OUT_PLAIN, false>(rows, w, out, s);
        if (rows.rows <= 32) return two ? w4_tile_launch<T, KIND, 2, 2, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, 1, 2, W4_OUT_PLAIN, false>(rows, w, out, s);
        return two ? w4_tile_launch<T, KIND, 2, 4, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, 1, 4, W4_OUT_PLAIN, false>(rows, w, out, s);
    }
    const bool few = rows.rows / rows.x_div <= 16;   // no expert has more than the tokens
    if (out_kind == W4_OUT_SWIGLU)
        return few ? w4_tile_launch<T, KIND, 2, 1, W4_OUT_SWIGLU, true>(rows, w, out, s) : w4_tile_launch<T, KIND, 2, 4, W4_OUT_SWIGLU, true>(rows, w, out, s);
    return few ? w4_tile_launch<T, KIND, 2, 1, W4_OUT_F32, true>(rows, w, out, s) : w4_tile_launch<T, KIND, 2, 4, W4_OUT_F32, true>(rows, w, out, s);
}

}  // namespace cch
