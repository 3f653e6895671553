// y = x w^T of a few 16-bit rows with 4-bit weights, on matrix instructions, for K a multiple of 32 and pointers on 16-byte boundaries.
//
// A workgroup has NT tiles of 16 rows of weights and MT tiles of 16 rows of x; its waves split K in blocks of 128, and their sums meet in LDS at the end.  In the
// loop a wave shares nothing: no barrier.  A block's codes (64 bytes of each row) and x (256 bytes of each row) are requested DEPTH blocks ahead in runs that
// the memory system takes whole, four lanes to a row of codes, sixteen to a row of x, and pass through LDS of the wave's own to become operands of
// v_mfma_f32_16x16x32, whose lanes each want another row.  (Loaded by the lanes that need them a block of codes costs the vector cache 64 accesses instead of 16 and x
// as many per instruction: 16 tokens through 2048 x 7168 MXFP4 took 10.0 us.)
//
// A sum over K may be taken in any order, so the instruction's 32 values of K are whichever lie ready.  A code of 4 bits becomes a 16-bit number with one shift and
// one and-or: 16 + q, the code in the leading bits of 1.xxxx * 2^4.  Masks with two nibbles 16 bits apart give pairs (j, j + 4) of a dword's eight elements, and x is
// put in the same order on its way into LDS.  The 16 and the zero point leave by a second instruction with the constant -(16 + z) as its right operand, exactly: in
// fp32 the products of a group sum to what (q - z) gives, and one fused multiply-add per group brings its scale in, which is never rounded into a weight.
// That asks for a group's values to meet in one instruction and no others, which the way the dwords are read from LDS sees to.  MXFP4 with bf16 needs none of
// it: the conversion instruction applies the power of two, exactly.
//
// Bound: the weights' bytes from HBM, below some 100 rows.
#pragma once
#include <algorithm>
#include <atomic>
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
    static constexpr uint32_t MINUS_24 = 0xC1C0C1C0u;
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
    static constexpr uint32_t SIXTEEN = 0x4C004C00u, MASK = 0x03C003C0u, MINUS_24 = 0xCE00CE00u;
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

// Loads of a lane at base + lane offset + wave offset; zeros where the lane's offset is W4_NOWHERE.  No lane's branch, so that any number of them stay in flight.
constexpr uint32_t W4_NOWHERE = 0x80000000u, W4_REACH = 0x7FFFFFFFu;
typedef __amdgpu_buffer_rsrc_t w4_buffer;
__device__ __forceinline__ w4_buffer w4_buffer_at(const void *p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, W4_REACH, 0x00027000); }
__device__ __forceinline__ w4_u32x4 w4_load128(w4_buffer b, uint32_t lane, uint32_t wave) { return __builtin_amdgcn_raw_buffer_load_b128(b, lane, wave, 0); }
__device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T, int KIND, bool ZEROS>
struct W4Tile {
    typedef W4Type<T> Type;
    static constexpr bool MX = KIND == W4_MX, IN_WEIGHT = MX && std::is_same_v<T, __bf16>;   // the scale is in the weight
    static constexpr int GROUP = KIND == W4_I4_G128 ? 128 : KIND == W4_I4_G64 ? 64 : 32;
    static constexpr int GROUPS = 128 / GROUP, PER = 4 / GROUPS;   // of a block; matrix instructions of a group
    static constexpr bool BY_DWORD = GROUPS > 1 && !IN_WEIGHT;     // instruction i takes K = 32 i + 8 (lane / 16) on, otherwise 32 (lane / 16) + 8 i

    // Scale and zero point of a group as one dword: MXFP4 the scale in fp32; otherwise the scale's bits and those of -(16 + z).
    static __device__ __forceinline__ uint32_t param(uint32_t scale, uint32_t zero)
    {
        if (MX) return __float_as_uint(w4_e8m0(scale));
        return ZEROS ? scale | Type::bits(-16.0f - (float)zero) << 16 : scale;
    }
    static __device__ __forceinline__ float scale_of(uint32_t p)
    {
        if (MX) return __uint_as_float(p);
        if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(p << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)p);
    }
    static __device__ __forceinline__ w4_u32x4 zero_of(uint32_t p)
    {
        const uint32_t z = ZEROS ? __builtin_amdgcn_perm(p, p, 0x03020302u) : Type::MINUS_24;
        return (w4_u32x4){z, z, z, z};
    }

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
    // Eight values of x in the order of a dword's operand.
    static __device__ __forceinline__ w4_u32x4 x_order(w4_u32x4 v)
    {
        if (MX) return v;
        return (w4_u32x4){__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                          __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
    }
};

// What a workgroup multiplies: uniform but for x_row.
struct W4Job {
    w4_buffer codes[2];          // from the first row of the tiles on; of SwiGLU's gate and up halves
    const uint8_t *scales[2], *zeros[2];
    w4_buffer x;
    int rows;                    // of weights in either half, up to 16 per tile
};

// Scales and zero points of groups [g0, g0 + count) of all tiles to LDS, `pitch` dwords a row (an odd number: rows on different banks).
template <class T, int KIND, bool ZEROS, int NT, int HALVES>
__device__ __forceinline__ void w4_stage_params(const W4Matrix &w, const W4Job &job, uint32_t *params, int pitch, int g0, int count)
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    typedef uint8_t u8x8 __attribute__((ext_vector_type(8)));
    constexpr int ROWS = 16 * NT / HALVES;
    constexpr int SIZE = Tile::MX ? 1 : 2;
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        uint32_t *to = params + h * ROWS * pitch;
        // groups behind K's last one (a last block that K fills in part) stand for nothing: zeros
        for (int i = threadIdx.x; i < ROWS * pitch; i += W4_THREADS)
            if (i % pitch >= count) to[i] = 0;
        if (count == w.row_groups && aligned16(job.scales[h]) && (!ZEROS || aligned16(job.zeros[h]))) {
            // the rows lie back to back: runs of eight (16 rows have a multiple of 16)
            for (int i = threadIdx.x * 8; i < job.rows * count; i += W4_THREADS * 8) {
                uint32_t s[8], z[8];
                if constexpr (Tile::MX) {
                    const u8x8 v = *reinterpret_cast<const u8x8 *>(job.scales[h] + i);
#pragma unroll
                    for (int u = 0; u < 8; u++) s[u] = v[u];
                } else {
                    const u16x8 v = *reinterpret_cast<const u16x8 *>(job.scales[h] + 2 * i);
#pragma unroll
                    for (int u = 0; u < 8; u++) s[u] = v[u];
                }
                if constexpr (ZEROS) {
                    const u8x8 v = *reinterpret_cast<const u8x8 *>(job.zeros[h] + i);
#pragma unroll
                    for (int u = 0; u < 8; u++) z[u] = v[u];
                }
                int row = i / count, g = i - row * count;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    if (row < job.rows) to[row * pitch + g] = Tile::param(s[u], ZEROS ? z[u] : 0);
                    if (++g == count) {
                        g = 0;
                        row++;
                    }
                }
            }
        } else {
            for (int i = threadIdx.x; i < job.rows * count; i += W4_THREADS) {
                const int row = i / count, g = i - row * count;
                const int64_t at = (int64_t)row * w.row_groups + g0 + g;
                uint32_t s;
                if (SIZE == 1) s = job.scales[h][at];
                else s = reinterpret_cast<const uint16_t *>(job.scales[h])[at];
                to[row * pitch + g] = Tile::param(s, ZEROS ? job.zeros[h][at] : 0);
            }
        }
    }
}

// Bytes of LDS of one wave: a block's x and codes; and in their place its sums at the end.
template <int NT, int MT, int XR>
constexpr int w4_wave_bytes()
{
    return std::max(XR * 1024 + NT * 1024, NT * MT * 1024);
}

// The wave's sums over all its blocks.  XR: four rows of x each are loaded (MT = 1: as few as there are).
template <class T, int KIND, bool ZEROS, int NT, int MT, int XR, int HALVES>
__device__ __forceinline__ void w4_sums(const W4Matrix &w, const W4Job &job, const uint32_t (&x_row)[XR], uint32_t *params, int pitch, int chunk, uint8_t *mine,
                                        w4_f32x4 (&acc)[NT][MT])
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    static_assert(XR <= 4 * MT && (MT == 1 || XR == 4 * MT));
    constexpr int COLS = NT / HALVES, STAGE = NT + XR;
    constexpr int DEPTH = STAGE <= 2 ? 5 : STAGE <= 3 ? 3 : STAGE <= 12 ? 2 : 1;   // blocks in flight
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n = lane & 15, g = lane >> 4, last = (w.k - 1) / 128;
    uint8_t *const x_lds = mine, *const w_lds = mine + XR * 1024;
    // this lane's loads of a block: 16 bytes of codes of row lane / 4, of x of row lane / 16; of the last block perhaps none
    uint32_t code_at[NT], code_last[NT], x_last[XR];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int row = 16 * (j % COLS) + (lane >> 2);
        code_at[j] = row < job.rows ? row * w.row_bytes + 16 * (lane & 3) : W4_NOWHERE;
        code_last[j] = last * 128 + 32 * (lane & 3) < w.k ? code_at[j] : W4_NOWHERE;
    }
#pragma unroll
    for (int u = 0; u < XR; u++) x_last[u] = last * 128 + 8 * (lane & 15) < w.k ? x_row[u] : W4_NOWHERE;
    // where they go: 16-byte pieces of a row exchanged so that lanes of different rows meet different banks
    const int code_to = (lane >> 2) * 64 + ((lane & 3) ^ (lane >> 4)) * 16;
    int x_to[XR];
#pragma unroll
    for (int u = 0; u < XR; u++) x_to[u] = (4 * u + g) * 256 + ((lane & 15) ^ ((4 * u + g) & 15)) * 16;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++) acc[j][mt] = (w4_f32x4){0, 0, 0, 0};

    struct Stage {
        w4_u32x4 q[NT], x[XR];
    } stage[DEPTH];
    auto fetch = [&](Stage &s, int block, int end) {
        const bool none = block >= end, part = block == last;
        const int at = none ? 0 : block;
#pragma unroll
        for (int j = 0; j < NT; j++) s.q[j] = w4_load128(job.codes[j / COLS], none ? W4_NOWHERE : part ? code_last[j] : code_at[j], at * 64);
#pragma unroll
        for (int u = 0; u < XR; u++) s.x[u] = w4_load128(job.x, none ? W4_NOWHERE : part ? x_last[u] : x_row[u], at * 256);
    };
    const int blocks = last + 1, groups = Tile::GROUPS;
    for (int b0 = 0; b0 < blocks; b0 += chunk) {
        const int here = min(chunk, blocks - b0);
        const int begin = b0 + here * wave / W4_WAVES, end = b0 + here * (wave + 1) / W4_WAVES;
#pragma unroll
        for (int d = 0; d < DEPTH; d++) fetch(stage[d], begin + d, end);
        if (b0 > 0) __syncthreads();
        w4_stage_params<T, KIND, ZEROS, NT, HALVES>(w, job, params, pitch, b0 * groups, min(here * groups, w.row_groups - b0 * groups));
        __syncthreads();
        for (int block = begin; block < end; block += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                Stage &s = stage[d];
                if (DEPTH > 1 && block + d >= end) break;
#pragma unroll
                for (int j = 0; j < NT; j++) *reinterpret_cast<w4_u32x4 *>(w_lds + j * 1024 + code_to) = s.q[j];
#pragma unroll
                for (int u = 0; u < XR; u++) *reinterpret_cast<w4_u32x4 *>(x_lds + x_to[u]) = Tile::x_order(s.x[u]);
                fetch(s, block + d + DEPTH, end);
                // (a wave's LDS accesses execute in program order; the fences keep the compiler to it)
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                w4_u32x4 q[NT];
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if constexpr (Tile::BY_DWORD) {
#pragma unroll
                        for (int i = 0; i < 4; i++) q[j][i] = *reinterpret_cast<const uint32_t *>(w_lds + j * 1024 + n * 64 + (i ^ (n >> 2)) * 16 + 4 * g);
                    } else {
                        q[j] = *reinterpret_cast<const w4_u32x4 *>(w_lds + j * 1024 + n * 64 + (g ^ (n >> 2)) * 16);
                    }
                }
                const uint32_t *const p = params + n * pitch + (block + d - b0) * groups;
                w4_f32x4 part[NT][MT];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (STAGE > 4) __builtin_amdgcn_sched_barrier(0);
                    w4_u32x4 x[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const int row = MT == 1 ? n & (4 * XR - 1) : 16 * mt + n, piece = Tile::BY_DWORD ? 4 * i + g : 4 * g + i;
                        x[mt] = *reinterpret_cast<const w4_u32x4 *>(x_lds + row * 256 + (piece ^ (row & 15)) * 16);
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        if constexpr (Tile::IN_WEIGHT) {
                            const w4_u32x4 b = Tile::operand(q[j][i], __uint_as_float(p[j * 16 * pitch + g]));
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) acc[j][mt] = Tile::Type::mfma(x[mt], b, acc[j][mt]);
                        } else {
                            const w4_u32x4 b = Tile::operand(q[j][i], 1.0f);
                            const uint32_t pj = p[j * 16 * pitch + i / Tile::PER];
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                if (i % Tile::PER == 0) part[j][mt] = (w4_f32x4){0, 0, 0, 0};
                                if (!Tile::MX) part[j][mt] = Tile::Type::mfma(x[mt], Tile::zero_of(pj), part[j][mt]);
                                part[j][mt] = Tile::Type::mfma(x[mt], b, part[j][mt]);
                                if (i % Tile::PER == Tile::PER - 1) {
#pragma unroll
                                    for (int r = 0; r < 4; r++) acc[j][mt][r] += Tile::scale_of(pj) * part[j][mt][r];
                                }
                            }
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_sched_barrier(0);   // (a block's operands are not made before its turn: registers)
            }
        }
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
template <class T, int KIND, bool ZEROS, int NT, int MT, int XR, int OUT, bool GROUPED>
__device__ __forceinline__ void w4_pass(const W4Rows &rows, const W4Matrix &w, int64_t matrix, const int *list, int m0, int total, int pitch, int chunk, uint8_t *lds,
                                        void *out)
{
    constexpr int HALVES = OUT == W4_OUT_SWIGLU ? 2 : 1, COLS = NT / HALVES, WAVE_BYTES = w4_wave_bytes<NT, MT, XR>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t cols = w.rows / HALVES, n0 = (int64_t)blockIdx.x * (16 * COLS);
    W4Job job;
    job.rows = (int)min((int64_t)(16 * COLS), cols - n0);
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        const int64_t first = matrix * w.rows + n0 + h * cols;
        job.codes[h] = w4_buffer_at(w.codes + first * w.row_bytes);
        job.scales[h] = static_cast<const uint8_t *>(w.scales) + first * w.row_groups * (KIND == W4_MX ? 1 : 2);
        job.zeros[h] = ZEROS ? w.zeros + first * w.row_groups : nullptr;
    }
    uint32_t x_row[XR];
#pragma unroll
    for (int u = 0; u < XR; u++) {
        const int at = min(m0 + 4 * u + (lane >> 4), total - 1);
        x_row[u] = (uint32_t)(GROUPED ? list[at] / rows.x_div : at - m0) * (uint32_t)(2 * w.k) + 16 * (lane & 15);
    }
    job.x = w4_buffer_at(static_cast<const T *>(rows.x) + (GROUPED ? 0 : (int64_t)m0 * w.k));
    uint8_t *const waves = lds, *const mine = waves + wave * WAVE_BYTES;
    uint32_t *const params = reinterpret_cast<uint32_t *>(lds + W4_WAVES * WAVE_BYTES);
    w4_f32x4 acc[NT][MT];
    w4_sums<T, KIND, ZEROS, NT, MT, XR, HALVES>(w, job, x_row, params, pitch, chunk, mine, acc);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) reinterpret_cast<float *>(mine)[((mt * NT + j) * 4 + r) * 64 + lane] = acc[j][mt][r];
    __syncthreads();
    // the sums of one row and column of the tiles, over the waves in their order
    constexpr int LANES = MT == 1 ? 16 * XR : 64;                // that hold rows there are
    for (int i = threadIdx.x; i < MT * COLS * 4 * LANES; i += W4_THREADS) {
        const int l = i % LANES, r = i / LANES & 3, j = i / (4 * LANES) % COLS, mt = i / (4 * LANES * COLS);
        const int m = m0 + 16 * mt + 4 * (l >> 4) + r;
        const int64_t n = n0 + 16 * j + (l & 15);
        if (m >= total || n >= cols) continue;
        float y[HALVES];
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            y[h] = 0.0f;
#pragma unroll
            for (int v = 0; v < W4_WAVES; v++) y[h] += reinterpret_cast<const float *>(waves + v * WAVE_BYTES)[((mt * NT + j + h * COLS) * 4 + r) * 64 + l];
        }
        const int64_t at = (GROUPED ? list[m] : m) * cols + n;
        if (OUT == W4_OUT_SWIGLU) static_cast<T *>(out)[at] = (T)(y[0] / (1.0f + __expf(-y[0])) * y[1]);
        else if (OUT == W4_OUT_F32) static_cast<float *>(out)[at] = y[0];
        else static_cast<T *>(out)[at] = (T)y[0];
    }
}

template <class T, int KIND, bool ZEROS, int NT, int MT, int XR, int OUT, bool GROUPED>
__global__ __launch_bounds__(W4_THREADS, MT == 1 ? 4 : 2) void w4_tile_kernel(W4Rows rows, W4Matrix w, int pitch, int chunk, void *__restrict__ out)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t w4_lds[];
    if constexpr (!GROUPED) {
        const int total = (int)rows.rows;
        for (int m0 = (int)blockIdx.y * (16 * MT); m0 < total; m0 += (int)gridDim.y * (16 * MT)) {
            w4_pass<T, KIND, ZEROS, NT, MT, XR, OUT, false>(rows, w, 0, nullptr, m0, total, pitch, chunk, w4_lds, out);
            __syncthreads();
        }
    } else {
        __shared__ int list[W4_LIST], scratch[1024 + 2];
        int expert = 0;
        const int total = w4_routes(rows, blockIdx.y, list, scratch, expert);
        for (int m0 = 0; m0 < total;) {
            if (MT == 1 || total - m0 <= 16) {
                constexpr int X = MT == 1 ? XR : 4;
                w4_pass<T, KIND, ZEROS, NT, 1, X, OUT, true>(rows, w, expert, list, m0, total, pitch, chunk, w4_lds, out);
                m0 += 4 * X;
            } else {
                w4_pass<T, KIND, ZEROS, NT, MT, XR, OUT, true>(rows, w, expert, list, m0, total, pitch, chunk, w4_lds, out);
                m0 += 16 * MT;
            }
            __syncthreads();
        }
    }
}

// The launch of one instantiation.
template <class T, int KIND, bool ZEROS, int NT, int MT, int XR, int OUT, bool GROUPED>
int w4_tile_launch(const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    auto kern = w4_tile_kernel<T, KIND, ZEROS, NT, MT, XR, OUT, GROUPED>;
    constexpr int HALVES = OUT == W4_OUT_SWIGLU ? 2 : 1, WAVES_BYTES = W4_WAVES * w4_wave_bytes<NT, MT, XR>();
    constexpr int PARAMS = std::min(32 * 1024, 160 * 1024 - WAVES_BYTES - (GROUPED ? 4 * (W4_LIST + 1024 + 2) : 0));   // bytes of LDS for scales and zero points, at most
    // blocks whose scales are in LDS at a time, evenly
    const int blocks = (w.k + 127) / 128, most = (PARAMS / (16 * NT * 4) - 1) / Tile::GROUPS, chunks = (blocks + most - 1) / most;
    const int chunk = (blocks + chunks - 1) / chunks, pitch = (chunk * Tile::GROUPS) | 1, lds = WAVES_BYTES + 16 * NT * pitch * 4;
    if (WAVES_BYTES + PARAMS > 48 * 1024) {
        // set once per device and kernel; setting it twice from two threads is harmless
        static std::atomic<uint64_t> attr_set{0};
        int dev = 0;
        CCH_HIP(hipGetDevice(&dev));
        const uint64_t dev_bit = (uint64_t)1 << (dev & 63);
        if (dev >= 64 || !(attr_set.load(std::memory_order_acquire) & dev_bit)) {
            CCH_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, WAVES_BYTES + PARAMS));
            attr_set.fetch_or(dev_bit, std::memory_order_release);
        }
    }
    const int64_t cols = w.rows / HALVES, per = 16 * (NT / HALVES);
    const int64_t y = GROUPED ? (rows.rows <= 64 ? rows.rows : std::min<int64_t>(rows.num_experts, rows.rows)) : std::min<int64_t>((rows.rows + 16 * MT - 1) / (16 * MT), 65535);
    hipLaunchKernelGGL(kern, dim3((unsigned)((cols + per - 1) / per), (unsigned)y), dim3(W4_THREADS), lds, s, rows, w, pitch, chunk, out);
    return launch_status("w4_tile_kernel");
}

// The number of columns says how many tiles a workgroup takes: as many as leave all CUs one.
template <class T, int KIND, bool ZEROS>
int w4_tile_choose(int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    if (out_kind == W4_OUT_PLAIN) {
        const bool two = w.rows >= 16 * 2 * 256;
        if (rows.rows <= 4)
            return two ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 1, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, ZEROS, 1, 1, 1, W4_OUT_PLAIN, false>(rows, w, out, s);
        if (rows.rows <= 16)
            return two ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 4, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, ZEROS, 1, 1, 4, W4_OUT_PLAIN, false>(rows, w, out, s);
        if (rows.rows <= 32)
            return two ? w4_tile_launch<T, KIND, ZEROS, 2, 2, 8, W4_OUT_PLAIN, false>(rows, w, out, s) : w4_tile_launch<T, KIND, ZEROS, 1, 2, 8, W4_OUT_PLAIN, false>(rows, w, out, s);
        return w4_tile_launch<T, KIND, ZEROS, 2, 4, 16, W4_OUT_PLAIN, false>(rows, w, out, s);
    }
    const int64_t tokens = rows.rows / rows.top_k;   // no expert has more of them
    if (out_kind == W4_OUT_SWIGLU)
        return tokens <= 4    ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 1, W4_OUT_SWIGLU, true>(rows, w, out, s)
               : tokens <= 16 ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 4, W4_OUT_SWIGLU, true>(rows, w, out, s)
                              : w4_tile_launch<T, KIND, ZEROS, 2, 2, 8, W4_OUT_SWIGLU, true>(rows, w, out, s);
    return tokens <= 4    ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 1, W4_OUT_F32, true>(rows, w, out, s)
           : tokens <= 16 ? w4_tile_launch<T, KIND, ZEROS, 2, 1, 4, W4_OUT_F32, true>(rows, w, out, s)
                          : w4_tile_launch<T, KIND, ZEROS, 2, 2, 8, W4_OUT_F32, true>(rows, w, out, s);
}

}  // namespace cch
