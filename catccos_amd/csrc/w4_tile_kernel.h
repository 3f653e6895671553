// y = x w^T of few 16-bit rows with 4-bit weights, on matrix instructions, for K a multiple of 32 and pointers on 16-byte boundaries.
//
// A workgroup has WN * NT tiles of 16 rows of weights and MT tiles of 16 rows of x, and walks K in blocks of 128.  Its waves are WN columns, NT tiles each, times
// WK parts of K, whose sums meet in LDS at the end.  A block's codes (64 bytes of each row, a wave's own) and x (256 bytes of each row, shared by a part's WN
// waves) come from memory straight into rings of two blocks in LDS, in runs that the memory system takes whole: four lanes to a row of codes, sixteen to a row of x.
// (Loaded by the lanes that need them, every lane of 16 another row, a block of codes costs the vector cache 64 accesses instead of 16, and x as many per instruction;
// through registers the loop needs its blocks unrolled, and its code is what a small launch waits for.)  One barrier a block, none where WN is 1.
//
// A sum over K may be taken in any order, so a matrix instruction's 32 values of K are whichever lie ready.  A code of 4 bits becomes a 16-bit number with one shift and
// one and-or: 16 + q, the code in the leading bits of 1.xxxx * 2^4.  Masks with two nibbles 16 bits apart give pairs (j, j + 4) of a dword's eight elements, and x is
// put in the same order.  The 16 and the zero point leave by a second instruction with the constant -(16 + z) as its right operand, and one fused multiply-add
// per group brings its scale in, which is never rounded into a weight.  Exact in this are the 16-bit operands.  The two halves of a group's sum are fp32 and round at their own size before
// they cancel: the error is that of a sum of |x| (31 + |q - z|) |scale|, for z up to 15 at most 31 / |q - z| + 1 times that of the products themselves, some bits more where a group's x
// have one sign.  (4096 x 7168: 2.4e-5 between this and (q - z) scale in fp32, of results whose rounding to bf16 is 1.7e-3.)  And they have to stay finite: a group of bf16 x whose sum of
// |x| passes 2^128 / 31 (about 1.1e37; 2^128 / 256 with zero points up to 240) gives NaN, as an infinite x does.
// That asks for a group's values to meet in one instruction and no others, which the way the dwords are read from LDS sees to.  MXFP4 with bf16 needs none of
// it: the conversion instruction applies the power of two, exactly.
//
// The sums and the groups' scales stay in fp32; rounded to 16 bits are the results alone.  Zero points that -(16 + z) holds exactly, up to 240 in bf16.
//
// Bound, one row: the weights' bytes, after a launch, two waits for memory and the sum over K's parts: 4096 x 7168 in 5.9 us, 2.5 TB/s (reading alone 3.6, an empty launch
// 2.4), 32768 x 7168 in 22 to 26 us, 4.6 TB/s.  61 rows x 32768 x 7168, groups of 64 with zero points: 61 to 71 us by card, 1.7 TB/s and 0.41 PFLOP/s at the latter.  A tile of
// weights and 64 rows of x take, per block of K, about 130 vector instructions of 4 clocks (conversion, scales, x and addresses), 32 matrix instructions of 16 and 18 KB from LDS, 16 of
// them x: 24, 24 and 27 us for all tiles at 2.4 GHz and 128 bytes a clock and CU, and the launch takes nearly their sum.  16 waves overlap them better than 8 (77 us), whatever order the
// compiler is asked for; two tiles of columns to a wave read x half as often but leave eight waves.
#pragma once
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gemm_device.h"
#include "w4_decode.h"

namespace cch {

__device__ __forceinline__ uint32_t w4_lds_address(const uint8_t *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p; }

typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));


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

// A lane's offset that no buffer reaches: zeros arrive.
constexpr uint32_t W4_NOWHERE = 0x80000000u, W4_REACH = 0x7FFFFFFFu;
__device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T, int KIND, bool ZEROS>
struct W4Tile {
    typedef W4Type<T> Type;
    static constexpr bool MX = KIND == W4_MX, IN_WEIGHT = MX && std::is_same_v<T, __bf16>;   // the scale is in the weight
    static constexpr int GROUP = KIND == W4_I4_G128 ? 128 : KIND == W4_I4_G64 ? 64 : 32;
    static constexpr int GROUPS = 128 / GROUP, PER = 4 / GROUPS;   // of a block; matrix instructions of a group
    static constexpr bool BY_DWORD = GROUPS > 1 && !IN_WEIGHT;     // instruction i takes K = 32 i + 8 (lane / 16) on, otherwise 32 (lane / 16) + 8 i

    // A group's scale, and with zero points the bits of -(16 + z) behind it, as LDS holds them.
    static constexpr int PARAM = MX ? 1 : ZEROS ? 4 : 2;
    static __device__ __forceinline__ void put_param(uint8_t *to, uint32_t scale, uint32_t zero)
    {
        if (MX) *to = (uint8_t)scale;
        else if (ZEROS) *reinterpret_cast<uint32_t *>(to) = scale | Type::bits(-16.0f - (float)zero) << 16;
        else *reinterpret_cast<uint16_t *>(to) = (uint16_t)scale;
    }
    static __device__ __forceinline__ uint32_t get_param(const uint8_t *from)
    {
        return MX ? *from : ZEROS ? *reinterpret_cast<const uint32_t *>(from) : *reinterpret_cast<const uint16_t *>(from);
    }
    static __device__ __forceinline__ float scale_of(uint32_t p)
    {
        if (MX) return w4_e8m0(p);
        if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(p << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)p);
    }
    static __device__ __forceinline__ w4_u32x4 zero_of(uint32_t p)
    {
        const uint32_t z = ZEROS ? __builtin_amdgcn_perm(p, p, 0x03020302u) : Type::MINUS_24;
        return (w4_u32x4){z, z, z, z};
    }

    static __device__ __forceinline__ w4_u32x4 operand(uint32_t q, float scale, uint32_t mask, uint32_t sixteen)
    {
        w4_u32x4 r;
        if (MX) {
            r[0] = Type::template fp4<0>(q, scale);
            r[1] = Type::template fp4<1>(q, scale);
            r[2] = Type::template fp4<2>(q, scale);
            r[3] = Type::template fp4<3>(q, scale);
        } else {
            constexpr int S = Type::SHIFT;
            r[0] = (q << S & mask) | sixteen;
            r[1] = ((S >= 4 ? q << (S >= 4 ? S - 4 : 0) : q >> (S >= 4 ? 0 : 4 - S)) & mask) | sixteen;
            r[2] = (q >> (8 - S) & mask) | sixteen;
            r[3] = (q >> (12 - S) & mask) | sixteen;
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

// What a workgroup multiplies, from the first row of its tiles on; two halves for SwiGLU's gate and up columns.
struct W4Job {
    const uint8_t *codes[2], *scales[2], *zeros[2];
    const void *x;
    int rows;                    // of weights in either half, up to 16 per tile
};

// Bytes of LDS: a wave's codes and a part's x of one block; a row of scales (an odd number of dwords: rows on different banks).
constexpr int W4_CODES = 1024, W4_X4 = 1024;   // of a tile, of four rows of x
__host__ __device__ inline int w4_param_pitch(int groups, int param) { return ((groups * param + 3) / 4 | 1) * 4; }

// What is exchanged: piece p of a row of codes lies at p ^ turn(row / 4), of x at p ^ x_turn(row).  A 16-byte read serves 16 lanes at a time, and
// these are lanes 0-3, 12-15, 20-23, 24-27 and so on: rows of fours from two neighbouring lane groups, which have to differ.
__device__ __forceinline__ int w4_turn(int fours) { return -fours & 3; }
__device__ __forceinline__ int w4_x_turn(int row) { return (row & 3) | w4_turn(row >> 2) << 2; }

// Scales and zero points of groups [g0, g0 + count) of all tiles to LDS, eight at a time where they lie back to back on 16-byte boundaries.  One row by 32768, K = 7168: 26.0 /
// 29.4 / 39.9 / 27.6 us (groups of 128, of 64 and of 32 with zero points, MXFP4), one at a time 27.2 / 33.1 / 52.5 / 28.5; by 4096, K = 2048, 4.2 / 3.9 / 4.1 / 3.4 against 3.6 / 3.5 /
// 3.9 / 3.5.
template <class T, int KIND, bool ZEROS, int TILES, int HALVES, int THREADS>
__device__ __forceinline__ void w4_stage_params(const int row_groups, const W4Job &job, uint8_t *params, int pitch, int g0, int count)
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    typedef uint8_t u8x8 __attribute__((ext_vector_type(8)));
    constexpr int ROWS = 16 * TILES / HALVES, SIZE = Tile::MX ? 1 : 2, P = Tile::PARAM;
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        uint8_t *to = params + h * ROWS * pitch;
        if (count == row_groups && aligned16(job.scales[h]) && (!ZEROS || aligned16(job.zeros[h]))) {
            // the rows lie back to back: runs of eight (a last one may end behind the last row, in the next one's)
            const int total = job.rows * count;
            for (int i = threadIdx.x * 8; i < total; i += THREADS * 8) {
                uint32_t s[8], z[8];
                if (i + 8 <= total) {
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
                } else {
                    for (int u = 0; u < 8; u++) {
                        const int at = min(i + u, total - 1);
                        s[u] = SIZE == 1 ? job.scales[h][at] : reinterpret_cast<const uint16_t *>(job.scales[h])[at];
                        z[u] = ZEROS ? job.zeros[h][at] : 0;
                    }
                }
                int row = i / count, g = i - row * count;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    if (row < job.rows) Tile::put_param(to + row * pitch + g * P, s[u], ZEROS ? z[u] : 0);
                    if (++g == count) {
                        g = 0;
                        row++;
                    }
                }
            }
        } else {
            for (int i = threadIdx.x; i < job.rows * count; i += THREADS) {
                const int row = i / count, g = i - row * count;
                const int64_t at = (int64_t)row * row_groups + g0 + g;
                const uint32_t s = SIZE == 1 ? job.scales[h][at] : reinterpret_cast<const uint16_t *>(job.scales[h])[at];
                Tile::put_param(to + row * pitch + g * P, s, ZEROS ? job.zeros[h][at] : 0);
            }
        }
    }
}

// The shape of a workgroup: NT tiles of weights to a wave, MT tiles of x, WN waves by columns, WK by parts of K.  XR: four rows of x each are loaded (MT = 1: as few as there are).
template <int NT_, int MT_, int XR_, int WN_, int WK_>
struct W4Shape {
    static constexpr int NT = NT_, MT = MT_, XR = XR_, WN = WN_, WK = WK_, W = WN * WK, THREADS = 64 * W, TILES = WN * NT;
    static constexpr int XU = XR / WN;                                       // x loads of a wave and block
    static constexpr int X_RING = 2 * XR * W4_X4, CODE_RING = 2 * NT * W4_CODES;
    static constexpr int RINGS = WK * X_RING + W * CODE_RING, SUMS = W * NT * MT * 1024;
    static constexpr int FIXED = RINGS > SUMS ? RINGS : SUMS;                // LDS in front of the scales
    static_assert(XR % WN == 0 && XR <= 4 * MT && (MT == 1 || XR == 4 * MT));
};

// The wave's sums of its tiles over its part of K.
template <class T, int KIND, bool ZEROS, class S, int HALVES>
__device__ __forceinline__ void w4_sums(const W4Matrix &w, const W4Job &job, const uint32_t (&x_row)[S::XU], int pitch, int chunk, w4_f32x4 (&acc)[S::NT][S::MT])
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    constexpr int NT = S::NT, MT = S::MT, XU = S::XU, COLS = NT / HALVES;
    // x's order: by the wave that loaded it, in LDS; or, where no wave shares it, with the operands
    constexpr bool ORDER_IN_LDS = !Tile::MX && S::WN > 1, ORDER_LATE = !Tile::MX && !ORDER_IN_LDS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wave % S::WN, wk = wave / S::WN, n = lane & 15, g = lane >> 4, last = (w.k - 1) / 128, f = w4_turn(n >> 2);
    uint8_t *const params = smem + S::FIXED, *const x_ring = smem + wk * S::X_RING, *const code_ring = smem + S::WK * S::X_RING + wave * S::CODE_RING;
    const uint32_t x_lds = w4_lds_address(x_ring) + wn * XU * W4_X4, code_lds = w4_lds_address(code_ring);
    // this lane's loads of a block: 16 bytes of codes of row lane / 4, of x of row lane / 16, pieces of a row exchanged so that an operand's lanes, of different
    // rows, meet different banks; of the last block perhaps none
    const int code_piece = (lane & 3) ^ w4_turn(lane >> 4), tile0 = wn * COLS;
    const uint32_t code_at = (lane >> 2) * w.row_bytes + 16 * code_piece;
    const bool code_in_last = last * 128 + 32 * code_piece < w.k;
    bool code_row[COLS], x_in_last[XU];
    uint32_t x_at[XU];
#pragma unroll
    for (int j = 0; j < COLS; j++) code_row[j] = 16 * (tile0 + j) + (lane >> 2) < job.rows;
#pragma unroll
    for (int u = 0; u < XU; u++) {
        const int piece = (lane & 15) ^ w4_x_turn(4 * (wn * XU + u) + g);
        x_at[u] = x_row[u] + 16 * piece;
        x_in_last[u] = last * 128 + 8 * piece < w.k;
    }
    const int x_n = MT == 1 ? n & (4 * S::XR - 1) : n;
    const uint32_t code_from = n * 64 + (Tile::BY_DWORD ? f * 16 + 4 * g : (g ^ f) * 16), x_from = x_n * 256 + ((Tile::BY_DWORD ? g : 4 * g) ^ w4_x_turn(x_n)) * 16;
    const Rsrc codes[2] = {make_rsrc(job.codes[0], W4_REACH), make_rsrc(job.codes[HALVES - 1], W4_REACH)}, xs = make_rsrc(job.x, W4_REACH);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++) acc[j][mt] = (w4_f32x4){0, 0, 0, 0};

    uint32_t mask = Tile::Type::MASK, sixteen = Tile::Type::SIXTEEN;
    asm volatile("" : "+s"(mask), "+v"(sixteen));               // (in registers: one instruction takes both, none takes two literals)

    auto request = [&](int block, int end, int slot) {
        const bool none = block >= end, part = block == last;
        const uint32_t at = none ? 0 : block;
#pragma unroll
        for (int j = 0; j < NT; j++)
            load16_to_lds(codes[j / COLS], none || !code_row[j % COLS] || (part && !code_in_last) ? W4_NOWHERE : code_at, at * 64 + 16 * (tile0 + j % COLS) * w.row_bytes,
                          code_lds + (slot * NT + j) * W4_CODES);
#pragma unroll
        for (int u = 0; u < XU; u++)
            load16_to_lds(xs, none || (part && !x_in_last[u]) ? W4_NOWHERE : x_at[u], at * 256, x_lds + (slot * S::XR + u) * W4_X4);
    };
    auto order = [&](int slot) {
#pragma unroll
        for (int u = 0; u < XU; u++) {
            w4_u32x4 *p = reinterpret_cast<w4_u32x4 *>(x_ring + (slot * S::XR + wn * XU + u) * W4_X4 + 16 * lane);
            *p = Tile::x_order(*p);
        }
    };
    // What a block's products take from LDS; read while the block before is multiplied.
    struct Operands {
        w4_u32x4 q[NT], x[MT][4];
        uint32_t p[NT][Tile::IN_WEIGHT ? 1 : Tile::GROUPS];
    };
    auto read = [&](Operands &o, int slot, int first, int own) {       // first: group of the block in the scales there are; own: end of this part's
        const uint8_t *const c = code_ring + slot * NT * W4_CODES, *const xb = x_ring + slot * S::XR * W4_X4;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if constexpr (Tile::BY_DWORD) {
#pragma unroll
                for (int i = 0; i < 4; i++) o.q[j][i] = *reinterpret_cast<const uint32_t *>(c + j * W4_CODES + (code_from ^ (16 * i)));
            } else {
                o.q[j] = *reinterpret_cast<const w4_u32x4 *>(c + j * W4_CODES + code_from);
            }
            // Behind the part's last group, where codes and x read as zeros, lie another part's scale, or the byte that pads MXFP4's rows to pairs: whatever it is (NaN or an
            // infinity times zero is NaN), none is taken.
            const int row = (j / COLS) * (16 * S::WN * COLS) + 16 * (tile0 + j % COLS) + n;
            if constexpr (Tile::IN_WEIGHT) {
                o.p[j][0] = first + g < own ? Tile::get_param(params + row * pitch + (first + g) * Tile::PARAM) : 0;
            } else {
#pragma unroll
                for (int i = 0; i < Tile::GROUPS; i++) o.p[j][i] = first + i < own ? Tile::get_param(params + row * pitch + (first + i) * Tile::PARAM) : 0;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o.x[mt][i] = *reinterpret_cast<const w4_u32x4 *>(xb + mt * 4 * W4_X4 + (x_from ^ ((Tile::BY_DWORD ? 64 : 16) * i)));
    };
    auto multiply = [&](Operands &o) {
        w4_f32x4 part[NT][MT];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (ORDER_LATE) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) o.x[mt][i] = Tile::x_order(o.x[mt][i]);
            }
#pragma unroll
            for (int j = 0; j < NT; j++) {
                if constexpr (Tile::IN_WEIGHT) {
                    const w4_u32x4 b = Tile::operand(o.q[j][i], Tile::scale_of(o.p[j][0]), 0, 0);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) acc[j][mt] = Tile::Type::mfma(o.x[mt][i], b, acc[j][mt]);
                } else {
                    const w4_u32x4 b = Tile::operand(o.q[j][i], 1.0f, mask, sixteen);
                    const uint32_t pj = o.p[j][i / Tile::PER];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (i % Tile::PER == 0) part[j][mt] = (w4_f32x4){0, 0, 0, 0};
                        if (!Tile::MX) part[j][mt] = Tile::Type::mfma(o.x[mt][i], Tile::zero_of(pj), part[j][mt]);
                        part[j][mt] = Tile::Type::mfma(o.x[mt][i], b, part[j][mt]);
                        if (i % Tile::PER == Tile::PER - 1) {
#pragma unroll
                            for (int r = 0; r < 4; r++) acc[j][mt][r] += Tile::scale_of(pj) * part[j][mt][r];
                        }
                    }
                }
            }
        }
    };
    const int blocks = last + 1;
    for (int b0 = 0; b0 < blocks; b0 += chunk) {
        const int here = min(chunk, blocks - b0), begin = b0 + here * wk / S::WK, end = b0 + here * (wk + 1) / S::WK, steps = (here + S::WK - 1) / S::WK;
        if (b0 > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < 2; d++) request(begin + d, end, d);
        int row_groups = w.row_groups;
        asm volatile("" : "+s"(row_groups));   // (nothing of what follows is worked out in front of the requests)
        const int g0 = b0 * Tile::GROUPS, count = min(here * Tile::GROUPS, row_groups - g0);
        w4_stage_params<T, KIND, ZEROS, S::TILES, HALVES, S::THREADS>(row_groups, job, params, pitch, g0, count);
        CCH_WAIT_VM(0);                // (the compiler knows of the loads above, not of the requests: with some of its own open it would wait for all in the loop)
        asm volatile("" ::: "memory");
        if (ORDER_IN_LDS) order(0);
        CCH_WAIT_LGKM0();
        CCH_BARRIER();
        Operands a, b;
        const int group0 = (begin - b0) * Tile::GROUPS, own = min(end * Tile::GROUPS, (w.k + Tile::GROUP - 1) / Tile::GROUP) - g0;
        read(a, 0, group0, own);
        // ring slot `SLOT` holds block `step`, whose operands are read or on their way; the other one the next
        auto advance = [&](auto which, Operands &o, int step) {
            constexpr int SLOT = decltype(which)::value;
            CCH_WAIT_VM(0);
            asm volatile("" ::: "memory");
            if (ORDER_IN_LDS) order(1 - SLOT);
            CCH_WAIT_LGKM0();          // (and this wave has the operands of block `step`)
            if (S::WN > 1) CCH_BARRIER();
            request(begin + step + 2, end, SLOT);
            read(o, 1 - SLOT, group0 + (step + 1) * Tile::GROUPS, own);
        };
        for (int step = 0; step < steps; step += 2) {
            advance(IC<0>{}, b, step);
            multiply(a);
            if (step + 1 == steps) break;
            advance(IC<1>{}, a, step + 1);
            multiply(b);
        }
        CCH_WAIT_VM(0);                // (requests of no block write zeros)
        CCH_WAIT_LGKM0();
    }
}

// Which matrix, and which rows of x: workgroup column `slot` of the grid takes the slot-th expert that some route names (up to 64 routes: the expert of route
// `slot`, if no earlier one names it; one look at all of them, where counting takes four barriers: one token's two products with 8 of 64 experts 6.0 + 4.3 us, counted 6.7 +
// 5.0).  Returns the number of its routes, their numbers in `list`; 0: nothing to do.  (Every workgroup sorts for itself: a launch that did it for all would take longer.)
template <int W>
__device__ __forceinline__ int w4_routes(const W4Rows &rows, int slot, int *list, int *scratch, int &expert)
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
    for (int e = threadIdx.x; e < 1024; e += 64 * W) count[e] = 0;
    __syncthreads();
    int mine[W4_LIST / (64 * W)];
#pragma unroll
    for (int u = 0; u < W4_LIST / (64 * W); u++) {
        const int r = u * (64 * W) + (int)threadIdx.x;
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
    for (int u = 0; u < W4_LIST / (64 * W); u++)
        if (mine[u] == expert) list[atomicAdd(&scratch[1025], 1)] = u * (64 * W) + (int)threadIdx.x;   // (any order: rows do not touch one another)
    __syncthreads();
    return total;
}

// The workgroup's tiles of columns (for SwiGLU half of them gate columns, the others the up columns of the same places) times MT tiles of rows.
template <class T, int KIND, bool ZEROS, class S, int OUT, bool GROUPED>
__device__ __forceinline__ void w4_pass(const W4Rows &rows, const W4Matrix &w, int64_t matrix, const int *list, int m0, int total, int pitch, int chunk, void *out)
{
    constexpr int NT = S::NT, MT = S::MT, HALVES = OUT == W4_OUT_SWIGLU ? 2 : 1, COLS = NT / HALVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t cols = w.rows / HALVES, n0 = (int64_t)blockIdx.x * (16 * S::WN * COLS);
    W4Job job;
    job.rows = (int)min((int64_t)(16 * S::WN * COLS), cols - n0);
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        const int64_t first = matrix * w.rows + n0 + h * cols;
        job.codes[h] = w.codes + first * w.row_bytes;
        job.scales[h] = static_cast<const uint8_t *>(w.scales) + first * w.row_groups * (KIND == W4_MX ? 1 : 2);
        job.zeros[h] = ZEROS ? w.zeros + first * w.row_groups : nullptr;
    }
    uint32_t x_row[S::XU];
#pragma unroll
    for (int u = 0; u < S::XU; u++) {
        const int at = min(m0 + 4 * ((wave % S::WN) * S::XU + u) + (lane >> 4), total - 1);
        x_row[u] = (uint32_t)(GROUPED ? list[at] / rows.x_div : at - m0) * (uint32_t)(2 * w.k);
    }
    job.x = static_cast<const T *>(rows.x) + (GROUPED ? 0 : (int64_t)m0 * w.k);
    w4_f32x4 acc[NT][MT];
    w4_sums<T, KIND, ZEROS, S, HALVES>(w, job, x_row, pitch, chunk, acc);
    __syncthreads();                                             // (the sums lie where others' rings were)
    float *const sums = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) sums[(((wave * MT + mt) * NT + j) * 4 + r) * 64 + lane] = acc[j][mt][r];
    __syncthreads();
    // the sums of one row and column of the tiles, over the parts of K in their order
    constexpr int LANES = MT == 1 ? 16 * S::XR : 64;             // that hold rows there are
    for (int i = threadIdx.x; i < S::WN * MT * COLS * 4 * LANES; i += S::THREADS) {
        const int l = i % LANES, r = i / LANES & 3, j = i / (4 * LANES) % COLS, mt = i / (4 * LANES * COLS) % MT, wn = i / (4 * LANES * COLS * MT);
        const int m = m0 + 16 * mt + 4 * (l >> 4) + r;
        const int64_t n = n0 + 16 * (wn * COLS + j) + (l & 15);
        if (m >= total || n >= cols) continue;
        float y[HALVES];
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            y[h] = 0.0f;
#pragma unroll
            for (int v = 0; v < S::WK; v++) y[h] += sums[((((v * S::WN + wn) * MT + mt) * NT + j + h * COLS) * 4 + r) * 64 + l];
        }
        const int64_t at = (GROUPED ? list[m] : m) * cols + n;
        if (OUT == W4_OUT_SWIGLU) static_cast<T *>(out)[at] = (T)(y[0] / (1.0f + __expf(-y[0])) * y[1]);
        else if (OUT == W4_OUT_F32) static_cast<float *>(out)[at] = y[0];
        else static_cast<T *>(out)[at] = (T)y[0];
    }
}

template <class T, int KIND, bool ZEROS, class S, int OUT, bool GROUPED>
__global__ __launch_bounds__(S::THREADS, S::NT * S::MT <= 2 ? 4 : 2) void w4_tile_kernel(W4Rows rows, W4Matrix w, int pitch, int chunk, int list_at, void *__restrict__ out)
{
    if constexpr (!GROUPED) {
        w4_pass<T, KIND, ZEROS, S, OUT, false>(rows, w, 0, nullptr, (int)blockIdx.y * (16 * S::MT), (int)rows.rows, pitch, chunk, out);
    } else {
        int *const scratch = reinterpret_cast<int *>(smem), *const list = reinterpret_cast<int *>(smem + list_at);   // (the rings come later)
        int expert = 0;
        const int total = w4_routes<S::W>(rows, blockIdx.y, list, scratch, expert);
        __syncthreads();
        for (int m0 = 0; m0 < total; m0 += S::MT == 1 ? 4 * S::XR : 16 * S::MT) {
            w4_pass<T, KIND, ZEROS, S, OUT, true>(rows, w, expert, list, m0, total, pitch, chunk, out);
            __syncthreads();
        }
    }
}

// The launch of one instantiation.
template <class T, int KIND, bool ZEROS, class S, int OUT, bool GROUPED>
int w4_tile_launch(const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    typedef W4Tile<T, KIND, ZEROS> Tile;
    auto kern = w4_tile_kernel<T, KIND, ZEROS, S, OUT, GROUPED>;
    constexpr int HALVES = OUT == W4_OUT_SWIGLU ? 2 : 1, COLS = S::NT / HALVES;
    // blocks whose scales are in LDS at a time, evenly
    constexpr int ROOM = 160 * 1024 - S::FIXED - (GROUPED ? 4 * W4_LIST : 0), PARAMS = ROOM < 32 * 1024 ? ROOM : 32 * 1024;
    static_assert(PARAMS >= 16 * S::TILES * 4 * 8);
    const int blocks = (w.k + 127) / 128, most = ((PARAMS / (16 * S::TILES) - 4) / 4 * 4) / (Tile::GROUPS * Tile::PARAM), chunks = (blocks + most - 1) / most;
    const int chunk = (blocks + chunks - 1) / chunks, pitch = w4_param_pitch(chunk * Tile::GROUPS, Tile::PARAM), list_at = S::FIXED + 16 * S::TILES * pitch;
    const int lds = list_at + (GROUPED ? 4 * (int)rows.rows : 0);
    static_assert(S::FIXED >= 4 * (1024 + 2));
    if (S::FIXED + PARAMS + (GROUPED ? 4 * W4_LIST : 0) > 48 * 1024) {
        // set once per device and kernel; setting it twice from two threads is harmless
        static std::atomic<uint64_t> attr_set{0};
        int dev = 0;
        CCH_HIP(hipGetDevice(&dev));
        const uint64_t dev_bit = (uint64_t)1 << (dev & 63);
        if (dev >= 64 || !(attr_set.load(std::memory_order_acquire) & dev_bit)) {
            CCH_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        S::FIXED + PARAMS + (GROUPED ? 4 * W4_LIST : 0)));
            attr_set.fetch_or(dev_bit, std::memory_order_release);
        }
    }
    const int64_t cols = w.rows / HALVES, per = 16 * S::WN * COLS;
    const int64_t y = GROUPED ? (rows.rows <= 64 ? rows.rows : std::min<int64_t>(rows.num_experts, rows.rows))
                              : (rows.rows + 16 * S::MT - 1) / (16 * S::MT);
    hipLaunchKernelGGL(kern, dim3((unsigned)((cols + per - 1) / per), (unsigned)y), dim3(S::THREADS), lds, s, rows, w, pitch, chunk, list_at, out);
    return launch_status("w4_tile_kernel");
}

// Which shape.  256 CUs are full with one or two workgroups each: as long as there are fewer, more waves share a tile (K in more parts), and where there are more tiles
// a workgroup takes several (x comes from the caches less often, K is in fewer parts).  Measured in us, int4 in groups of 128 / MXFP4, bf16 x, random codes:
//
//   dense, K = 7168, by n:            4096          8192          16384         32768         65536
//   1 row      1 tile, K in 8      *  6.0 /  5.7  *  9.1 /  7.8    15.3 / 14.4   31.7 / 31.5
//              2 tiles, K in 4        9.4 /  9.6    10.2 / 10.5  * 14.5 / 13.9 * 27.3 / 27.2
//   8 rows     1 tile, 8 rows of x *  6.6 /  6.2  *  9.7 /  9.1
//              1 tile, 16             7.1 /  6.7    12.7 / 12.3
//   16 rows    1 tile, K in 8      *  7.5 /  7.5    13.8 / 14.0    25.4 / 26.2   60.3 / 61.5   118 / 121
//              2 tiles, K in 8        8.7 /  9.0  * 10.4 / 11.0    18.7 / 20.1   43.1 / 45.6    84 / 89
//              2 waves of 1, in 4    11.6 /  9.9    13.4 / 12.6  * 18.8 / 16.2   38.6 / 34.1    74 / 67
//              4 waves of 1, in 2    16.8 / 14.8    18.6 / 17.9    21.3 / 19.9 * 33.3 / 29.1    65 / 62
//              4 waves of 2, in 2    23.6 / 22.3    24.0 / 23.4    25.4 / 25.4   35.5 / 34.5  * 53 / 52
//   32 rows    2 of 1, in 4        * 15.9 / 12.5  * 18.4 / 16.2    34.0 / 30.5   71.5 / 63.0          (more rows: whichever of the three has
//              4 of 1, in 4          18.3 / 14.6    19.8 / 17.0  * 22.5 / 21.3   48.5 / 42.8           no more than 256 workgroups)
//              4 of 2, in 4          26.1 / 21.4    27.2 / 22.5    27.7 / 24.1 * 39.4 / 34.4
//   64 rows    tiles of 32, best   * 17.4 / 13.9  * 21.6 / 18.2  * 31.6 / 25.5   70.3 / 60.2
//              64 rows, 8 of 1, in 2 44.2 / 30.4    45.2 / 30.8    45.4 / 31.9 * 58.2 / 43.1
//              64 rows, 4 of 2, in 2 49.5 / 35.6    49.5 / 36.4    49.7 / 37.3   60.3 / 47.0          (two waves to a SIMD, four above)
//
//   grouped, 16 experts, K = 7168, n = 4096, 6 routes a token; 64 experts, K = 2048, n = 1024, 8 routes; by an expert's routes, on average (tokens, experts):
//                  1 token         8 (64, 64)      12 (32, 16)     16 (128, 64)    24 (64, 16)     32 (256, 64)    36 (96, 16)
//   up, 4 rows   * 19.2 / 20.0     45.2 / 39.1     152 / 143       67.5 / 61.1     260 / 256       126 / 112
//       16         30.1 / 29.7   * 18.1 / 17.0     73.0 / 74.5     29.9 / 27.5     110 / 110       44.1 / 41.7
//       32         46.6 / 44.3     23.4 / 19.9   * 68.7 / 61.8   * 24.9 / 21.0     110 / 102       44.3 / 36.6     129 / 113
//       48                         28.4 / 22.3     88.8 / 67.2     29.3 / 24.0   *  90 /  70     * 32.1 / 25.8   *  93 /  74
//       64         65.1 / 51.8     33.1 / 24.6     101 / 73.4      34.4 / 25.6     101 /  76       36.3 / 28.1     106 /  77      (48 routes: * 115 / 78, 48 rows 157 / 121)
//   down, 4 rows * 13.8 / 12.9     35.5 / 33.7     81.5 / 71.9     55.0 / 52.2     142 / 128       106 / 101
//       16         16.0 / 15.5   * 14.6 / 13.2     40.8 / 41.5     23.1 / 20.6      62 /  61       32.0 / 30.6
//       32         19.4 / 15.5     17.9 / 16.2   * 44.3 / 38.7   * 19.1 / 17.7   *  53 /  47     * 32.0 / 26.9      81 /  66
//       48                         25.3 / 20.6     56.1 / 47.5     26.7 / 23.1      59 /  51       31.7 / 26.9   *  63 /  53      (96 routes: * 143 / 114, 32 rows 142 / 117)
//
// These are the layers that were swept.  Below 4096 columns the dense rule was measured afterwards and not tuned: K = 7168, 512 to 2048 columns 6.0 us for one row, 6.6 for 16, 15.1 to
// 16.4 for 17 to 128 (16 to 256 workgroups of eight waves).  The grouped rule looks at tokens and routes alone: with few experts or a narrow up projection its larger shapes are few workgroups that walk
// all of K (two of 4 experts, n = 512, K = 8192, 64 tokens: 77 us for the block, 16 of them in the up projection's launch; its weights are 3 us at the rate of a copy).
template <class T, int KIND, bool ZEROS>
int w4_tile_choose(int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
#define W4_GO(OUT, GROUPED, ...) w4_tile_launch<T, KIND, ZEROS, W4Shape<__VA_ARGS__>, OUT, GROUPED>(rows, w, out, s)
    if (out_kind == W4_OUT_PLAIN) {
        constexpr bool G = false;
        constexpr int64_t CUS = 256;
        const int64_t m = rows.rows, m32 = (m + 31) / 32, tiles = (w.rows + 15) / 16;
        if (m <= 4) return tiles <= 2 * CUS ? W4_GO(W4_OUT_PLAIN, G, 1, 1, 1, 1, 8) : W4_GO(W4_OUT_PLAIN, G, 2, 1, 1, 1, 4);
        if (m <= 8 && tiles <= 2 * CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 1, 2, 1, 8);
        if (m <= 16) {
            if (tiles <= CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 1, 4, 1, 8);
            if (tiles <= 2 * CUS) return W4_GO(W4_OUT_PLAIN, G, 2, 1, 4, 1, 8);
            if (tiles <= 4 * CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 1, 4, 2, 4);
            if (tiles <= 8 * CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 1, 4, 4, 2);
            return W4_GO(W4_OUT_PLAIN, G, 2, 1, 4, 4, 2);
        }
        if (m32 * ((tiles + 1) / 2) <= CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 2, 8, 2, 4);
        if (m32 * ((tiles + 3) / 4) <= CUS) return W4_GO(W4_OUT_PLAIN, G, 1, 2, 8, 4, 4);
        if (m32 == 1 || m32 * ((tiles + 7) / 8) <= CUS) return W4_GO(W4_OUT_PLAIN, G, 2, 2, 8, 4, 4);
        return W4_GO(W4_OUT_PLAIN, G, 1, 4, 16, 8, 2);
    }
    constexpr bool G = true;
    const int64_t tokens = rows.rows / rows.top_k;   // no expert has more of them
    if (out_kind == W4_OUT_SWIGLU) {
        if (tokens <= 4) return W4_GO(W4_OUT_SWIGLU, G, 2, 1, 1, 1, 4);
        if (tokens <= 16 || rows.rows <= 8 * rows.num_experts) return W4_GO(W4_OUT_SWIGLU, G, 2, 1, 4, 4, 2);
        if (tokens <= 32 || rows.rows <= 16 * rows.num_experts) return W4_GO(W4_OUT_SWIGLU, G, 2, 2, 8, 4, 1);
        if (tokens <= 48 || rows.rows <= 36 * rows.num_experts) return W4_GO(W4_OUT_SWIGLU, G, 2, 3, 12, 4, 1);
        return W4_GO(W4_OUT_SWIGLU, G, 2, 4, 16, 4, 1);
    }
    if (tokens <= 4) return W4_GO(W4_OUT_F32, G, 2, 1, 1, 1, 4);
    if (tokens <= 16 || rows.rows <= 8 * rows.num_experts) return W4_GO(W4_OUT_F32, G, 2, 1, 4, 4, 1);
    if (tokens <= 32 || rows.rows <= 32 * rows.num_experts) return W4_GO(W4_OUT_F32, G, 1, 2, 8, 8, 1);
    return W4_GO(W4_OUT_F32, G, 2, 3, 12, 4, 1);
#undef W4_GO
}

}  // namespace cch
