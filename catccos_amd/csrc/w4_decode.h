// Weights of 4 bits with a scale per group along K, as they lie in memory, and what one of them stands for.
//
//   codes   [rows, ceil(K/2)] bytes, element 2j in the low nibble
//   int4    value (q - z) * s: s bf16 or half (the activations' type) [rows, ceil(K/G)], z bytes of the same shape, or 8 everywhere
//   E2M1    value v(q) * 2^(s - 127): s E8M0 [rows, 2*ceil(K/64)], G = 32, the layout that the MX row quantiser writes
#pragma once
#include "common.h"

namespace cch {

constexpr int64_t W4_MAX_ROWS = 1 << 25;   // of a matrix: a launch has below 2^32 threads, and the kernel for any K has 64 to a row

// One matrix [rows, k] or a stack of them, `rows` apart.
struct W4Matrix {
    const uint8_t *codes;
    const void *scales;
    const uint8_t *zeros;   // int4: or null
    int k, group, row_bytes, row_groups;
    int64_t rows;
};

__device__ __forceinline__ float w4_e8m0(uint32_t s) { return s == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(s ? s << 23 : 0x00400000u); }

__device__ __forceinline__ float w4_e2m1(uint32_t q)
{
    const uint32_t size = q & 7;
    const float v = size < 2 ? 0.5f * (float)size : __uint_as_float((126 + (size >> 1)) << 23 | (size & 1) << 22);
    return q & 8 ? -v : v;
}

inline W4Matrix w4_matrix(const void *codes, const void *scales, const void *zeros, int64_t rows, int64_t k, int fmt, int group)
{
    W4Matrix w{};
    w.codes = static_cast<const uint8_t *>(codes);
    w.scales = scales;
    w.zeros = fmt == CCH_FMT_INT4 ? static_cast<const uint8_t *>(zeros) : nullptr;
    w.k = (int)k;
    w.group = fmt == CCH_FMT_INT4 ? group : 32;
    w.row_bytes = (int)((k + 1) / 2);
    w.row_groups = fmt == CCH_FMT_INT4 ? (int)((k + group - 1) / group) : 2 * (int)((k + 63) / 64);
    w.rows = rows;
    return w;
}

// Where a product's left rows and its weights are: output row r takes row r / x_div of x and, with `experts`, matrix experts[r]
// (entries outside [0, num_experts): a dropped route, nothing is read or written), top_k of a token back to back.
struct W4Rows {
    const void *x;
    const int32_t *experts;
    int64_t rows;
    int num_experts, x_div, top_k;
};

// What a product leaves: out[r, n] in the activations' type; silu(gate) * up of columns n and n + N/2 in that type; fp32.
enum { W4_OUT_PLAIN = 0, W4_OUT_SWIGLU = 1, W4_OUT_F32 = 2 };

constexpr int W4_LIST = 2048;   // routes that a workgroup of the tiled kernel sorts out for itself
enum { W4_I4_G32 = 0, W4_I4_G64 = 1, W4_I4_G128 = 2, W4_MX = 3 };   // kinds of weights it knows

int w4_product(int out_kind, int fmt, int dtype, const W4Rows &rows, const W4Matrix &w, void *out, void *stream);

}  // namespace cch
