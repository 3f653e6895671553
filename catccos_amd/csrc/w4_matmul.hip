// Products of a few 16-bit rows with weights of 4 bits (w4_decode.h): y[m, n] = sum_k x[m, k] w[n, k], sums in fp32.
#include <algorithm>

#include "w4_decode.h"

namespace cch {

constexpr int W4_SIMPLE_THREADS = 256;

// The dot product of x's row with one row of weights, in every lane of the wave.
template <class T, bool INT4>
__device__ __forceinline__ float w4_dot(const T *__restrict__ x, const W4Matrix &w, int64_t row)
{
    const int lane = threadIdx.x & 63;
    const uint8_t *codes = w.codes + row * w.row_bytes;
    float acc = 0.0f;
    for (int b = lane; b < w.row_bytes; b += 64) {
        const uint32_t q = codes[b];
        const int64_t g = row * w.row_groups + 2 * b / w.group;
        const float x0 = (float)x[2 * b], x1 = 2 * b + 1 < w.k ? (float)x[2 * b + 1] : 0.0f;
        if (INT4) {
            const float z = w.zeros ? (float)w.zeros[g] : 8.0f;
            acc += (x0 * ((float)(q & 15) - z) + x1 * ((float)(q >> 4) - z)) * (float)static_cast<const T *>(w.scales)[g];
        } else {
            const float s = w4_e8m0(static_cast<const uint8_t *>(w.scales)[g]);
            acc += x0 * (w4_e2m1(q & 15) * s) + x1 * (w4_e2m1(q >> 4) * s);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) acc += __shfl_xor(acc, off, 64);
    return acc;
}

// A wave to an output element, a byte of codes to a lane: any K, any alignment.  Bound by its loads of single bytes and elements of x: 4096 rows of weights with K = 7168 take
// 23 us for one row of x and 252 for 16, where the tiled kernel takes 5.8 and 7.0; it is there for rows and pointers that the other does not take.
template <class T, bool INT4, int OUT>
__global__ __launch_bounds__(W4_SIMPLE_THREADS) void w4_simple_kernel(W4Rows rows, W4Matrix w, void *__restrict__ out, int64_t row0)
{
    const int64_t r = row0 + blockIdx.y;
    const int64_t cols = OUT == W4_OUT_SWIGLU ? w.rows / 2 : w.rows;
    const int64_t n = (int64_t)blockIdx.x * (W4_SIMPLE_THREADS / 64) + (threadIdx.x >> 6);
    if (n >= cols) return;
    int64_t first = 0;
    if (rows.experts) {
        const int e = rows.experts[r];
        if (e < 0 || e >= rows.num_experts) return;
        first = e * w.rows;
    }
    const T *x = static_cast<const T *>(rows.x) + r / rows.x_div * w.k;
    float y = w4_dot<T, INT4>(x, w, first + n);
    if (OUT == W4_OUT_SWIGLU) {
        const float up = w4_dot<T, INT4>(x, w, first + cols + n);
        y = y / (1.0f + __expf(-y)) * up;
    }
    if ((threadIdx.x & 63) != 0) return;
    if (OUT == W4_OUT_F32) static_cast<float *>(out)[r * cols + n] = y;
    else static_cast<T *>(out)[r * cols + n] = (T)y;
}

template <class T, bool INT4>
static int w4_simple(int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s)
{
    const int64_t cols = out_kind == W4_OUT_SWIGLU ? w.rows / 2 : w.rows;
    auto kern = out_kind == W4_OUT_PLAIN    ? w4_simple_kernel<T, INT4, W4_OUT_PLAIN>
                : out_kind == W4_OUT_SWIGLU ? w4_simple_kernel<T, INT4, W4_OUT_SWIGLU>
                                            : w4_simple_kernel<T, INT4, W4_OUT_F32>;
    for (int64_t r = 0; r < rows.rows; r += 65535) {
        const unsigned some = (unsigned)std::min<int64_t>(65535, rows.rows - r);
        hipLaunchKernelGGL(kern, dim3((unsigned)((cols + 3) / 4), some), dim3(W4_SIMPLE_THREADS), 0, s, rows, w, out, r);
    }
    return launch_status("w4_simple_kernel");
}

int w4_tile_int4_bf16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s);   // w4_tile_*.hip
int w4_tile_int4_f16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s);
int w4_tile_mx_bf16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s);
int w4_tile_mx_f16(int kind, int out_kind, const W4Rows &rows, const W4Matrix &w, void *out, hipStream_t s);

int w4_product(int out_kind, int fmt, int dtype, const W4Rows &rows, const W4Matrix &w, void *out, void *stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool half = dtype == CCH_DTYPE_F16, ints = fmt == CCH_FMT_INT4;
    // (16-byte loads straight to LDS, and groups that end where a lane's eight elements end; offsets of lanes are 32 bits: 128 rows of codes, and all rows of x that a
    // workgroup can meet)
    const int64_t x_rows = rows.experts ? std::min<int64_t>(rows.rows, W4_LIST) : 64;
    if (w.k > 0 && w.k % 32 == 0 && w.k <= 1 << 24 && x_rows * w.k < (int64_t)1 << 30 && aligned(w.codes, 16) && aligned(rows.x, 16) && (!ints || aligned(w.scales, 2))) {
        const int kind = !ints ? W4_MX : w.group == 32 ? W4_I4_G32 : w.group == 64 ? W4_I4_G64 : W4_I4_G128;
        const auto tile = ints ? (half ? w4_tile_int4_f16 : w4_tile_int4_bf16) : (half ? w4_tile_mx_f16 : w4_tile_mx_bf16);
        if (!rows.experts) {
            // as many rows as the grid's second dimension has tiles of 16 for
            for (int64_t r = 0; r < rows.rows; r += 65535 * 16) {
                W4Rows some = rows;
                some.rows = std::min<int64_t>(65535 * 16, rows.rows - r);
                some.x = static_cast<const uint16_t *>(rows.x) + r * w.k;
                const int rc = tile(kind, out_kind, some, w, static_cast<uint16_t *>(out) + r * w.rows, s);
                if (rc != CCH_OK) return rc;
            }
            return CCH_OK;
        }
        // routes in windows of as many whole tokens as a workgroup sorts out for itself
        const int64_t window = W4_LIST / rows.top_k * rows.top_k, cols = out_kind == W4_OUT_SWIGLU ? w.rows / 2 : w.rows;
        for (int64_t r = 0; r < rows.rows; r += window) {
            W4Rows some = rows;
            some.rows = std::min(window, rows.rows - r);
            some.experts = rows.experts + r;
            some.x = static_cast<const uint16_t *>(rows.x) + r / rows.x_div * w.k;
            const int rc = tile(kind, out_kind, some, w, static_cast<uint8_t *>(out) + r * cols * (out_kind == W4_OUT_F32 ? 4 : 2), s);
            if (rc != CCH_OK) return rc;
        }
        return CCH_OK;
    }
    if (half) return ints ? w4_simple<_Float16, true>(out_kind, rows, w, out, s) : w4_simple<_Float16, false>(out_kind, rows, w, out, s);
    return ints ? w4_simple<__bf16, true>(out_kind, rows, w, out, s) : w4_simple<__bf16, false>(out_kind, rows, w, out, s);
}

// What every product of this kind asks of its weights.
int w4_check(const char *what, int fmt, int group_size, int dtype)
{
    CCH_REQUIRE(fmt == CCH_FMT_INT4 || fmt == CCH_FMT_E2M1, "%s: weights of format %d (CCH_FMT_INT4 or CCH_FMT_E2M1)", what, fmt);
    CCH_REQUIRE(fmt == CCH_FMT_E2M1 || group_size == 32 || group_size == 64 || group_size == 128, "%s: group_size %d (32, 64 or 128)", what, group_size);
    CCH_REQUIRE(dtype == CCH_DTYPE_BF16 || dtype == CCH_DTYPE_F16, "%s: activations of type %d", what, dtype);
    return CCH_OK;
}

}  // namespace cch

extern "C" int64_t cch_w4a16_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k) { return 0; }

extern "C" int cch_w4a16_matmul(const void *x, const void *w, const void *scales, const void *zeros, void *out, int64_t m, int64_t n, int64_t k, int fmt, int group_size,
                                int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace cch;
    CCH_REQUIRE(m >= 0 && n >= 0 && k >= 0 && !(m >> 31) && n <= W4_MAX_ROWS && !(k >> 30), "cch_w4a16_matmul: bad shape m=%lld n=%lld k=%lld", (long long)m, (long long)n,
                (long long)k);
    if (const int rc = w4_check("cch_w4a16_matmul", fmt, group_size, dtype)) return rc;
    if (m == 0 || n == 0) return CCH_OK;
    CCH_REQUIRE(out && (k == 0 || (x && w && scales)), "cch_w4a16_matmul: null pointer");
    return w4_product(W4_OUT_PLAIN, fmt, dtype, W4Rows{x, nullptr, m, 1, 1, 1}, w4_matrix(w, scales, zeros, n, k, fmt, group_size), out, stream);
}
