// The mixture-of-experts feed-forward of few tokens with weights of 4 bits: for every route (t, j) to expert e = expert_idx[t, j]
//   h = silu(g) * u, [g | u] = W1_e x_t,  y = W2_e h,  out[t] = sum_j probs[t, j] y_tj
// Up projection and activation are one launch, down projection the next (fp32), then the sum over a token's routes in their order, so that the same inputs give the same bits.
// h is rounded to the activations' type, as between two layers that are separate calls: it is the next product's 16-bit operand, and two such parts of it would be twice the rows for
// the matrix instructions and for LDS.  Of results in bf16 it takes the error against 64 bits from 1.7e-3, their own rounding, to 2.3e-3 or 2.4e-3; in half an h past 65504 is an infinity.
//
// Bound by the weights of the experts that some route names, once each: one token, 6 of 16 experts, k = 7168, n = 4096 (136 MB) 21.2 + 15.3 + 3.8 us in its three launches, 3.7 TB/s over the
// products (fastest of a kernel trace; 36 to 40 us a call); 64 tokens (374 MB) 71 + 51 + 4.4 fastest, 80 + 57 + 5.2 in the median, 113 to 153 a call by card and inputs.  Down projection and sum in one launch, a workgroup having its columns of all routes, measured about the same for one token (14.4 us for 13.2 +
// 4.7) and far worse for twelve (26 for 11.8 + 4.7, the experts one after another): not kept.
#include <algorithm>

#include "w4_decode.h"

namespace cch {

int w4_check(const char *what, int fmt, int group_size, int dtype);   // w4_matmul.hip

constexpr int MW4_MAX_TOPK = 8, MW4_MAX_EXPERTS = 1024, MW4_THREADS = 256;

// out[t] = sum over the token's routes, in their order, of probs * y.  The routes' loads are issued together: one after another, each behind its expert's, and with a
// 64-bit division to find the token, the launch took 12 tokens of 8 routes 1024 wide 8 us, now 4.7, an empty one 2.4.  Loads of routes that were dropped or are not
// there (ROUTES above top_k) are not used; for one and two routes 8 loads cost the block 3 and 1 %, for four less than 0.5 %.  Four columns to a thread where rows are
// that aligned, else one: 0.1 % of the block for one token, 0.5 % for 512 with 8 routes, 4 % with one.
template <class T, int ROUTES, int CHUNK>
__global__ __launch_bounds__(MW4_THREADS) void moe_w4_combine_kernel(const float *__restrict__ y, const int32_t *__restrict__ expert_idx, const float *__restrict__ probs,
                                                                    T *__restrict__ out, int k, int top_k, int experts)
{
    typedef float In __attribute__((ext_vector_type(CHUNK)));
    typedef T Out __attribute__((ext_vector_type(CHUNK)));
    const int64_t t = blockIdx.y, first = t * top_k;
    const int c = ((int)blockIdx.x * MW4_THREADS + (int)threadIdx.x) * CHUNK;
    if (c >= k) return;
    In v[ROUTES];
#pragma unroll
    for (int j = 0; j < ROUTES; j++) v[j] = *reinterpret_cast<const In *>(y + (first + min(j, top_k - 1)) * k + c);
    In sum = 0.0f;
#pragma unroll
    for (int j = 0; j < ROUTES; j++) {
        const int at = min(j, top_k - 1), e = expert_idx[first + at];
        const float p = probs[first + at];
        const bool there = j < top_k && e >= 0 && e < experts;
#pragma unroll
        for (int i = 0; i < CHUNK; i++) sum[i] = there ? sum[i] + p * v[j][i] : sum[i];
    }
    Out o;
#pragma unroll
    for (int i = 0; i < CHUNK; i++) o[i] = (T)sum[i];
    *reinterpret_cast<Out *>(out + t * k + c) = o;
}

template <class T>
static int moe_w4_combine(const float *y, const int32_t *expert_idx, const float *probs, void *out, int64_t m, int64_t k, int top_k, int experts, hipStream_t s)
{
    const bool four = k % 4 == 0 && aligned(out, 8);
    auto kern = top_k <= 2 ? (four ? moe_w4_combine_kernel<T, 2, 4> : moe_w4_combine_kernel<T, 2, 1>) : (four ? moe_w4_combine_kernel<T, 8, 4> : moe_w4_combine_kernel<T, 8, 1>);
    const int per = MW4_THREADS * (four ? 4 : 1);
    for (int64_t t = 0; t < m; t += 65535)   // tokens of the grid's second dimension
        hipLaunchKernelGGL(kern, dim3((unsigned)((k + per - 1) / per), (unsigned)std::min<int64_t>(65535, m - t)), dim3(MW4_THREADS), 0, s, y + t * top_k * k,
                           expert_idx + t * top_k, probs + t * top_k, static_cast<T *>(out) + t * k, (int)k, top_k, experts);
    return launch_status("moe_w4_combine_kernel");
}

struct MoeW4Workspace {
    int64_t h, y, end;
};
static MoeW4Workspace moe_w4_workspace(int64_t m, int64_t k, int64_t top_k, int64_t n)
{
    MoeW4Workspace w{};
    auto piece = [&](int64_t bytes) {
        const int64_t at = w.end;
        w.end += (bytes + 511) & ~(int64_t)511;
        return at;
    };
    w.h = piece(m * top_k * (n / 2) * 2);
    w.y = piece(m * top_k * k * 4);
    return w;
}

}  // namespace cch

extern "C" int64_t cch_moe_ffn_w4a16_workspace_bytes(int64_t m, int64_t k, int top_k, int64_t num_experts, int64_t n)
{
    if (m < 0 || k < 0 || top_k < 1 || num_experts < 1 || n < 0 || m >> 31 || k > cch::W4_MAX_ROWS || n > cch::W4_MAX_ROWS || num_experts >> 31 || top_k > 1024) return 0;
    return std::max<int64_t>(cch::moe_w4_workspace(m, k, top_k, n).end, 1);
}

extern "C" int cch_moe_ffn_w4a16(const void *x, const int32_t *expert_idx, const float *probs, const void *w1, const void *s1, const void *z1, const void *w2,
                                 const void *s2, const void *z2, void *out, int64_t m, int64_t k, int top_k, int64_t num_experts, int64_t n, int fmt, int group_size,
                                 int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace cch;
    CCH_REQUIRE(m >= 0 && k >= 0 && n >= 0 && !(m >> 31) && k <= W4_MAX_ROWS && n <= W4_MAX_ROWS, "cch_moe_ffn_w4a16: bad shape m=%lld k=%lld n=%lld", (long long)m, (long long)k,
                (long long)n);
    CCH_REQUIRE(top_k >= 1 && top_k <= MW4_MAX_TOPK, "cch_moe_ffn_w4a16: top_k=%d outside 1..%d", top_k, MW4_MAX_TOPK);
    CCH_REQUIRE(num_experts >= 1 && num_experts <= MW4_MAX_EXPERTS, "cch_moe_ffn_w4a16: num_experts=%lld outside 1..%d", (long long)num_experts, MW4_MAX_EXPERTS);
    CCH_REQUIRE(n % 2 == 0, "cch_moe_ffn_w4a16: n=%lld must be even (gate | up halves)", (long long)n);
    CCH_REQUIRE(!(m * top_k >> 31), "cch_moe_ffn_w4a16: %lld routes", (long long)(m * top_k));
    if (const int rc = w4_check("cch_moe_ffn_w4a16", fmt, group_size, dtype)) return rc;
    if (m == 0 || k == 0) return CCH_OK;
    const MoeW4Workspace at = moe_w4_workspace(m, k, top_k, n);
    CCH_REQUIRE(x && expert_idx && probs && out && (n == 0 || (w1 && s1 && w2 && s2)), "cch_moe_ffn_w4a16: null pointer");
    CCH_REQUIRE(workspace && aligned(workspace, 512) && workspace_bytes >= at.end, "cch_moe_ffn_w4a16: workspace of %lld bytes, need %lld on a 512-byte boundary",
                (long long)workspace_bytes, (long long)at.end);
    uint8_t *p = static_cast<uint8_t *>(workspace);
    const int64_t routes = m * top_k;
    if (n > 0)
        if (const int rc = w4_product(W4_OUT_SWIGLU, fmt, dtype, W4Rows{x, expert_idx, routes, (int)num_experts, top_k, top_k},
                                      w4_matrix(w1, s1, z1, n, k, fmt, group_size), p + at.h, stream))
            return rc;
    if (const int rc = w4_product(W4_OUT_F32, fmt, dtype, W4Rows{p + at.h, expert_idx, routes, (int)num_experts, 1, top_k}, w4_matrix(w2, s2, z2, k, n / 2, fmt, group_size),
                                  p + at.y, stream))
        return rc;
    const float *y = reinterpret_cast<const float *>(p + at.y);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == CCH_DTYPE_F16 ? moe_w4_combine<_Float16>(y, expert_idx, probs, out, m, k, top_k, (int)num_experts, s)
                                  : moe_w4_combine<__bf16>(y, expert_idx, probs, out, m, k, top_k, (int)num_experts, s);
}
