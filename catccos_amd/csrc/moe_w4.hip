// The mixture-of-experts feed-forward of few tokens with weights of 4 bits: for every route (t, j) to expert e = expert_idx[t, j]
//   h = silu(g) * u, [g | u] = W1_e x_t,  y = W2_e h,  out[t] = sum_j probs[t, j] y_tj
// Up projection and activation are one launch (h in the activations' type: it is the next product's operand), down projection the next (fp32), then the sum
// over a token's routes in their order.
#include <algorithm>

#include "w4_decode.h"

namespace cch {

int w4_check(const char *what, int fmt, int group_size, int dtype);   // w4_matmul.hip

constexpr int MW4_MAX_TOPK = 8, MW4_MAX_EXPERTS = 1024, MW4_THREADS = 256;

template <class T>
__global__ __launch_bounds__(MW4_THREADS) void moe_w4_combine_kernel(const float *__restrict__ y, const int32_t *__restrict__ expert_idx, const float *__restrict__ probs,
                                                                    T *__restrict__ out, int64_t total, int k, int top_k, int experts)
{
    const int64_t i = (int64_t)blockIdx.x * MW4_THREADS + threadIdx.x;
    if (i >= total) return;
    const int64_t t = i / k, c = i - t * k;
    float sum = 0.0f;
    for (int j = 0; j < top_k; j++) {
        const int e = expert_idx[t * top_k + j];
        if (e >= 0 && e < experts) sum += probs[t * top_k + j] * y[(t * top_k + j) * k + c];
    }
    out[i] = (T)sum;
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
    if (m < 0 || k < 0 || top_k < 1 || num_experts < 1 || n < 0 || m >> 31 || k >> 30 || n >> 31 || num_experts >> 31) return 0;
    return std::max<int64_t>(cch::moe_w4_workspace(m, k, top_k, n).end, 1);
}

extern "C" int cch_moe_ffn_w4a16(const void *x, const int32_t *expert_idx, const float *probs, const void *w1, const void *s1, const void *z1, const void *w2,
                                 const void *s2, const void *z2, void *out, int64_t m, int64_t k, int top_k, int64_t num_experts, int64_t n, int fmt, int group_size,
                                 int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace cch;
    CCH_REQUIRE(m >= 0 && k >= 0 && n >= 0 && !(m >> 31) && !(k >> 30) && !(n >> 30), "cch_moe_ffn_w4a16: bad shape m=%lld k=%lld n=%lld", (long long)m, (long long)k,
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
    const dim3 grid((unsigned)((m * k + MW4_THREADS - 1) / MW4_THREADS));
    if (dtype == CCH_DTYPE_F16)
        hipLaunchKernelGGL(moe_w4_combine_kernel<_Float16>, grid, dim3(MW4_THREADS), 0, static_cast<hipStream_t>(stream), y, expert_idx, probs,
                           static_cast<_Float16 *>(out), m * k, (int)k, top_k, (int)num_experts);
    else
        hipLaunchKernelGGL(moe_w4_combine_kernel<__bf16>, grid, dim3(MW4_THREADS), 0, static_cast<hipStream_t>(stream), y, expert_idx, probs, static_cast<__bf16 *>(out),
                           m * k, (int)k, top_k, (int)num_experts);
    return launch_status("moe_w4_combine_kernel");
}
