// Entry points of the products of 16-bit operands: grouped by expert, and dense with bias, activation and residual; forward and backward.
#include <algorithm>

#include "gemm16.h"

namespace cch {

constexpr int64_t MAX_ROWS16 = (int64_t)1 << 30;

static bool fits16(int64_t m, int64_t n, int64_t k) { return m >= 0 && n >= 0 && k >= 0 && m <= MAX_ROWS16 && n <= MAX_PITCH16 && k <= MAX_PITCH16; }

static int check_shape16(const char *what, int64_t m, int64_t n, int64_t k, int trans_b, int dtype)
{
    CCH_REQUIRE(fits16(m, n, k), "%s: bad shape, %lld rows, n=%lld k=%lld (at most 2^30, 2^22, 2^22)", what, (long long)m, (long long)n, (long long)k);
    CCH_REQUIRE(trans_b == 0 || trans_b == 1, "%s: trans_b=%d", what, trans_b);
    CCH_REQUIRE(dtype == CCH_DTYPE_BF16 || dtype == CCH_DTYPE_F16, "%s: operands of type %d", what, dtype);
    return CCH_OK;
}

static int check_workspace16(const char *what, const void *ws, int64_t have, int64_t need)
{
    CCH_REQUIRE(need == 0 || (ws && aligned(ws, 256) && have >= need), "%s: workspace of %lld bytes, need %lld on a 256-byte boundary", what, (long long)(ws ? have : 0), (long long)need);
    return CCH_OK;
}

static const uint16_t *u16(const void *p) { return static_cast<const uint16_t *>(p); }
static uint16_t *u16(void *p) { return static_cast<uint16_t *>(p); }

static bool groups_fit(int64_t e) { return e >= 1 && e <= MAX_GROUPS16; }

// Bytes of the padded copies of x (rows of k), grad_out or dz (rows of n) and w.
static int64_t weights16_bytes(int64_t e, int64_t n, int64_t k, int trans_b) { return trans_b ? padded16_bytes(e * n, k) : padded16_bytes(e * k, n); }

// The product x [m, k] times w: rows of `out` [m, n]; dense (groups 1, no sizes) or grouped.
static Gemm16 product16(const uint16_t *x, int64_t pitch_x, const uint16_t *w, int64_t pitch_w, uint16_t *out, int64_t m, int64_t n, int64_t k, int trans_b, int dtype)
{
    Gemm16 p{};
    p.a = x;
    p.b = w;
    p.out = out;
    p.pitch_a = pitch_x;
    p.pitch_b = pitch_w;
    p.pitch_out = n;
    p.m = (int)m;
    p.n = (int)n;
    p.k = (int)k;
    p.b_stride = (trans_b ? n : k) * pitch_w;
    p.groups = 1;
    p.half = dtype == CCH_DTYPE_F16;
    return p;
}

// The two products of a backward pass, pointers apart: grad_x's and grad_w's.
static Gemm16 grad_x_product(const int32_t *sizes, int64_t e, int64_t t, int64_t n, int64_t k, int trans_b, int dtype)
{
    // W^T of weights [n, k] is weights [k', n'] with k' = n
    Gemm16 p = product16(nullptr, pitch16(n), nullptr, pitch16(trans_b ? k : n), nullptr, t, k, n, !trans_b, dtype);
    p.b_stride = (trans_b ? n : k) * p.pitch_b;
    p.group_sizes = sizes;
    p.groups = (int)e;
    p.zero_rest = sizes != nullptr;
    return p;
}
static Gemm16 grad_w_product(const int32_t *sizes, int64_t e, int64_t t, int64_t n, int64_t k, int trans_b, int dtype)
{
    Gemm16 p = trans_b ? product16(nullptr, pitch16(n), nullptr, pitch16(k), nullptr, n, k, t, 0, dtype) : product16(nullptr, pitch16(k), nullptr, pitch16(n), nullptr, k, n, t, 0, dtype);
    p.b_stride = 0;
    p.out_stride = n * k;
    p.group_sizes = sizes;
    p.groups = (int)e;
    p.k_grouped = 1;
    return p;
}
static Gemm16 grouped_product(const uint16_t *x, const uint16_t *w, const int32_t *sizes, uint16_t *out, int64_t e, int64_t t, int64_t n, int64_t k, int trans_b, int dtype)
{
    Gemm16 p = product16(x, pitch16(k), w, pitch16(trans_b ? k : n), out, t, n, k, trans_b, dtype);
    p.group_sizes = sizes;
    p.groups = (int)e;
    p.zero_rest = 1;
    return p;
}
static const int32_t SOME_SIZES = 0;   // stands for sizes that are there, where only that counts
static int64_t backward_partial16(const int32_t *sizes, int64_t e, int64_t t, int64_t n, int64_t k, int trans_b)
{
    return std::max(partial16_bytes(grad_x_product(sizes, e, t, n, k, trans_b, CCH_DTYPE_BF16), trans_b ? ROWS_NN : ROWS_NK, EPI16_OUT),
                    partial16_bytes(grad_w_product(sizes, e, t, n, k, trans_b, CCH_DTYPE_BF16), ROWS_TN, EPI16_OUT));
}

// grad_x [t, k] = grad [t, n] W^T and grad_w = x^T grad (or its transpose), per group.
static int backward_products16(const uint16_t *grad, const uint16_t *x, const uint16_t *w, const int32_t *sizes, int64_t e, uint16_t *grad_x, uint16_t *grad_w, int64_t t, int64_t n,
                               int64_t k, int trans_b, int dtype, const Carve &ws, void *workspace, int64_t workspace_bytes, hipStream_t stream)
{
    if (grad_x && t > 0 && k > 0) {
        Gemm16 p = grad_x_product(sizes, e, t, n, k, trans_b, dtype);
        p.a = grad;
        p.b = w;
        p.out = grad_x;
        ws.rest(p, workspace, workspace_bytes);
        if (const int rc = gemm16_launch(p, trans_b ? ROWS_NN : ROWS_NK, EPI16_OUT, stream)) return rc;
    }
    if (grad_w && n > 0 && k > 0) {
        Gemm16 p = grad_w_product(sizes, e, t, n, k, trans_b, dtype);
        p.a = trans_b ? grad : x;
        p.b = trans_b ? x : grad;
        p.out = grad_w;
        ws.rest(p, workspace, workspace_bytes);
        if (const int rc = gemm16_launch(p, ROWS_TN, EPI16_OUT, stream)) return rc;
    }
    return CCH_OK;
}

}  // namespace cch

using namespace cch;

extern "C" int64_t cch_grouped_matmul_workspace_bytes(int64_t num_experts, int64_t t, int64_t n, int64_t k, int trans_b)
{
    if (!fits16(t, n, k) || !groups_fit(num_experts)) return 0;
    return padded16_bytes(t, k) + weights16_bytes(num_experts, n, k, trans_b) + partial16_bytes(grouped_product(nullptr, nullptr, &SOME_SIZES, nullptr, num_experts, t, n, k, trans_b, CCH_DTYPE_BF16), trans_b ? ROWS_NK : ROWS_NN, EPI16_OUT);
}

extern "C" int cch_grouped_matmul(const void *x, const void *w, const int32_t *group_sizes, void *out, int64_t num_experts, int64_t t, int64_t n, int64_t k, int trans_b,
                                  int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_shape16("cch_grouped_matmul", t, n, k, trans_b, dtype)) return rc;
    CCH_REQUIRE(groups_fit(num_experts), "cch_grouped_matmul: num_experts=%lld outside 1..%d", (long long)num_experts, MAX_GROUPS16);
    if (t == 0 || n == 0) return CCH_OK;
    CCH_REQUIRE(out && group_sizes && (k == 0 || (x && w)), "cch_grouped_matmul: null pointer");
    CCH_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(out, 2), "cch_grouped_matmul: x and w must lie on 16-byte boundaries");
    if (const int rc = check_workspace16("cch_grouped_matmul", workspace, workspace_bytes, cch_grouped_matmul_workspace_bytes(num_experts, t, n, k, trans_b))) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Carve ws{static_cast<uint8_t *>(workspace)};
    Operand16 in[2] = {{u16(x), t, k}, {u16(w), num_experts * (trans_b ? n : k), trans_b ? k : n, group_sizes, trans_b ? n : k}};
    if (const int rc = whole_operands16(in, 2, ws, s)) return rc;
    Gemm16 p = grouped_product(in[0].at, in[1].at, group_sizes, u16(out), num_experts, t, n, k, trans_b, dtype);
    ws.rest(p, workspace, workspace_bytes);
    return gemm16_launch(p, trans_b ? ROWS_NK : ROWS_NN, EPI16_OUT, s);
}

extern "C" int64_t cch_grouped_matmul_backward_workspace_bytes(int64_t num_experts, int64_t t, int64_t n, int64_t k, int trans_b)
{
    if (!fits16(t, n, k) || !groups_fit(num_experts)) return 0;
    return padded16_bytes(t, k) + padded16_bytes(t, n) + weights16_bytes(num_experts, n, k, trans_b) + backward_partial16(&SOME_SIZES, num_experts, t, n, k, trans_b);
}

extern "C" int cch_grouped_matmul_backward(const void *grad_out, const void *x, const void *w, const int32_t *group_sizes, void *grad_x, void *grad_w, int64_t num_experts,
                                           int64_t t, int64_t n, int64_t k, int trans_b, int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_shape16("cch_grouped_matmul_backward", t, n, k, trans_b, dtype)) return rc;
    CCH_REQUIRE(groups_fit(num_experts), "cch_grouped_matmul_backward: num_experts=%lld outside 1..%d", (long long)num_experts, MAX_GROUPS16);
    CCH_REQUIRE(group_sizes && (t == 0 || n == 0 || grad_out) && (!grad_w || t == 0 || k == 0 || x) && (!grad_x || n == 0 || k == 0 || w), "cch_grouped_matmul_backward: null pointer");
    CCH_REQUIRE(aligned(grad_out, 16) && aligned(x, 16) && aligned(w, 16) && aligned(grad_x, 2) && aligned(grad_w, 2),
                "cch_grouped_matmul_backward: grad_out, x and w must lie on 16-byte boundaries");
    if (const int rc = check_workspace16("cch_grouped_matmul_backward", workspace, workspace_bytes, cch_grouped_matmul_backward_workspace_bytes(num_experts, t, n, k, trans_b)))
        return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Carve ws{static_cast<uint8_t *>(workspace)};
    Operand16 in[3] = {{u16(grad_out), t, n}, {grad_w ? u16(x) : nullptr, t, k}, {grad_x ? u16(w) : nullptr, num_experts * (trans_b ? n : k), trans_b ? k : n, group_sizes, trans_b ? n : k}};
    if (const int rc = whole_operands16(in, 3, ws, s)) return rc;
    return backward_products16(in[0].at, in[1].at, in[2].at, group_sizes, num_experts, u16(grad_x), u16(grad_w), t, n, k, trans_b, dtype, ws, workspace, workspace_bytes, s);
}

static int check_act(const char *what, int act)
{
    CCH_REQUIRE(act >= CCH_ACT_NONE && act <= CCH_ACT_GELU_TANH, "%s: activation %d", what, act);
    return CCH_OK;
}

extern "C" int64_t cch_matmul_bias_act_workspace_bytes(int64_t m, int64_t n, int64_t k, int trans_b)
{
    if (!fits16(m, n, k)) return 0;
    return padded16_bytes(m, k) + weights16_bytes(1, n, k, trans_b) +
           partial16_bytes(product16(nullptr, pitch16(k), nullptr, pitch16(trans_b ? k : n), nullptr, m, n, k, trans_b, CCH_DTYPE_BF16), trans_b ? ROWS_NK : ROWS_NN, EPI16_ACT);
}

extern "C" int cch_matmul_bias_act(const void *x, const void *w, const void *bias, const void *residual, void *preact, void *out, int64_t m, int64_t n, int64_t k, int trans_b,
                                   int activation, int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_shape16("cch_matmul_bias_act", m, n, k, trans_b, dtype)) return rc;
    if (const int rc = check_act("cch_matmul_bias_act", activation)) return rc;
    if (m == 0 || n == 0) return CCH_OK;
    CCH_REQUIRE(out && (k == 0 || (x && w)), "cch_matmul_bias_act: null pointer");
    CCH_REQUIRE(aligned(x, 16) && aligned(w, 16), "cch_matmul_bias_act: x and w must lie on 16-byte boundaries");
    CCH_REQUIRE(aligned(out, 2) && aligned(preact, 2) && aligned(bias, 2) && aligned(residual, 2), "cch_matmul_bias_act: a tensor on an odd address");
    if (const int rc = check_workspace16("cch_matmul_bias_act", workspace, workspace_bytes, cch_matmul_bias_act_workspace_bytes(m, n, k, trans_b))) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Carve ws{static_cast<uint8_t *>(workspace)};
    Operand16 in[2] = {{u16(x), m, k}, {u16(w), trans_b ? n : k, trans_b ? k : n}};
    if (const int rc = whole_operands16(in, 2, ws, s)) return rc;
    Gemm16 p = product16(in[0].at, pitch16(k), in[1].at, pitch16(trans_b ? k : n), u16(out), m, n, k, trans_b, dtype);
    p.bias = u16(bias);
    p.residual = u16(residual);
    p.preact = u16(preact);
    p.act = activation;
    ws.rest(p, workspace, workspace_bytes);
    return gemm16_launch(p, trans_b ? ROWS_NK : ROWS_NN, EPI16_ACT, s);
}

extern "C" int64_t cch_matmul_bias_act_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, int trans_b, int activation)
{
    if (!fits16(m, n, k)) return 0;
    const int64_t dz = activation == CCH_ACT_NONE ? padded16_bytes(m, n) : round256(m * pitch16(n) * 2);
    return dz + column_sum_bytes(m, n) + padded16_bytes(m, k) + weights16_bytes(1, n, k, trans_b) + backward_partial16(nullptr, 1, m, n, k, trans_b);
}

extern "C" int cch_matmul_bias_act_backward(const void *grad_out, const void *x, const void *w, const void *preact, void *grad_x, void *grad_w, void *grad_bias, int64_t m,
                                            int64_t n, int64_t k, int trans_b, int activation, int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_shape16("cch_matmul_bias_act_backward", m, n, k, trans_b, dtype)) return rc;
    if (const int rc = check_act("cch_matmul_bias_act_backward", activation)) return rc;
    const bool none = m == 0 || n == 0;
    CCH_REQUIRE((none || (grad_out && (activation == CCH_ACT_NONE || preact))) && (!grad_w || none || k == 0 || x) && (!grad_x || none || k == 0 || w),
                "cch_matmul_bias_act_backward: null pointer");
    CCH_REQUIRE(aligned(grad_out, 16) && aligned(x, 16) && aligned(w, 16) && aligned(preact, 2), "cch_matmul_bias_act_backward: grad_out, x and w must lie on 16-byte boundaries");
    CCH_REQUIRE(aligned(grad_x, 2) && aligned(grad_w, 2) && aligned(grad_bias, 2), "cch_matmul_bias_act_backward: a tensor on an odd address");
    if (const int rc = check_workspace16("cch_matmul_bias_act_backward", workspace, workspace_bytes, cch_matmul_bias_act_backward_workspace_bytes(m, n, k, trans_b, activation)))
        return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Carve ws{static_cast<uint8_t *>(workspace)};
    // dz = grad_out * act'(preact), rounded to the operands' type like every operand of a product here; without an activation it is grad_out
    const bool own = activation != CCH_ACT_NONE || !whole16(n);
    uint16_t *dz = own ? ws.take<uint16_t>(m * pitch16(n) * 2) : nullptr;
    float *partial = ws.take<float>(column_sum_bytes(m, n));
    if (m == 0 && grad_bias && n > 0) {
        // no rows: zeros from the same sum over none
        if (const int rc = fill_zero16(u16(grad_bias), n, s)) return rc;
    }
    if (const int rc = act_backward16(u16(grad_out), u16(preact), dz, u16(grad_bias), partial, m, n, activation, dtype == CCH_DTYPE_F16, s)) return rc;
    Operand16 in[2] = {{grad_w ? u16(x) : nullptr, m, k}, {grad_x ? u16(w) : nullptr, trans_b ? n : k, trans_b ? k : n}};
    if (const int rc = whole_operands16(in, 2, ws, s)) return rc;
    return backward_products16(own ? dz : u16(grad_out), in[0].at, in[1].at, nullptr, 1, u16(grad_x), u16(grad_w), m, n, k, trans_b, dtype, ws, workspace, workspace_bytes, s);
}
