// The gate of a mixture of experts: what makes the expert_idx and probs that the routing sort, the grouped products and the combine take.
//
// Of a token's logits l over E experts: scores s = softmax(l), or sigmoid(l) of each; the top_k experts by score, or by score + bias where a bias steers
// the load (it only selects); weights w_j = scale s_j, or scale s_j / sum of the selected s ("renormalised").  Scores grow with the logits, so
// without a bias the logits themselves are compared: what is selected then depends on no rounding.  Equal keys go to the lower index.  An expert
// whose logit is -inf or NaN is not there; where fewer than top_k are, or the token is masked, the remaining routes are -1 with weight 0, which
// the routing sort drops.  With a bias softmax scores are compared over the candidates alone, and logits of +inf share the whole of them.
//
// Backward, g the weights' gradient, p = softmax(l):
//   softmax                  dl_e = p_e (scale g_e [e selected] - sum_j g_j w_j)
//   softmax, renormalised    dl_j = w_j (g_j - sum_i g_i w_i / scale), the selected experts only
//   sigmoid                  dl_j = w_j (1 - s_j) g_j
//   sigmoid, renormalised    dl_j = w_j (1 - s_j) (g_j - sum_i g_i w_i / scale)
// Everything is fp32 in registers; a row of logits is read once, and in the backward pass of three of the four forms not at all but for the selected ones.  The
// selection is top_k times the maximum over a lane's keys and over the lanes, the lowest index that holds it, and that key's removal: for few experts and few routes
// less than sorting anything, and ties need no extra step.
//
// Bound: on paper the bytes (16384 tokens of 64 experts in bf16, 8 routes: 3.1 MB forward, 5.2 MB backward, 1.6 us for both at the rate of a large copy), in fact the
// launch (an empty one 2.4 us) and the selection's instructions, some 2 V + 20 to a route: that case takes 4.8 + 4.0 us, 4099 tokens of 256 experts (fp32, sigmoid) 5.4 +
// 4.0, 64 tokens of 16 experts 2.2; 16384 x 1024 in bf16 28.0 + 16.7 (1.2 and 4.0 TB/s).  A bias costs the scores of all experts, a division each for softmax: 64 x 256 4.3 -> 6.5 us,
// 16384 x 64 4.4 -> 5.6, x 256 8.5 -> 15.1, x 1024 25.6 -> 46.7.  Backward, the selected experts' terms reach the lanes that hold them through LDS: one
// write for all routes, where comparing every expert with every route is 2 V instructions a route (16384 x 1024 23.6 us, x 256 9.1 against 6.5, x 64 4.3 against 3.8).
#include <algorithm>

#include "router_lanes.h"

namespace cch {

constexpr int ROUTER_THREADS = 256;

// This lane's selected logit l (lane `at` < top_k of its token; `there`: it is one) to its weight.  `top`: the largest selected logit, or, for
// softmax over all experts, of all of them with `denominator` their sum.
template <int L, bool SIGMOID, bool RENORM>
__device__ __forceinline__ float route_weight(float l, bool there, float top, float denominator, float scale)
{
    if (SIGMOID && !RENORM) return there ? scale * sigmoid(l) : 0.0f;
    if (!RENORM) return there ? scale * (exp_of(l - top) / denominator) : 0.0f;
    const float c = SIGMOID ? fminf(top, 0.0f) : top;
    const float s = !there ? 0.0f : SIGMOID ? scaled_sigmoid(l, c, exp_of(c)) : exp_of(l - c);
    const float sum = lanes_sum<L>(s);
    return there ? scale * (s / sum) : 0.0f;
}

template <class T, int V, int L, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(ROUTER_THREADS) void moe_router_kernel(const T *__restrict__ logits, const float *__restrict__ bias, const uint8_t *__restrict__ token_mask,
                                                                   float *__restrict__ probs, int32_t *__restrict__ expert_idx, int tokens, int experts, int top_k,
                                                                   float scale, bool vec)
{
    const int lane = threadIdx.x & 63, at = lane & (L - 1), base = lane & ~(L - 1);
    const int64_t t = ((int64_t)blockIdx.x * ROUTER_THREADS + threadIdx.x) / L;
    const bool inside = t < tokens;
    float l[V], key[V];
    load_row<T, V>(logits + (inside ? t : 0) * experts, at * V, experts, vec, l);
    const bool counted = inside && (token_mask == nullptr || token_mask[t] != 0);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        key[i] = l[i] == l[i] && counted ? l[i] : -INFINITY;
        top = fmaxf(top, key[i]);
    }
    float denominator = 1.0f, x[V];
    if (!SIGMOID && (!RENORM || bias)) {
        top = lanes_max<L>(top);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            x[i] = exp_of(l[i] - top);
            sum += at * V + i < experts ? x[i] : 0.0f;
        }
        denominator = lanes_sum<L>(sum);
    }
    if (bias) {
        float of_candidates = denominator;
        if (!SIGMOID && __ballot(denominator != denominator) != 0) {
            // Of a logit that is no candidate nothing, of one of +inf (as top is then) 1, the limit.  The weights' denominator keeps every logit as it is, so that what is
            // not finite shows there; in the scores it would take all of the token's candidates away.  (Always, without a look at the sum: 64 x 256 7.1 us for 6.5.)
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) {
                x[i] = key[i] == top ? 1.0f : key[i] > -INFINITY ? x[i] : 0.0f;
                sum += x[i];
            }
            of_candidates = lanes_sum<L>(sum);
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = at * V + i;
            if (e >= experts || key[i] == -INFINITY) continue;
            key[i] = (SIGMOID ? sigmoid(l[i]) : x[i] / of_candidates) + bias[e];
            if (!(key[i] == key[i])) key[i] = -INFINITY;
        }
    }
    int mine_idx = -1;
    float mine_l = -INFINITY;
    for (int j = 0; j < top_k; j++) {
        float best = key[0];
#pragma unroll
        for (int i = 1; i < V; i++) best = fmaxf(best, key[i]);
        const float all = lanes_max<L>(best);
        const uint64_t holders = (__ballot(best == all) >> base) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1);
        const int owner = __ffsll((unsigned long long)holders) - 1;   // (at least one lane holds the maximum)
        const bool found = all > -INFINITY;
        int which = 0;
#pragma unroll
        for (int i = V - 1; i >= 0; i--) which = key[i] == all ? i : which;
        const int taken = found && at == owner ? which : V;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i == taken) key[i] = -INFINITY;
        const int idx = __shfl(at * V + which, base + owner, 64);
        if (at == j && found) {
            mine_idx = idx;
            mine_l = all;
        }
    }
    const bool there = mine_idx >= 0;
    if (bias && there) mine_l = to_f32(logits[t * experts + mine_idx]);   // (keys were scores)
    if (RENORM) top = lanes_max<L>(mine_l);
    const float w = route_weight<L, SIGMOID, RENORM>(mine_l, there, top, denominator, scale);
    if (inside && at < top_k) {
        probs[t * top_k + at] = w;
        expert_idx[t * top_k + at] = mine_idx;
    }
}

template <class T, int V, int L, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(ROUTER_THREADS) void moe_router_backward_kernel(const float *__restrict__ grad_probs, const T *__restrict__ logits,
                                                                            const int32_t *__restrict__ expert_idx, T *__restrict__ grad_logits, int tokens, int experts,
                                                                            int top_k, float scale, bool vec)
{
    const int lane = threadIdx.x & 63, at = lane & (L - 1);
    const int64_t t = ((int64_t)blockIdx.x * ROUTER_THREADS + threadIdx.x) / L;
    const bool inside = t < tokens;
    const T *row = logits + (inside ? t : 0) * experts;
    int idx = -1;
    float g = 0.0f, sel = -INFINITY;
    if (inside && at < top_k) {
        idx = expert_idx[t * top_k + at];
        if (idx < 0 || idx >= experts) idx = -1;
        if (idx >= 0) {
            g = grad_probs[t * top_k + at];
            sel = to_f32(row[idx]);
        }
    }
    const bool there = idx >= 0;
    float d[V], top, denominator = 1.0f;
    if (!SIGMOID && !RENORM) {
        load_row<T, V>(row, at * V, experts, vec, d);
        top = d[0];
#pragma unroll
        for (int i = 1; i < V; i++) top = fmaxf(top, d[i]);
        top = lanes_max<L>(top);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            d[i] = at * V + i < experts ? exp_of(d[i] - top) : 0.0f;
            sum += d[i];
        }
        denominator = lanes_sum<L>(sum);
    } else {
        top = RENORM ? lanes_max<L>(sel) : 0.0f;
    }
    const float w = route_weight<L, SIGMOID, RENORM>(sel, there, top, denominator, 1.0f);   // of scale 1
    const float dot = lanes_sum<L>(there ? g * w : 0.0f);
    float own = RENORM ? w * (g - dot) : w * g;
    if (SIGMOID) own *= 1.0f / (1.0f + exp_of(sel));   // 1 - sigmoid
    own = there ? own * scale : 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) d[i] = !SIGMOID && !RENORM && dot != 0.0f ? -scale * dot * (d[i] / denominator) : 0.0f;
    // the selected experts' own terms, by way of the token's row in LDS; its lanes are of one wave, whose LDS accesses are in order
    // (pieces of four experts, all lanes' first ones first: neighbouring lanes on neighbouring banks)
    constexpr int PIECE = V < 4 ? V : 4;
    typedef float Piece __attribute__((ext_vector_type(PIECE)));
    __shared__ Piece rows[ROUTER_THREADS / L][V / PIECE][L];
    Piece (*const mine)[L] = rows[threadIdx.x / L];
#pragma unroll
    for (int c = 0; c < V / PIECE; c++) mine[c][at] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (there) atomicAdd(reinterpret_cast<float *>(&mine[idx % V / PIECE][idx / V]) + idx % PIECE, own);   // (an expert that a caller names twice gets both)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < V; i++) d[i] += mine[i / PIECE][at][i % PIECE];
    if (inside) store_row<T, V>(grad_logits + t * experts, at * V, experts, vec, d);
}

static int router_shape(const char *what, int dtype, int64_t tokens, int64_t experts, int top_k, int scoring)
{
    CCH_REQUIRE(logits_type_ok(dtype), "%s: logits of type %d", what, dtype);
    CCH_REQUIRE(tokens >= 0 && tokens <= ROUTER_MAX_TOKENS, "%s: %lld tokens", what, (long long)tokens);
    CCH_REQUIRE(experts >= 1 && experts <= ROUTER_MAX_EXPERTS, "%s: num_experts=%lld outside 1..%d", what, (long long)experts, ROUTER_MAX_EXPERTS);
    CCH_REQUIRE(top_k >= 1 && top_k <= ROUTER_MAX_TOPK && top_k <= experts, "%s: top_k=%d outside 1..min(%d, num_experts)", what, top_k, ROUTER_MAX_TOPK);
    CCH_REQUIRE(scoring == CCH_SCORING_SOFTMAX || scoring == CCH_SCORING_SIGMOID, "%s: scoring %d", what, scoring);
    return CCH_OK;
}

// f(first token, tokens) for launches of up to 2^25 tokens: one has below 2^32 threads.
template <class F>
static int router_launches(int64_t tokens, F f)
{
    for (int64_t t = 0; t < tokens; t += 1 << 25) {
        const int rc = f(t, (int)std::min<int64_t>(1 << 25, tokens - t));
        if (rc != CCH_OK) return rc;
    }
    return CCH_OK;
}
template <int L>
static unsigned router_grid(int tokens)
{
    return (unsigned)((tokens + ROUTER_THREADS / L - 1) / (ROUTER_THREADS / L));
}

}  // namespace cch

extern "C" int cch_moe_router(const void *logits, int dtype, int64_t tokens, int64_t num_experts, int top_k, int scoring, int renormalize, float scale, const float *bias,
                              const uint8_t *token_mask, float *probs, int32_t *expert_idx, void *stream)
{
    using namespace cch;
    if (const int rc = router_shape("cch_moe_router", dtype, tokens, num_experts, top_k, scoring)) return rc;
    CCH_REQUIRE(renormalize == 0 || renormalize == 1, "cch_moe_router: renormalize %d", renormalize);
    if (tokens == 0) return CCH_OK;
    CCH_REQUIRE(logits && probs && expert_idx, "cch_moe_router: null pointer");
    return with_logits_type(dtype, [&](auto *type) {
        return with_lanes((int)num_experts, [&](auto v, auto lanes) {
            typedef std::remove_pointer_t<decltype(type)> T;
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value;
            auto kern = scoring == CCH_SCORING_SIGMOID ? (renormalize ? moe_router_kernel<T, V, L, true, true> : moe_router_kernel<T, V, L, true, false>)
                                                       : (renormalize ? moe_router_kernel<T, V, L, false, true> : moe_router_kernel<T, V, L, false, false>);
            return router_launches(tokens, [&](int64_t t, int some) {
                hipLaunchKernelGGL(kern, dim3(router_grid<L>(some)), dim3(ROUTER_THREADS), 0, static_cast<hipStream_t>(stream),
                                   static_cast<const T *>(logits) + t * num_experts, bias, token_mask ? token_mask + t : nullptr, probs + t * top_k, expert_idx + t * top_k,
                                   some, (int)num_experts, top_k, scale, LanePieces<T, V>::vec(logits, num_experts));
                return launch_status("moe_router_kernel");
            });
        });
    });
}

extern "C" int cch_moe_router_backward(const float *grad_probs, const void *logits, int dtype, const int32_t *expert_idx, int64_t tokens, int64_t num_experts, int top_k,
                                       int scoring, int renormalize, float scale, void *grad_logits, void *stream)
{
    using namespace cch;
    if (const int rc = router_shape("cch_moe_router_backward", dtype, tokens, num_experts, top_k, scoring)) return rc;
    CCH_REQUIRE(renormalize == 0 || renormalize == 1, "cch_moe_router_backward: renormalize %d", renormalize);
    if (tokens == 0) return CCH_OK;
    CCH_REQUIRE(grad_probs && logits && expert_idx && grad_logits, "cch_moe_router_backward: null pointer");
    return with_logits_type(dtype, [&](auto *type) {
        return with_lanes((int)num_experts, [&](auto v, auto lanes) {
            typedef std::remove_pointer_t<decltype(type)> T;
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value;
            auto kern = scoring == CCH_SCORING_SIGMOID
                            ? (renormalize ? moe_router_backward_kernel<T, V, L, true, true> : moe_router_backward_kernel<T, V, L, true, false>)
                            : (renormalize ? moe_router_backward_kernel<T, V, L, false, true> : moe_router_backward_kernel<T, V, L, false, false>);
            const bool vec = LanePieces<T, V>::vec(logits, num_experts) && aligned(grad_logits, 16);
            return router_launches(tokens, [&](int64_t t, int some) {
                hipLaunchKernelGGL(kern, dim3(router_grid<L>(some)), dim3(ROUTER_THREADS), 0, static_cast<hipStream_t>(stream), grad_probs + t * top_k,
                                   static_cast<const T *>(logits) + t * num_experts, expert_idx + t * top_k, static_cast<T *>(grad_logits) + t * num_experts, some,
                                   (int)num_experts, top_k, scale, vec);
                return launch_status("moe_router_backward_kernel");
            });
        });
    });
}
