// The balance loss of a mixture of experts, the z loss and the routes per expert, and the gradient of the logits.
//
// Of a sequence s with N_s tokens that count (not masked, at least one logit above -inf), c_se routes to expert e and k routes per token, E experts:
//   f_se = E c_se / (k N_s),  P_se = mean over its tokens of p_te,  p = softmax(l), or sigmoid(l) / sum over experts of sigmoid(l)
//   loss = coef * mean over sequences with N_s > 0 of sum_e f_se P_se  +  z_coef * mean over all N tokens of lse_t^2,  lse_t = log sum_e exp(l_te)
// Without sequence offsets the whole batch is one sequence.  Routes are whole numbers without a gradient, so
//   dl_te = coef / (S' N_s) p_te (f_se - sum_i p_ti f_si) [(1 - sigmoid(l_te)) for sigmoid scores] + z_coef 2 lse_t softmax(l)_te / N
// times the loss's own gradient.
//
// Forward: workgroups take tokens of one sequence each, keep P in registers (fp32) and the routes in LDS, and leave their sums in the workspace;
// the sequences' workgroups add those up in a fixed order, so that the same inputs give the same bits.  Backward: one pass, logits in, gradient out.
#include <algorithm>

#include "router_lanes.h"

namespace cch {

constexpr int BAL_THREADS = 256, BAL_WAVES = BAL_THREADS / 64;
constexpr int BAL_MAX_SEQUENCES = 65535;

struct Span {
    int begin, end;
};
__device__ __forceinline__ Span span_of(const int32_t *offsets, int s, int tokens)
{
    if (offsets == nullptr) return {0, tokens};
    const int b = min(max(offsets[s], 0), tokens);
    return {b, min(max(offsets[s + 1], b), tokens)};
}

// A token's p (in place of l), and with Z softmax(l) in `q` and the log of the sum of exponentials.  False: no logit is above -inf (NaN is not).
template <int V, int L, bool SIGMOID, bool Z>
__device__ __forceinline__ bool token_shares(float (&l)[V], float (&q)[V], float &lse)
{
    float top = l[0];
#pragma unroll
    for (int i = 1; i < V; i++) top = fmaxf(top, l[i]);
    top = lanes_max<L>(top);
    if (SIGMOID && Z) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            q[i] = __expf(l[i] - top);
            sum += q[i];
        }
        sum = lanes_sum<L>(sum);
        lse = __logf(sum) + top;
#pragma unroll
        for (int i = 0; i < V; i++) q[i] /= sum;
    }
    float sum = 0.0f;
    const float c = fminf(top, 0.0f), ec = __expf(c);
#pragma unroll
    for (int i = 0; i < V; i++) {
        l[i] = SIGMOID ? scaled_sigmoid(l[i], c, ec) : __expf(l[i] - top);
        sum += l[i];
    }
    sum = lanes_sum<L>(sum);
    if (!SIGMOID && Z) lse = __logf(sum) + top;
#pragma unroll
    for (int i = 0; i < V; i++) {
        l[i] /= sum;
        if (!SIGMOID && Z) q[i] = l[i];
    }
    return top > -INFINITY;
}

// Sums of workgroup (c, s) in part[(s * gridDim.x + c) * (2 experts + 2)]: P per expert, routes per expert, sum of lse^2, tokens.
template <class T, int V, int L, bool SIGMOID, bool Z>
__global__ __launch_bounds__(BAL_THREADS) void moe_balance_sums_kernel(const T *__restrict__ logits, const int32_t *__restrict__ expert_idx,
                                                                      const uint8_t *__restrict__ token_mask, const int32_t *__restrict__ seq_offsets, int tokens,
                                                                      int experts, int top_k, float *__restrict__ part, bool vec)
{
    constexpr int TPW = 64 / L;   // tokens of a wave at a time
    __shared__ float shares[BAL_WAVES][V * L], rest[BAL_WAVES];
    __shared__ int32_t routes[V * L], counted[BAL_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & (L - 1);
    for (int e = threadIdx.x; e < V * L; e += BAL_THREADS) routes[e] = 0;
    __syncthreads();
    const Span span = span_of(seq_offsets, blockIdx.y, tokens);
    float acc[V], zsum = 0.0f;
    int n = 0;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    const int64_t step = (int64_t)gridDim.x * BAL_WAVES * TPW;
    for (int64_t t0 = span.begin + ((int64_t)blockIdx.x * BAL_WAVES + wave) * TPW; t0 < span.end; t0 += step) {
        const int64_t t = t0 + lane / L;
        const bool inside = t < span.end && (token_mask == nullptr || token_mask[t] != 0);
        float l[V], q[V], lse = 0.0f;
        LaneRow<T, V>::load(logits + (inside ? t : t0) * experts, at * V, experts, vec, l);
        const bool valid = token_shares<V, L, SIGMOID, Z>(l, q, lse) && inside;
        if (valid) {
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] += l[i];
            if (at == 0) {
                n++;
                if (Z) zsum += lse * lse;
            }
            if (at < top_k) {
                const int e = expert_idx[t * top_k + at];
                if (e >= 0 && e < experts) atomicAdd(&routes[e], 1);
            }
        }
    }
#pragma unroll
    for (int off = L; off < 64; off <<= 1) {
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += __shfl_xor(acc[i], off, 64);
        zsum += __shfl_xor(zsum, off, 64);
        n += __shfl_xor(n, off, 64);
    }
    if (lane < L) {
#pragma unroll
        for (int i = 0; i < V; i++) shares[wave][at * V + i] = acc[i];
    }
    if (lane == 0) {
        rest[wave] = zsum;
        counted[wave] = n;
    }
    __syncthreads();
    float *out = part + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * (2 * experts + 2);
    for (int e = threadIdx.x; e < experts; e += BAL_THREADS) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < BAL_WAVES; w++) sum += shares[w][e];
        out[e] = sum;
        out[experts + e] = __int_as_float(routes[e]);
    }
    if (threadIdx.x == 0) {
        float sum = 0.0f;
        int all = 0;
#pragma unroll
        for (int w = 0; w < BAL_WAVES; w++) {
            sum += rest[w];
            all += counted[w];
        }
        out[2 * experts] = sum;
        out[2 * experts + 1] = __int_as_float(all);
    }
}

// The sum over the workgroup, in thread 0.
template <class N>
__device__ __forceinline__ N block_sum(N x, N (&scratch)[BAL_WAVES])
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    N sum = 0;
#pragma unroll
    for (int w = 0; w < BAL_WAVES; w++) sum += scratch[w];
    return sum;
}

// Workgroup s: the sequence's sums, counts and tokens; its loss to of_seq[2 s] and its sum of lse^2 behind it, or, of one sequence, the whole loss.
__global__ __launch_bounds__(BAL_THREADS) void moe_balance_sequence_kernel(const float *__restrict__ part, int chunks, int experts, int top_k, float coef, float z_coef,
                                                                          int32_t *__restrict__ counts, int32_t *__restrict__ seq_tokens, float *__restrict__ of_seq,
                                                                          float *__restrict__ loss)
{
    __shared__ float fs[BAL_WAVES];
    __shared__ int is[BAL_WAVES];
    const int pitch = 2 * experts + 2;
    const float *mine = part + (size_t)blockIdx.x * chunks * pitch;
    float zsum = 0.0f;
    int n = 0;
    for (int c = threadIdx.x; c < chunks; c += BAL_THREADS) {
        zsum += mine[(size_t)c * pitch + 2 * experts];
        n += __float_as_int(mine[(size_t)c * pitch + 2 * experts + 1]);
    }
    zsum = block_sum(zsum, fs);
    n = block_sum(n, is);
    float sum = 0.0f;
    for (int e = threadIdx.x; e < experts; e += BAL_THREADS) {
        float p = 0.0f;
        int routes = 0;
#pragma unroll 8
        for (int c = 0; c < chunks; c++) {
            p += mine[(size_t)c * pitch + e];
            routes += __float_as_int(mine[(size_t)c * pitch + experts + e]);
        }
        counts[(size_t)blockIdx.x * experts + e] = routes;
        sum += p * (float)routes;
    }
    sum = block_sum(sum, fs);
    if (threadIdx.x == 0) {
        seq_tokens[blockIdx.x] = n;
        const float tokens = (float)max(n, 1), r = sum / tokens * ((float)experts / ((float)top_k * tokens));
        if (gridDim.x == 1) {
            *loss = coef * r + z_coef * (zsum / tokens);
        } else {
            of_seq[2 * blockIdx.x] = r;
            of_seq[2 * blockIdx.x + 1] = zsum;
        }
    }
}

__global__ __launch_bounds__(BAL_THREADS) void moe_balance_loss_kernel(const float *__restrict__ of_seq, const int32_t *__restrict__ seq_tokens, int sequences, float coef,
                                                                      float z_coef, float *__restrict__ loss)
{
    __shared__ float fs[BAL_WAVES];
    __shared__ int is[BAL_WAVES];
    float r = 0.0f, z = 0.0f;
    int alive = 0, n = 0;
    for (int s = threadIdx.x; s < sequences; s += BAL_THREADS) {
        r += of_seq[2 * s];
        z += of_seq[2 * s + 1];
        n += seq_tokens[s];
        alive += seq_tokens[s] > 0;
    }
    r = block_sum(r, fs);
    z = block_sum(z, fs);
    n = block_sum(n, is);
    alive = block_sum(alive, is);
    if (threadIdx.x == 0) *loss = coef * (r / (float)max(alive, 1)) + z_coef * (z / (float)max(n, 1));
}

// Workgroup (c, s): tokens of sequence s; the first and the last sequence's also write the zeros of tokens before and behind all sequences.
template <class T, int V, int L, bool SIGMOID, bool Z>
__global__ __launch_bounds__(BAL_THREADS) void moe_balance_backward_kernel(const float *__restrict__ grad_loss, const T *__restrict__ logits,
                                                                          const uint8_t *__restrict__ token_mask, const int32_t *__restrict__ seq_offsets,
                                                                          const int32_t *__restrict__ counts, const int32_t *__restrict__ seq_tokens, int tokens, int experts,
                                                                          int top_k, float coef, float z_coef, T *__restrict__ grad_logits, bool vec)
{
    constexpr int TPW = 64 / L;
    __shared__ int is[BAL_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & (L - 1);
    const int sequences = gridDim.y, s = blockIdx.y;
    int alive = 0, all = 0;
    if (sequences > 1) {
        for (int i = threadIdx.x; i < sequences; i += BAL_THREADS) {
            all += seq_tokens[i];
            alive += seq_tokens[i] > 0;
        }
        all = block_sum(all, is);
        alive = block_sum(alive, is);
    } else {
        all = seq_tokens[0];
        alive = 1;
    }
    const float g = *grad_loss, n = (float)max(seq_tokens[s], 1);
    const float unit = g * coef / ((float)max(alive, 1) * n) * ((float)experts / ((float)top_k * n)), zunit = 2.0f * g * z_coef / (float)max(all, 1);
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = at * V + i < experts ? unit * (float)counts[(size_t)s * experts + at * V + i] : 0.0f;
    const Span span = span_of(seq_offsets, s, tokens);
    const int begin = s == 0 ? 0 : span.begin, end = s == sequences - 1 ? tokens : span.end;
    const int64_t step = (int64_t)gridDim.x * BAL_WAVES * TPW;
    for (int64_t t0 = begin + ((int64_t)blockIdx.x * BAL_WAVES + wave) * TPW; t0 < end; t0 += step) {
        const int64_t t = t0 + lane / L;
        const bool inside = t >= span.begin && t < span.end && (token_mask == nullptr || token_mask[t] != 0);
        float l[V], q[V], d[V], keep[V], lse = 0.0f;
        LaneRow<T, V>::load(logits + (t < end ? t : t0) * experts, at * V, experts, vec, l);
        if (SIGMOID) {
#pragma unroll
            for (int i = 0; i < V; i++) keep[i] = 1.0f / (1.0f + __expf(l[i]));   // 1 - sigmoid
        }
        const bool valid = token_shares<V, L, SIGMOID, Z>(l, q, lse) && inside;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) dot += l[i] * v[i];
        dot = lanes_sum<L>(dot);
#pragma unroll
        for (int i = 0; i < V; i++) {
            d[i] = l[i] * (v[i] - dot);
            if (SIGMOID) d[i] *= keep[i];
            if (Z) d[i] += zunit * lse * q[i];
            if (!valid) d[i] = 0.0f;
        }
        if (t < end) LaneRow<T, V>::store(grad_logits + t * experts, at * V, experts, vec, d);
    }
}

static int balance_shape(const char *what, int dtype, int64_t tokens, int64_t experts, int top_k, int64_t sequences, const int32_t *seq_offsets, int scoring)
{
    CCH_REQUIRE(logits_type_ok(dtype), "%s: logits of type %d", what, dtype);
    CCH_REQUIRE(tokens >= 0 && tokens < (int64_t)1 << 31, "%s: %lld tokens", what, (long long)tokens);
    CCH_REQUIRE(experts >= 1 && experts <= ROUTER_MAX_EXPERTS, "%s: num_experts=%lld outside 1..%d", what, (long long)experts, ROUTER_MAX_EXPERTS);
    CCH_REQUIRE(top_k >= 1 && top_k <= ROUTER_MAX_TOPK, "%s: top_k=%d outside 1..%d", what, top_k, ROUTER_MAX_TOPK);
    CCH_REQUIRE(sequences >= 1 && sequences <= BAL_MAX_SEQUENCES && (seq_offsets || sequences == 1), "%s: num_sequences=%lld (1..%d, 1 without offsets)", what,
                (long long)sequences, BAL_MAX_SEQUENCES);
    CCH_REQUIRE(tokens * top_k < (int64_t)1 << 31, "%s: %lld routes", what, (long long)(tokens * top_k));
    CCH_REQUIRE(scoring == CCH_SCORING_SOFTMAX || scoring == CCH_SCORING_SIGMOID, "%s: scoring %d", what, scoring);
    return CCH_OK;
}

// Workgroups per sequence.
static int64_t balance_chunks(int64_t tokens, int64_t experts, int64_t sequences)
{
    const int64_t per = BAL_WAVES * (experts <= 64 ? 8 : experts <= 256 ? 4 : experts <= 512 ? 2 : 1);   // tokens of a workgroup at a time
    const int64_t fill = (256 + sequences - 1) / sequences, need = (tokens + per - 1) / per;
    return std::max<int64_t>(1, std::min(fill, need));
}

}  // namespace cch

extern "C" int64_t cch_moe_balance_loss_workspace_bytes(int64_t tokens, int64_t num_experts, int64_t num_sequences)
{
    if (tokens < 0 || num_experts < 1 || num_experts > cch::ROUTER_MAX_EXPERTS || num_sequences < 1 || num_sequences > cch::BAL_MAX_SEQUENCES) return 0;
    return 4 * (2 * num_sequences + num_sequences * cch::balance_chunks(tokens, num_experts, num_sequences) * (2 * num_experts + 2));
}

extern "C" int cch_moe_balance_loss(const void *logits, int dtype, const int32_t *expert_idx, const uint8_t *token_mask, const int32_t *seq_offsets, int64_t tokens,
                                    int64_t num_experts, int top_k, int64_t num_sequences, int scoring, float coef, float z_coef, float *loss, int32_t *counts,
                                    int32_t *seq_tokens, void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace cch;
    if (const int rc = balance_shape("cch_moe_balance_loss", dtype, tokens, num_experts, top_k, num_sequences, seq_offsets, scoring)) return rc;
    CCH_REQUIRE(loss && counts && seq_tokens && (tokens == 0 || (logits && expert_idx)), "cch_moe_balance_loss: null pointer");
    const int64_t need = cch_moe_balance_loss_workspace_bytes(tokens, num_experts, num_sequences);
    CCH_REQUIRE(workspace && aligned(workspace, 4) && workspace_bytes >= need, "cch_moe_balance_loss: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
                (long long)need);
    const int chunks = (int)balance_chunks(tokens, num_experts, num_sequences);
    float *of_seq = static_cast<float *>(workspace), *part = of_seq + 2 * num_sequences;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = with_logits_type(dtype, [&](auto *type) {
        return with_lanes((int)num_experts, [&](auto v, auto lanes) {
            typedef std::remove_pointer_t<decltype(type)> T;
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value;
            auto kern = scoring == CCH_SCORING_SIGMOID ? (z_coef != 0 ? moe_balance_sums_kernel<T, V, L, true, true> : moe_balance_sums_kernel<T, V, L, true, false>)
                                                       : (z_coef != 0 ? moe_balance_sums_kernel<T, V, L, false, true> : moe_balance_sums_kernel<T, V, L, false, false>);
            hipLaunchKernelGGL(kern, dim3((unsigned)chunks, (unsigned)num_sequences), dim3(BAL_THREADS), 0, s, static_cast<const T *>(logits), expert_idx, token_mask,
                               seq_offsets, (int)tokens, (int)num_experts, top_k, part, LaneRow<T, V>::vec(logits, num_experts));
            return launch_status("moe_balance_sums_kernel");
        });
    });
    if (rc != CCH_OK) return rc;
    hipLaunchKernelGGL(moe_balance_sequence_kernel, dim3((unsigned)num_sequences), dim3(BAL_THREADS), 0, s, part, chunks, (int)num_experts, top_k, coef, z_coef, counts,
                       seq_tokens, of_seq, loss);
    if (num_sequences > 1)
        hipLaunchKernelGGL(moe_balance_loss_kernel, dim3(1), dim3(BAL_THREADS), 0, s, of_seq, seq_tokens, (int)num_sequences, coef, z_coef, loss);
    return launch_status("moe_balance_sequence_kernel");
}

extern "C" int cch_moe_balance_loss_backward(const float *grad_loss, const void *logits, int dtype, const uint8_t *token_mask, const int32_t *seq_offsets,
                                             const int32_t *counts, const int32_t *seq_tokens, int64_t tokens, int64_t num_experts, int top_k, int64_t num_sequences,
                                             int scoring, float coef, float z_coef, void *grad_logits, void *stream)
{
    using namespace cch;
    if (const int rc = balance_shape("cch_moe_balance_loss_backward", dtype, tokens, num_experts, top_k, num_sequences, seq_offsets, scoring)) return rc;
    if (tokens == 0) return CCH_OK;
    CCH_REQUIRE(grad_loss && logits && counts && seq_tokens && grad_logits, "cch_moe_balance_loss_backward: null pointer");
    return with_logits_type(dtype, [&](auto *type) {
        return with_lanes((int)num_experts, [&](auto v, auto lanes) {
            typedef std::remove_pointer_t<decltype(type)> T;
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value, PER = BAL_WAVES * (64 / L);
            const int64_t need = (tokens + PER - 1) / PER, fill = (2048 + num_sequences - 1) / num_sequences;
            auto kern = scoring == CCH_SCORING_SIGMOID
                            ? (z_coef != 0 ? moe_balance_backward_kernel<T, V, L, true, true> : moe_balance_backward_kernel<T, V, L, true, false>)
                            : (z_coef != 0 ? moe_balance_backward_kernel<T, V, L, false, true> : moe_balance_backward_kernel<T, V, L, false, false>);
            hipLaunchKernelGGL(kern, dim3((unsigned)std::max<int64_t>(1, std::min(need, fill)), (unsigned)num_sequences), dim3(BAL_THREADS), 0,
                               static_cast<hipStream_t>(stream), grad_loss, static_cast<const T *>(logits), token_mask, seq_offsets, counts, seq_tokens, (int)tokens,
                               (int)num_experts, top_k, coef, z_coef, static_cast<T *>(grad_logits),
                               LaneRow<T, V>::vec(logits, num_experts) && aligned(grad_logits, 16));
            return launch_status("moe_balance_backward_kernel");
        });
    });
}
