// The balance loss of a mixture of experts, the z loss and the routes per expert, and the gradient of the logits.
//
// Of a sequence s with N_s tokens that count (not masked, at least one logit above -inf), c_se routes to expert e and k routes per token, E experts:
//   f_se = E c_se / (k N_s),  P_se = mean over its tokens of p_te,  p = softmax(l), or sigmoid(l) / sum over experts of sigmoid(l)
//   loss = coef * mean over sequences with N_s > 0 of sum_e f_se P_se  +  z_coef * mean over all N tokens of lse_t^2,  lse_t = log sum_e exp(l_te)
// Without sequence offsets the whole batch is one sequence.  Routes are whole numbers without a gradient, so
//   dl_te = coef / (S' N_s) p_te (f_se - sum_i p_ti f_si) [(1 - sigmoid(l_te)) for sigmoid scores] + z_coef 2 lse_t softmax(l)_te / N
// times the loss's own gradient.
//
// Forward, where one workgroup is not enough: a workgroup takes a run of tokens, whatever sequences they belong to; of each of those it leaves the sums of p (fp32 in registers) and the routes
// (LDS) in the workspace, and a second launch adds a sequence's sums up, in their order, so that the same inputs give the same bits.  The last workgroup of that
// launch has the loss.  Backward: one pass, logits in, gradient out.
//
// Bound by the logits' bytes on paper (16384 tokens of 256 experts, bf16: 8.4 MB read, then 16.8 MB read and written, 5.1 us at the rate of a large copy), by launches
// and waits for memory in fact: that batch in 13 sequences with sigmoid scores takes 8.6 to 11 + 4.5 + 2.4 us forward and 10 backward, where an empty launch takes 2.4 and every
// workgroup has two steps of 16 tokens, the exponentials of all being 1.3 us of the card's time.
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

// Where a workgroup of token `first` on stands among the sequences, from one look at all of them: the sequence that holds `first`, or the one before it where none
// does (as many sequences begin at or before it, less one; -1: none), the number of sequences with tokens, and the tokens of all.  `staged` (the workgroup's, in
// LDS) then holds the offsets of up to THREADS - 1 sequences.
struct Place {
    int s, alive, all;
};
template <int THREADS, bool COUNTS, bool ALL>
__device__ __forceinline__ Place place_of(const int32_t *offsets, const int32_t *seq_tokens, int sequences, int first, int32_t *staged, int (&scratch)[3][THREADS / 64])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0, alive = 0, all = 0;
    for (int i0 = 0; i0 <= sequences; i0 += THREADS) {
        const int i = i0 + (int)threadIdx.x;
        int offset = 0, n = 0;
        if (offsets && i <= sequences) offset = offsets[i];
        if (COUNTS && i < sequences) n = seq_tokens[i];
        if (i0 == 0) staged[threadIdx.x] = offset;
        before += __builtin_popcountll(__ballot(i < sequences && offset <= first));
        if (COUNTS) alive += __builtin_popcountll(__ballot(n > 0));
        if (ALL) all += n;
    }
    if (ALL) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off, 64);
    }
    if (lane == 0) {
        scratch[0][wave] = before;
        scratch[1][wave] = alive;
        scratch[2][wave] = all;
    }
    __syncthreads();
    Place p = {-1, 0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) {
        p.s += scratch[0][w];
        p.alive += scratch[1][w];
        p.all += scratch[2][w];
    }
    if (offsets == nullptr) p.s = 0;
    p.s = __builtin_amdgcn_readfirstlane(p.s);
    return p;
}

// A token's p (in place of l) and for sigmoid scores `rest` = 1 - sigmoid(l); with z also softmax(l) in `q` and the log of the sum of exponentials.  False: no logit
// is above -inf (NaN is not).
template <int V, int L, bool SIGMOID>
__device__ __forceinline__ bool token_shares(float (&l)[V], float (&rest)[V], float (&q)[V], float &lse, bool z)
{
    float top = l[0];
#pragma unroll
    for (int i = 1; i < V; i++) top = fmaxf(top, l[i]);
    top = lanes_max<L>(top);
    float sum = 0.0f;
    if (!SIGMOID || z) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            q[i] = exp_of(l[i] - top);
            sum += q[i];
        }
        sum = lanes_sum<L>(sum);
        if (z) lse = __logf(sum) + top;
        const float over = reciprocal(sum);
#pragma unroll
        for (int i = 0; i < V; i++) q[i] *= over;
    }
    if (!SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; i++) l[i] = q[i];
        return top > -INFINITY;
    }
    sum = 0.0f;
    if (__ballot(!(top >= SIGMOID_IN_RANGE)) == 0) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            sigmoid_pair(l[i], l[i], rest[i]);
            sum += l[i];
        }
    } else {
        const float c = fminf(top, 0.0f), ec = exp_of(c);
#pragma unroll
        for (int i = 0; i < V; i++) {
            rest[i] = reciprocal(1.0f + exp_of(l[i]));
            l[i] = scaled_sigmoid(l[i], c, ec);
            sum += l[i];
        }
    }
    const float over = reciprocal(lanes_sum<L>(sum));
#pragma unroll
    for (int i = 0; i < V; i++) l[i] *= over;
    return top > -INFINITY;
}

// The sum over the workgroup, in every thread.
template <int WAVES, class N>
__device__ __forceinline__ N block_sum(N x, N (&scratch)[WAVES])
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    N sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) sum += scratch[w];
    return sum;
}

// What is read of a token; all of it at once, a step ahead.  (The mask, then the experts of those that it leaves, are two waits for memory in every step, which other workgroups
// hide: 16384 tokens of 256 experts in 13 sequences 10.1 and 11.2 us in the median that way, 11.5 and 11.0 this way.)
template <class T, int V, bool VEC>
struct TokenIn {
    LaneRow<T, V, VEC> row;
    uint32_t mask;
    int e;
    __device__ __forceinline__ void load(const T *logits, const uint8_t *token_mask, const int32_t *expert_idx, int t, int at, int experts, int top_k)
    {
        row.load(logits + (int64_t)t * experts, at * V, experts);
        mask = token_mask ? token_mask[t] : 1;
        e = -1;
        if (at < top_k) e = expert_idx[(int64_t)t * top_k + at];
    }
    __device__ __forceinline__ void load(const T *logits, const uint8_t *token_mask, int t, int at, int experts)
    {
        row.load(logits + (int64_t)t * experts, at * V, experts);
        mask = token_mask ? token_mask[t] : 1;
    }
};

// The workgroup's sums over tokens [from, to), STEP at a time, the first of them in `token`: in lanes 0 .. L - 1 of a wave p per expert, in every lane sum of lse^2 and
// tokens of the wave; routes per expert in LDS.
template <class T, int V, int L, bool SIGMOID, bool VEC, int STEP>
__device__ __forceinline__ void add_tokens(TokenIn<T, V, VEC> &token, const T *logits, const int32_t *expert_idx, const uint8_t *token_mask, int from, int to, int mine,
                                           int experts, int top_k, bool z, int32_t *routes, float (&acc)[V], float &zsum, int &n)
{
    const int lane = threadIdx.x & 63, at = lane & (L - 1);
    zsum = 0.0f;
    n = 0;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    for (int t1 = from; t1 < to; t1 += STEP) {
        const int t = t1 + mine;
        TokenIn<T, V, VEC> next;
        next.load(logits, token_mask, expert_idx, min(t + STEP, to - 1), at, experts, top_k);
        const bool inside = t < to && token.mask != 0;
        float l[V], rest[V], q[V], lse = 0.0f;
        token.row.values(at * V, experts, l);
        const bool valid = token_shares<V, L, SIGMOID>(l, rest, q, lse, z) && inside;
        if (valid) {
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] += l[i];
            if (at == 0) {
                n++;
                if (z) zsum += lse * lse;
            }
            if (token.e >= 0 && token.e < experts) atomicAdd(&routes[token.e], 1);
        }
        token = next;
    }
#pragma unroll
    for (int off = L; off < 64; off <<= 1) {
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += __shfl_xor(acc[i], off, 64);
        zsum += __shfl_xor(zsum, off, 64);
        n += __shfl_xor(n, off, 64);
    }
    zsum = __shfl(zsum, 0, 64);
    n = __shfl(n, 0, 64);
}

// All of it in one workgroup, for one sequence of few tokens.  In us, sigmoid scores, against the launches below: 512 tokens of 16 experts 5.4 / 6.5, 1024 tokens 7.3 / 6.6;
// 64 experts, 256 tokens 6.0 / 6.7, 512 tokens 7.9 / 6.9; 256 experts, 128 tokens 8.0 / 10.0, 256 tokens 12.0 / 10.0; 1024 experts, 32 tokens 8.6 / 11.1, 64 tokens
// 13.5 / 11.2.  So: four steps at most, and 2^14 logits, 2^15 of more than 64 experts, where the launches below are three.
template <int L>
constexpr int ONE_THREADS = L > 32 ? 512 : 1024;   // (the waves' sums fit LDS)
constexpr int ONE_STEPS = 4;
template <class T, int V, int L, bool SIGMOID, bool VEC>
__global__ __launch_bounds__(ONE_THREADS<L>) void moe_balance_one_kernel(const T *__restrict__ logits, const int32_t *__restrict__ expert_idx,
                                                                     const uint8_t *__restrict__ token_mask, const int32_t *__restrict__ seq_offsets, int tokens, int experts,
                                                                     int top_k, float coef, float z_coef, float *__restrict__ loss, int32_t *__restrict__ counts,
                                                                     int32_t *__restrict__ seq_tokens)
{
    constexpr int THREADS = ONE_THREADS<L>, WAVES = THREADS / 64, TPW = 64 / L, STEP = WAVES * TPW;
    __shared__ float shares[WAVES][V * L], fs[WAVES];
    __shared__ int32_t routes[V * L], is[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & (L - 1), mine = wave * TPW + lane / L;
    const Span span = span_of(seq_offsets, 0, tokens);
    TokenIn<T, V, VEC> token;
    if (span.begin < span.end) token.load(logits, token_mask, expert_idx, min(span.begin + mine, span.end - 1), at, experts, top_k);
    for (int e = threadIdx.x; e < V * L; e += THREADS) routes[e] = 0;
    __syncthreads();
    float acc[V], zsum;
    int n;
    add_tokens<T, V, L, SIGMOID, VEC, STEP>(token, logits, expert_idx, token_mask, span.begin, span.end, mine, experts, top_k, z_coef != 0, routes, acc, zsum, n);
    if (lane < L) {
#pragma unroll
        for (int i = 0; i < V; i++) shares[wave][at * V + i] = acc[i];
    }
    zsum = block_sum(lane == 0 ? zsum : 0.0f, fs);
    n = block_sum(lane == 0 ? n : 0, is);
    float sum = 0.0f;
    for (int e = threadIdx.x; e < experts; e += THREADS) {
        float p = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) p += shares[w][e];
        counts[e] = routes[e];
        sum += p * (float)routes[e];
    }
    sum = block_sum(sum, fs);
    if (threadIdx.x == 0) {
        const float counted = (float)max(n, 1);
        *seq_tokens = n;
        *loss = coef * (sum / counted * ((float)experts / ((float)top_k * counted))) + z_coef * (zsum / counted);
    }
}

// Tokens [run * blockIdx.x, ...) of `run`; what they add to sequence s goes to part[(blockIdx.x + s) * (2 experts + 2)]: p per expert, routes per expert, sum of
// lse^2, tokens.  (Workgroups in order and sequences in order: no two meet.)
template <class T, int V, int L, bool SIGMOID, bool VEC>
__global__ __launch_bounds__(BAL_THREADS) void moe_balance_sums_kernel(const T *__restrict__ logits, const int32_t *__restrict__ expert_idx,
                                                                      const uint8_t *__restrict__ token_mask, const int32_t *__restrict__ seq_offsets, int tokens,
                                                                      int experts, int top_k, int sequences, int run, float *__restrict__ part, bool z)
{
    constexpr int TPW = 64 / L, STEP = BAL_WAVES * TPW;   // tokens of a wave and of the workgroup at a time
    __shared__ float shares[BAL_WAVES][V * L], zsums[BAL_WAVES];
    __shared__ int32_t routes[V * L], counted[BAL_WAVES], staged[BAL_THREADS], scratch[3][BAL_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), at = lane & (L - 1);
    const int first = (int)blockIdx.x * run, end = min(first + run, tokens);
    const int mine = wave * TPW + lane / L;
    if (first >= end) return;
    // the first rows are on their way while the sequences are looked at
    TokenIn<T, V, VEC> token;
    token.load(logits, token_mask, expert_idx, min(first + mine, end - 1), at, experts, top_k);
    int s = max(place_of<BAL_THREADS, false, false>(seq_offsets, nullptr, sequences, first, staged, scratch).s, 0);
    const int32_t *const offsets = seq_offsets && sequences < BAL_THREADS ? staged : seq_offsets;
    for (; s < sequences; s++) {
        const Span span = span_of(offsets, s, tokens);
        if (span.begin >= end) break;
        const int from = max(span.begin, first), to = min(span.end, end);
        if (from >= to) continue;
        if (from > first) token.load(logits, token_mask, expert_idx, min(from + mine, to - 1), at, experts, top_k);
        for (int e = threadIdx.x; e < V * L; e += BAL_THREADS) routes[e] = 0;
        __syncthreads();
        float acc[V], zsum;
        int n;
        add_tokens<T, V, L, SIGMOID, VEC, STEP>(token, logits, expert_idx, token_mask, from, to, mine, experts, top_k, z, routes, acc, zsum, n);
        if (lane < L) {
#pragma unroll
            for (int i = 0; i < V; i++) shares[wave][at * V + i] = acc[i];
        }
        if (lane == 0) {
            zsums[wave] = zsum;
            counted[wave] = n;
        }
        __syncthreads();
        float *out = part + ((size_t)blockIdx.x + s) * (2 * experts + 2);
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
                sum += zsums[w];
                all += counted[w];
            }
            out[2 * experts] = sum;
            out[2 * experts + 1] = __int_as_float(all);
        }
        __syncthreads();
    }
}

// Workgroup (b, s): experts 64 b ... of sequence s, a wave to every sixteenth workgroup's sums, sixteen of them on their way together (four: 16384 tokens of 16 experts
// 9.8 us for the whole forward pass instead of 8.9).  One workgroup alone has the loss; of several each leaves its
// share, the sum of lse^2 and the tokens in of_seq, for the launch below.  (The last of them to come could add these up instead, but publishing them to one
// another takes longer than a launch: 9.5 us against 3.0 for 16 experts, the caches of the card's parts being written back.)
constexpr int FIN_THREADS = 1024, FIN_WAVES = FIN_THREADS / 64;
__global__ __launch_bounds__(FIN_THREADS) void moe_balance_finish_kernel(const float *__restrict__ part, const int32_t *__restrict__ seq_offsets, int tokens, int experts,
                                                                        int top_k, int run, float coef, float z_coef, int32_t *__restrict__ counts,
                                                                        int32_t *__restrict__ seq_tokens, float *__restrict__ of_seq, float *__restrict__ loss)
{
    __shared__ float fs[FIN_WAVES], shares[FIN_WAVES][64];
    __shared__ int is[FIN_WAVES], routes[FIN_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.y, sequences = gridDim.y, blocks = gridDim.x;
    const int e = (int)blockIdx.x * 64 + lane, pitch = 2 * experts + 2;
    const Span span = span_of(seq_offsets, s, tokens);
    const int c0 = span.begin / run, c1 = span.end > span.begin ? (span.end - 1) / run + 1 : c0;
    const float *mine = part + (size_t)s * pitch;
    float p = 0.0f, zsum = 0.0f;
    int r = 0, n = 0;
    if (e < experts) {
        constexpr int MANY = 16;   // on their way together
        for (int first = c0 + wave; first < c1; first += MANY * FIN_WAVES) {
            float v[MANY];
            int q[MANY];
#pragma unroll
            for (int u = 0; u < MANY; u++) {
                const float *from = mine + (size_t)min(first + u * FIN_WAVES, c1 - 1) * pitch + e;
                v[u] = from[0];
                q[u] = __float_as_int(from[experts]);
            }
#pragma unroll
            for (int u = 0; u < MANY; u++) {
                p += first + u * FIN_WAVES < c1 ? v[u] : 0.0f;
                r += first + u * FIN_WAVES < c1 ? q[u] : 0;
            }
        }
    }
    for (int c = c0 + (int)threadIdx.x; c < c1; c += FIN_THREADS) {
        zsum += mine[(size_t)c * pitch + 2 * experts];
        n += __float_as_int(mine[(size_t)c * pitch + 2 * experts + 1]);
    }
    shares[wave][lane] = p;
    routes[wave][lane] = r;
    zsum = block_sum(zsum, fs);
    n = block_sum(n, is);
    const float counted = (float)max(n, 1);
    if (wave == 0) {
        p = 0.0f;
        r = 0;
#pragma unroll
        for (int w = 0; w < FIN_WAVES; w++) {
            p += shares[w][lane];
            r += routes[w][lane];
        }
        if (e < experts) counts[(size_t)s * experts + e] = r;
        float sum = p * (float)r;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if (lane == 0) {
            sum = sum / counted * ((float)experts / ((float)top_k * counted));
            if (blockIdx.x == 0) seq_tokens[s] = n;
            if (blocks * sequences == 1) {
                *loss = coef * sum + z_coef * (zsum / counted);
            } else {
                float *to = of_seq + ((size_t)s * blocks + blockIdx.x) * 3;
                to[0] = sum;
                to[1] = zsum;
                to[2] = __int_as_float(n);
            }
        }
    }
}

__global__ __launch_bounds__(BAL_THREADS) void moe_balance_loss_kernel(const float *__restrict__ of_seq, int blocks, int sequences, float coef, float z_coef,
                                                                      float *__restrict__ loss)
{
    __shared__ float fs[BAL_WAVES];
    __shared__ int is[BAL_WAVES];
    float total = 0.0f, z = 0.0f;
    int alive = 0, all = 0;
    for (int i = threadIdx.x; i < sequences; i += BAL_THREADS) {
        const float *from = of_seq + (size_t)i * blocks * 3;
        for (int b = 0; b < blocks; b++) total += from[3 * b];
        z += from[1];
        const int m = __float_as_int(from[2]);
        all += m;
        alive += m > 0;
    }
    total = block_sum(total, fs);
    z = block_sum(z, fs);
    all = block_sum(all, is);
    alive = block_sum(alive, is);
    if (threadIdx.x == 0) *loss = coef * (total / (float)max(alive, 1)) + z_coef * (z / (float)max(all, 1));
}

// Tokens [run * blockIdx.x, ...) of `run`, sequence by sequence; those before and behind all sequences get zeros.
template <class T, int V, int L, bool SIGMOID, bool VEC>
__global__ __launch_bounds__(BAL_THREADS) void moe_balance_backward_kernel(const float *__restrict__ grad_loss, const T *__restrict__ logits,
                                                                          const uint8_t *__restrict__ token_mask, const int32_t *__restrict__ seq_offsets,
                                                                          const int32_t *__restrict__ counts, const int32_t *__restrict__ seq_tokens, int tokens, int experts,
                                                                          int top_k, int sequences, int run, float coef, float z_coef, T *__restrict__ grad_logits)
{
    constexpr int TPW = 64 / L, STEP = BAL_WAVES * TPW;
    __shared__ int32_t staged[BAL_THREADS];
    __shared__ int scratch[3][BAL_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), at = lane & (L - 1);
    const int first = (int)blockIdx.x * run, end = min(first + run, tokens), mine = wave * TPW + lane / L;
    TokenIn<T, V, VEC> token;
    token.load(logits, token_mask, min(first + mine, end - 1), at, experts);
    const float g = *grad_loss;
    const bool z = z_coef != 0;
    const Place place = place_of<BAL_THREADS, true, true>(seq_offsets, seq_tokens, sequences, first, staged, scratch);
    const int32_t *const offsets = seq_offsets && sequences < BAL_THREADS ? staged : seq_offsets;
    const float zunit = 2.0f * g * z_coef / (float)max(place.all, 1);
    for (int s = place.s; s <= sequences; s++) {
        const bool real = s >= 0 && s < sequences;
        Span span = {0, 0};
        if (real) span = span_of(offsets, s, tokens);
        else if (offsets) span = s < 0 ? Span{0, min(max(offsets[0], 0), tokens)} : Span{min(max(offsets[sequences], 0), tokens), tokens};
        if (span.begin >= end) break;
        const int from = max(span.begin, first), to = min(span.end, end);
        if (from >= to) continue;
        if (from > first) token.load(logits, token_mask, min(from + mine, to - 1), at, experts);
        float v[V];
        const float n = real ? (float)max(seq_tokens[s], 1) : 1.0f, unit = g * coef / ((float)max(place.alive, 1) * n) * ((float)experts / ((float)top_k * n));
        constexpr int FEW = VEC && V >= 4 ? 4 : VEC ? 2 : 1;   // counts of one access
        typedef int32_t Counts __attribute__((ext_vector_type(FEW)));
#pragma unroll
        for (int i = 0; i < V; i += FEW) {
            Counts c = {};
            if (real && at * V + i < experts) c = *reinterpret_cast<const Counts *>(counts + (size_t)s * experts + at * V + i);
#pragma unroll
            for (int u = 0; u < FEW; u++) v[i + u] = unit * (float)c[u];
        }
        for (int t1 = from; t1 < to; t1 += STEP) {
            const int t = t1 + mine;
            TokenIn<T, V, VEC> next;
            next.load(logits, token_mask, min(t + STEP, to - 1), at, experts);
            const bool inside = real && t < to && token.mask != 0;
            float l[V], rest[V], q[V], d[V], lse = 0.0f;
            token.row.values(at * V, experts, l);
            const bool valid = token_shares<V, L, SIGMOID>(l, rest, q, lse, z) && inside;
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) dot += l[i] * v[i];
            dot = lanes_sum<L>(dot);
#pragma unroll
            for (int i = 0; i < V; i++) {
                d[i] = l[i] * (v[i] - dot);
                if (SIGMOID) d[i] *= rest[i];
                if (z) d[i] += zunit * lse * q[i];
                if (!valid) d[i] = 0.0f;
            }
            if (t < to) LaneRow<T, V, VEC>::store(grad_logits + (int64_t)t * experts, at * V, experts, d);
            token = next;
        }
    }
}

static int balance_shape(const char *what, int dtype, int64_t tokens, int64_t experts, int top_k, int64_t sequences, const int32_t *seq_offsets, int scoring)
{
    CCH_REQUIRE(logits_type_ok(dtype), "%s: logits of type %d", what, dtype);
    CCH_REQUIRE(tokens >= 0 && tokens <= ROUTER_MAX_TOKENS, "%s: %lld tokens", what, (long long)tokens);
    CCH_REQUIRE(experts >= 1 && experts <= ROUTER_MAX_EXPERTS, "%s: num_experts=%lld outside 1..%d", what, (long long)experts, ROUTER_MAX_EXPERTS);
    CCH_REQUIRE(top_k >= 1 && top_k <= ROUTER_MAX_TOPK, "%s: top_k=%d outside 1..%d", what, top_k, ROUTER_MAX_TOPK);
    CCH_REQUIRE(sequences >= 1 && sequences <= BAL_MAX_SEQUENCES && (seq_offsets || sequences == 1), "%s: num_sequences=%lld (1..%d, 1 without offsets)", what,
                (long long)sequences, BAL_MAX_SEQUENCES);
    CCH_REQUIRE(tokens * top_k < (int64_t)1 << 31, "%s: %lld routes", what, (long long)(tokens * top_k));
    CCH_REQUIRE(scoring == CCH_SCORING_SOFTMAX || scoring == CCH_SCORING_SIGMOID, "%s: scoring %d", what, scoring);
    return CCH_OK;
}

// Tokens of a workgroup: several steps of it, so that the sums left in the workspace stay fewer than the logits and reading the sequences is paid once, but two
// workgroups to a CU where there are tokens for them (262144 tokens of 64 experts, forward with up to 4 / 16 / 64 steps 28.7 / 21.6 / 21.7 us, backward with 1 / 4 / 16
// 20.3 / 15.5 / 16.7; of 256 experts 52.6 / 42.6 / 45.0 and 71 / 44 / 45); more steps than `most` only where the launch would have 2^32 threads.
template <int L>
static int balance_run(int64_t tokens, int most)
{
    constexpr int STEP = BAL_WAVES * (64 / L);
    return STEP * (int)std::max<int64_t>({1, std::min<int64_t>(most, tokens / (512 * STEP)), tokens / ((int64_t)STEP << 23)});
}
constexpr int BAL_STEPS = 16, BAL_BACKWARD_STEPS = 4;   // at most

static int64_t balance_runs(int64_t tokens, int64_t experts)
{
    return with_lanes((int)experts, [&](auto, auto lanes) {
        const int run = balance_run<decltype(lanes)::value>(tokens, BAL_STEPS);
        return (int)((tokens + run - 1) / run);
    });
}
struct BalanceWorkspace {
    int64_t part, end;
};
static BalanceWorkspace balance_workspace(int64_t tokens, int64_t experts, int64_t sequences)
{
    BalanceWorkspace w{};
    w.part = sequences * ((experts + 63) / 64) * 3 * 4;
    w.end = w.part + (balance_runs(tokens, experts) + sequences) * (2 * experts + 2) * 4;
    return w;
}

}  // namespace cch

extern "C" int64_t cch_moe_balance_loss_workspace_bytes(int64_t tokens, int64_t num_experts, int64_t num_sequences)
{
    if (tokens < 0 || tokens > cch::ROUTER_MAX_TOKENS || num_experts < 1 || num_experts > cch::ROUTER_MAX_EXPERTS || num_sequences < 1 || num_sequences > cch::BAL_MAX_SEQUENCES) return 0;
    return cch::balance_workspace(tokens, num_experts, num_sequences).end;
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
    const BalanceWorkspace at = balance_workspace(tokens, num_experts, num_sequences);
    uint8_t *p = static_cast<uint8_t *>(workspace);
    float *of_seq = reinterpret_cast<float *>(p), *part = reinterpret_cast<float *>(p + at.part);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int run = 1;
    bool one = false;
    const int rc = with_logits_type(dtype, [&](auto *type) {
        return with_lanes((int)num_experts, [&](auto v, auto lanes) {
            typedef std::remove_pointer_t<decltype(type)> T;
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value;
            run = balance_run<L>(tokens, BAL_STEPS);
            const bool vec = LanePieces<T, V>::vec(logits, num_experts);
            // (its comment has both sides)
            one = tokens > 0 && num_sequences == 1 && tokens <= ONE_STEPS * (ONE_THREADS<L> / L) && tokens * V * L <= (V * L <= 64 ? 1 << 14 : 1 << 15);
            if (one) {
                auto kern = scoring == CCH_SCORING_SIGMOID ? (vec ? moe_balance_one_kernel<T, V, L, true, true> : moe_balance_one_kernel<T, V, L, true, false>)
                                                           : (vec ? moe_balance_one_kernel<T, V, L, false, true> : moe_balance_one_kernel<T, V, L, false, false>);
                hipLaunchKernelGGL(kern, dim3(1), dim3(ONE_THREADS<L>), 0, s, static_cast<const T *>(logits), expert_idx, token_mask, seq_offsets, (int)tokens, (int)num_experts,
                                   top_k, coef, z_coef, loss, counts, seq_tokens);
                return launch_status("moe_balance_one_kernel");
            }
            auto kern = scoring == CCH_SCORING_SIGMOID ? (vec ? moe_balance_sums_kernel<T, V, L, true, true> : moe_balance_sums_kernel<T, V, L, true, false>)
                                                       : (vec ? moe_balance_sums_kernel<T, V, L, false, true> : moe_balance_sums_kernel<T, V, L, false, false>);
            hipLaunchKernelGGL(kern, dim3((unsigned)std::max<int64_t>(1, (tokens + run - 1) / run)), dim3(BAL_THREADS), 0, s, static_cast<const T *>(logits), expert_idx,
                               token_mask, seq_offsets, (int)tokens, (int)num_experts, top_k, (int)num_sequences, run, part,
                               z_coef != 0);
            return launch_status("moe_balance_sums_kernel");
        });
    });
    if (rc != CCH_OK || one) return rc;
    const dim3 grid((unsigned)((num_experts + 63) / 64), (unsigned)num_sequences);
    hipLaunchKernelGGL(moe_balance_finish_kernel, grid, dim3(FIN_THREADS), 0, s, part, seq_offsets, (int)tokens, (int)num_experts, top_k, run, coef, z_coef, counts, seq_tokens,
                       of_seq, loss);
    if (grid.x * grid.y > 1)
        hipLaunchKernelGGL(moe_balance_loss_kernel, dim3(1), dim3(BAL_THREADS), 0, s, of_seq, (int)grid.x, (int)num_sequences, coef, z_coef, loss);
    return launch_status("moe_balance_finish_kernel");
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
            constexpr int V = decltype(v)::value, L = decltype(lanes)::value;
            const int run = balance_run<L>(tokens, BAL_BACKWARD_STEPS);
            const bool vec = LanePieces<T, V>::vec(logits, num_experts) && aligned(grad_logits, 16) && aligned(counts, 16);
            auto kern = scoring == CCH_SCORING_SIGMOID ? (vec ? moe_balance_backward_kernel<T, V, L, true, true> : moe_balance_backward_kernel<T, V, L, true, false>)
                                                       : (vec ? moe_balance_backward_kernel<T, V, L, false, true> : moe_balance_backward_kernel<T, V, L, false, false>);
            hipLaunchKernelGGL(kern, dim3((unsigned)((tokens + run - 1) / run)), dim3(BAL_THREADS), 0, static_cast<hipStream_t>(stream), grad_loss,
                               static_cast<const T *>(logits), token_mask, seq_offsets, counts, seq_tokens, (int)tokens, (int)num_experts, top_k, (int)num_sequences, run, coef,
                               z_coef, static_cast<T *>(grad_logits));
            return launch_status("moe_balance_backward_kernel");
        });
    });
}
