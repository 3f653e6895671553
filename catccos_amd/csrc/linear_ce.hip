// Softmax cross entropy of hidden states x [t, h] against an output projection w [v, h], without the logits:
//   l = x w^T,  lse_i = log sum_j exp l_ij,  nll_i = lse_i - l_i,target;  loss = mean (or sum) of nll + z lse^2 over the tokens that count
//   d_ij = g (p_ij (1 + 2 z lse_i) - [j = target_i]),  p = exp(l - lse);  dx = d w,  dw = d^T x
// Tokens whose target lies outside the vocabulary do not count: the ones that do are numbered first, and every product is over those rows alone, so that masked ones cost
// nothing and what they hold (an infinity, a NaN) reaches nothing.  Forward: the product's epilogue leaves each row's largest logit and sum of exponentials per 64 columns
// and the target's logit, a second launch joins them.  Backward: a piece of the vocabulary at a time, its logits are computed again, the epilogue turns them into d, rounded to
// 16 bits (it is the next two products' operand), which the products for dw and dx read; with more than one piece dx is added up in fp32.
#include <algorithm>

#include "gemm16_device.h"

namespace cch {

constexpr int64_t CE_MAX_TOKENS = (int64_t)1 << 30, CE_MAX_VOCAB = (int64_t)1 << 30;
constexpr int CE_STAT = 64;                                   // columns of one pair of statistics
constexpr int64_t CE_PIECE_BYTES = (int64_t)256 << 20;        // of d at a time
// Half cannot hold p of a large vocabulary: d is kept times 2^11 there, which leaves p above 2^-25 at full precision.  |d| can be as large as |1 + 2 z lse|, or as that
// number's distance to 1: where this passes 31 for some token, d is kept times the largest power of two that leaves it at 31 * 2^11 or less (half ends at 65504).
constexpr float CE_HALF_SCALE = 2048.0f, CE_HALF_MOST = 31.0f;

static int64_t ce_piece(int64_t t, int64_t v)
{
    const int64_t most = std::min<int64_t>(std::max<int64_t>(CE_PIECE_BYTES / 2 / std::max<int64_t>(t, 1) / 256 * 256, 1024), 1 << 20);
    if (v <= most) return v;
    const int64_t pieces = (v + most - 1) / most;
    return std::min<int64_t>(((v + pieces - 1) / pieces + 255) / 256 * 256, v);
}

// ---- the tokens that count, in their order: src[i] the i-th one, target[i] its target, count[0] how many; scalars[0] what the gradient's products are multiplied by, scalars[1]
// what d is kept times.  The others' nll and lse are zero.  One workgroup, four tokens to a thread and round.
constexpr int CE_THREADS = 1024, CE_PER = 4;
struct CeTokens {
    const void *targets;
    int target_bytes;
    int t, v;
    int32_t *src, *pos, *target, *count;
    const float *lse_in;         // backward: gathered to lse
    float *lse;
    float *nll_out, *lse_out;    // forward
    int32_t *tokens;             // forward
    const float *grad_loss;      // backward
    const int32_t *divisor;
    float *scalars;
    float z2;                    // 2 * z_coef
    int half, mean;
};
__global__ __launch_bounds__(CE_THREADS) void ce_tokens_kernel(CeTokens p)
{
    __shared__ int sums[2][CE_THREADS / 64];
    __shared__ float largest[CE_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0, par = 0;
    float most = 0.0f;   // of |d|, this thread's tokens
    for (int base = 0; base < p.t; base += CE_THREADS * CE_PER, par ^= 1) {
        const int first = base + (int)threadIdx.x * CE_PER;
        int64_t tg[CE_PER];
        int n = 0;
#pragma unroll
        for (int i = 0; i < CE_PER; i++) {
            tg[i] = -1;
            if (first + i < p.t) tg[i] = p.target_bytes == 8 ? static_cast<const int64_t *>(p.targets)[first + i] : (int64_t)static_cast<const int32_t *>(p.targets)[first + i];
            if (tg[i] >= p.v) tg[i] = -1;
            n += tg[i] >= 0;
        }
        const int incl = (int)wave_scan_sat((uint32_t)n);
        if (lane == 63) sums[par][wave] = incl;
        __syncthreads();   // (the buffer's other half is read until the next round's barrier)
        int at = before + incl - n;
#pragma unroll
        for (int w = 0; w < CE_THREADS / 64; w++) {
            const int s = sums[par][w];
            if (w < wave) at += s;
            before += s;
        }
#pragma unroll
        for (int i = 0; i < CE_PER; i++) {
            const int t = first + i;
            if (t >= p.t) break;
            if (p.pos) p.pos[t] = tg[i] >= 0 ? at : -1;
            if (tg[i] >= 0) {
                p.src[at] = t;
                p.target[at] = (int32_t)tg[i];
                if (p.lse) {
                    const float lse = p.lse_in[t], f = 1.0f + p.z2 * lse, d = fmaxf(f, 1.0f - f);
                    p.lse[at] = lse;
                    if (d < INFINITY) most = fmaxf(most, d);   // (not a NaN's either: such a token's row says so itself)
                }
                at++;
            } else if (p.nll_out) {
                p.nll_out[t] = 0.0f;
                p.lse_out[t] = 0.0f;
            }
        }
    }
    if (threadIdx.x == 0) {
        p.count[0] = before;
        if (p.tokens) p.tokens[0] = before;
    }
    if (!p.scalars) return;
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) largest[wave] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        float scale = p.half ? CE_HALF_SCALE : 1.0f;
        for (int w = 0; w < CE_THREADS / 64; w++) most = fmaxf(most, largest[w]);
        if (p.half)
            for (; most > CE_HALF_MOST; most *= 0.5f) scale *= 0.5f;
        p.scalars[0] = p.grad_loss[0] / (p.mean ? (float)max(p.divisor[0], 1) : 1.0f) / scale;
        p.scalars[1] = scale;
    }
}

// One wave to a counted token and turn: its partial statistics joined.  (A launch holds fewer than 2^32 threads: beyond, it is cut short without an error.)
constexpr int CE_JOIN_BLOCKS = 1 << 16;
__global__ __launch_bounds__(256) void ce_join_kernel(const float2 *__restrict__ stats, const float *__restrict__ logit, const int32_t *__restrict__ src,
                                                      const int32_t *__restrict__ count, float *__restrict__ nll, float *__restrict__ lse, int cols)
{
    const int lane = threadIdx.x & 63, tokens = count[0];
    for (int i = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6); i < tokens; i += (int)gridDim.x * 4) {
        const float2 *s = stats + (int64_t)i * cols;
        float top = -INFINITY, sum = 0.0f;
        for (int c = lane; c < cols; c += 64) {
            const float2 v = s[c];
            const float m = fmaxf(top, v.x);
            sum = (top > -INFINITY || sum != sum ? sum * __expf(top - m) : 0.0f) + (v.x > -INFINITY || v.y != v.y ? v.y * __expf(v.x - m) : 0.0f);
            top = m;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const float ot = __shfl_xor(top, d), os = __shfl_xor(sum, d), m = fmaxf(top, ot);
            sum = (sum == 0.0f ? 0.0f : sum * __expf(top - m)) + (os == 0.0f ? 0.0f : os * __expf(ot - m));
            top = m;
        }
        if (lane == 0) {
            const float l = top + logf(sum);
            const int t = src[i];
            lse[t] = l;
            nll[t] = l - logit[i];
        }
    }
}

// loss = (sum of nll + z * sum of lse^2) / tokens, sums in 64 bits in a fixed order: one workgroup.
__global__ __launch_bounds__(CE_THREADS) void ce_loss_kernel(const float *__restrict__ nll, const float *__restrict__ lse, const int32_t *__restrict__ tokens, float *loss, int t,
                                                             float z, int mean)
{
    __shared__ double sums[CE_THREADS / 64];
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < t; i += CE_THREADS) s += (double)nll[i] + (double)z * ((double)lse[i] * (double)lse[i]);
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < CE_THREADS / 64; w++) all += sums[w];
        loss[0] = (float)(mean ? all / max(tokens[0], 1) : all);
    }
}

// Rows of x that count, one behind the other (rows of pitch16(h), zeros behind h); the others' rows of grad_x are zeros.  pos: a token's place or -1.
__global__ __launch_bounds__(256) void ce_gather_kernel(const uint16_t *__restrict__ x, const int32_t *__restrict__ pos, uint16_t *__restrict__ rows, uint16_t *__restrict__ grad_x,
                                                        int64_t chunks, int64_t h, int64_t per_row)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per_row, c = (i - t * per_row) * 8;
        const int at = pos[t];
        const int left = (int)min(h - c, (int64_t)8);
        if (at >= 0) {
            if (!rows) continue;
            const uint16_t *s = x + t * h + c;
            v4i o = {};
            if (left >= 8) o = reinterpret_cast<const Unaligned16 *>(s)->v;
            else
#pragma unroll
                for (int k = 0; k < 7; k++)
                    if (k < left) o[k >> 1] |= (int)((uint32_t)s[k] << (16 * (k & 1)));
            *reinterpret_cast<v4i *>(rows + (int64_t)at * per_row * 8 + c) = o;
        } else if (grad_x) {
            uint16_t *o = grad_x + t * h + c;
            if (left >= 8) reinterpret_cast<Unaligned16 *>(o)->v = (v4i){0, 0, 0, 0};
            else
#pragma unroll
                for (int k = 0; k < 7; k++)
                    if (k < left) o[k] = 0;
        }
    }
}

static int ce_gather(const uint16_t *x, const int32_t *pos, uint16_t *rows, uint16_t *grad_x, int64_t t, int64_t h, hipStream_t s)
{
    const int64_t per_row = pitch16(h) / 8, chunks = t * per_row;
    if (chunks == 0) return CCH_OK;
    hipLaunchKernelGGL(ce_gather_kernel, dim3((unsigned)std::min<int64_t>((chunks + 255) / 256, 1 << 16)), dim3(256), 0, s, x, pos, rows, grad_x, chunks, h, per_row);
    return launch_status("ce_gather_kernel");
}

// Rows of x are picked by the product's requests where it runs on tiles of 128 x 128, offsets of 32 bits reach them all and none needs padding; else they are copied.
static bool ce_picks(int64_t t, int64_t h, int64_t v) { return whole16(h) && t * h * 2 <= 0x7FFFFFF0 && ((t + 255) / 256) * ((v + 255) / 256) < BIG_TILES16; }

// The two products of a piece of c columns of the gradient, pointers apart.
static const int32_t CE_COUNT = 0;   // stands for the number of tokens that count, where only that there is one matters
static Gemm16 ce_grad_w(const int32_t *count, int64_t t, int64_t h, int64_t c)
{
    Gemm16 p{};
    p.pitch_a = pitch16(c);
    p.pitch_b = pitch16(h);
    p.pitch_out = h;
    p.m = (int)c;
    p.n = (int)h;
    p.k = (int)t;
    p.k_grouped = 1;
    p.groups = 1;
    p.group_sizes = count;
    return p;
}
static Gemm16 ce_grad_x(const int32_t *count, const int32_t *src, float *sums, int64_t t, int64_t h, int64_t c)
{
    Gemm16 p{};
    p.pitch_a = pitch16(c);
    p.pitch_b = pitch16(h);
    p.pitch_out = h;
    p.m = (int)t;
    p.n = (int)h;
    p.k = (int)c;
    p.groups = 1;
    p.group_sizes = count;
    p.out_rows = src;
    p.sums = sums;
    return p;
}

struct CeWorkspace {
    int64_t src, pos, target, lse, count, scalars, logit, stats, rows, w, d, sums, parts, end;
};
static CeWorkspace ce_workspace(int64_t t, int64_t h, int64_t v, bool backward)
{
    CeWorkspace at{};
    auto piece = [&](int64_t bytes) {
        const int64_t a = at.end;
        at.end += round256(bytes);
        return a;
    };
    at.src = piece(t * 4);
    at.target = piece(t * 4);
    at.count = piece(4);
    at.w = piece(padded16_bytes(v, h));
    if (backward || !ce_picks(t, h, v)) {
        at.pos = piece(t * 4);
        at.rows = piece(t * pitch16(h) * 2);
    }
    if (!backward) {
        at.logit = piece(t * 4);
        at.stats = piece(t * ((v + CE_STAT - 1) / CE_STAT) * 8);
    } else {
        const int64_t c = ce_piece(t, v);
        float some;   // (stands for sums that are there)
        at.lse = piece(t * 4);
        at.scalars = piece(8);
        at.d = piece(t * pitch16(c) * 2);
        if (c < v) at.sums = piece(t * h * 4);
        at.parts = piece(std::max(partial16_bytes(ce_grad_w(&CE_COUNT, t, h, c), ROWS_TN, EPI16_OUT),
                                  partial16_bytes(ce_grad_x(&CE_COUNT, &CE_COUNT, c < v ? &some : nullptr, t, h, c), ROWS_NN, EPI16_OUT)));
    }
    return at;
}

static bool ce_fits(int64_t t, int64_t h, int64_t v) { return t >= 0 && t <= CE_MAX_TOKENS && h >= 1 && h <= MAX_PITCH16 && v >= 1 && v <= CE_MAX_VOCAB; }

static int ce_check(const char *what, int64_t t, int64_t h, int64_t v, int target_bytes, int reduction, int dtype)
{
    CCH_REQUIRE(ce_fits(t, h, v), "%s: bad shape t=%lld h=%lld v=%lld (at most 2^30, 2^22, 2^30)", what, (long long)t, (long long)h, (long long)v);
    CCH_REQUIRE(target_bytes == 4 || target_bytes == 8, "%s: targets of %d bytes (4 or 8)", what, target_bytes);
    CCH_REQUIRE(reduction == CCH_REDUCE_MEAN || reduction == CCH_REDUCE_SUM, "%s: reduction %d", what, reduction);
    CCH_REQUIRE(dtype == CCH_DTYPE_BF16 || dtype == CCH_DTYPE_F16, "%s: operands of type %d", what, dtype);
    return CCH_OK;
}

}  // namespace cch

using namespace cch;

extern "C" int64_t cch_linear_cross_entropy_workspace_bytes(int64_t t, int64_t h, int64_t v) { return ce_fits(t, h, v) ? ce_workspace(t, h, v, false).end : 0; }
extern "C" int64_t cch_linear_cross_entropy_backward_workspace_bytes(int64_t t, int64_t h, int64_t v) { return ce_fits(t, h, v) ? ce_workspace(t, h, v, true).end : 0; }

extern "C" int cch_linear_cross_entropy(const void *x, const void *w, const void *targets, int target_bytes, float *loss, float *nll, float *lse, int32_t *tokens, int64_t t,
                                        int64_t h, int64_t v, int reduction, float z_coef, int dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = ce_check("cch_linear_cross_entropy", t, h, v, target_bytes, reduction, dtype)) return rc;
    const CeWorkspace at = ce_workspace(t, h, v, false);
    CCH_REQUIRE(loss && tokens && w && (t == 0 || (x && targets && nll && lse)), "cch_linear_cross_entropy: null pointer");
    CCH_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(targets, target_bytes), "cch_linear_cross_entropy: x and w must lie on 16-byte boundaries");
    CCH_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= at.end, "cch_linear_cross_entropy: workspace of %lld bytes, need %lld on a 256-byte boundary",
                (long long)(workspace ? workspace_bytes : 0), (long long)at.end);
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    auto i32 = [&](int64_t o) { return reinterpret_cast<int32_t *>(ws + o); };
    auto f32 = [&](int64_t o) { return reinterpret_cast<float *>(ws + o); };
    const bool picks = ce_picks(t, h, v);

    CeTokens tk{};
    tk.targets = targets;
    tk.target_bytes = target_bytes;
    tk.t = (int)t;
    tk.v = (int)v;
    tk.src = i32(at.src);
    tk.pos = picks ? nullptr : i32(at.pos);
    tk.target = i32(at.target);
    tk.count = i32(at.count);
    tk.nll_out = nll;
    tk.lse_out = lse;
    tk.tokens = tokens;
    hipLaunchKernelGGL(ce_tokens_kernel, dim3(1), dim3(CE_THREADS), 0, s, tk);
    if (const int rc = launch_status("ce_tokens_kernel")) return rc;
    if (t > 0) {
        Gemm16 p{};
        p.a = static_cast<const uint16_t *>(x);
        p.pitch_a = pitch16(h);
        if (picks) {
            p.a_rows = tk.src;
            p.m_src = (int)t;
        } else {
            uint16_t *rows = reinterpret_cast<uint16_t *>(ws + at.rows);
            if (const int rc = ce_gather(p.a, tk.pos, rows, nullptr, t, h, s)) return rc;
            p.a = rows;
        }
        Carve wc{ws + at.w};
        Operand16 in{static_cast<const uint16_t *>(w), v, h};
        if (const int rc = whole_operands16(&in, 1, wc, s)) return rc;
        p.b = in.at;
        p.pitch_b = pitch16(h);
        p.m = (int)t;
        p.n = (int)v;
        p.k = (int)h;
        p.group_sizes = tk.count;
        p.groups = 1;
        p.half = dtype == CCH_DTYPE_F16;
        p.targets = tk.target;
        p.target_logit = f32(at.logit);
        p.stats = reinterpret_cast<float2 *>(ws + at.stats);
        p.stat_cols = (int)((v + CE_STAT - 1) / CE_STAT);
        if (const int rc = gemm16_launch(p, ROWS_NK, EPI16_STATS, s)) return rc;
        hipLaunchKernelGGL(ce_join_kernel, dim3((unsigned)std::min<int64_t>((t + 3) / 4, CE_JOIN_BLOCKS)), dim3(256), 0, s, p.stats, p.target_logit, tk.src, tk.count, nll, lse, p.stat_cols);
        if (const int rc = launch_status("ce_join_kernel")) return rc;
    }
    hipLaunchKernelGGL(ce_loss_kernel, dim3(1), dim3(CE_THREADS), 0, s, nll, lse, tokens, loss, (int)t, z_coef, (int)(reduction == CCH_REDUCE_MEAN));
    return launch_status("ce_loss_kernel");
}

extern "C" int cch_linear_cross_entropy_backward(const float *grad_loss, const void *x, const void *w, const void *targets, int target_bytes, const float *lse,
                                                 const int32_t *tokens, void *grad_x, void *grad_w, int64_t t, int64_t h, int64_t v, int reduction, float z_coef, int dtype,
                                                 void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = ce_check("cch_linear_cross_entropy_backward", t, h, v, target_bytes, reduction, dtype)) return rc;
    const CeWorkspace at = ce_workspace(t, h, v, true);
    CCH_REQUIRE(grad_loss && tokens && w && (t == 0 || (x && targets && lse)), "cch_linear_cross_entropy_backward: null pointer");
    CCH_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(targets, target_bytes) && aligned(grad_x, 2) && aligned(grad_w, 2),
                "cch_linear_cross_entropy_backward: x and w must lie on 16-byte boundaries");
    CCH_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= at.end, "cch_linear_cross_entropy_backward: workspace of %lld bytes, need %lld on a 256-byte boundary",
                (long long)(workspace ? workspace_bytes : 0), (long long)at.end);
    if (!grad_x && !grad_w) return CCH_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    auto i32 = [&](int64_t o) { return reinterpret_cast<int32_t *>(ws + o); };
    auto f32 = [&](int64_t o) { return reinterpret_cast<float *>(ws + o); };
    const int half = dtype == CCH_DTYPE_F16;
    uint16_t *gx = static_cast<uint16_t *>(grad_x), *gw = static_cast<uint16_t *>(grad_w);

    CeTokens tk{};
    tk.targets = targets;
    tk.target_bytes = target_bytes;
    tk.t = (int)t;
    tk.v = (int)v;
    tk.src = i32(at.src);
    tk.pos = i32(at.pos);
    tk.target = i32(at.target);
    tk.count = i32(at.count);
    tk.lse_in = lse;
    tk.lse = f32(at.lse);
    tk.grad_loss = grad_loss;
    tk.divisor = tokens;
    tk.scalars = f32(at.scalars);
    tk.z2 = 2.0f * z_coef;
    tk.half = half;
    tk.mean = reduction == CCH_REDUCE_MEAN;
    hipLaunchKernelGGL(ce_tokens_kernel, dim3(1), dim3(CE_THREADS), 0, s, tk);
    if (const int rc = launch_status("ce_tokens_kernel")) return rc;
    uint16_t *rows = reinterpret_cast<uint16_t *>(ws + at.rows), *d = reinterpret_cast<uint16_t *>(ws + at.d);
    if (const int rc = ce_gather(static_cast<const uint16_t *>(x), tk.pos, rows, gx, t, h, s)) return rc;
    Operand16 in{static_cast<const uint16_t *>(w), v, h};
    Carve wc{ws + at.w};
    if (const int rc = whole_operands16(&in, 1, wc, s)) return rc;
    const uint16_t *pw = in.at;
    const int64_t ldw = pitch16(h);

    const int64_t piece = ce_piece(t, v);
    for (int64_t v0 = 0; v0 < v; v0 += piece) {
        const int64_t c = std::min(piece, v - v0);
        if (t > 0) {
            Gemm16 p{};
            p.half = half;
            p.groups = 1;
            p.group_sizes = tk.count;
            p.a = rows;
            p.pitch_a = pitch16(h);
            p.b = pw + v0 * ldw;
            p.pitch_b = ldw;
            p.out = d;
            p.pitch_out = pitch16(c);
            p.m = (int)t;
            p.n = (int)c;
            p.k = (int)h;
            p.v0 = (int)v0;
            p.targets = tk.target;
            p.lse = tk.lse;
            p.z2 = tk.z2;
            p.grad_scale = half ? tk.scalars + 1 : nullptr;
            if (const int rc = gemm16_launch(p, ROWS_NK, EPI16_GRAD, s)) return rc;
        }
        const Carve parts{ws + at.parts};
        if (gw) {
            Gemm16 q = ce_grad_w(tk.count, t, h, c);
            q.half = half;
            q.a = d;
            q.b = rows;
            q.out = gw + v0 * h;
            q.scale = tk.scalars;
            parts.rest(q, workspace, workspace_bytes);
            if (const int rc = gemm16_launch(q, ROWS_TN, EPI16_OUT, s)) return rc;
        }
        if (gx && t > 0) {
            Gemm16 q = ce_grad_x(tk.count, tk.src, piece < v ? f32(at.sums) : nullptr, t, h, c);
            q.half = half;
            q.a = d;
            q.b = pw + v0 * ldw;
            q.out = gx;
            q.scale = tk.scalars;
            q.sums_in = v0 > 0;
            q.sums_out = v0 + piece < v;
            parts.rest(q, workspace, workspace_bytes);
            if (const int rc = gemm16_launch(q, ROWS_NN, EPI16_OUT, s)) return rc;
        }
    }
    return CCH_OK;
}
