// Products of bf16 or half operands with fp32 sums: the problem that the kernels take (gemm16_kernel.h), how it is launched, and the preparation of
// operands whose rows start on no 16-byte boundary.
#pragma once
#include <atomic>

#include "common.h"

namespace cch {

constexpr int MAX_GROUPS16 = 1024;
constexpr int64_t MAX_PITCH16 = (int64_t)1 << 22;   // elements of a row as stored: 256 of them stay below 2^31 bytes, which a request's offset holds

enum Layout16 { ROWS_NK = 0, ROWS_NN = 1, ROWS_TN = 2 };
// ROWS_NK: A [M, K], B [N, K].  ROWS_NN: A [M, K], B [K, N].  ROWS_TN: A [K, M], B [K, N].
enum Epilogue16 {
    EPI16_OUT = 0,    // out = scale * sum, rounded; or fp32 sums kept and added to (`sums`)
    EPI16_ACT = 1,    // z = sum + bias, kept if asked for; out = act(z) + residual
    EPI16_STATS = 2,  // cross entropy: a row's largest logit and sum of exponentials per 64 columns, and its target's logit
    EPI16_GRAD = 3,   // cross entropy: the logits' gradient times grad_scale
};

// The kernels, numbered as the switch "matmul16_kernel" names them: tiles of 128 x 128, 256 x 256, and of few rows.
enum Kernel16 { KERNEL16_128 = 0, KERNEL16_256 = 1, KERNEL16_ROWS = 2, NUM_KERNELS16 };
constexpr int64_t BIG_TILES16 = 192;     // tiles of 256 x 256 from which on they are taken: three quarters of the CUs
struct Plan16 {
    int kernel, splits, deep;   // Kernel16, parts of K, four stages (tiles of 128 x 128)
    int tail;                   // tiles of 256 x 256: how many parts of its last round's tiles there may be (0: that round is not split)
};
// Tiles of 256 x 256: in how many parts the K of the last round's `left` tiles is worked on by `grid` workgroups, at most `most` parts in all.  In ns, measured: a step of a tile; a
// part's sums to memory and back (256 KiB each way); the second launch.  Integers: the product's kernel and the one that joins the parts decide it alike.
constexpr int TAIL16_MOST = 8, TAIL16_STEPS = 64;   // (from TAIL16_MOST^2 steps on every part has some)
constexpr int64_t TAIL16_BYTES = 256 * 256 * 4;
__host__ __device__ inline int tail_parts16(int left, int grid, int steps, int most)
{
    constexpr int STEP = 1450, PART = 110, JOIN = 6000;
    int parts = 1, best = STEP * steps;
    if (left <= 0 || steps < TAIL16_STEPS) return 1;
    for (int s = 2; s <= TAIL16_MOST && left * s <= most; s++) {
        const int ns = (left * s + grid - 1) / grid * ((steps + s - 1) / s) * STEP + left * s * PART + JOIN;
        if (ns < best) {
            best = ns;
            parts = s;
        }
    }
    return parts;
}
Plan16 plan16(const struct Gemm16 &p, int layout, int epilogue);
extern std::atomic<int> g_kernel16;   // -1: chosen per problem; else that one wherever it takes the problem

struct Gemm16 {
    const uint16_t *a, *b;
    uint16_t *out;
    int64_t pitch_a, pitch_b, pitch_out;   // elements between rows as stored: multiples of 8 for a and b, whose addresses are multiples of 16 bytes
    int m, n, k;                           // with groups: all groups' rows (or, k_grouped, all groups' K)
    int64_t b_stride, out_stride;          // elements between the groups' B (rows grouped), outputs (K grouped)
    const int32_t *group_sizes;            // device, or nullptr: one group of everything.  Clipped to 0..what is left
    int groups;
    int k_grouped;                         // 0: a group is a range of rows of A and of the output; 1: a range of K (ROWS_TN)
    int zero_rest;                         // rows behind the last group are written as zeros
    const int32_t *a_rows;                 // ROWS_NK: row of A that is row i of the product (m_src rows there; below 2^31 bytes), or nullptr
    int m_src;
    const int32_t *out_rows;               // row of the output that row i goes to, or nullptr
    int half;                              // IEEE half, else bf16
    float *partial;                        // fp32, for sums of parts of K; K is not split where partial_bytes are too few
    int64_t partial_bytes;
    int splits;                            // parts of K (set by the launch)
    int tail;                              // Plan16::tail (set by the launch)
    // EPI16_OUT
    const float *scale;                    // device, or nullptr: 1
    float *sums;                           // fp32 [m, n], or nullptr: a product in pieces of K.  sums_in: added to the sum; sums_out: takes it in place of out
    int sums_in, sums_out;
    // EPI16_ACT
    const uint16_t *bias, *residual;
    uint16_t *preact;
    int act;
    // EPI16_STATS, EPI16_GRAD (columns are v0 + 0..n-1 of the vocabulary)
    int v0;
    const int32_t *targets;                // per row of the product
    float2 *stats;                         // [m, stat_cols]
    int stat_cols;
    float *target_logit;
    const float *lse;                      // per row of the product
    float z2;                              // 2 * z_coef
    const float *grad_scale;               // device, or nullptr: 1
};

// Bytes of `partial` that the product may use (its sizes, groups and pointers' being there or not as at the launch; no GPU needed).
int64_t partial16_bytes(const Gemm16 &p, int layout, int epilogue);
int gemm16_launch(const Gemm16 &p, int layout, int epilogue, hipStream_t stream);

// Tiles that a launch may have: the groups' sizes are on the device.
inline int64_t tiles16(const Gemm16 &p, int tm, int tn)
{
    const int64_t cols = (p.n + tn - 1) / tn;
    if (p.k_grouped) return (int64_t)p.groups * ((p.m + tm - 1) / tm) * cols;
    return (p.group_sizes ? p.m / tm + (p.groups < p.m ? p.groups : p.m) : (p.m + tm - 1) / tm) * cols;
}
// Rows of a tile of the kernel for few rows: a group's share of them.
inline int rows16(const Gemm16 &p)
{
    const int share = (int)(((int64_t)p.m + p.groups - 1) / p.groups);
    return share <= 8 ? 8 : share <= 16 ? 16 : 32;
}

inline bool whole16(int64_t cols) { return cols % 8 == 0; }
inline int64_t pitch16(int64_t cols) { return (cols + 7) & ~(int64_t)7; }
inline int64_t round256(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }
// Bytes of the copy that rows of `cols` elements need (0: none, they are whole multiples of 16 bytes).
inline int64_t padded16_bytes(int64_t rows, int64_t cols) { return whole16(cols) ? 0 : round256(rows * pitch16(cols) * 2); }

// A workspace handed out front to back.
struct Carve {
    uint8_t *at;
    template <class T> T *take(int64_t bytes)
    {
        T *p = reinterpret_cast<T *>(at);
        at += round256(bytes);
        return p;
    }
    // What is left of a workspace to a product's parts.
    void rest(Gemm16 &p, void *workspace, int64_t bytes) const
    {
        p.partial = reinterpret_cast<float *>(at);
        p.partial_bytes = workspace ? static_cast<uint8_t *>(workspace) + bytes - at : 0;
    }
};

// An operand's rows of `cols` elements, back to back.  `whole_operands16` makes copies in rows of pitch16(cols), zeros behind them, of those that are no whole multiples of 16 bytes
// (space from `ws`), and points `at` there; an operand that is not there (nullptr) stays so.  With sizes (device), `group_rows` rows belong to a group each, and those of groups without
// rows of their own are not copied (9 tokens over 128 experts x 1152 x 1007, K-major: 222 us with all of them, 39 so).
struct Operand16 {
    const uint16_t *at;
    int64_t rows, cols;
    const int32_t *sizes = nullptr;
    int64_t group_rows = 1;
};
int whole_operands16(Operand16 *operands, int n, Carve &ws, hipStream_t stream);

int fill_zero16(uint16_t *dst, int64_t n, hipStream_t stream);
// dz = grad_out * act'(preact) in rows of pitch16(n) and its column sums; either may be left out.  partial: column_sum_bytes(...) of fp32
int64_t column_sum_bytes(int64_t m, int64_t n);
int act_backward16(const uint16_t *grad_out, const uint16_t *preact, uint16_t *dz, uint16_t *grad_bias, float *partial, int64_t m, int64_t n, int act, int half, hipStream_t stream);

}  // namespace cch
