// What the products of 16-bit operands need around their kernels: the choice by type, copies of operands whose rows start on no 16-byte boundary, and the
// first step of a layer's backward pass.
#include <algorithm>

#include "gemm16_device.h"

namespace cch {

int gemm16_launch_bf16(const Gemm16 &p, const Plan16 &plan, int layout, int epilogue, hipStream_t stream);   // gemm16_bf16.hip
int gemm16_launch_f16(const Gemm16 &p, const Plan16 &plan, int layout, int epilogue, hipStream_t stream);    // gemm16_f16.hip
std::atomic<int> g_kernel16{-1};

// ---- which kernel, and K in how many parts: by sizes alone, so that what a call's workspace holds does not depend on the device.
// Estimates in us beyond an empty launch, fitted to products of 1 to 512 rows, 512 to 7168 columns and K of 512 to 8192.
Plan16 plan16(const Gemm16 &p, int layout, int epilogue)
{
    constexpr int CUS = 256;
    constexpr double MEMORY = 5.1e6;   // bytes a us
    const int asked = g_kernel16.load();
    Plan16 plan{KERNEL16_128, 1, 0, 0};
    const bool results = epilogue == EPI16_OUT || epilogue == EPI16_ACT;
    const bool rows_kernel = layout != ROWS_TN && results && !p.a_rows && !p.sums && !p.out_rows && !p.scale;
    if (rows_kernel && asked == KERNEL16_ROWS) return {KERNEL16_ROWS, 1, 0, 0};
    const bool big = !p.a_rows && p.pitch_out < MAX_PITCH16 / 2;
    const int64_t big_tiles = tiles16(p, 256, 256);
    Plan16 on_big{KERNEL16_256, 1, 0, 0};
    const int big_steps = (p.k + 63) / 64;
    if (layout != ROWS_TN && results && big_steps >= TAIL16_STEPS) {
        on_big.tail = (int)std::min<int64_t>(2 * CUS, TAIL16_MOST * big_tiles);
        if (!p.group_sizes && tail_parts16((int)(big_tiles % CUS), CUS, big_steps, on_big.tail) == 1) on_big.tail = 0;
    }
    if (big && (asked == KERNEL16_256 || (asked < 0 && big_tiles >= BIG_TILES16))) return on_big;
    // tiles of 128 x 128, about: a group's rows or K are taken to be its share
    const int64_t groups = p.k_grouped || !p.group_sizes ? p.groups : std::max(std::min(p.groups, p.m), 1);   // that may have rows
    const int64_t share = p.k_grouped || !p.group_sizes ? p.m : (p.m + groups - 1) / groups, each = (share + 127) / 128 * ((p.n + 127) / 128);
    const int64_t tiles = each * groups, steps = ((p.k_grouped ? (p.k + groups - 1) / groups : p.k) + 63) / 64;
    const double weights = 2.0 * p.n * p.k * groups / MEMORY;
    double best = 0;
    for (int s = 1; s <= 32 && (s == 1 || (s <= steps && results && !p.sums && tiles < CUS)); s++) {
        // a step of a workgroup with four stages, longer the more of them share the caches; the second launch, and the parts' way to memory and back (128 x 1024 x 8192 in 1, 2,
        // 4, 8, 16 parts: 47, 30, 21, 17.5, 18.7 us; 256 x 4096 x 7168 in 1, 2, 4, 8: 45, 32, 34, 33; 512 x 1024 x 1024: 12.2, 13.5, 14.4, 19.9)
        const double STEP = 0.32, SHARED = 0.18, JOIN = 1.7, PER_BYTE = 0.6e-6;
        const double fill = (double)(tiles * s) / CUS, rounds = fill <= 1 ? 1 : (double)((tiles * s + CUS - 1) / CUS);
        const double us = rounds * (double)((steps + s - 1) / s) * (STEP + SHARED * (fill < 1 ? fill : 1)) +
                          (s > 1 ? JOIN + s * 4.0 * p.m * p.n * (p.k_grouped ? groups : 1) * PER_BYTE : 0);
        if (s == 1 || us < best) {
            best = us;
            plan.splits = s;
        }
    }
    if (big && asked < 0 && on_big.tail) {
        // Few tiles of 256 x 256 and a long K, whose parts fill the chip (2000 of 4999 rows x 1984, K = 20011: 289 us on tiles of 128 x 128)
        const int parts = tail_parts16((int)big_tiles, CUS, big_steps, on_big.tail);
        const double us = (double)((big_tiles * parts + CUS - 1) / CUS) * ((big_steps + parts - 1) / parts) * 1.45 + (double)big_tiles * parts * 0.11 + 12;
        if (us < best) return on_big;
    }
    plan.deep = tiles * plan.splits <= CUS;
    if (rows_kernel && asked < 0 && share <= 128) {
        // The kernel for few rows: an eighth of the steps in a row, or the weights' way from memory, again for every tile of rows (from the caches).  K-major weights come in half
        // lines.  4096 x 7168: 1 row 15.4 us (128 x 128 tiles 18.3), 32 22.4 (19.3), K-major 29 (18.7); 7168 x 2048: 1 row 8.7 (13.9), 64 17.1 (16.7), K-major 12.1 (13.8);
        // 1024 x 1024: 1 row 4.9 (9.4), 96 5.9 (11.3), K-major 6.0 (9.5).  Its launch, prologue and epilogue take 2 us less than the others'.  Weights from memory in all of these;
        // where the caches hold them, 4096 x 7168: 1 row 11.5 (17.2), 32 15.6 (18.4), K-major 18.5 (17.8).  The estimate is off in two places: 17 to 32 rows of 4096 x 7168 come here, 3 to 12 %
        // slower than tiles with weights from memory; K-major 7168 x 2048 goes to tiles up to 32 rows, 15.1 to 16.0 where this kernel takes 12.3 to 14.6.
        const int mr = rows16(p);
        const int64_t row_tiles = (share + mr - 1) / mr, workgroups = row_tiles * groups * ((p.n + 31) / 32);
        const double step = (layout == ROWS_NN ? 0.9 : 0.31) * (mr == 32 ? 1.2 : 1.0) * (double)((workgroups + CUS - 1) / CUS);
        const double fetch = weights * (layout == ROWS_NN ? 2.0 : 1.0) * (1 + 0.4 * (row_tiles - 1));
        const double us = std::max((double)((steps + 7) / 8) * step, fetch);
        if (us <= std::max(best, weights) + 2.0) return {KERNEL16_ROWS, 1, 0, 0};
    }
    return plan;
}

static int64_t parts_bytes(const Gemm16 &p, int splits) { return splits > 1 ? round256((int64_t)splits * (p.k_grouped ? p.groups : 1) * p.m * p.n * 4) : 0; }
int64_t partial16_bytes(const Gemm16 &p, int layout, int epilogue)
{
    const Plan16 plan = plan16(p, layout, epilogue);
    return std::max(parts_bytes(p, plan.splits), plan.tail * TAIL16_BYTES);
}

// ---- the parts of K added up in their order, with the product's epilogue.  VEC elements of a row to a thread.
template <class T, int EPI, int VEC> __global__ __launch_bounds__(256) void join16_kernel(Gemm16 p, int64_t outputs, int64_t per_row)
{
    __shared__ int used;
    if (!p.k_grouped && p.group_sizes) {
        if (threadIdx.x < 64) {
            uint32_t sum = 0;
            for (int g = threadIdx.x; g < p.groups; g += 64) sum = sat_add(sum, (uint32_t)min(max(p.group_sizes[g], 0), p.m));
            const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_sat(sum), 63);
            if (threadIdx.x == 0) used = (int)min(all, (uint32_t)p.m);
        }
        __syncthreads();
    } else {
        if (threadIdx.x == 0) used = p.m;
        __syncthreads();
    }
    const float scale = EPI == EPI16_OUT && p.scale ? *p.scale : 1.0f;
    const int64_t one = (int64_t)p.m * p.n, all = one * (p.k_grouped ? p.groups : 1);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < outputs; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, m = p.k_grouped ? row % p.m : row, e = p.k_grouped ? row / p.m : 0;
        const int n = (int)(i - row * per_row) * VEC;
        if (m >= used && !p.zero_rest) continue;
        float v[VEC] = {};
        if (m < used) {
            typedef float F __attribute__((ext_vector_type(VEC)));
            const float *from = p.partial + row * p.n + n;
            // (eight parts' loads on their way together; those past the last are not added)
            for (int s = 0; s < p.splits; s += 8) {
                F part[8];
#pragma unroll
                for (int y = 0; y < 8; y++) part[y] = *reinterpret_cast<const F *>(from + min(s + y, p.splits - 1) * all);
#pragma unroll
                for (int y = 0; y < 8; y++)
#pragma unroll
                    for (int x = 0; x < VEC; x++) v[x] = s + y < p.splits ? v[x] + part[y][x] : v[x];
            }
        }
        const int64_t to = e * p.out_stride + (EPI == EPI16_OUT && p.out_rows ? p.out_rows[m] : m) * p.pitch_out + n;
#pragma unroll
        for (int x = 0; x < VEC; x++) {
            if constexpr (EPI == EPI16_ACT) {
                if (p.bias) v[x] += T::to(p.bias[n + x]);
                if (p.preact) p.preact[to + x] = T::from(v[x]);
                v[x] = act_value(v[x], p.act);
                if (p.residual) v[x] += T::to(p.residual[to + x]);
            } else {
                v[x] *= scale;
            }
            p.out[to + x] = T::from(v[x]);
        }
    }
}

template <class T> static int join16(const Gemm16 &p, int epilogue, hipStream_t stream)
{
    const bool four = p.n % 4 == 0;
    const int64_t per_row = four ? p.n / 4 : p.n, outputs = per_row * p.m * (p.k_grouped ? p.groups : 1);
    auto kern = epilogue == EPI16_ACT ? (four ? join16_kernel<T, EPI16_ACT, 4> : join16_kernel<T, EPI16_ACT, 1>)
                                      : (four ? join16_kernel<T, EPI16_OUT, 4> : join16_kernel<T, EPI16_OUT, 1>);
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>((outputs + 255) / 256, 1 << 16)), dim3(256), 0, stream, p, outputs, per_row);
    return launch_status("join16_kernel");
}

int gemm16_launch(const Gemm16 &problem, int layout, int epilogue, hipStream_t stream)
{
    Gemm16 p = problem;
    Plan16 plan = plan16(p, layout, epilogue);
    if (!p.partial || parts_bytes(p, plan.splits) > p.partial_bytes) plan.splits = 1;
    if (!p.partial || plan.tail * TAIL16_BYTES > p.partial_bytes) plan.tail = 0;
    p.splits = plan.splits;
    if (const int rc = p.half ? gemm16_launch_f16(p, plan, layout, epilogue, stream) : gemm16_launch_bf16(p, plan, layout, epilogue, stream)) return rc;
    if (p.splits == 1) return CCH_OK;
    return p.half ? join16<F16>(p, epilogue, stream) : join16<Bf16>(p, epilogue, stream);
}

// Copies of rows; up to two operands in a launch.  A row has a power of two of a workgroup's threads, 16 bytes to each and turn, so that no thread divides (2684
// rows, 20 experts' 3840 x 1449: one chunk of the whole copy to a thread 247 us a call, so 210).
struct PadRows16 {
    const uint16_t *src;
    uint16_t *dst;
    int64_t rows, cols, per_row;
    int threads_log2;
    const int32_t *sizes;
    int64_t group_rows;
};
__global__ __launch_bounds__(256) void pad_rows16_kernel(PadRows16 a, PadRows16 b)
{
    const PadRows16 &o = blockIdx.y ? b : a;
    const int threads = 1 << o.threads_log2, at_once = 256 >> o.threads_log2;
    for (int64_t row = (int64_t)blockIdx.x * at_once + (threadIdx.x >> o.threads_log2); row < o.rows; row += (int64_t)gridDim.x * at_once) {
        if (o.sizes && o.sizes[row / o.group_rows] <= 0) continue;
        const uint16_t *s = o.src + row * o.cols;
        uint16_t *d = o.dst + row * o.per_row * 8;
        for (int64_t c = (threadIdx.x & (threads - 1)) * 8; c < o.per_row * 8; c += threads * 8) {
            v4i v = {};
            if (c + 8 <= o.cols) v = reinterpret_cast<const Unaligned16 *>(s + c)->v;
            else
#pragma unroll
                for (int x = 0; x < 7; x++)
                    if (c + x < o.cols) v[x >> 1] |= (int)((uint32_t)s[c + x] << (16 * (x & 1)));
            *reinterpret_cast<v4i *>(d + c) = v;
        }
    }
}

int whole_operands16(Operand16 *operands, int n, Carve &ws, hipStream_t stream)
{
    PadRows16 pads[2];
    int used = 0;
    auto copy = [&] {
        int64_t blocks = 1;
        for (int i = 0; i < used; i++) blocks = std::max(blocks, (pads[i].rows << pads[i].threads_log2) / 256 + 1);
        hipLaunchKernelGGL(pad_rows16_kernel, dim3((unsigned)std::min<int64_t>(blocks, 2048), (unsigned)used), dim3(256), 0, stream, pads[0], pads[used - 1]);
        used = 0;
        return launch_status("pad_rows16_kernel");
    };
    for (int i = 0; i < n; i++) {
        Operand16 &o = operands[i];
        if (!o.at || whole16(o.cols) || o.rows == 0 || o.cols == 0) continue;
        uint16_t *to = ws.take<uint16_t>(padded16_bytes(o.rows, o.cols));
        const int64_t per_row = pitch16(o.cols) / 8;
        int log2 = 0;
        while (log2 < 8 && (1 << log2) < per_row) log2++;
        pads[used++] = PadRows16{o.at, to, o.rows, o.cols, per_row, log2, o.sizes, o.group_rows};
        o.at = to;
        if (used == 2)
            if (const int rc = copy()) return rc;
    }
    return used ? copy() : CCH_OK;
}

__global__ __launch_bounds__(256) void fill_zero16_kernel(uint16_t *dst, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = 0;
}
int fill_zero16(uint16_t *dst, int64_t n, hipStream_t stream)
{
    hipLaunchKernelGGL(fill_zero16_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 14)), dim3(256), 0, stream, dst, n);
    return launch_status("fill_zero16_kernel");
}

// ---- dz = grad_out * act'(preact) and the bias' gradient.  A workgroup has 256 columns, 8 to a thread, and a run of rows, every eighth to a thread; its columns' sums over
// the run go to `partial`, which a second launch adds up in the runs' order.  Sums are of the products before their rounding.  Bound by memory (two reads, one write) in wide layers:
// 8192 x 7168 68 us.  At most 64 runs, so that the second launch stays short: narrow layers of many rows leave CUs without work (without dz, 16384 x 256 43 us, 65536 x 1024 243).
constexpr int SUM_COLS = 256, SUM_RUNS = 64;
static int64_t sum_runs(int64_t m) { return std::max<int64_t>(1, std::min<int64_t>((m + 7) / 8, SUM_RUNS)); }
int64_t column_sum_bytes(int64_t m, int64_t n) { return round256(sum_runs(m) * n * 4); }

template <class T>
__global__ __launch_bounds__(256) void act_backward16_kernel(const uint16_t *__restrict__ grad, const uint16_t *__restrict__ pre, uint16_t *__restrict__ dz,
                                                             float *__restrict__ partial, int m, int n, int64_t pitch, int run, int act)
{
    __shared__ float sums[8][SUM_COLS];
    const int tc = threadIdx.x & 31, tr = threadIdx.x >> 5;
    const int c = (int)blockIdx.x * SUM_COLS + tc * 8, left = n - c;
    const int first = (int)blockIdx.y * run, last = min(m, first + run);
    float sum[8] = {};
    if (left > 0)
        for (int row = first + tr; row < last; row += 8) {
            float v[8], z[8];
            load8<T>(grad + (int64_t)row * n + c, left, v);
            if (act != CCH_ACT_NONE) {
                load8<T>(pre + (int64_t)row * n + c, left, z);
#pragma unroll
                for (int x = 0; x < 8; x++) v[x] = x < left ? v[x] * act_slope(z[x], act) : 0.0f;
            }
            if (dz) *reinterpret_cast<v4i *>(dz + (int64_t)row * pitch + c) = pack8<T>(v);
#pragma unroll
            for (int x = 0; x < 8; x++) sum[x] += v[x];
        }
    if (!partial) return;
#pragma unroll
    for (int x = 0; x < 8; x++) sums[tr][tc * 8 + x] = sum[x];
    __syncthreads();
    const int col = (int)blockIdx.x * SUM_COLS + (int)threadIdx.x;
    if (col < n) {
        float s = 0.0f;
#pragma unroll
        for (int x = 0; x < 8; x++) s += sums[x][threadIdx.x];
        partial[(int64_t)blockIdx.y * n + col] = s;
    }
}

template <class T> __global__ __launch_bounds__(256) void column_sum16_kernel(const float *__restrict__ partial, uint16_t *__restrict__ out, int n, int runs)
{
    const int col = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (col >= n) return;
    float s = 0.0f;
#pragma unroll 16
    for (int i = 0; i < runs; i++) s += partial[(int64_t)i * n + col];
    out[col] = T::from(s);
}

int act_backward16(const uint16_t *grad_out, const uint16_t *preact, uint16_t *dz, uint16_t *grad_bias, float *partial, int64_t m, int64_t n, int act, int half, hipStream_t stream)
{
    if (m == 0 || n == 0 || (!dz && !grad_bias)) return CCH_OK;
    const int64_t runs = sum_runs(m), run = (m + runs - 1) / runs;
    auto kern = half ? act_backward16_kernel<F16> : act_backward16_kernel<Bf16>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((n + SUM_COLS - 1) / SUM_COLS), (unsigned)runs), dim3(256), 0, stream, grad_out, preact, dz, grad_bias ? partial : nullptr, (int)m,
                       (int)n, pitch16(n), (int)run, act);
    if (const int rc = launch_status("act_backward16_kernel")) return rc;
    if (!grad_bias) return CCH_OK;
    auto sum = half ? column_sum16_kernel<F16> : column_sum16_kernel<Bf16>;
    hipLaunchKernelGGL(sum, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, partial, grad_bias, (int)n, (int)runs);
    return launch_status("column_sum16_kernel");
}

}  // namespace cch
