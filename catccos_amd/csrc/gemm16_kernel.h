// Products of 16-bit operands on tiles of (32 MT WM) x (32 NT WN): WM x WN waves of MT x NT blocks of 32 x 32, K in steps of 64 elements, DEPTH stages in LDS that are
// filled straight from memory, DEPTH - 1 steps ahead; one barrier a step publishes what has landed and frees what was read.  A 128 x 128 step is 512 clocks of matrix
// instructions, while memory answers in 1500 to 2500: with two stages two workgroups share a CU, so that one's waits and epilogue pass under the other's matrix instructions; where there are not
// that many workgroups, one has four stages (256 x 4096 x 7168 on 64 tiles: 97 us with two).  Tiles too few for the chip are split along K (p.splits): each part leaves fp32 sums,
// which join16_kernel adds up in the parts' order.
#pragma once
#include <atomic>

#include "gemm16_device.h"

namespace cch {

constexpr int min_c(int a, int b) { return a < b ? a : b; }

template <int MT_, int NT_, int WM_, int WN_, int DEPTH_> struct Shape16 {
    static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, WAVES = WM * WN, THREADS = 64 * WAVES, DEPTH = DEPTH_, PER_CU = DEPTH == 2 ? 2 : 1;
    static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN;      // tile
    static constexpr int A_BYTES = TM * 128, B_BYTES = TN * 128, STAGE = A_BYTES + B_BYTES, LDS = DEPTH * STAGE;
    static constexpr int NJA = A_BYTES / 1024 / WAVES, NJB = B_BYTES / 1024 / WAVES;   // requests of a wave and step
};

template <class T, int LAYOUT, int EPI, class S>
__global__ __launch_bounds__(S::THREADS, S::PER_CU * S::WAVES / 4) void gemm16_kernel(Gemm16 p)
{
    constexpr bool A_KM = LAYOUT == ROWS_TN, B_KM = LAYOUT != ROWS_NK;   // K-major operands
    constexpr int MT = S::MT, NT = S::NT, NJA = S::NJA, NJB = S::NJB;
    using KA = KMajor<S::TM>;
    using KB = KMajor<S::TN>;
    __shared__ GroupTable16 tab;
    const bool rows_grouped = !p.k_grouped;
    if (threadIdx.x < 64) build_groups16(tab, p.group_sizes, p.groups, rows_grouped ? p.m : p.k, S::TM);
    __syncthreads();
    if (p.zero_rest) zero_rest16(p, tab.start[p.groups]);
    const bool leave_empty = !rows_grouped && p.splits == 1;
    if (leave_empty) zero_groups16(p, tab);

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
    const int r = lane & 31, g = lane >> 5, tq = lane >> 4, ti = lane & 15;
    const uint32_t lds = (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem);
    const int col_tiles = (p.n + S::TN - 1) / S::TN;
    const int row_tiles = uniform(rows_grouped ? tab.tile[p.groups] : (p.m + S::TM - 1) / S::TM);
    const int per_list = row_tiles * col_tiles * p.splits, end = lists_end16(per_list, rows_grouped ? 1 : p.groups);   // (below 2^31: the launch checks)
    const bool whole = whole_rows(p);

    // this lane's fragment reads in stage 0
    uint32_t fr_a[4], fr_b[4], ft_a[MT], ft_b[NT];
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        const uint32_t chunk = ((uint32_t)(2 * kk + g) ^ swizzle_of_row(r)) << 4;
        fr_a[kk] = lds + (uint32_t)(wm * MT * 32 + r) * 128u + chunk;
        fr_b[kk] = lds + S::A_BYTES + (uint32_t)(wn * NT * 32 + r) * 128u + chunk;
    }
    const int krow = (tq >> 1) * 8 + (ti >> 2);                                 // (and 4 more by the second load)
    const uint32_t quarter = (uint32_t)((tq & 1) * 2 + ((ti & 3) >> 1));        // chunk among a block's four
#pragma unroll
    for (int i = 0; i < MT; i++) ft_a[i] = lds + (uint32_t)krow * KA::ROW + ((((uint32_t)(wm * MT + i) * 4 + quarter) ^ KA::swizzle(krow)) << 4) + (ti & 1) * 8u;
#pragma unroll
    for (int j = 0; j < NT; j++)
        ft_b[j] = lds + S::A_BYTES + (uint32_t)krow * KB::ROW + ((((uint32_t)(wn * NT + j) * 4 + quarter) ^ KB::swizzle(krow)) << 4) + (ti & 1) * 8u;

    for (int64_t t = blockIdx.x; t < end; t += gridDim.x) {
        int e = 0, rt, ct, m0, m_end, k_begin = 0, k_end = p.k;
        const int at = place_in_lists16((int)t, per_list, e);
        if (at < 0) continue;
        const int part = at % p.splits;
        tile_of16(at / p.splits, row_tiles, col_tiles, rt, ct);
        if (rows_grouped) {
            e = uniform(group_of_tile16(tab, p.groups, rt));
            m0 = uniform(tab.start[e] + (rt - tab.tile[e]) * S::TM);
            m_end = uniform(tab.start[e + 1]);
        } else {
            m0 = rt * S::TM;
            m_end = p.m;
            k_begin = uniform(tab.start[e]);
            k_end = uniform(tab.start[e + 1]);
            if (leave_empty && k_end == k_begin) continue;
        }
        const int n0 = ct * S::TN;
        // this part's steps: `first`.. of the group's K
        const int rows = min(m_end - m0, S::TM), cols = min(p.n - n0, S::TN), k_all = k_end - k_begin, steps_all = (k_all + 63) >> 6;
        const int each = (steps_all + p.splits - 1) / p.splits, first = min(part * each, steps_all), steps = min(each, steps_all - first);
        const int k_stop = min((first + steps) * 64, k_all);   // from k_begin

        // requests: descriptors and this lane's offsets
        uint32_t off_a[NJA], off_b[NJB];
        Rsrc rs_a{}, rs_b{};
        const int k8 = (p.k + 7) & ~7;   // (rows of other lengths are padded with zeros)
        const uint16_t *a0 = p.a + (A_KM ? (int64_t)k_begin * p.pitch_a : p.a_rows ? 0 : (int64_t)m0 * p.pitch_a);
        const uint16_t *b0 = p.b + (rows_grouped ? (int64_t)e * p.b_stride : (int64_t)0) + (B_KM ? (int64_t)k_begin * p.pitch_b : (int64_t)n0 * p.pitch_b);
        if constexpr (!A_KM) {
            const int last = p.a_rows ? p.m_src - 1 : rows - 1;
            rs_a = make_rsrc(a0, (uint32_t)min(((int64_t)last * p.pitch_a + k8) * 2, (int64_t)0x7FFFFFF0));
        }
        if constexpr (!B_KM) rs_b = make_rsrc(b0, (uint32_t)min(((int64_t)(cols - 1) * p.pitch_b + k8) * 2, (int64_t)0x7FFFFFF0));
#pragma unroll
        for (int j = 0; j < NJA; j++) {
            if constexpr (A_KM) {
                const int kr = (wave * NJA + j) * KA::ROWS_PER_KIB + lane / KA::CHUNKS;
                off_a[j] = (uint32_t)kr * (uint32_t)p.pitch_a * 2u + (((uint32_t)(lane % KA::CHUNKS) ^ KA::swizzle(kr)) << 4);
            } else {
                const int row = (wave * NJA + j) * 8 + (lane >> 3);
                uint32_t src = (uint32_t)row;
                if (p.a_rows) src = row < rows ? (uint32_t)p.a_rows[m0 + row] : 0u;
                off_a[j] = row < rows ? src * (uint32_t)p.pitch_a * 2u + (((uint32_t)(lane & 7) ^ swizzle_of_row(row)) << 4) : NO_FETCH;
            }
        }
#pragma unroll
        for (int j = 0; j < NJB; j++) {
            if constexpr (B_KM) {
                const int kr = (wave * NJB + j) * KB::ROWS_PER_KIB + lane / KB::CHUNKS;
                off_b[j] = (uint32_t)kr * (uint32_t)p.pitch_b * 2u + (((uint32_t)(lane % KB::CHUNKS) ^ KB::swizzle(kr)) << 4);
            } else {
                const int row = (wave * NJB + j) * 8 + (lane >> 3);
                off_b[j] = row < cols ? (uint32_t)row * (uint32_t)p.pitch_b * 2u + (((uint32_t)(lane & 7) ^ swizzle_of_row(row)) << 4) : NO_FETCH;
            }
        }
        // (K contiguous: a lane whose 8 elements begin at or past K fetches nothing; K is a multiple of 8 or its rows are padded with zeros)
        int k_left = 0;
        uint32_t k_at = 0;
        uint32_t stage_at = 0;
        auto prepare = [&](int step) {
            const int k0 = (first + step) * 64;
            if constexpr (A_KM) rs_a = kmajor_rsrc(a0, p.pitch_a, k0, k_stop, m0, p.m);
            if constexpr (B_KM) rs_b = kmajor_rsrc(b0, p.pitch_b, k0, k_stop, n0, p.n);
            k_left = k_stop - k0;
            k_at = (uint32_t)k0 * 2u;
            stage_at = lds + (uint32_t)(step % S::DEPTH) * S::STAGE;
        };
        // request q of a wave's NJA + NJB of a step
        auto request = [&](auto q_c) {
            constexpr int q = decltype(q_c)::value, j = q < NJA ? q : q - NJA;
            constexpr bool is_a = q < NJA, km = is_a ? A_KM : B_KM;
            const int row = (wave * (is_a ? NJA : NJB) + j) * 8 + (lane >> 3);
            const bool in = km || (int)(((uint32_t)(lane & 7) ^ swizzle_of_row(row)) * 8u) < k_left;
            const uint32_t off = is_a ? off_a[j] : off_b[j];
            load16_to_lds(is_a ? rs_a : rs_b, in ? off : NO_FETCH, km ? 0u : k_at, stage_at + (is_a ? 0u : (uint32_t)S::A_BYTES) + (uint32_t)(wave * (is_a ? NJA : NJB) + j) * 1024u);
        };

        v16f acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = (v16f)(0.0f);
        // Operands are read a step ahead: while one set is multiplied the other is filled, and the step's requests, DEPTH ahead into the stage that was read last, go
        // between the matrix instructions too.  (Requests past the last step fetch nothing: every wait counts the same.)
        static_for<S::DEPTH>([&](auto i) { prepare(i); static_for<NJA + NJB>(request); });
        CCH_WAIT_VM((S::DEPTH - 1) * (NJA + NJB));
        CCH_BARRIER();
        v4i fa[2][MT][4], fb[2][NT][4];
        uint32_t read_at = 0;   // the stage to read next
        auto read = [&](auto set_c, auto i_c) {   // the i-th of a step's fragments, sixteenth by sixteenth
            constexpr int set = decltype(set_c)::value, kk = decltype(i_c)::value / (MT + NT), f = decltype(i_c)::value % (MT + NT);
            if constexpr (f < NT) fb[set][f][kk] = B_KM ? read_transposed(ft_b[f] + read_at + (uint32_t)kk * 16u * KB::ROW, KB::ROW) : lds_read16_abs(fr_b[kk] + read_at + (uint32_t)f * 4096u);
            else fa[set][f - NT][kk] = A_KM ? read_transposed(ft_a[f - NT] + read_at + (uint32_t)kk * 16u * KA::ROW, KA::ROW) : lds_read16_abs(fr_a[kk] + read_at + (uint32_t)(f - NT) * 4096u);
        };
        constexpr int READS = 4 * (MT + NT), MMAS = 4 * MT * NT;
        static_for<READS>([&](auto i) { read(IC<0>{}, i); });
        auto multiply = [&](auto set_c, int step) {
            constexpr int set = decltype(set_c)::value;
            read_at = read_at + S::STAGE == S::LDS ? 0u : read_at + (uint32_t)S::STAGE;
            CCH_WAIT_VM_LGKM0((S::DEPTH - 2) * (NJA + NJB));
            CCH_BARRIER();
            prepare(step + S::DEPTH);
            static_for<MMAS>([&](auto m_c) {
                constexpr int m = decltype(m_c)::value, kk = m / (MT * NT), i = m / NT % MT, j = m % NT;
                acc[i][j] = T::mfma(fb[set][j][kk], fa[set][i][kk], acc[i][j]);
                // reads in the first three quarters, requests over all
                constexpr int r0 = min_c(m * READS * 4 / (MMAS * 3), READS), r1 = min_c((m + 1) * READS * 4 / (MMAS * 3), READS);
                static_for<r1 - r0>([&](auto x) { read(IC<1 - set>{}, IC<r0 + decltype(x)::value>{}); });
                constexpr int q0 = m * (NJA + NJB) / MMAS, q1 = (m + 1) * (NJA + NJB) / MMAS;
                static_for<q1 - q0>([&](auto x) { request(IC<q0 + decltype(x)::value>{}); });
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        int step = 0;
        for (; step + 2 <= steps; step += 2) {
            multiply(IC<0>{}, step);
            multiply(IC<1>{}, step + 1);
        }
        if (step < steps) multiply(IC<0>{}, step);
        CCH_WAIT_VM_LGKM0(0);
        CCH_BARRIER();
        if constexpr (EPI == EPI16_OUT || EPI == EPI16_ACT) {
            if (p.splits > 1) {
                store_part16<MT, NT>(p, acc, p.partial + ((int64_t)part * (rows_grouped ? 1 : p.groups) + (rows_grouped ? 0 : e)) * p.m * p.n, m0 + wm * MT * 32, m_end, n0 + wn * NT * 32);
                continue;
            }
        }
        epilogue16<T, EPI, MT, NT, 32>(p, acc, e, m0, m_end, n0, wm * MT * 32, wn * NT * 32, whole, false);
    }
}

// Lets a kernel have more than 64 KB of LDS: once per device; doing it twice from two threads is harmless.
inline int allow_lds16(const void *kernel, int bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    CCH_HIP(hipGetDevice(&dev));
    const uint64_t bit = (uint64_t)1 << (dev & 63);
    if (dev >= 64 || !(done.load(std::memory_order_acquire) & bit)) {
        CCH_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit, std::memory_order_release);
    }
    return CCH_OK;
}

template <class T, int LAYOUT, int EPI, class S> int launch16(const Gemm16 &p, int64_t tiles, hipStream_t stream)
{
    static_assert(S::A_BYTES % (1024 * S::WAVES) == 0 && S::B_BYTES % (1024 * S::WAVES) == 0, "whole requests");
    static std::atomic<uint64_t> attr_set{0};
    auto kernel = gemm16_kernel<T, LAYOUT, EPI, S>;
    if (const int rc = allow_lds16(reinterpret_cast<const void *>(kernel), S::LDS, attr_set)) return rc;
    const int64_t groups = p.k_grouped ? p.groups : 1, grid = std::min<int64_t>((tiles / groups * p.splits + 7) / 8 * 8 * groups, (int64_t)1 << 22);   // (a multiple of 8: place16)
    kernel<<<dim3((uint32_t)grid), dim3(S::THREADS), S::LDS, stream>>>(p);
    return launch_status("gemm16_kernel");
}

}  // namespace cch
