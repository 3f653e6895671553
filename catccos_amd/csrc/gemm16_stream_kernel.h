// Products of a few rows: bound by the weights' way from memory.  A workgroup has MR rows (8, 16 or 32) of a group and 32 columns; its waves take K's steps of 64 elements in
// turn, each with a ring of DEPTH stages in LDS of its own that is filled straight from memory, so that the loop over K has no barrier and 64 KiB or more of weights are on their way to
// a CU at any time.  1 x 4096 x 7168 from memory 15.4 us, 3.8 TB/s: 128 columns' workgroups are half of the CUs; again from the caches 11.5.  In the end the waves' sums are added up in LDS, in their order.
#pragma once
#include <atomic>

#include "gemm16_kernel.h"

namespace cch {

// A step's weights are 32 rows of 128 bytes, or (K-major) 64 of 64: half lines, whose other halves a neighbouring workgroup of the same XCD asks for.
template <int LAYOUT, int MR_> struct Stream16 {
    static constexpr int MR = MR_, WAVES = 8, THREADS = 64 * WAVES, TN = 32;
    static constexpr int W_BYTES = TN * 128, X_BYTES = MR * 128, STAGE = W_BYTES + X_BYTES;
    static constexpr int DEPTH = MR == 32 ? 2 : 3, RW = W_BYTES / 1024, RX = X_BYTES / 1024;
    static constexpr int RING = WAVES * DEPTH * STAGE, PITCH = 36, SUMS = WAVES * 32 * PITCH * 4, LDS = (RING > SUMS ? RING : SUMS);
};

template <class T, int LAYOUT, int EPI, class S>
__global__ __launch_bounds__(S::THREADS) void gemm16_stream_kernel(Gemm16 p)
{
    constexpr bool B_KM = LAYOUT != ROWS_NK;
    constexpr int DEPTH = S::DEPTH;
    using KB = KMajor<S::TN>;
    __shared__ GroupTable16 tab;
    if (threadIdx.x < 64) build_groups16(tab, p.group_sizes, p.groups, p.m, S::MR);
    __syncthreads();
    if (p.zero_rest) zero_rest16(p, tab.start[p.groups]);

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5, tq = lane >> 4, ti = lane & 15;
    const uint32_t lds = (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem);
    const uint32_t ring = lds + (uint32_t)wave * (DEPTH * S::STAGE);
    const int col_tiles = (p.n + S::TN - 1) / S::TN, row_tiles = uniform(tab.tile[p.groups]), total = row_tiles * col_tiles;
    const int steps = (p.k + 63) >> 6, mine = (steps - wave + S::WAVES - 1) / S::WAVES;   // of this wave: wave, wave + WAVES, ...
    const int k8 = (p.k + 7) & ~7;

    uint32_t fr_x[4], fr_w[4];
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        const int row = r & (S::MR - 1);   // (rows of the block that there are none of are not stored: any will do)
        fr_w[kk] = ring + (uint32_t)r * 128u + (((uint32_t)(2 * kk + g) ^ swizzle_of_row(r)) << 4);
        fr_x[kk] = ring + S::W_BYTES + (uint32_t)row * 128u + (((uint32_t)(2 * kk + g) ^ swizzle_of_row(row)) << 4);
    }
    const int krow = (tq >> 1) * 8 + (ti >> 2);
    const uint32_t ft_w = ring + (uint32_t)krow * KB::ROW + ((uint32_t)((tq & 1) * 2 + ((ti & 3) >> 1)) << 4) + (ti & 1) * 8u;

    for (int64_t t = blockIdx.x; t < ((total + 7) & ~7); t += gridDim.x) {
        const int at = place16((int)t, total);
        if (at < 0) continue;
        const int rt = at / col_tiles, n0 = (at - rt * col_tiles) * S::TN;
        const int e = uniform(group_of_tile16(tab, p.groups, rt));
        const int m0 = uniform(tab.start[e] + (rt - tab.tile[e]) * S::MR), m_end = uniform(tab.start[e + 1]);
        const int rows = min(m_end - m0, S::MR), cols = min(p.n - n0, S::TN);
        const uint16_t *x0 = p.a + (int64_t)m0 * p.pitch_a, *w0 = p.b + (int64_t)e * p.b_stride + (B_KM ? 0 : (int64_t)n0 * p.pitch_b);
        const Rsrc rs_x = make_rsrc(x0, (uint32_t)min(((int64_t)(rows - 1) * p.pitch_a + k8) * 2, (int64_t)0x7FFFFFF0));
        Rsrc rs_w{};
        if constexpr (!B_KM) rs_w = make_rsrc(w0, (uint32_t)min(((int64_t)(cols - 1) * p.pitch_b + k8) * 2, (int64_t)0x7FFFFFF0));
        uint32_t off_x[S::RX], off_w[S::RW];
#pragma unroll
        for (int q = 0; q < S::RX; q++) {
            const int row = q * 8 + (lane >> 3);
            off_x[q] = row < rows ? (uint32_t)row * (uint32_t)p.pitch_a * 2u + (((uint32_t)(lane & 7) ^ swizzle_of_row(row)) << 4) : NO_FETCH;
        }
#pragma unroll
        for (int q = 0; q < S::RW; q++) {
            const int row = q * 8 + (lane >> 3);
            if (B_KM) {
                const int kr = q * KB::ROWS_PER_KIB + lane / KB::CHUNKS;
                off_w[q] = (uint32_t)kr * (uint32_t)p.pitch_b * 2u + (((uint32_t)(lane % KB::CHUNKS) ^ KB::swizzle(kr)) << 4);
            }
            else off_w[q] = row < cols ? (uint32_t)row * (uint32_t)p.pitch_b * 2u + (((uint32_t)(lane & 7) ^ swizzle_of_row(row)) << 4) : NO_FETCH;
        }
        // the wave's i-th step into stage `at`; past the last one nothing is fetched, so that waits count the same
        auto request = [&](int i, uint32_t at) {
            const int k0 = (wave + i * S::WAVES) * 64, left = i < mine ? p.k - k0 : 0;
            if constexpr (B_KM) rs_w = kmajor_rsrc(w0, p.pitch_b, k0, i < mine ? p.k : 0, n0, p.n);
#pragma unroll
            for (int q = 0; q < S::RW; q++) {
                const bool in = B_KM || (int)(((uint32_t)(lane & 7) ^ swizzle_of_row(q * 8 + (lane >> 3))) * 8u) < left;
                load16_to_lds(rs_w, in ? off_w[q] : NO_FETCH, B_KM ? 0u : (uint32_t)k0 * 2u, ring + at + (uint32_t)q * 1024u);
            }
#pragma unroll
            for (int q = 0; q < S::RX; q++) {
                const bool in = (int)(((uint32_t)(lane & 7) ^ swizzle_of_row(q * 8 + (lane >> 3))) * 8u) < left;
                load16_to_lds(rs_x, in ? off_x[q] : NO_FETCH, (uint32_t)k0 * 2u, ring + at + (uint32_t)(S::W_BYTES + q * 1024));
            }
        };
        v16f acc = (v16f)(0.0f);
#pragma unroll
        for (int i = 0; i < DEPTH; i++) request(i, (uint32_t)(i * S::STAGE));
        uint32_t stage = 0;
        for (int i = 0; i < mine; i++) {
            CCH_WAIT_VM((DEPTH - 1) * (S::RW + S::RX));
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            v4i fx[4], fw[4];
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
                fx[kk] = lds_read16_abs(fr_x[kk] + stage);
                fw[kk] = B_KM ? read_transposed(ft_w + stage + (uint32_t)kk * 16u * KB::ROW, KB::ROW) : lds_read16_abs(fr_w[kk] + stage);
            }
            __builtin_amdgcn_sched_barrier(0);
            CCH_WAIT_LGKM0();   // (in registers: the stage is free)
            __builtin_amdgcn_sched_barrier(0);
            request(i + DEPTH, stage);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < 4; kk++) acc = T::mfma(fw[kk], fx[kk], acc);
            stage = stage + S::STAGE == DEPTH * S::STAGE ? 0u : stage + S::STAGE;
        }
        CCH_WAIT_VM_LGKM0(0);
        CCH_BARRIER();   // all rings are done with: the sums take their place, [wave][32 rows][32 columns and 4 more, so that rows begin on other banks]
        float *sums = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int q = 0; q < 4; q++)
            *reinterpret_cast<f32x4 *>(sums + (wave * 32 + r) * S::PITCH + 8 * q + 4 * g) = (f32x4){acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        CCH_WAIT_LGKM0();
        CCH_BARRIER();
        for (int i = threadIdx.x; i < rows * S::TN; i += S::THREADS) {
            const int row = i / S::TN, col = i % S::TN, n = n0 + col, m = m0 + row;
            if (n >= p.n) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < S::WAVES; w++) v += sums[(w * 32 + row) * S::PITCH + col];
            const int64_t to = (int64_t)m * p.pitch_out + n;
            if constexpr (EPI == EPI16_ACT) {
                if (p.bias) v += T::to(p.bias[n]);
                if (p.preact) p.preact[to] = T::from(v);
                v = act_value(v, p.act);
                if (p.residual) v += T::to(p.residual[to]);
            }
            p.out[to] = T::from(v);
        }
        CCH_WAIT_LGKM0();
        CCH_BARRIER();   // (the next tile's requests overwrite the sums)
    }
}

template <class T, int LAYOUT, int EPI, int MR> int launch16_stream_rows(const Gemm16 &p, int64_t tiles, hipStream_t stream)
{
    using S = Stream16<LAYOUT, MR>;
    static std::atomic<uint64_t> attr_set{0};
    auto kernel = gemm16_stream_kernel<T, LAYOUT, EPI, S>;
    if (const int rc = allow_lds16(reinterpret_cast<const void *>(kernel), S::LDS, attr_set)) return rc;
    const int64_t grid = std::min<int64_t>((tiles + 7) & ~(int64_t)7, (int64_t)1 << 22);   // (a multiple of 8: place16)
    kernel<<<dim3((uint32_t)grid), dim3(S::THREADS), S::LDS, stream>>>(p);
    return launch_status("gemm16_stream_kernel");
}

}  // namespace cch
