// Products of 16-bit operands on tiles of 256 x 256: one persistent workgroup of eight waves to a CU walks the tiles; K in steps of 64 elements, two stages in LDS.
//
// The waves form two groups of four, one wave of each on every SIMD; a wave owns 128 x 64 outputs.  A step is four slots between workgroup barriers, memory, matrix, memory, matrix
// (L0 C0 L1 C1), and the second group runs one slot behind the first: while one wave of a SIMD reads its operands from LDS, the other one's matrix instructions run.  Both memory
// slots read at most 64 KiB for a group, which takes about as long as the 16 matrix instructions of a slot.  In a group's 128 rows the tile's blocks of 32 rows alternate with
// the other group's.
//
// A K-contiguous panel's rows hold both halves of a step, so that nothing of it is free before all of it is read; a K-major panel's halves are separate rows.  Requests, by
// layout (s: the step; a request lands in the stage that the step two before it has just read):
//   ROWS_NK  L0: A blocks 2-3 of s + 1   C0: A blocks 0-1 of s + 2   L1, C1: half of B of s + 2 each; L0 reads all of B and A blocks 0-1, L1 A blocks 2-3
//   ROWS_NN  L0: second half of B of s + 1   L1: first half of B of s + 2   C1: A of s + 2; L0 reads the first half of the step, L1 the second
//   ROWS_TN  L0: second halves of A and B of s + 1   L1: first halves of s + 2; reads likewise
// Where the tiles leave part of the last round's workgroups idle and K is long, that round's tiles are worked on in parts of K (tail_parts16): each leaves its fp32 sums as its lanes hold them, and a
// second launch adds a tile's parts up in their order and writes the results.
// A group's A rows are read by that group alone (K contiguous), so they are free one slot earlier than B.  Every wave issues the same number of requests in every step (what lies
// past the operand fetches nothing), so every wait is a constant: requests complete in order.  The last two steps of a tile request the next one's first two; past the last tile
// the descriptors are empty.
#pragma once
#include <atomic>

#include "gemm16_kernel.h"

namespace cch {

struct Big16 {
    static constexpr int MT = 4, NT = 2, TM = 256, TN = 256, THREADS = 512;
    static constexpr int PANEL = 32768, A_AT = 0, B_AT = 2 * PANEL, TABLE = 4 * PANEL, LDS = TABLE + (int)sizeof(GroupTable16);
};

template <class T, int LAYOUT, int EPI>
__global__ __launch_bounds__(Big16::THREADS, 2) void gemm16_big_kernel(Gemm16 p)
{
    using S = Big16;
    constexpr bool A_KM = LAYOUT == ROWS_TN, B_KM = LAYOUT != ROWS_NK, HALVES = LAYOUT != ROWS_NK;
    constexpr bool TAIL = LAYOUT != ROWS_TN && (EPI == EPI16_OUT || EPI == EPI16_ACT);
    constexpr int MT = S::MT, NT = S::NT, PANEL = S::PANEL;
    using KM = KMajor<256>;
    GroupTable16 &tab = *reinterpret_cast<GroupTable16 *>(smem + S::TABLE);
    const bool rows_grouped = !p.k_grouped;
    if (threadIdx.x < 64) build_groups16(tab, p.group_sizes, p.groups, rows_grouped ? p.m : p.k, S::TM);
    __syncthreads();
    if (p.zero_rest) zero_rest16(p, uniform(tab.start[p.groups]));
    if (!rows_grouped) zero_groups16(p, tab);

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int r = lane & 31, g = lane >> 5, tq = lane >> 4, ti = lane & 15;
    const uint32_t lds = (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem);
    const int col_tiles = (p.n + S::TN - 1) / S::TN;
    const int row_tiles = uniform(rows_grouped ? tab.tile[p.groups] : (p.m + S::TM - 1) / S::TM);
    const int per_list = row_tiles * col_tiles, end = lists_end16(per_list, rows_grouped ? 1 : p.groups);   // (below 2^31: the launch checks)

    int parts = 1, left = 0, full = 0;   // of K; tiles of the last round, and before it
    if (TAIL && p.tail) {
        left = per_list % (int)gridDim.x;
        full = per_list - left;
        parts = uniform(tail_parts16(left, (int)gridDim.x, (p.k + 63) >> 6, p.tail));
    }
    const int tiles_end = TAIL && parts > 1 ? full + ((left * parts + 7) & ~7) : end, part_k = TAIL ? (((p.k + 63) >> 6) + parts - 1) / parts * 64 : 0;

    // ---- this lane's fragment reads (the current stage's; moved by a panel from step to step)
    // A, K contiguous: panel position 128 wm + 32 i + r holds tile row 64 i + 32 wm + r; K-major: column = tile row
    uint32_t fr_a[4], fr_b[4], ft_a[MT], ft_b[NT];
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        const uint32_t chunk = ((uint32_t)(2 * kk + g) ^ swizzle_of_row(r)) << 4;
        fr_a[kk] = lds + S::A_AT + (uint32_t)(wm * 128 + r) * 128u + chunk;
        fr_b[kk] = lds + S::B_AT + (uint32_t)(wn * 64 + r) * 128u + chunk;
    }
    const int krow = (tq >> 1) * 8 + (ti >> 2);
    const uint32_t part = (uint32_t)((tq & 1) * 2 + ((ti & 3) >> 1));
#pragma unroll
    for (int i = 0; i < MT; i++) ft_a[i] = lds + S::A_AT + (uint32_t)krow * KM::ROW + ((((uint32_t)(2 * i + wm) * 4 + part) ^ KM::swizzle(krow)) << 4) + (ti & 1) * 8u;
#pragma unroll
    for (int j = 0; j < NT; j++) ft_b[j] = lds + S::B_AT + (uint32_t)krow * KM::ROW + ((((uint32_t)(wn * 2 + j) * 4 + part) ^ KM::swizzle(krow)) << 4) + (ti & 1) * 8u;

    // ---- requests: this lane's offsets from a descriptor's start, the same for every tile.  K contiguous: request q of a wave fills 8 rows; A: blocks q / 2 of the wave's
    // group; K-major: request q fills 2 K-rows of half q / 2
    uint32_t off_a[4], off_b[4], dst_a[4], dst_b[4];
    int chunk_a[4], chunk_b[4];   // K contiguous: the chunk's first element in the step
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int kr = (q >> 1) * 32 + wave * 4 + (q & 1) * 2 + (lane >> 5);
        const uint32_t kpart = (((uint32_t)(lane & 31) ^ KM::swizzle(kr)) << 4);
        if (A_KM) {
            off_a[q] = (uint32_t)kr * (uint32_t)p.pitch_a * 2u + kpart;
            dst_a[q] = (uint32_t)(kr & ~1) * KM::ROW;
        } else {
            const int pos = wm * 128 + q * 32 + wn * 8, row = q * 64 + wm * 32 + wn * 8 + (lane >> 3);   // block q, eight of its rows
            const uint32_t c = (uint32_t)(lane & 7) ^ swizzle_of_row(wn * 8 + (lane >> 3));
            off_a[q] = (uint32_t)row * (uint32_t)p.pitch_a * 2u + (c << 4);
            chunk_a[q] = (int)c * 8;
            dst_a[q] = (uint32_t)pos * 128u;
        }
        if (B_KM) {
            off_b[q] = (uint32_t)kr * (uint32_t)p.pitch_b * 2u + kpart;
            dst_b[q] = (uint32_t)(kr & ~1) * KM::ROW;
        } else {
            const int row = (wave * 4 + q) * 8 + (lane >> 3);
            const uint32_t c = (uint32_t)(lane & 7) ^ swizzle_of_row(row);
            off_b[q] = (uint32_t)row * (uint32_t)p.pitch_b * 2u + (c << 4);
            chunk_b[q] = (int)c * 8;
            dst_b[q] = (uint32_t)(wave * 4 + q) * 1024u;
        }
        dst_a[q] = (uint32_t)uniform((int)(dst_a[q] + lds + S::A_AT));
        dst_b[q] = (uint32_t)uniform((int)(dst_b[q] + lds + S::B_AT));
    }

    struct Tile {
        bool valid;
        int slot;                    // of a part of K: where its sums go; else -1
        int e, m0, m_end, n0, k_len, steps;
        const uint16_t *a, *b;       // first element of the first step
        int64_t left_a, left_b;      // bytes from there to the operand's end
    };
    const int64_t adv_a = A_KM ? p.pitch_a * 128 : 128, adv_b = B_KM ? p.pitch_b * 128 : 128;   // bytes from step to step
    const int k8 = (p.k + 7) & ~7, n8 = (p.n + 7) & ~7, m8 = (p.m + 7) & ~7;
    // The tile at t, or the next one there is of this workgroup's (t moves on).
    auto decode = [&](int &t, Tile &c) {
        int at = -1, list = 0, part = 0;
        c.slot = -1;
        for (; t < tiles_end; t += (int)gridDim.x) {
            if (!TAIL || parts == 1) {
                at = place_in_lists16(t, per_list, list);
                if (!rows_grouped && uniform(tab.start[list + 1] - tab.start[list]) == 0) at = -1;   // (zero_groups16)
            } else if (t < full) {
                at = place16(t, full);
            } else {
                const int v = place16(t - full, left * parts);
                if (v >= 0) {
                    part = v / left;
                    at = full + v - part * left;
                    c.slot = v;
                }
            }
            if (at >= 0) break;
        }
        c.valid = at >= 0;
        c.steps = 2;
        c.k_len = 0;
        c.left_a = c.left_b = 0;
        c.a = p.a;
        c.b = p.b;
        c.e = c.m0 = c.m_end = c.n0 = 0;
        if (!c.valid) return;
        int rt, ct, k0 = 0;
        c.k_len = p.k;
        tile_of16(at, row_tiles, col_tiles, rt, ct);
        if (rows_grouped) {
            c.e = uniform(group_of_tile16(tab, p.groups, rt));
            c.m0 = uniform(tab.start[c.e] + (rt - tab.tile[c.e]) * S::TM);
            c.m_end = uniform(tab.start[c.e + 1]);
            if (TAIL && c.slot >= 0) {
                k0 = part * part_k;
                c.k_len = min(p.k - k0, part_k);
            }
        } else {
            c.e = list;
            c.m0 = rt * S::TM;
            c.m_end = p.m;
            k0 = uniform(tab.start[c.e]);
            c.k_len = uniform(tab.start[c.e + 1]) - k0;
        }
        c.n0 = ct * S::TN;
        c.steps = max((c.k_len + 63) >> 6, 2);
        if (A_KM) {
            c.a = p.a + (int64_t)k0 * p.pitch_a + c.m0;
            c.left_a = c.k_len ? ((int64_t)(c.k_len - 1) * p.pitch_a + m8 - c.m0) * 2 : 0;
        } else {
            c.a = p.a + (int64_t)c.m0 * p.pitch_a + k0;
            c.left_a = ((int64_t)(min(c.m_end - c.m0, S::TM) - 1) * p.pitch_a + k8 - k0) * 2;
        }
        const uint16_t *b = p.b + (rows_grouped ? (int64_t)c.e * p.b_stride : (int64_t)0);
        if (B_KM) {
            c.b = b + (int64_t)k0 * p.pitch_b + c.n0;
            c.left_b = c.k_len ? ((int64_t)(c.k_len - 1) * p.pitch_b + n8 - c.n0) * 2 : 0;
        } else {
            c.b = b + (int64_t)c.n0 * p.pitch_b + k0;
            c.left_b = ((int64_t)(min(p.n - c.n0, S::TN) - 1) * p.pitch_b + k8 - k0) * 2;
        }
    };

    // What the requests two steps ahead are for; moved on once a step.
    struct Ahead {
        const uint16_t *a, *b;
        int64_t left_a, left_b;
        int k_left;
    } rq;
    Rsrc ra2, rb2, ra1, rb1;    // descriptors two steps ahead, one step ahead
    int k2, k1;                 // elements of K that are left there
    auto open = [&](const Tile &c) { rq = Ahead{c.a, c.b, c.left_a, c.left_b, c.k_len}; };
    auto describe = [&]() {
        ra2 = make_rsrc(rq.a, (uint32_t)max(min(rq.left_a, (int64_t)0x7FFFFFF0), (int64_t)0));
        rb2 = make_rsrc(rq.b, (uint32_t)max(min(rq.left_b, (int64_t)0x7FFFFFF0), (int64_t)0));
        k2 = uniform(rq.k_left);
    };
    auto advance = [&]() {
        rq.a = reinterpret_cast<const uint16_t *>(reinterpret_cast<const uint8_t *>(rq.a) + adv_a);
        rq.b = reinterpret_cast<const uint16_t *>(reinterpret_cast<const uint8_t *>(rq.b) + adv_b);
        rq.left_a -= adv_a;
        rq.left_b -= adv_b;
        rq.k_left -= 64;
    };
    auto request_a = [&](const Rsrc &rs, int k_left, uint32_t stage, auto q_c) {
        constexpr int q = decltype(q_c)::value;
        load16_to_lds(rs, A_KM || chunk_a[q] < k_left ? off_a[q] : NO_FETCH, 0u, dst_a[q] + stage);
    };
    auto request_b = [&](const Rsrc &rs, int k_left, uint32_t stage, auto q_c) {
        constexpr int q = decltype(q_c)::value;
        load16_to_lds(rs, B_KM || chunk_b[q] < k_left ? off_b[q] : NO_FETCH, 0u, dst_b[q] + stage);
    };

    Tile cur, nxt;
    int t = (int)blockIdx.x;
    decode(t, cur);
    if (!cur.valid) return;
    t += (int)gridDim.x;
    decode(t, nxt);

    uint32_t stage = 0;   // byte offset of the current step's panels in the ring: 0 or PANEL
    open(cur);
    describe();
    static_for<4>([&](auto q) { request_b(rb2, k2, 0u, q); });
    static_for<4>([&](auto q) { request_a(ra2, k2, 0u, q); });
    advance();
    describe();
    if constexpr (!HALVES) {
        static_for<4>([&](auto q) { request_b(rb2, k2, (uint32_t)PANEL, q); });
        request_a(ra2, k2, (uint32_t)PANEL, IC<0>{});
        request_a(ra2, k2, (uint32_t)PANEL, IC<1>{});
    } else {
        request_b(rb2, k2, (uint32_t)PANEL, IC<0>{});
        request_b(rb2, k2, (uint32_t)PANEL, IC<1>{});
        request_a(ra2, k2, (uint32_t)PANEL, IC<0>{});
        request_a(ra2, k2, (uint32_t)PANEL, IC<1>{});
        if constexpr (!A_KM) {
            request_a(ra2, k2, (uint32_t)PANEL, IC<2>{});
            request_a(ra2, k2, (uint32_t)PANEL, IC<3>{});
        }
    }
    CCH_WAIT_VM_LGKM0(0);
    CCH_BARRIER();
    if (wm == 1) CCH_BARRIER();   // one slot behind

    v16f acc[MT][NT];
    // Output stores of a wave that its next tile's first step may leave in flight: they are younger than what that step waits for.  Counted only where they are always issued.
    const bool whole = whole_rows(p), counted = whole && counted_stores<EPI>(p);
    const int more = !counted ? 0 : EPI == EPI16_ACT && p.preact ? 2 : 1;   // times 16
    int young = 0;   // what the current tile's first step finds

    // What a wait of n requests allows in step `first_c`: those, and in a tile's first step the stores
    auto wait = [&](auto first_c, auto n_c) {
        constexpr int n = decltype(n_c)::value;
        if constexpr (decltype(first_c)::value != 0) {
            if (young == 2) CCH_WAIT_VM(n + 32);
            else if (young == 1) CCH_WAIT_VM(n + 16);
            else CCH_WAIT_VM(n);
        } else {
            CCH_WAIT_VM(n);
        }
    };
    auto mma = [&](auto first_c, v16f &c, const v4i &b, const v4i &a) {
        if constexpr (decltype(first_c)::value != 0) c = T::mfma(b, a, (v16f)(0.0f));
        else c = T::mfma(b, a, c);
    };
    auto step = [&](auto first_c, int kt) {
        // descriptors: one step ahead are what two steps ahead were
        ra1 = ra2;
        rb1 = rb2;
        k1 = k2;
        if (kt + 2 == cur.steps) open(nxt);
        else advance();
        describe();
        const uint32_t other = (uint32_t)PANEL - stage;
        if constexpr (!HALVES) {
            v4i fb[NT][4], fa[2][4];
            // L0
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
#pragma unroll
                for (int j = 0; j < NT; j++) fb[j][kk] = lds_read16_abs(fr_b[kk] + (uint32_t)j * 4096u);
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) fa[i][kk] = lds_read16_abs(fr_a[kk] + (uint32_t)i * 4096u);
            __builtin_amdgcn_sched_barrier(0);
            request_a(ra1, k1, other, IC<2>{});
            request_a(ra1, k1, other, IC<3>{});
            CCH_WAIT_LGKM0();
            CCH_BARRIER();
            // C0
            static_for<4>([&](auto kk_c) {
                constexpr int kk = decltype(kk_c)::value;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++) mma(IC<(kk == 0 && decltype(first_c)::value)>{}, acc[i][j], fb[j][kk], fa[i][kk]);
                if constexpr (kk == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    request_a(ra2, k2, stage, IC<0>{});
                    request_a(ra2, k2, stage, IC<1>{});
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
            wait(first_c, IC<10>{});
            CCH_BARRIER();
            // L1
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) fa[i][kk] = lds_read16_abs(fr_a[kk] + (uint32_t)(2 + i) * 4096u);
            __builtin_amdgcn_sched_barrier(0);
            request_b(rb2, k2, stage, IC<0>{});
            request_b(rb2, k2, stage, IC<1>{});
            wait(first_c, IC<6>{});
            CCH_WAIT_LGKM0();
            CCH_BARRIER();
            // C1
            static_for<4>([&](auto kk_c) {
                constexpr int kk = decltype(kk_c)::value;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++) mma(IC<(kk == 0 && decltype(first_c)::value)>{}, acc[2 + i][j], fb[j][kk], fa[i][kk]);
                if constexpr (kk == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    request_b(rb2, k2, stage, IC<2>{});
                    request_b(rb2, k2, stage, IC<3>{});
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        } else {
            v4i fb[NT][2], fa[MT][2];
            static_for<2>([&](auto h_c) {
                constexpr int h = decltype(h_c)::value;
                // L0, L1
#pragma unroll
                for (int kk = 0; kk < 2; kk++)
#pragma unroll
                    for (int j = 0; j < NT; j++) fb[j][kk] = read_transposed(ft_b[j] + (uint32_t)(2 * h + kk) * 16u * KM::ROW, KM::ROW);
#pragma unroll
                for (int kk = 0; kk < 2; kk++)
#pragma unroll
                    for (int i = 0; i < MT; i++)
                        fa[i][kk] = A_KM ? read_transposed(ft_a[i] + (uint32_t)(2 * h + kk) * 16u * KM::ROW, KM::ROW) : lds_read16_abs(fr_a[2 * h + kk] + (uint32_t)i * 4096u);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (h == 0) {
                    request_b(rb1, k1, other, IC<2>{});
                    request_b(rb1, k1, other, IC<3>{});
                    if constexpr (A_KM) {
                        request_a(ra1, k1, other, IC<2>{});
                        request_a(ra1, k1, other, IC<3>{});
                    }
                } else {
                    request_b(rb2, k2, stage, IC<0>{});
                    request_b(rb2, k2, stage, IC<1>{});
                    if constexpr (A_KM) {
                        request_a(ra2, k2, stage, IC<0>{});
                        request_a(ra2, k2, stage, IC<1>{});
                    }
                }
                if (wm == 1) wait(first_c, IC<8>{});
                CCH_WAIT_LGKM0();
                CCH_BARRIER();
                // C0, C1
                static_for<2>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value;
                    static_for<MT>([&](auto i_c) {
                        constexpr int i = decltype(i_c)::value;
#pragma unroll
                        for (int j = 0; j < NT; j++) mma(IC<(h == 0 && kk == 0 && decltype(first_c)::value)>{}, acc[i][j], fb[j][kk], fa[i][kk]);
                        if constexpr (h == 1 && !A_KM && kk == 0) {
                            __builtin_amdgcn_sched_barrier(0);
                            request_a(ra2, k2, stage, i_c);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                });
                __builtin_amdgcn_sched_barrier(0);
                if (wm == 0 || (h == 1 && !A_KM)) wait(first_c, IC<8>{});
                if constexpr (h == 0) CCH_BARRIER();
            });
        }
        // the other stage
        const uint32_t move = other - stage;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            if (!A_KM) fr_a[x] += move;
            if (!B_KM) fr_b[x] += move;
            if (A_KM) ft_a[x] += move;
        }
#pragma unroll
        for (int j = 0; j < NT; j++)
            if (B_KM) ft_b[j] += move;
        stage = other;
    };

    while (true) {
        step(IC<1>{}, 0);
        for (int kt = 1; kt < cur.steps; kt++) {
            CCH_BARRIER();
            step(IC<0>{}, kt);
        }
        // Both groups write their results in the same slot: the first behind the barrier that ends its last matrix slot, the second, one slot behind, before it.
        if (wm == 0) CCH_BARRIER();
        if (TAIL && cur.slot >= 0) {
            // (blocks of rows that there are none of stay out, so these stores are not counted on)
            f32x4 *to = reinterpret_cast<f32x4 *>(p.partial) + (int64_t)cur.slot * (TAIL16_BYTES / 16) + threadIdx.x;
            static_for<MT>([&](auto i_c) {
                static_for<NT>([&](auto j_c) {
                    constexpr int i = decltype(i_c)::value, j = decltype(j_c)::value;
                    if (cur.m0 + wm * 32 + i * 64 >= cur.m_end) return;
#pragma unroll
                    for (int q = 0; q < 4; q++) to[((i * NT + j) * 4 + q) * S::THREADS] = (f32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                });
            });
        } else {
            epilogue16<T, EPI, MT, NT, 64>(p, acc, cur.e, cur.m0, cur.m_end, cur.n0, wm * 32, wn * 64, whole, counted);
        }
        if (!nxt.valid) break;
        young = TAIL && cur.slot >= 0 ? 0 : more;
        cur = nxt;
        t += (int)gridDim.x;
        decode(t, nxt);
        if (wm == 1) CCH_BARRIER();
    }
    CCH_WAIT_VM_LGKM0(0);   // (requests past the last tile fetch nothing, but they write zeros to LDS)
}

// The last round's tiles whose K was split: their parts added up in order, 64 rows (a block of each group of waves) to a workgroup and turn, then what the product does with a result.
template <class T, int EPI> __global__ __launch_bounds__(Big16::THREADS) void gemm16_tail_kernel(Gemm16 p, int grid)
{
    using S = Big16;
    __shared__ GroupTable16 tab;
    if (threadIdx.x < 64) build_groups16(tab, p.group_sizes, p.groups, p.m, S::TM);
    __syncthreads();
    const int wave = uniform(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int row_tiles = uniform(tab.tile[p.groups]), col_tiles = (p.n + S::TN - 1) / S::TN, all = row_tiles * col_tiles, left = all % grid;
    const int parts = uniform(tail_parts16(left, grid, (p.k + 63) >> 6, p.tail));
    if (parts == 1) return;
    const bool whole = whole_rows(p);
    for (int t = blockIdx.x; t < left * S::MT; t += gridDim.x) {
        const int tile = t / S::MT, i = t % S::MT;
        int rt, ct;
        tile_of16(all - left + tile, row_tiles, col_tiles, rt, ct);
        const int e = uniform(group_of_tile16(tab, p.groups, rt)), m0 = uniform(tab.start[e] + (rt - tab.tile[e]) * S::TM), m_end = uniform(tab.start[e + 1]);
        if (m0 + i * 64 >= m_end) continue;
        const f32x4 *from = reinterpret_cast<const f32x4 *>(p.partial) + (int64_t)tile * (TAIL16_BYTES / 16) + i * (S::NT * 4 * S::THREADS) + threadIdx.x;
        f32x4 sum[S::NT * 4];
#pragma unroll
        for (int q = 0; q < S::NT * 4; q++) sum[q] = from[q * S::THREADS];
#pragma unroll 2
        for (int s = 1; s < parts; s++)
#pragma unroll
            for (int q = 0; q < S::NT * 4; q++) sum[q] += from[(int64_t)s * left * (TAIL16_BYTES / 16) + q * S::THREADS];
        v16f acc[1][S::NT];
#pragma unroll
        for (int q = 0; q < S::NT * 4; q++)
#pragma unroll
            for (int x = 0; x < 4; x++) acc[0][q >> 2][4 * (q & 3) + x] = sum[q][x];
        epilogue16<T, EPI, 1, S::NT, 64>(p, acc, e, m0, m_end, ct * S::TN, wm * 32 + i * 64, wn * 64, whole, false);
    }
}

template <class T, int LAYOUT, int EPI> int launch16_big(const Gemm16 &p, int64_t tiles, hipStream_t stream)
{
    static std::atomic<uint64_t> attr_set{0};
    auto kernel = gemm16_big_kernel<T, LAYOUT, EPI>;
    int dev = 0, cus = 0;
    CCH_HIP(hipGetDevice(&dev));
    CCH_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    if (const int rc = allow_lds16(reinterpret_cast<const void *>(kernel), Big16::LDS, attr_set)) return rc;
    const int64_t most = std::max(cus & ~7, 8), grid = p.tail ? most : std::min<int64_t>((tiles + 7) & ~(int64_t)7, most);   // (a multiple of 8: place16)
    kernel<<<dim3((uint32_t)grid), dim3(Big16::THREADS), Big16::LDS, stream>>>(p);
    if (const int rc = launch_status("gemm16_big_kernel")) return rc;
    if constexpr (LAYOUT != ROWS_TN && (EPI == EPI16_OUT || EPI == EPI16_ACT)) {
        if (p.tail) {
            gemm16_tail_kernel<T, EPI><<<dim3((uint32_t)(2 * grid)), dim3(Big16::THREADS), 0, stream>>>(p, (int)grid);
            return launch_status("gemm16_tail_kernel");
        }
    }
    return CCH_OK;
}

}  // namespace cch
