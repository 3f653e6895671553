// What the kernels of 16-bit products share: types, the panels' way from memory through LDS to the matrix instructions' operands, the group table, the
// activations, and the epilogues.
#pragma once
#include "gemm16.h"
#include "gemm_device.h"

namespace cch {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
    using V8 = bf16x8;
    static __device__ __forceinline__ v16f mfma(v4i a, v4i b, v16f c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint16_t from(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest even
    static __device__ __forceinline__ uint32_t two(float a, float b) { return __builtin_bit_cast(uint32_t, (bf16x2){(__bf16)a, (__bf16)b}); }
    static __device__ __forceinline__ float to(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
};
struct F16 {
    using V8 = f16x8;
    static __device__ __forceinline__ v16f mfma(v4i a, v4i b, v16f c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint16_t from(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ uint32_t two(float a, float b) { return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b}); }
    static __device__ __forceinline__ float to(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
};

// ---- activations, fp32.  gelu_tanh(z) = z (1 + tanh u) / 2 with u = sqrt(2/pi) (z + 0.044715 z^3), which is z / (1 + exp(-2u)).
__device__ __forceinline__ float sigmoid16(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
constexpr float GELU_A = 1.5957691216057308f, GELU_B = 0.044715f;   // 2 sqrt(2/pi)
__device__ __forceinline__ float act_value(float z, int act)
{
    switch (act) {
    case CCH_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case CCH_ACT_SILU: return z * sigmoid16(z);
    case CCH_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.7071067811865476f));
    case CCH_ACT_GELU_TANH: return z * sigmoid16(GELU_A * (z + GELU_B * z * z * z));
    default: return z;
    }
}
// (one branch for all of them)
template <int N> __device__ __forceinline__ void apply_act(float (&v)[N], int act)
{
    switch (act) {
#define CCH_EACH(ACT) case ACT: _Pragma("unroll") for (int x = 0; x < N; x++) v[x] = act_value(v[x], ACT); break
    CCH_EACH(CCH_ACT_RELU);
    CCH_EACH(CCH_ACT_SILU);
    CCH_EACH(CCH_ACT_GELU);
    CCH_EACH(CCH_ACT_GELU_TANH);
#undef CCH_EACH
    }
}
__device__ __forceinline__ float act_slope(float z, int act)
{
    switch (act) {
    case CCH_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case CCH_ACT_SILU: {
        const float s = sigmoid16(z), c = fminf(fmaxf(z, -1e3f), 1e3f);   // (c: past it s (1 - s) is 0, and infinity times it would not be)
        return s + c * (s * (1.0f - s));
    }
    case CCH_ACT_GELU: {
        const float c = fminf(fmaxf(z, -1e3f), 1e3f);
        return 0.5f * (1.0f + erff(z * 0.7071067811865476f)) + c * 0.3989422804014327f * __expf(-0.5f * c * c);
    }
    case CCH_ACT_GELU_TANH: {
        const float s = sigmoid16(GELU_A * (z + GELU_B * z * z * z)), c = fminf(fmaxf(z, -1e3f), 1e3f);
        return s + c * (s * (1.0f - s)) * GELU_A * (1.0f + 3.0f * GELU_B * c * c);
    }
    default: return 1.0f;
    }
}

// ---- groups.  start[g] .. start[g + 1]: group g's rows (or K); tile[g]: its first row tile among all groups'.
struct GroupTable16 {
    int start[MAX_GROUPS16 + 1];
    int tile[MAX_GROUPS16 + 1];
};
// By one wave.  `all`: rows (or K) that there are; sizes are clipped to what the groups before leave (no sizes: one group of all).  bm: rows of a tile.
__device__ inline void build_groups16(GroupTable16 &tab, const int32_t *sizes, int groups, int all, int bm)
{
    const int lane = threadIdx.x & 63;
    if (!sizes) {
        if (lane == 0) {
            tab.start[0] = tab.tile[0] = 0;
            tab.start[1] = all;
            tab.tile[1] = (all + bm - 1) / bm;
        }
        return;
    }
    uint32_t before = 0;
    int tiles_before = 0;
    for (int b = 0; b < groups; b += 64) {
        const int g = b + lane;
        uint32_t sz = 0;
        if (g < groups) sz = (uint32_t)min(max(sizes[g], 0), all);
        const uint32_t incl = sat_add(before, wave_scan_sat(sz));
        const uint32_t prev = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)incl, 0x138, 0xF, 0xF, false);   // the neighbour's: wave_shr:1
        const int hi = (int)min(incl, (uint32_t)all), lo = (int)min(lane == 0 ? before : prev, (uint32_t)all);
        const int tiles = (hi - lo + bm - 1) / bm;
        const int tincl = (int)wave_scan_sat((uint32_t)tiles);
        if (g < groups) {
            tab.start[g] = lo;
            tab.tile[g] = tiles_before + tincl - tiles;
        }
        before = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
        tiles_before += __builtin_amdgcn_readlane(tincl, 63);
    }
    if (lane == 0) {
        tab.start[groups] = (int)min(before, (uint32_t)all);
        tab.tile[groups] = tiles_before;
    }
}
// The last group whose first tile is not behind `t`: the one that t belongs to, as groups without tiles begin where the next one does.
__device__ __forceinline__ int group_of_tile16(const GroupTable16 &tab, int groups, int t)
{
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.tile[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// Place of the launch's t-th tile in the list of `total`: consecutive workgroups run on the 8 XCDs in turn, and each XCD takes a run of consecutive
// tiles, so that its L2 sees neighbours.  -1: none.
__device__ __forceinline__ int place16(int t, int total)
{
    const int per = (int)(((uint32_t)total + 7) >> 3), i = t >> 3;
    const int64_t at = (int64_t)(t & 7) * per + i;
    return i < per && at < total ? (int)at : -1;
}
// The launch's t-th tile of `groups` lists of `per` tiles each: the list in `e`, the place in it returned, -1 for none.  Every list is spread over all XCDs, as lists
// whose tiles take different times (groups of K) would otherwise leave some XCDs behind.  `lists_end`: from where on there is none.
__device__ __forceinline__ int lists_end16(int per, int groups) { return ((per + 7) & ~7) * groups; }
__device__ __forceinline__ int place_in_lists16(int t, int per, int &e)
{
    const int whole = (per + 7) & ~7;
    e = t / whole;
    return place16(t - e * whole, per);
}

// Tiles are walked in bands of 8 row tiles, column by column: the 32 to 64 tiles that an XCD works on at a time then share 8 panels of A and 4 to 8 of B.
constexpr int BAND16 = 8;
__device__ __forceinline__ void tile_of16(int at, int row_tiles, int col_tiles, int &rt, int &ct)
{
    const int per = BAND16 * col_tiles, band = at / per, in = at - band * per;
    const int rows = min(BAND16, row_tiles - band * BAND16);
    ct = in / rows;
    rt = band * BAND16 + in - ct * rows;
}

// ---- panels.  A step is 64 elements of K.
// K contiguous: a row is 128 bytes, its 16-byte chunk c at position c ^ ((row >> 1) & 7) (gemm_device.h).  Lane (r, g) of a 32 x 32 x 16 instruction holds
// elements 8g..8g+7 of a sixteenth: chunk 2 kk + g.
// K-major: a K-row is COLS * 2 bytes; a transposing LDS load hands 16 lanes four K-rows of 16 columns, lane i addressing columns 4 (i % 4) .. of row i / 4 and
// receiving column i.  32 lanes, one pass of the load, touch 64 bytes of each of four rows that lie a multiple of 256 bytes apart: the chunk
// position's bits 2 and 3 are those of the chunk xor the row's, which puts them on all banks once.  (Four rows of 64 bytes are on all banks as they are.)
template <int COLS> struct KMajor {
    static constexpr int ROW = COLS * 2, CHUNKS = COLS / 8, ROWS_PER_KIB = 512 / COLS;
    static_assert(COLS == 32 || COLS % 128 == 0, "64 columns would need a swizzle of their own");
    static __device__ __forceinline__ uint32_t swizzle(int row) { return COLS >= 128 ? (uint32_t)(row & 3) << 2 : 0u; }
};
__device__ __forceinline__ v4i read_transposed(uint32_t addr, uint32_t row_bytes)
{
    typedef __attribute__((address_space(3))) v4s *P;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)addr);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)(addr + 4 * row_bytes));
    const v2i l = __builtin_bit_cast(v2i, lo), h = __builtin_bit_cast(v2i, hi);
    return (v4i){l[0], l[1], h[0], h[1]};
}

// A descriptor of what is left of a K-major operand from K-row k0 and column c0 on: the last of its `k` rows ends with its n-th column (the 16 bytes that hold it).
__device__ __forceinline__ Rsrc kmajor_rsrc(const uint16_t *base, int64_t pitch, int k0, int k, int c0, int n)
{
    const int64_t left = k0 < k ? ((int64_t)(k - k0 - 1) * pitch + (((n + 7) & ~7) - c0)) * 2 : 0;
    return make_rsrc(base + (int64_t)k0 * pitch + c0, (uint32_t)min(left, (int64_t)0x7FFFFFF0));
}

// Sixteen bytes anywhere: global memory takes them on any element's address, where rows do not start on 16-byte boundaries (1733 x 307, K = 512, with a residual and preact: 18.8 us, element by element 35.8).
struct __attribute__((packed, aligned(2))) Unaligned16 {
    v4i v;
};

// ---- epilogues.  The matrix instructions take B's fragment first: lane (r, g) then holds, of a 32 x 32 block, row r and columns 8 q + 4 g + x at 4 q + x.
template <class T> __device__ __forceinline__ v4i pack8(const float v[8])
{
    v4i o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (int)((uint32_t)T::from(v[2 * i]) | (uint32_t)T::from(v[2 * i + 1]) << 16);
    return o;
}
template <class T> __device__ __forceinline__ void unpack8(v4i o, float v[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = T::to((uint16_t)(uint32_t)o[i]);
        v[2 * i + 1] = T::to((uint16_t)((uint32_t)o[i] >> 16));
    }
}
// Eight elements, of which `there` exist.
template <class T> __device__ __forceinline__ void load8(const uint16_t *p, int there, float v[8])
{
    if (there >= 8) {
        unpack8<T>(reinterpret_cast<const Unaligned16 *>(p)->v, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < there ? T::to(p[i]) : 0.0f;
}

// Whether the epilogue's tensors have rows on 16-byte boundaries: then p.n is a multiple of 8, or (EPI16_GRAD) rows have room for whole pieces.
__device__ __forceinline__ bool whole_rows(const Gemm16 &p)
{
    return p.pitch_out % 8 == 0 && ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0 && (((uintptr_t)p.bias | (uintptr_t)p.residual | (uintptr_t)p.preact) & 15) == 0;
}
// Whether every tile of such a problem stores the same number of times, whatever of it exists: 16 stores of a wave with 128 x 64 outputs, twice that with preact.
template <int EPI> __device__ __forceinline__ bool counted_stores(const Gemm16 &p) { return EPI != EPI16_STATS && !p.sums && !p.out_rows; }

// A block's 16 values of a lane as memory wants them.  Rounded to pairs (q, w) of columns 8 q + 4 g + 2 w, + 1; a swap between the wave's halves of pairs 2 h and 2 h + 1 makes that 16 bytes of
// columns 16 h + 8 g; a swap of rows of 16 lanes between h = 0 and 1 then brings four lanes, 64 bytes, to a row: out[0] has rows 0..15 of the block, out[1] rows 16..31, the lane's row among them
// being lane & 15 and its columns lane_columns(lane) + 0..7.  Both swaps undo themselves.  Pairs are swapped, not the fp32 values: the epilogue of a tile is its vector instructions, four clocks
// each and two waves to a SIMD.  (Stored as the lanes hold them, 32 bytes a row, a 256 x 256 tile's epilogue took 11 us; 64 bytes a row is as fast as whole lines by way of LDS.)
__device__ __forceinline__ int lane_columns(int lane) { return (lane >> 4 & 1) * 16 + (lane >> 5) * 8; }
__device__ __forceinline__ void swap32(uint32_t &x, uint32_t &y)
{
    const auto s = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = s[0];
    y = s[1];
}
__device__ __forceinline__ void swap16(uint32_t &x, uint32_t &y)
{
    const auto s = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = s[0];
    y = s[1];
}
template <class T> __device__ __forceinline__ void to_rows(const float (&v)[16], v4i (&out)[2])
{
    uint32_t p[4][2];
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int w = 0; w < 2; w++) p[q][w] = T::two(v[4 * q + 2 * w], v[4 * q + 2 * w + 1]);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int w = 0; w < 2; w++) swap32(p[2 * h][w], p[2 * h + 1][w]);
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
        for (int w = 0; w < 2; w++) swap16(p[q][w], p[q + 2][w]);
#pragma unroll
    for (int h = 0; h < 2; h++) out[h] = (v4i){(int)p[2 * h][0], (int)p[2 * h][1], (int)p[2 * h + 1][0], (int)p[2 * h + 1][1]};
}
template <class T> __device__ __forceinline__ void from_rows(const v4i (&in)[2], float (&v)[16])
{
    uint32_t p[4][2];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int x = 0; x < 4; x++) p[2 * h + (x >> 1)][x & 1] = (uint32_t)in[h][x];
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
        for (int w = 0; w < 2; w++) swap16(p[q][w], p[q + 2][w]);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int w = 0; w < 2; w++) swap32(p[2 * h][w], p[2 * h + 1][w]);
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int w = 0; w < 2; w++) {
            v[4 * q + 2 * w] = T::to((uint16_t)p[q][w]);
            v[4 * q + 2 * w + 1] = T::to((uint16_t)(p[q][w] >> 16));
        }
}

// The results of one wave: MT x NT blocks of 32 x 32, every RS rows from row mw on and side by side from column nw of the tile that begins at row m0 and column n0 of the
// product, of which rows below m_end exist.  group: the output that K-grouped problems write.  counted: whole pieces are stored
// by way of a descriptor that drops what lies outside, always the same number of times (counted_stores).
template <class T, int EPI, int MT, int NT, int RS>
__device__ __forceinline__ void epilogue16(const Gemm16 &p, v16f (&acc)[MT][NT], int group, int tile_m, int m_end, int tile_n, int mw, int nw, bool whole, bool counted)
{
    static_assert(NT == 2, "64 columns to a wave");
    // (opaque: what depends on the lane would otherwise be worked out before the loop over tiles and take registers from the loop over K)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int r = lane & 31, g = lane >> 5, m0 = tile_m + mw, n0 = tile_n + nw;
    if (!counted && n0 >= p.n) return;
    // this lane's columns of block j: n0 + 32 j + 8 q + 4 g + x at 4 q + x; those from `left` on do not exist
    const int left = p.n - n0 - 4 * g;
    auto column = [](int j, int x) { return 32 * j + 8 * (x >> 2) + (x & 3); };
    const bool edge = n0 + 32 * NT > p.n;
    if constexpr (EPI == EPI16_STATS) {
        // 64 columns' largest logit and sum of exponentials, the two halves of the wave joined; a target's logit on the way
        static_for<MT>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            const int m = m0 + RS * i + r;
            const bool there = m < m_end;
            const int want = there ? p.targets[m] - p.v0 - n0 - 4 * g : -1;
            if (__any(want >= 0 && want < 32 * NT)) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 16; x++)
                        if (column(j, x) == want) p.target_logit[m] = acc[i][j][x];
            }
            if (edge) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 16; x++)
                        if (column(j, x) >= left) acc[i][j][x] = -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int x = 0; x < 16; x++) top = fmaxf(top, acc[i][j][x]);
            top = fmaxf(top, __shfl_xor(top, 32));
            // (all of them -inf: a sum of 0; a NaN among them: NaN)
            const float base = top > -INFINITY ? top : 0.0f;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int x = 0; x < 16; x++) sum += __expf(acc[i][j][x] - base);
            sum += __shfl_xor(sum, 32);
            if (there && g == 0) p.stats[(int64_t)m * p.stat_cols + (p.v0 + n0) / (32 * NT)] = make_float2(top, sum);
        });
    } else {
        uint16_t *const out = p.out + (int64_t)group * p.out_stride;
        const bool scaled = EPI == EPI16_OUT && p.scale, summed = EPI == EPI16_OUT && p.sums;
        const float scale = scaled ? *p.scale : 1.0f, grad_scale = EPI == EPI16_GRAD && p.grad_scale ? *p.grad_scale : 1.0f;
        const int lc = lane_columns(lane);
        // counted: descriptors of the tile's rows that exist; a lane whose columns do not starts 2^31 bytes behind, past any of them
        const int64_t tile_at = (int64_t)tile_m * p.pitch_out + tile_n;
        const int tile_bytes = (int)min(((int64_t)max(m_end - tile_m, 0) * p.pitch_out - tile_n) * 2, (int64_t)0x7FFFFFF0);
        const uint32_t pitch = (uint32_t)p.pitch_out * 2u;
        uint32_t lane_at[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) lane_at[j] = (uint32_t)(mw + (lane & 15)) * pitch + (uint32_t)(nw + 32 * j + lc) * 2u + (n0 + 32 * j + lc < p.n ? 0u : 0x80000000u);
        float bias[NT][16];
        if constexpr (EPI == EPI16_ACT) {
            if (p.bias) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 16; x++) bias[j][x] = column(j, x) < left ? T::to(p.bias[n0 + 4 * g + column(j, x)]) : 0.0f;
            }
        }
        static_for<MT>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            const int first = m0 + RS * i, m = first + r;
            if (!counted && first >= m_end) return;
            const bool there = m < m_end;
            float lse = 0.0f, slope = 0.0f;
            int want = -1;
            bool wanted = false;
            if constexpr (EPI == EPI16_GRAD) {
                lse = there ? p.lse[m] : 0.0f;
                slope = (1.0f + p.z2 * lse) * grad_scale;
                want = there ? p.targets[m] - p.v0 - n0 - 4 * g : -1;
                wanted = __any(want >= 0 && want < 32 * NT);
            }
            static_for<NT>([&](auto j_c) {
                constexpr int j = decltype(j_c)::value;
                float v[16];
#pragma unroll
                for (int x = 0; x < 16; x++) v[x] = acc[i][j][x];
                // sixteen bytes of `base` in rows' layout: store (or load) row `row` of the block, columns lane_at
                auto each_row = [&](auto &&at_row) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int at = first + 16 * h + (lane & 15), c = n0 + 32 * j + lc;
                        if (at >= m_end || c >= p.n) continue;
                        const int64_t to = EPI == EPI16_OUT && p.out_rows ? p.out_rows[at] : at;
                        at_row(h, to * p.pitch_out + c);
                    }
                };
                auto store = [&](uint16_t *base) {
                    v4i rows[2];
                    to_rows<T>(v, rows);
                    if (whole) {
                        if (counted) {
                            const auto rs = __builtin_amdgcn_make_buffer_rsrc(base + tile_at, 0, tile_bytes, 0x00020000);
#pragma unroll
                            for (int h = 0; h < 2; h++)
                                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, rows[h]), rs, lane_at[j] + (uint32_t)(RS * i + 16 * h) * pitch, 0, 0);
                        } else {
                            each_row([&](int h, int64_t at) { *reinterpret_cast<v4i *>(base + at) = rows[h]; });
                        }
                    } else {
                        each_row([&](int h, int64_t at) {
                            const int there = p.n - n0 - 32 * j - lc;
                            if (there >= 8) reinterpret_cast<Unaligned16 *>(base + at)->v = rows[h];
                            else
#pragma unroll
                                for (int x = 0; x < 7; x++)
                                    if (x < there) base[at + x] = (uint16_t)((uint32_t)rows[h][x >> 1] >> (16 * (x & 1)));
                        });
                    }
                };
                if constexpr (EPI == EPI16_OUT) {
                    if (summed) {
                        float *s = p.sums + (int64_t)m * p.n + n0 + 4 * g;
                        if (there)
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const int c = column(j, 4 * q);
                                if (p.n % 4 == 0 && c < left) {
                                    f32x4 *at = reinterpret_cast<f32x4 *>(s + c);
                                    f32x4 a = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                                    if (p.sums_in) a += *at;
                                    if (p.sums_out) *at = a;
#pragma unroll
                                    for (int x = 0; x < 4; x++) v[4 * q + x] = a[x];
                                } else {
#pragma unroll
                                    for (int x = 0; x < 4; x++)
                                        if (c + x < left) {
                                            if (p.sums_in) v[4 * q + x] += s[c + x];
                                            if (p.sums_out) s[c + x] = v[4 * q + x];
                                        }
                                }
                            }
                        if (p.sums_out) return;
                    }
                    if (scaled) {
#pragma unroll
                        for (int x = 0; x < 16; x++) v[x] *= scale;
                    }
                    store(out);
                } else if constexpr (EPI == EPI16_ACT) {
                    if (p.bias) {
#pragma unroll
                        for (int x = 0; x < 16; x++) v[x] += bias[j][x];
                    }
                    if (p.preact) store(p.preact);
                    apply_act(v, p.act);
                    if (p.residual) {
                        float add[16] = {};
                        v4i rows[2] = {};
                        each_row([&](int h, int64_t at) {
                            const int there = whole ? 8 : p.n - n0 - 32 * j - lc;
                            if (there >= 8) rows[h] = reinterpret_cast<const Unaligned16 *>(p.residual + at)->v;
                            else
#pragma unroll
                                for (int x = 0; x < 7; x++)
                                    if (x < there) rows[h][x >> 1] |= (int)((uint32_t)p.residual[at + x] << (16 * (x & 1)));
                        });
                        from_rows<T>(rows, add);
#pragma unroll
                        for (int x = 0; x < 16; x++) v[x] += add[x];
                    }
                    store(out);
                } else {
                    // rows of the gradient end on 16-byte boundaries, zeros behind the last column: the next product reads it along K
#pragma unroll
                    for (int x = 0; x < 16; x++) v[x] = __expf(v[x] - lse) * slope;
                    if (wanted) {
#pragma unroll
                        for (int x = 0; x < 16; x++)
                            if (column(j, x) == want) v[x] -= grad_scale;
                    }
                    if (edge) {
#pragma unroll
                        for (int x = 0; x < 16; x++)
                            if (column(j, x) >= left) v[x] = 0.0f;
                    }
                    store(out);
                }
            });
        });
    }
}

// The fp32 sums of one part of K: MT x NT blocks from row m0 and column n0 on, rows below m_end, to rows of n.
template <int MT, int NT> __device__ __forceinline__ void store_part16(const Gemm16 &p, const v16f (&acc)[MT][NT], float *to, int m0, int m_end, int n0)
{
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int m = m0 + 32 * i + r;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int n = n0 + 32 * j + 8 * q + 4 * g, left = p.n - n;
                if (m >= m_end || left <= 0) continue;
                float *s = to + (int64_t)m * p.n + n;
                const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (p.n % 4 == 0) {
                    *reinterpret_cast<f32x4 *>(s) = v;
                } else {
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (x < left) s[x] = v[x];
                }
            }
    }
}

// Rows behind the last group: zeros.
__device__ __forceinline__ void zero_rest16(const Gemm16 &p, int first)
{
    const int64_t begin = (int64_t)first * p.pitch_out, end = (int64_t)p.m * p.pitch_out, threads = (int64_t)gridDim.x * blockDim.x;
    const int64_t me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (((uintptr_t)p.out & 15) == 0 && p.pitch_out % 8 == 0) {
        v4i *o = reinterpret_cast<v4i *>(p.out);
        for (int64_t i = begin / 8 + me; i < end / 8; i += threads) o[i] = (v4i){0, 0, 0, 0};
    } else {
        for (int64_t i = begin + me; i < end; i += threads) p.out[i] = 0;
    }
}

// K grouped: zeros to the outputs of groups without a K, which the kernel then leaves out (backward of 9 rows over 128 experts, 1152 x 1007: 190 -> 127 us).
__device__ __forceinline__ void zero_groups16(const Gemm16 &p, const GroupTable16 &tab)
{
    const int64_t n = (int64_t)p.m * p.pitch_out, threads = (int64_t)gridDim.x * blockDim.x, me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int g = 0; g < p.groups; g++) {
        if (uniform(tab.start[g + 1] - tab.start[g]) > 0) continue;
        uint16_t *o = p.out + g * p.out_stride;
        for (int64_t i = me; i < n / 8; i += threads) reinterpret_cast<Unaligned16 *>(o)[i].v = (v4i){0, 0, 0, 0};
        if (me < n % 8) o[n / 8 * 8 + me] = 0;
    }
}

}  // namespace cch
