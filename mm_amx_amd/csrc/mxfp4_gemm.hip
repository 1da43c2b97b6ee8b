// Products in microscaled 4-bit floating point: C = PP( sum over blocks kb of 32 k of sA[m][kb] sB[n][kb] (A_kb . B_kb) ).
//
// The matrix cores apply both scales themselves, so all sums stay in them.  The weights are the first operand: a lane then holds neighbouring columns of one row of C.  An instruction's
// sum came out within 2^-20 of its largest term over random values and scales, and exact wherever it can be held in 24 bits; scales of 255 make a NaN of their row, products from 2^128 on an infinity.
#include "mxfp4.hpp"

namespace mmx {

int num_cus();

__device__ __forceinline__ i32x8 mx_operand(u32x4 a) { return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}; }

// ---- few rows: every wavefront multiplies its own chunks of k --------------------------------------------------------------
// A workgroup computes 16 NT columns of 16 MT rows; its eight wavefronts take chunks of 256 k in turn, straight from memory into registers, and add their sums in LDS in the order of the
// wavefronts.  The 16 x 16 x 128 form of the instruction (half the rate of the other, which does not matter here) lets a workgroup have half a panel.
// PAIR: the four column tiles are both halves of a gate panel and of its up panel, 32 columns of the result, a whole block of it.
// QUANTIZE: A is bf16 rows, which every workgroup quantises into LDS while its first weights are on their way.
// Bound: HBM, at M = 1 the launch too.  1 x 4096 x 11008 6.4 us from bf16 rows (3.8 TB/s of weights; a quantiser of its own in front costs 4 us more), 16 x 4096 x 22016 as a pair 10.3,
// 24 x 11008 x 4096 6.9 (16 rows a workgroup 7.9, 64 8.0, 32 columns 8.5).
template <int MT, int NT, bool PAIR, bool QUANTIZE>
__global__ __launch_bounds__(512) void mxfp4_rows_kernel(const Mxfp4Gemm g) {
    static_assert(!PAIR || NT == 4, "both halves of a gate and an up panel");
    constexpr int NW = 8;
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][MT * NT][64];
    extern __shared__ __attribute__((aligned(16))) char rows[];  // QUANTIZE: M rows of pitch bytes, then their scales, M rows of 8 chunks bytes
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, quad = lane >> 4;
    const int m0 = blockIdx.y * (16 * MT);
    const int pitch = g.chunks * 128 + 16;  // (16 bytes more: neighbouring rows in other banks)
    // this lane's place in a chunk: of its row c, block 4 kk + quad for the instructions kk = 0, 1
    const uint32_t place = (quad >> 1) * 1024 + (quad & 1) * 512 + c * 16, scale_place = MX_SCALES_AT + (quad & 1) * 128 + c * 4;
    const int turn = 8 * (quad >> 1);

    const char* w_at[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int tile = PAIR ? blockIdx.x * 4 + j : blockIdx.x * NT + j;
        const int panel = tile >> 1 < g.npanels ? tile >> 1 : g.npanels - 1;
        w_at[j] = g.B + (int64_t)panel * g.ldb + (tile & 1) * 256;  // (its scales: 64 bytes on)
    }
    const int w_scale = (int)scale_place;
    const char* x_at[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        int m = m0 + i * 16 + c;
        m = m < g.M ? m : g.M - 1;
        // (a row past the last one: the last again, never stored)
        x_at[i] = QUANTIZE ? rows + m * pitch + quad * 16 : g.A + (int64_t)(m >> 5) * g.lda + ((m & 31) - c) * 16 + place;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // U chunks: ch, ch + NW, ...
    constexpr int U = MT * NT <= 2 ? 2 : 1;
    auto load = [&](auto n_c, int ch, u32x4 (&w)[U][NT][2], uint32_t (&sw)[U][NT]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < decltype(n_c)::value; u++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const char* const p = w_at[j] + (int64_t)(ch + u * NW) * MX_CHUNK_BYTES;
                w[u][j][0] = *reinterpret_cast<const u32x4*>(p + place);
                w[u][j][1] = *reinterpret_cast<const u32x4*>(p + place + 2048);
                const int half = (PAIR ? j : blockIdx.x * NT + j) & 1;
                sw[u][j] = *reinterpret_cast<const uint32_t*>(p + w_scale - half * 192) >> turn;
            }
    };
    auto multiply = [&](auto n_c, int ch, const u32x4 (&w)[U][NT][2], const uint32_t (&sw)[U][NT]) __attribute__((always_inline)) {
        constexpr int N = decltype(n_c)::value;
        u32x4 x[N][MT][2];
        uint32_t sx[N][MT];
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < MT; i++) {
                if constexpr (QUANTIZE) {
                    int m = m0 + i * 16 + c;
                    m = m < g.M ? m : g.M - 1;
                    x[u][i][0] = *reinterpret_cast<const u32x4*>(x_at[i] + (ch + u * NW) * 128);
                    x[u][i][1] = *reinterpret_cast<const u32x4*>(x_at[i] + (ch + u * NW) * 128 + 64);
                    // bytes 0 and 2 are the ones that are taken
                    const char* const s = rows + g.M * pitch + (m * g.chunks + ch + u * NW) * 8 + quad;
                    sx[u][i] = (uint32_t)(uint8_t)s[0] | (uint32_t)(uint8_t)s[4] << 16;
                } else {
                    const char* const p = x_at[i] + (int64_t)(ch + u * NW) * MX_CHUNK_BYTES;
                    x[u][i][0] = *reinterpret_cast<const u32x4*>(p);
                    x[u][i][1] = *reinterpret_cast<const u32x4*>(p + 2048);
                    int m = m0 + i * 16 + c;
                    m = m < g.M ? m : g.M - 1;
                    sx[u][i] = *reinterpret_cast<const uint32_t*>(p - place - ((m & 31) - c) * 12 + scale_place) >> turn;
                }
            }
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(w[u][j][0]), mx_operand(x[u][i][0]), acc[i][j], 4, 4, 0, (int)sw[u][j], 0, (int)sx[u][i]);
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(w[u][j][1]), mx_operand(x[u][i][1]), acc[i][j], 4, 4, 2, (int)sw[u][j], 2, (int)sx[u][i]);
                }
    };
    typedef std::integral_constant<int, U> all_c;
    typedef std::integral_constant<int, 1> one_c;
    u32x4 w[U][NT][2];
    uint32_t sw[U][NT];
    int ch = wave;
    if constexpr (QUANTIZE) {
        const bool ahead = ch + (U - 1) * NW < g.chunks;
        if (ahead) load(all_c(), ch, w, sw);
        // four lanes a block
        for (int b = threadIdx.x >> 2; b < g.M * g.chunks * 8; b += NW * 16) {
            const int m = b / (g.chunks * 8), kb = b - m * (g.chunks * 8), part = threadIdx.x & 3;
            float v[8];
            load_row_f32(reinterpret_cast<const uint16_t*>(g.A + m * g.lda), kb * MX_BLOCK + part * 8, g.K, v);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) top = umax(top, abs_bits(v[e]));
#pragma unroll
            for (int d = 1; d < 4; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
            const uint32_t s = mx_scale_of(top);
            *reinterpret_cast<uint32_t*>(rows + m * pitch + kb * 16 + part * 4) = to_fp4x8(v, mx_value_of(s));
            if (part == 0) rows[g.M * pitch + b] = (char)s;
        }
        __syncthreads();
        if (ahead) {
            multiply(all_c(), ch, w, sw);
            ch += U * NW;
        }
    }
    for (; ch + (U - 1) * NW < g.chunks; ch += U * NW) {
        load(all_c(), ch, w, sw);
        multiply(all_c(), ch, w, sw);
    }
    for (; ch < g.chunks; ch += NW) {
        load(one_c(), ch, w, sw);
        multiply(one_c(), ch, w, sw);
    }

#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) red[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    auto sum = [&](int t, int l, float (&r)[4]) __attribute__((always_inline)) {
        f32x4 s = red[0][t][l];
#pragma unroll
        for (int w = 1; w < NW; w++) {
            const f32x4 a = red[w][t][l];
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = s[e] + a[e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = s[e];
    };
    if constexpr (PAIR) {
        // 16 rows x 32 columns of the result: a row's columns 4 q ... 4 q + 3 of half h in lane l = 16 q + row % 16 of tile h; eight neighbouring threads take a row's eight fours
        for (int t = threadIdx.x; t < MT * 128; t += NW * 64) {
            const int row = t >> 3, part = t & 7, i = row >> 4, l = (part & 3) * 16 + (row & 15), half = part >> 2;
            const int m = m0 + row;
            float r[4], up[4];
            sum(i * NT + half, l, r);
            sum(i * NT + 2 + half, l, up);
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = silu32(r[e]) * up[e];
            if (!g.packed_out) {
                if (m < g.M) store4(g.ep, m, blockIdx.x * 32 + part * 4, g.N / 2, r);
                continue;
            }
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = umax(top, abs_bits(r[e]));
#pragma unroll
            for (int d = 1; d < 8; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
            const uint32_t s = mx_scale_of(top);
            if (m < g.M) {
                char* const panel = g.packed_out + (int64_t)(m >> 5) * g.ld_out;
                const uint16_t w = (uint16_t)to_fp4x4(r[0], r[1], r[2], r[3], mx_value_of(s));
                *reinterpret_cast<uint16_t*>(panel + mx_piece(m, blockIdx.x) + part * 2) = w;
                if (part == 0) panel[mx_scale_at(m, blockIdx.x)] = (char)s;
                if (blockIdx.x + 1 == gridDim.x) {  // what is left of the last chunk
                    for (int kb = blockIdx.x + 1; kb & 7; kb++) {
                        *reinterpret_cast<uint16_t*>(panel + mx_piece(m, kb) + part * 2) = 0;
                        if (part == 0) panel[mx_scale_at(m, kb)] = 127;
                    }
                }
            }
        }
    } else {
        for (int u = threadIdx.x; u < MT * NT * 64; u += NW * 64) {
            const int t = u >> 6, l = u & 63;
            const int m = m0 + (t / NT) * 16 + (l & 15);
            float r[4];
            sum(t, l, r);
            const int n = (blockIdx.x * NT + t % NT) * 16 + (l >> 4) * 4;
            if (m < g.M && n < g.N) {
                post4(g.ep, n, g.N, r);
                store4(g.ep, m, n, g.N, r);
            }
        }
    }
}

// ---- many rows: tiles ------------------------------------------------------------------------------------------------------
// A workgroup computes 32 PM WGM rows x 32 PN WGN columns, a wavefront PM x PN panels of them.  A stage is a chunk of 256 k: all the tile's panels' 4 KiB of values one behind the other,
// then their 256 bytes of scales, straight from memory into one of R slots of LDS; with the operands in the instruction's own order every LDS read is a KiB in a row.  A stage has four steps of 64 k;
// the operands of a step are read during the one before.  The one barrier per stage stands in front of its last step: all of it has been read into registers then, so its slot is free for
// stage t + R, whose loads are spread over the last step and the next stage's first two, and stage t + 1 has landed.
// Bound: what a CU gets from L2 into LDS (40 bytes a nanosecond in 256 x 192 tiles, two slots holding no more on its way) and the LDS itself, whose reads and writes a step of that tile take as long as
// its MFMAs; 2048 x 4096 x 11008 takes 61 to 65 us in a trace, by card, 2.8 to 3.0 PFLOP/s (57 with operands that stay in the caches, 3250 TFLOP/s, and 4096 x 4096 x 4096 3500), where the MFMAs alone reach
// 6670 on random values.  Refilling slots by halves, with loads R - 1 stages ahead, was no faster (57 -> 60 us),
// nor were 4 x 3 panels a wavefront with a third fewer LDS reads and one wavefront a SIMD (59).
// KG groups of wavefronts, each with a ring of its own, take the chunks in turn where there are fewer tiles than CUs; their sums are added in LDS, in order.
template <int PM, int PN, int WGM, int WGN, int R, int KG>
struct Mxfp4Tile {
    static constexpr int NW = WGM * WGN, BM = 32 * PM * WGM, BN = 32 * PN * WGN;
    static constexpr int PANELS = PM * WGM + PN * WGN;
    static constexpr int SCALES = PANELS * 4096;          // their place in a stage
    static constexpr int STAGE = SCALES + (PANELS + 3) / 4 * 1024;
    static constexpr int RING = R * STAGE, BIAS = KG * RING, BYTES = BIAS + 2 * BN * 4;  // (the columns' biases behind the rings, of this tile and the next)
    static_assert(BN % 64 == 0 || KG > 1, "64 biases at a time: those of 32 columns take the next tile's place, of which there is none where K is shared");
    static_assert((KG - 1) * BM * BN * 4 <= BIAS, "the groups' sums fit where the stages were");
    static constexpr int PIECES = PANELS * 4;             // KiB of values
    static constexpr int DATA_LOADS = PIECES / NW, SCALE_LOADS = ((PANELS + 3) / 4 + NW - 1) / NW, LOADS = DATA_LOADS + SCALE_LOADS;
    static_assert(PIECES % NW == 0 && BYTES <= 160 * 1024 && (R - 1) * LOADS < 64, "every wavefront issues the same number of loads, which a wait can count");
};

// A panel's 32 columns from n of row m, of which the lane holds 8 q + 4 half + 0..3: it takes its partner's (that of the same row) in exchange, so that each of the two has eight neighbours
// at a time, 16 or 32 bytes to store.
__device__ __forceinline__ void store16(const Epilogue& ep, int m, int M, int n, int n1, int half, const float (&r)[16]) {
    char* const row = ep.C + (int64_t)m * ep.ldc;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const int at = n + 16 * p + 8 * half;
        if (ep.out_dtype == MMX_F32) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const auto v = __builtin_amdgcn_permlane32_swap(f2u(r[8 * p + e]), f2u(r[8 * p + 4 + e]), false, false);
                w[e] = v[0], w[4 + e] = v[1];
            }
            float* const to = reinterpret_cast<float*>(row) + at;
            if (m >= M) continue;
            if (at + 8 <= n1) {
                __builtin_memcpy(__builtin_assume_aligned(to, 4), w, 32);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (at + e < n1) to[e] = u2f(w[e]);
            }
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const auto v = __builtin_amdgcn_permlane32_swap((uint32_t)to_bf16(r[8 * p + 2 * e]) | (uint32_t)to_bf16(r[8 * p + 2 * e + 1]) << 16,
                                                                (uint32_t)to_bf16(r[8 * p + 4 + 2 * e]) | (uint32_t)to_bf16(r[8 * p + 5 + 2 * e]) << 16, false, false);
                w[e] = v[0], w[2 + e] = v[1];
            }
            uint16_t* const to = reinterpret_cast<uint16_t*>(row) + at;
            if (m >= M) continue;
            if (at + 8 <= n1) {
                __builtin_memcpy(__builtin_assume_aligned(to, 2), w, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (at + e < n1) to[e] = (uint16_t)(w[e >> 1] >> 16 * (e & 1));
            }
        }
    }
}

template <int PM, int PN, int WGM, int WGN, int R, int KG>
__global__ __launch_bounds__(WGM * WGN * KG * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void mxfp4_tile_kernel(const Mxfp4Gemm g, int tiles_m, int tiles_n, int total, int per_xcd) {
    using T = Mxfp4Tile<PM, PN, WGM, WGN, R, KG>;
    static_assert(PM * PN <= 8, "sums of 128 registers at most");
    constexpr int NW = T::NW, STAGE = T::STAGE, LOADS = T::LOADS, DATA = T::DATA_LOADS;
    using lds_u32x4 = __attribute__((address_space(3))) const u32x4;
    using lds_u32 = __attribute__((address_space(3))) const uint32_t;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // Neighbouring workgroups go to different XCDs: each XCD gets a run of tiles, eight rows of them at a time and those fastest, so that the ones it works on share both operands in its L2.
    // A workgroup takes every stride-th tile of its XCD's run; the next one's first stages are on their way while its results are stored (2048 x 4096 x 11008 with a bias 62.5 -> 55 us).
    const int first = (blockIdx.x & 7) * per_xcd, stride = gridDim.x >> 3;
    int turn = blockIdx.x >> 3;
    if (first + turn >= total) return;
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all_waves % NW, group = all_waves / NW;
    const int wm = wave / WGN, wn = wave % WGN;
    const int half = lane >> 5, c = lane & 31;
    const int panels_m = (g.M + 31) >> 5;
    int panel_m0, panel_n0;
    const int steps = (g.chunks - group + KG - 1) / KG, most = (g.chunks + KG - 1) / KG;  // of this group, of any: chunks group, group + KG, ...

    // ---- loads: this wavefront's KiB of a stage.  A tile may reach past the last panel: that one again, never stored.
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem) + group * T::RING;
    auto panel_at = [&](int p) __attribute__((always_inline)) {
        if (p < PM * WGM) {
            const int panel = panel_m0 + p < panels_m ? panel_m0 + p : panels_m - 1;
            return g.A + (int64_t)panel * g.lda;
        }
        p -= PM * WGM;
        const int panel = panel_n0 + p < g.npanels ? panel_n0 + p : g.npanels - 1;
        return g.B + (int64_t)panel * g.ldb;
    };
    const char* from[LOADS];  // (uniform for values, each lane's own for scales)
    uint32_t to[LOADS];
    auto go_to = [&](int L) __attribute__((always_inline)) {
        const int band = L / (8 * tiles_n), in_band = L - band * (8 * tiles_n), high = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
        const int tn = in_band / high, tm = band * 8 + in_band - tn * high;
        panel_m0 = tm * (PM * WGM), panel_n0 = tn * (PN * WGN);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (i < DATA) {
                const int piece = i * NW + wave;
                from[i] = panel_at(piece >> 2) + (piece & 3) * 1024;
                to[i] = lds0 + piece * 1024;
            } else {
                // 16 lanes a panel's scales; what is past the last group of four panels again
                int four = (i - DATA) * NW + wave;
                four = four < (T::PANELS + 3) / 4 ? four : (T::PANELS + 3) / 4 - 1;
                const int p = four * 4 + (lane >> 4);
                from[i] = panel_at(p < T::PANELS ? p : T::PANELS - 1) + MX_SCALES_AT + (lane & 15) * 16;
                to[i] = lds0 + T::SCALES + four * 1024;
            }
        }
    };
    const uint32_t lane16 = lane * 16;
    auto load = [&](auto ic, int t, int slot) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(to[i] + slot * STAGE);
        if constexpr (i < DATA) {
            const char* const src = from[i] + (int64_t)(group + KG * t) * MX_CHUNK_BYTES;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(dst), "v"(lane16), "s"(src) : "memory");
        } else {
            const char* const src = from[i] + (int64_t)(group + KG * t) * MX_CHUNK_BYTES;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(dst), "v"(src) : "memory");
        }
    };

    f32x16 acc[PM][PN];
    u32x4 fa[2][PM], fb[2][PN];  // a step's operands, now and next
    uint32_t sa[2][PM], sb[2][PN];
    const uint32_t a_lane = wm * PM * 4096 + lane * 16, b_lane = (PM * WGM + wn * PN) * 4096 + lane * 16;
    const uint32_t sa_lane = T::SCALES + wm * PM * 256 + lane * 4, sb_lane = T::SCALES + (PM * WGM + wn * PN) * 256 + lane * 4;
    uint32_t at_a, at_b, at_sa, at_sb;
    auto places = [&](int slot) __attribute__((always_inline)) {
        const uint32_t st = lds0 + slot * STAGE;
        at_a = st + a_lane, at_b = st + b_lane, at_sa = st + sa_lane, at_sb = st + sb_lane;
        asm volatile("" : "+v"(at_a), "+v"(at_b), "+v"(at_sa), "+v"(at_sb));
    };
    auto read_a = [&](int i, int u) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32x4*>(at_a + i * 4096 + u * 1024); };
    auto read_b = [&](int j, int u) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32x4*>(at_b + j * 4096 + u * 1024); };
    auto read_sa = [&](int i) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32*>(at_sa + i * 256); };
    auto read_sb = [&](int j) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32*>(at_sb + j * 256); };

    // a tile's biases, 64 columns a wavefront, and its first stages
    const bool biased = g.ep.steps & MMX_PP_BIAS;
    auto start = [&](int parity) __attribute__((always_inline)) {
        if (biased && group == 0) {
#pragma unroll
            for (int b = 0; b < ((T::BN + 63) / 64 + NW - 1) / NW; b++) {
                const int part = b * NW + wave;
                if (part * 64 < T::BN) {
                    const int n = panel_n0 * 32 + part * 64 + lane;
                    const float* const src = g.ep.bias + (n < g.N ? n : g.N - 1);
                    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + T::BIAS + parity * (T::BN * 4) + part * 256);
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(dst), "v"(src) : "memory");
                }
            }
        }
        unrolled<0, R>([&](auto rc) __attribute__((always_inline)) {
            constexpr int r = decltype(rc)::value;
            unrolled<0, LOADS>([&](auto ic) __attribute__((always_inline)) { if (r < steps) load(ic, r, r); });
        });
    };
    go_to(first + turn);
    start(0);
    for (int parity = 0;; parity ^= 1) {
        // (behind the first tile its stores are among what is on its way, in an order of their own: all of it is waited for)
        if (parity == 0 && turn < stride && steps >= R) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((R - 1) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        places(0);
#pragma unroll
        for (int i = 0; i < PM; i++)
#pragma unroll
            for (int j = 0; j < PN; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < PM; i++) {
            fa[0][i] = read_a(i, 0);
            sa[0][i] = read_sa(i);
        }
#pragma unroll
        for (int j = 0; j < PN; j++) {
            fb[0][j] = read_b(j, 0);
            sb[0][j] = read_sb(j);
        }
        __builtin_amdgcn_sched_barrier(0);

        // One slot per MFMA, in this order and no other: the MFMA, an LDS read for the next step, a load.
        constexpr int PER = PM * PN, READS = PM + PN;
        int slot = 0;
        // ODD: which set of scales the stage has
        auto stage = [&](auto odd_c, int t) __attribute__((always_inline)) {
            constexpr int S = decltype(odd_c)::value;
            const int next = slot + 1 < R ? slot + 1 : 0, before = slot > 0 ? slot - 1 : R - 1;
            const bool more_before = t > 0 && t - 1 + R < steps, more = t + R < steps;
            unrolled<0, 4 * PER>([&](auto xc) __attribute__((always_inline)) {
                constexpr int x = decltype(xc)::value, u = x / PER, y = x % PER, i = y / PN, j = y % PN;
                if constexpr (x == 3 * PER) {
                    // all of this stage is in registers (its last step's operands arrive now); the next one has landed, R - 2 younger ones may be on their way
                    if (R > 2 && t + R - 1 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((R - 2) * LOADS) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                    places(next);
                }
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(fb[u & 1][j]), mx_operand(fa[u & 1][i]), acc[i][j], 4, 4, u, (int)sb[S][j], u, (int)sa[S][i]);
                // (else the compiler gathers the products behind the branches of the loads)
                asm volatile("" : "+v"(acc[i][j]));
                // the next step's operands (past the last stage what an earlier one left there: never used)
                unrolled<0, READS>([&](auto rc) __attribute__((always_inline)) {
                    constexpr int r = decltype(rc)::value;
                    if constexpr (r * PER / READS == y) {
                        // in the order in which the step uses them
                        if constexpr (r == 0) fa[(u + 1) & 1][0] = read_a(0, (u + 1) & 3);
                        else if constexpr (r <= PN) fb[(u + 1) & 1][r - 1] = read_b(r - 1, (u + 1) & 3);
                        else fa[(u + 1) & 1][r - PN] = read_a(r - PN, (u + 1) & 3);
                        if constexpr (u == 3) {
                            if constexpr (r == 0) sa[S ^ 1][0] = read_sa(0);
                            else if constexpr (r <= PN) sb[S ^ 1][r - 1] = read_sb(r - 1);
                            else sa[S ^ 1][r - PN] = read_sa(r - PN);
                        }
                    }
                });
                // stage t + R from the last step on; the rest of t - 1 + R before
                unrolled<0, LOADS>([&](auto lc) __attribute__((always_inline)) {
                    constexpr int l = decltype(lc)::value, when = l * 3 * PER / LOADS;  // of three steps, the first of which is a stage's last
                    if constexpr (when < PER) {
                        if constexpr (x == 3 * PER + when) {
                            if (more) load(lc, t + R, slot);
                        }
                    } else if constexpr (x == when - PER) {
                        if (more_before) load(lc, t - 1 + R, before);
                    }
                });
                __builtin_amdgcn_sched_barrier(0);
            });
            slot = next;
        };
        int t = 0;
        for (; t + 2 <= steps; t += 2) {
            stage(std::integral_constant<int, 0>(), t);
            stage(std::integral_constant<int, 1>(), t + 1);
        }
        if (t < steps) stage(std::integral_constant<int, 0>(), t);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if constexpr (KG > 1) {
            if (steps < most) __builtin_amdgcn_s_barrier();  // (the others have one stage more)
            __syncthreads();
            f32x4* const sums = reinterpret_cast<f32x4*>(smem) + threadIdx.x % (NW * 64);
            if (group > 0) {
#pragma unroll
                for (int i = 0; i < PM; i++)
#pragma unroll
                    for (int j = 0; j < PN; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            sums[((((group - 1) * PM + i) * PN + j) * 4 + q) * (NW * 64)] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            }
            __syncthreads();
            if (group > 0) return;
#pragma unroll
            for (int o = 0; o < KG - 1; o++)
#pragma unroll
                for (int i = 0; i < PM; i++)
#pragma unroll
                    for (int j = 0; j < PN; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const f32x4 v = sums[(((o * PM + i) * PN + j) * 4 + q) * (NW * 64)];
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][j][4 * q + e] += v[e];
                        }
        }

        const int done_m0 = panel_m0, done_n0 = panel_n0;
        bool more = false;
        if constexpr (KG == 1) {
            turn += stride;
            more = turn < per_xcd && first + turn < total;
            if (more) {
                go_to(first + turn);
                start(parity ^ 1);
            }
        }

        // ---- post-op: a lane holds columns 8 q + 4 half + 0..3, q = 0..3, of row c of each panel of 32 columns
        if (g.pair) {
            if constexpr (PN % 2 == 0) {
#pragma unroll
                for (int j = 0; j < PN / 2; j++) {
                    const int block = (done_n0 + wn * PN) / 2 + j;  // of 32 columns of the result
                    if (block * 64 >= g.N) continue;
#pragma unroll
                    for (int i = 0; i < PM; i++) {
                        const int m = (done_m0 + wm * PM + i) * 32 + c;
                        float r[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) r[e] = silu32(acc[i][2 * j][e]) * acc[i][2 * j + 1][e];
                        if (!g.packed_out) {
                            store16(g.ep, m, g.M, block * 32, g.N / 2, half, r);
                            continue;
                        }
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 16; e++) top = umax(top, abs_bits(r[e]));
                        top = umax(top, (uint32_t)__shfl_xor((int)top, 32));
                        const uint32_t b = mx_scale_of(top);
                        const float s = mx_value_of(b);
                        uint32_t mine[2], other[2];
#pragma unroll
                        for (int q = 0; q < 2; q++)
                            mine[q] = to_fp4x4(r[8 * q], r[8 * q + 1], r[8 * q + 2], r[8 * q + 3], s) | to_fp4x4(r[8 * q + 4], r[8 * q + 5], r[8 * q + 6], r[8 * q + 7], s) << 16;
#pragma unroll
                        for (int q = 0; q < 2; q++) other[q] = (uint32_t)__shfl_xor((int)mine[q], 32);
                        if (half == 0 && m < g.M) {
                            char* const panel = g.packed_out + (int64_t)(m >> 5) * g.ld_out;
                            *reinterpret_cast<u32x4*>(panel + mx_piece(m, block)) =
                                u32x4{(mine[0] & 0xffffu) | other[0] << 16, mine[0] >> 16 | (other[0] & 0xffff0000u), (mine[1] & 0xffffu) | other[1] << 16, mine[1] >> 16 | (other[1] & 0xffff0000u)};
                            panel[mx_scale_at(m, block)] = (char)b;
                            if ((block + 1) * 64 == g.N) {  // what is left of the last chunk
                                for (int kb = block + 1; kb & 7; kb++) {
                                    *reinterpret_cast<u32x4*>(panel + mx_piece(m, kb)) = u32x4{0, 0, 0, 0};
                                    panel[mx_scale_at(m, kb)] = 127;
                                }
                            }
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < PN; j++) {
                const int n = (done_n0 + wn * PN + j) * 32;
                if (n >= g.N) continue;
                float bias[16];
                if (biased) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(smem + T::BIAS + parity * (T::BN * 4) + ((wn * PN + j) * 32 + q * 8 + half * 4) * 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) bias[4 * q + e] = v[e];
                    }
                }
#pragma unroll
                for (int i = 0; i < PM; i++) {
                    float r[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) r[e] = acc[i][j][e];
                    if (biased) {
#pragma unroll
                        for (int e = 0; e < 16; e++) r[e] = r[e] + bias[e];
                    }
                    if (g.ep.steps & MMX_PP_GELU) {
#pragma unroll
                        for (int e = 0; e < 16; e++) r[e] = gelu_erf_minimax(r[e]);
                    }
                    store16(g.ep, (done_m0 + wm * PM + i) * 32 + c, g.M, n, g.N, half, r);
                }
            }
        }
        if (!more) return;
    }
}

template <int PM, int PN, int WGM, int WGN, int R, int KG = 1>
static int launch_tile(const Mxfp4Gemm& g, hipStream_t st, const char* name) {
    using T = Mxfp4Tile<PM, PN, WGM, WGN, R, KG>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = mxfp4_tile_kernel<PM, PN, WGM, WGN, R, KG>;
    const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), T::BYTES, done);
    if (rc) return rc;
    const int64_t tiles_m = (g.M + T::BM - 1) / T::BM, tiles_n = ((int64_t)g.npanels * 32 + T::BN - 1) / T::BN, total = tiles_m * tiles_n, per_xcd = (total + 7) / 8;
    if (per_xcd * 8 * (T::NW * KG * 64) > 0xffffffffll) return set_error(MMX_E_INVALID, "mmx_gemm_mxfp4: too many tiles for one launch");
    note_kernel(name);
    constexpr int by_lds = 160 * 1024 / T::BYTES, by_waves = 8 / (T::NW * KG);  // (of a CU: two wavefronts a SIMD)
    const int64_t at_once = (int64_t)num_cus() * (by_lds < by_waves ? by_lds : by_waves) / 8 * 8;
    const int64_t grid = KG > 1 || per_xcd * 8 < at_once ? per_xcd * 8 : at_once;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(T::NW * KG * 64), T::BYTES, st, g, (int)tiles_m, (int)tiles_n, (int)total, (int)per_xcd);
    return check_hip(hipGetLastError(), "mxfp4_tile_kernel launch");
}

static size_t quantized_in_lds(int M, int K) {
    const size_t chunks = (size_t)mx_chunks(K);
    return (size_t)M * (chunks * 128 + 16) + (size_t)M * chunks * 8;
}
template <int MT, int NT, bool PAIR, bool QUANTIZE = false>
static int launch_rows(const Mxfp4Gemm& g, hipStream_t st, const char* name) {
    note_kernel(name);
    const unsigned cols = PAIR ? (unsigned)g.npanels / 2 : (unsigned)((g.N + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((mxfp4_rows_kernel<MT, NT, PAIR, QUANTIZE>), dim3(cols, (unsigned)((g.M + 16 * MT - 1) / (16 * MT))), dim3(512), QUANTIZE ? quantized_in_lds(g.M, g.K) : 0, st, g);
    return check_hip(hipGetLastError(), "mxfp4_rows_kernel launch");
}

// Whether the kernel for few rows quantises bf16 rows on the way.  That saves a launch, 2.6 us, and costs (0.3 + workgroups / 1540) us for every 4096 values (a CU's workgroups do it again and again).
// On the way / by the quantiser, us: M 1, 2, 4, 8 x 4096 x 4096 4.3, 4.8, 5.6, 7.5 / 6.4; x 4096 x 11008 6.5, 7.4, 9.1, 12.9 / 8.6; x 4096 x 32000 13.1, 14.4, 17.5, 25.7 / 15.3.
// (A pair has fewer workgroups: where the plain product takes the rows, so does the pair.)
bool mx_takes_bf16(int M, int K, int N, bool pair) { return M <= 8 && (int64_t)M * K * (N / (pair ? 64 : 16) + 460) <= 16400000; }

// Which tile: the least of rounds * (fixed + chunks of 256 k * stage), a round being as many tiles as fit on the chip; one that is not full leaves each of its tiles more of the chip, down to `least` of
// the time.  The constants are fitted to 86 products of 33 to 4096 rows, 256 to 11008 k and 256 to 32000 columns in every tile, each by how near it comes to the fastest; among those same products the tile
// chosen was 0.5 % behind that on average, 10 % at most (times of all: profiles/mxfp4_tiles_by_size.txt).  us at 2048 x 4096 x 11008 / 4096 x 4096 x 4096 / 1024 x 11008 x 4096 / 256 x 4096 x 4096 / 64 x 11008 x 4096:
//     256 x 256            64 / 39 / 57 / 25 / 52
//     256 x 192            57 / 55 / 46 / 21 / 42
//     128 x 256            61 / 45 / 36 / 16 / 30
//     128 x 128            63 / 47 / 36 / 15 / 33
//     128 x 128, K by two  77 / 53 / 31 / 13 / 24
//      64 x 128, K by two  87 / 67 / 39 / 9.2 / 15
//      64 x 64             93 / 70 / 44 / 8.1 / 14
//      64 x 64, K by two  115 / 85 / 46 / 7.4 / 12
//      32 x 64, K by four   - / - / - / 10.5 / 9.3
//      32 x 32, K by eight  - / - / - / 15.4 / 9.0
// (64 x 128 with K whole, 73 / 54 / 33 / 10 / 19, a 192 x 256 for pairs and a 64 x 64 of their own came out first too rarely to be kept; without the last two here the mean was 4 % behind.)
struct TileCost {
    int bm, bn, per_cu;
    float fixed_us, stage_us, least;
    bool pair;  // (a wavefront of a pair has as many gate panels as up panels)
};
enum { T_256_256, T_256_192, T_128_256, T_128_128, T_128_128_BY_2, T_64_128_BY_2, T_64_64, T_64_64_BY_2, T_32_64_BY_4, T_32_32_BY_8, TILES };
static constexpr TileCost COSTS[TILES] = {{256, 256, 1, 10.3f, 1.70f, 0.62f, true}, {256, 192, 1, 8.4f, 1.32f, 0.64f, false}, {128, 256, 1, 7.5f, 0.90f, 0.67f, true},  {128, 128, 2, 6.3f, 1.01f, 0.63f, true},
                                          {128, 128, 1, 5.9f, 0.546f, 0.81f, true}, {64, 128, 1, 4.9f, 0.30f, 0.85f, true},  {64, 64, 2, 4.04f, 0.347f, 0.79f, false}, {64, 64, 1, 3.8f, 0.192f, 0.95f, true},
                                          {32, 64, 1, 3.55f, 0.133f, 0.94f, false}, {32, 32, 1, 3.57f, 0.10f, 0.92f, false}};

static int choose_tile(const Mxfp4Gemm& g) {
    int best = -1;
    double fastest = 0;
    for (int i = 0; i < TILES; i++) {
        if (g.pair && !COSTS[i].pair) continue;
        const TileCost& t = COSTS[i];
        const int64_t tiles = (int64_t)((g.M + t.bm - 1) / t.bm) * (((int64_t)g.npanels * 32 + t.bn - 1) / t.bn), at_once = (int64_t)num_cus() * t.per_cu;
        const double full = (double)(tiles / at_once), rest = (double)(tiles % at_once) / at_once;
        const double us = (full + (rest > 0 ? t.least + (1 - t.least) * rest : 0)) * (t.fixed_us + g.chunks * t.stage_us);
        if (best < 0 || us < fastest) {
            best = i;
            fastest = us;
        }
    }
    return best;
}

int launch_gemm_mxfp4(const Mxfp4Gemm& g, hipStream_t st) {
    if (g.a_bf16) return g.pair ? launch_rows<1, 4, true, true>(g, st, "mxfp4_rows_16_pair_bf16") : launch_rows<1, 1, false, true>(g, st, "mxfp4_rows_16_bf16");
    if (g.M <= 16) return g.pair ? launch_rows<1, 4, true>(g, st, "mxfp4_rows_16_pair") : launch_rows<1, 1, false>(g, st, "mxfp4_rows_16");
    if (g.M <= 32) return g.pair ? launch_rows<2, 4, true>(g, st, "mxfp4_rows_32_pair") : launch_rows<2, 1, false>(g, st, "mxfp4_rows_32");
    switch (choose_tile(g)) {
    case T_256_256: return launch_tile<4, 2, 2, 4, 2>(g, st, "mxfp4_256x256");
    case T_256_192: return launch_tile<2, 3, 4, 2, 2>(g, st, "mxfp4_256x192");
    case T_128_256: return launch_tile<2, 2, 2, 4, 3>(g, st, "mxfp4_128x256");
    case T_128_128: return launch_tile<2, 2, 2, 2, 2>(g, st, "mxfp4_128x128");
    case T_128_128_BY_2: return launch_tile<2, 2, 2, 2, 2, 2>(g, st, "mxfp4_128x128_k_by_2");
    case T_64_128_BY_2: return launch_tile<1, 2, 2, 2, 3, 2>(g, st, "mxfp4_64x128_k_by_2");
    case T_64_64: return launch_tile<1, 1, 2, 2, 4>(g, st, "mxfp4_64x64");
    case T_64_64_BY_2: return g.pair ? launch_tile<1, 2, 2, 1, 3, 2>(g, st, "mxfp4_64x64_k_by_2_pair") : launch_tile<1, 1, 2, 2, 3, 2>(g, st, "mxfp4_64x64_k_by_2");
    case T_32_64_BY_4: return launch_tile<1, 1, 1, 2, 3, 4>(g, st, "mxfp4_32x64_k_by_4");
    default: return launch_tile<1, 1, 1, 1, 2, 8>(g, st, "mxfp4_32x32_k_by_8");
    }
}

}  // namespace mmx
