// Products in e4m3 with a scale for each block of 128: C = PP( sum over kb of sA[kb][m] sB[n / 128][kb] * (A_kb . B_kb) ).
//
// v_mfma_f32_16x16x128_f8f6f4 multiplies one block of 128 k in one instruction, so its result, started from zero, is what the
// two scales are applied to; the sums over the blocks are kept in 32 bits by vector instructions, 4 fused multiply-adds per MFMA
// of 32 cycles.  (By the product of both scales, a multiplication for each MFMA: one after the other would be four more of them.)  The weights are the first operand: a lane then holds four neighbouring columns of one row of C, and its row's
// scale is one register for all of them.
#include "ffn.hpp"

namespace mmx {

int num_cus();

// C[m][n .. n + 3] = PP(r); the caller has checked m < M.  n1: columns of the result.
__device__ __forceinline__ void store4(const Epilogue& ep, int m, int n, int n1, const float (&r)[4]) {
    char* const row = ep.C + (int64_t)m * ep.ldc;
    if (ep.out_dtype == MMX_F32) {
        float* const p = reinterpret_cast<float*>(row) + n;
        if (n + 4 <= n1) {
            const u32x4 w = {f2u(r[0]), f2u(r[1]), f2u(r[2]), f2u(r[3])};
            __builtin_memcpy(__builtin_assume_aligned(p, 4), &w, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < n1) p[e] = r[e];
        }
    } else {
        uint16_t* const p = reinterpret_cast<uint16_t*>(row) + n;
        if (n + 4 <= n1) {
            const uint16_t w[4] = {to_bf16(r[0]), to_bf16(r[1]), to_bf16(r[2]), to_bf16(r[3])};
            __builtin_memcpy(__builtin_assume_aligned(p, 2), w, 8);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < n1) p[e] = to_bf16(r[e]);
        }
    }
}
// bias and GELU of four neighbouring columns
__device__ __forceinline__ void post4(const Epilogue& ep, int n, int n1, float (&r)[4]) {
    if (ep.steps & MMX_PP_BIAS) {
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = r[e] + ep.bias[n + e < n1 ? n + e : n1 - 1];
    }
    if (ep.steps & MMX_PP_GELU) {
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = gelu_erf_minimax(r[e]);
    }
}

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 a, i32x8 b) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);  // (no scales: the plain instruction)
}

// ---- few rows: every wavefront multiplies its own blocks of k ------------------------------------------------------------
// A workgroup computes 16 NT columns of 16 MT rows; its eight wavefronts take blocks of k in turn, straight from memory into
// registers, and add their sums in LDS in the order of the wavefronts.
// PAIR: the first column tile is gate's, the second up's, 16 columns of the result.
// QUANTIZE: A is bf16 rows, which every workgroup quantises into LDS while its first weights are on their way (one row of 4096 x 11008: 8.5 us on quantised rows, which take a launch of
// 2.5 us more, and 9.3 so; quantised in every wavefront's registers, whose number leaves two wavefronts on a SIMD, 16.5).
template <int MT, int NT, bool PAIR, bool QUANTIZE>
__global__ __launch_bounds__(512) void fp8_rows_kernel(const Fp8Gemm g) {
    static_assert(!PAIR || NT == 2, "a gate and an up tile");
    constexpr int NW = 8;
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][MT * NT][64];
    extern __shared__ __attribute__((aligned(16))) char rows[];  // QUANTIZE: M rows of row_pitch(K) bytes, then their scales [M][nkb]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, quad = lane >> 4;
    const int m0 = blockIdx.y * (16 * MT);
    const int pitch = g.nkb * 128 + 16;  // (16 bytes more: neighbouring rows in other banks)

    const char* w_at[NT];
    const float* s_at[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        // 16-column tile j of this workgroup: which half of which panel
        const int tile = PAIR ? 0 : blockIdx.x * NT + j;
        int panel = PAIR ? (int)(blockIdx.x >> 1) * 2 + j : tile >> 1;
        const int half = PAIR ? (int)blockIdx.x & 1 : tile & 1;
        panel = panel < g.npanels ? panel : g.npanels - 1;
        w_at[j] = g.Bp + (int64_t)panel * g.panel_stride + quad * 1024 + (half * 16 + c) * 16;
        s_at[j] = g.sB + (int64_t)scale_row(g, panel) * g.nkb;
    }
    const char* x_at[MT];
    const float* sx_at[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        int m = m0 + i * 16 + c;
        m = m < g.M ? m : g.M - 1;
        x_at[i] = (QUANTIZE ? rows + m * pitch : g.A + (int64_t)m * g.lda) + quad * 32;
        sx_at[i] = QUANTIZE ? reinterpret_cast<const float*>(rows + g.M * pitch) + m * g.nkb : g.sA + m;
    }
    const int64_t sx_step = QUANTIZE ? 1 : g.ld_sA;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // U blocks of k: kb, kb + NW, ...
    constexpr int U = MT * NT <= 2 ? 4 : 2;
    auto load = [&](auto n_c, int kb, u32x4 (&w)[U][NT][2], float (&sw)[U][NT]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < decltype(n_c)::value; u++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const u32x4* p = reinterpret_cast<const u32x4*>(w_at[j] + (int64_t)(kb + u * NW) * 4096);
                w[u][j][0] = p[0];
                w[u][j][1] = p[32];
                sw[u][j] = s_at[j][kb + u * NW];
            }
    };
    auto multiply = [&](auto n_c, int kb, const u32x4 (&w)[U][NT][2], const float (&sw)[U][NT]) __attribute__((always_inline)) {
        constexpr int N = decltype(n_c)::value;
        u32x4 x[N][MT][2];
        float sx[N][MT];
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const u32x4* p = reinterpret_cast<const u32x4*>(x_at[i] + (int64_t)(kb + u * NW) * 128);
                x[u][i][0] = p[0];
                x[u][i][1] = p[1];
                sx[u][i] = sx_at[i][(kb + u * NW) * sx_step];
            }
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const f32x4 p = mfma_e4m3(join(w[u][j][0], w[u][j][1]), join(x[u][i][0], x[u][i][1]));
                    const float s = sx[u][i] * sw[u][j];
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(p[e], s, acc[i][j][e]);
                }
    };
    typedef std::integral_constant<int, U> all_c;
    typedef std::integral_constant<int, 1> one_c;
    u32x4 w[U][NT][2];
    float sw[U][NT];
    int kb = wave;
    if constexpr (QUANTIZE) {
        const bool ahead = kb + (U - 1) * NW < g.nkb;
        if (ahead) load(all_c(), kb, w, sw);
        for (int b = threadIdx.x >> 3; b < g.M * g.nkb; b += NW * 8) {  // (whole groups of eight lanes)
            const int m = b / g.nkb, k = b - m * g.nkb, part = threadIdx.x & 7;
            float v[16];
            load_row_f32(reinterpret_cast<const uint16_t*>(g.A + m * g.lda), k * BLOCK + part * 16, g.K, v);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) top = umax(top, abs_bits(v[e]));
#pragma unroll
            for (int d = 1; d < 8; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
            const float s = fp8_scale_of(top);
            *reinterpret_cast<u32x4*>(rows + m * pitch + k * BLOCK + part * 16) = to_fp8x16(v, fp8_inverse(s));
            if (part == 0) reinterpret_cast<float*>(rows + g.M * pitch)[b] = s;
        }
        __syncthreads();
        if (ahead) {
            multiply(all_c(), kb, w, sw);
            kb += U * NW;
        }
    }
    for (; kb + (U - 1) * NW < g.nkb; kb += U * NW) {
        load(all_c(), kb, w, sw);
        multiply(all_c(), kb, w, sw);
    }
    for (; kb < g.nkb; kb += NW) {
        load(one_c(), kb, w, sw);
        multiply(one_c(), kb, w, sw);
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
    for (int u = threadIdx.x; u < MT * (PAIR ? 1 : NT) * 64; u += NW * 64) {
        const int t = u >> 6, l = u & 63;
        const int m = m0 + (PAIR ? t : t / NT) * 16 + (l & 15);
        float r[4];
        if constexpr (PAIR) {
            float up[4];
            sum(2 * t, l, r);
            sum(2 * t + 1, l, up);
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = silu32(r[e]) * up[e];
            if (m < g.M) store4(g.ep, m, blockIdx.x * 16 + (l >> 4) * 4, g.N / 2, r);
        } else {
            sum(t, l, r);
            const int n = (blockIdx.x * NT + t % NT) * 16 + (l >> 4) * 4;
            if (m < g.M && n < g.N) {
                post4(g.ep, n, g.N, r);
                store4(g.ep, m, n, g.N, r);
            }
        }
    }
}

// ---- many rows: tiles ----------------------------------------------------------------------------------------------------
// A workgroup computes BM rows x BN columns, its NW wavefronts a grid of WGM x (NW / WGM).  A stage is 128 k, one block.  A's rows of 128 bytes
// and the stage's scales go from memory straight into a ring of R LDS slots.  A wavefront walks its rows 16 at a time against all its
// columns' fragments, which it holds in registers.  The one barrier per stage stands in front of the last 16 rows: all of this
// stage has been read into registers then, so its slot is free for the loads of stage kb + R (issued during the next stage), and the next stage has landed, so its
// first fragments are fetched beside the last rows' products.
// KG groups of NW wavefronts, each with a ring of its own, take the blocks of k in turn where there are fewer tiles than CUs; their sums are added in LDS, in order.
// What bounds it: beside a product of 32 cycles each of a SIMD's two wavefronts issues 6 or 7 vector instructions of 4 cycles, and the chip's power holds the clock at 2.0 GHz; a loop of
// nothing but these products and multiply-adds runs at 3.2 PFLOP/s on random values, 4.3 on zeros.  By card 8192 x 8192 x 8192 runs at 1.9 to 2.0, 4096 x 4096 x 4096 at 1.75 to 1.9, 2048 x 4096 x 11008,
// whose tiles leave a fifth of the second round empty, at 1.6 (115 us; 100 to 107 where the operands stay in the caches, 7 more with a bias).  (Workgroups that walk over tiles, the next one's first loads on their way while results are stored: 0 to 2 %.)
// Where the chunks of a row of A lie in LDS: chunk ^ turn(row), 0 ... 7.  An LDS cycle serves 16 lanes of a ds_read_b128, 256 bytes, and takes them as
// lanes 0-3, 12-15, 20-23, 24-27 (and 4-11, 16-19, 28-31, and the same of the other half): eight rows' chunk c and the other eight's c ^ 2.  Two rows lie in
// 256 bytes, so row / 2 has to be spread over the eight positions, the first eight's and the second's without a common one: {0, 1, 6, 7} go to {0, 1, 2, 3},
// which c ^ 2 maps to itself.  (With row / 2 as it is, every read took twice its cycles.)
__device__ __forceinline__ int turn(int row) {
    const int x = row >> 1 & 7;
    return ((x >> 2 ^ x >> 1) & 1) << 2 | (x >> 2) << 1 | (x & 1);
}
template <int BM, int BN, int NW, int WGM, int R, int KG>
struct Fp8Tile {
    static constexpr int WGN = NW / WGM, WM = BM / WGM, WN = BN / WGN;
    static constexpr int MI = WM / 16, NJ = WN / 16;
    static constexpr int A_B = BM * 128, B_B = BN * 128, SA_B = BM * 4, SB_B = 256;
    static constexpr int STAGE = A_B + B_B + SA_B + SB_B;
    static constexpr int RING = R * STAGE, BYTES = KG * RING;
    static_assert((KG - 1) * BM * BN * 4 <= BYTES, "the groups' sums fit where the stages were");
    static constexpr int PIECES = (A_B + B_B) / 1024, LOADS = PIECES / NW;  // loads of 1 KiB: of a stage, of a wavefront
    static constexpr int A_LOADS = BM / 8 / NW;  // of them of A, the first ones
    static_assert(PIECES % NW == 0 && BM / 8 % NW == 0 && BM % 64 == 0, "every wavefront issues the same number of loads");
    // wavefront w < BM / 64 brings 64 rows' scales, the others B's (again): one load each
    static_assert(BM / 64 < NW, "a wavefront is left for B's scales");
    static_assert(MI >= 2 && NJ >= 2, "the loads of a stage go in front of its last 16 rows; a row's two halves are read in two slots");
};

template <int BM, int BN, int NW, int WGM, int R, int KG>
__global__ __launch_bounds__(NW * KG * 64) __attribute__((amdgpu_waves_per_eu(NW * KG > 8 ? NW * KG / 4 : 2, NW * KG > 8 ? NW * KG / 4 : 2))) void fp8_tile_kernel(const Fp8Gemm g, int tiles_m, int tiles_n, int total,
                                                                                                          int per_xcd) {
    using T = Fp8Tile<BM, BN, NW, WGM, R, KG>;
    constexpr int MI = T::MI, NJ = T::NJ, STAGE = T::STAGE, LOADS = T::LOADS;
    using lds_u32x4 = __attribute__((address_space(3))) const u32x4;
    using lds_float = __attribute__((address_space(3))) const float;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // Neighbouring workgroups go to different XCDs: each XCD gets a run of tiles, eight rows of them at a time and those fastest, so that the 32 it works on share both operands
    // in its L2 (all rows of tiles fastest: 8192 x 8192 x 8192 700 us in 256 x 192 and 582 in 128 x 256, now 596 and 553).
    const int L = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (L >= total) return;
    const int band = L / (8 * tiles_n), in_band = L - band * (8 * tiles_n), high = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    const int tn = in_band / high, tm = band * 8 + in_band - tn * high;
    const int m0 = tm * BM, panel0 = tn * (BN / 32);
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all_waves % NW, group = all_waves / NW;
    const int wm = wave / T::WGN, wn = wave % T::WGN;
    const int c = lane & 15, quad = lane >> 4;
    const int nkb = g.nkb;
    const bool younger = wave >= NW / 2;
    const int steps = (nkb - group + KG - 1) / KG, most = (nkb + KG - 1) / KG;  // of this group, of any: blocks group, group + KG, ...

    // ---- loads: this wavefront's pieces of 1 KiB of a stage, as offsets from the stage's place in A and B
    const char* const a_base = g.A + (int64_t)m0 * g.lda;
    const char* const b_base = g.Bp + (int64_t)panel0 * g.panel_stride;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem) + group * T::RING;
    auto panel_off = [&](int p) __attribute__((always_inline)) {  // of the tile's panel p; a tile may reach past the last panel: that one again, never stored
        const int panel = panel0 + p < g.npanels ? panel0 + p : g.npanels - 1;
        return (uint32_t)(panel - panel0) * (uint32_t)g.panel_stride;
    };
    uint32_t off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int piece = i * NW + wave;
        if (i < T::A_LOADS) {
            // 8 rows x 128 bytes, the 16-byte chunk c of row r at position c ^ turn(r)
            const int row = piece * 8 + (lane >> 3);
            int m = m0 + row;
            m = m < g.M ? m : g.M - 1;
            off[i] = (uint32_t)(m - m0) * (uint32_t)g.lda + (uint32_t)(((lane & 7) ^ turn(row)) * 16);
        } else {
            const int frag = piece - BM / 8;
            off[i] = panel_off(frag >> 2) + (uint32_t)((frag & 3) * 1024 + lane * 16);
        }
    }
    // The 16 columns that the wavefront's tile j is of, in halves of panels.  A gate/up pair has its gate columns in tiles 0 ... NJ / 2 - 1 and the same of up's
    // behind them.
    const bool pair = g.pair_up != 0;
    auto half_of = [&](int j) __attribute__((always_inline)) {
        if (!pair) return wn * NJ + j;
        const int col = wn * (NJ / 2) + (j < NJ / 2 ? j : j - NJ / 2);
        return (col >> 1) * 4 + (col & 1) + (j < NJ / 2 ? 0 : 2);
    };
    uint32_t b_off[NJ], sb_off[NJ];  // B's bytes of tile j in a stage, less the lane's place; and its scale
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int half = half_of(j);
        b_off[j] = __builtin_amdgcn_readfirstlane((uint32_t)(half >> 1) * 4096u + (uint32_t)(half & 1) * 256u);
        sb_off[j] = __builtin_amdgcn_readfirstlane((uint32_t)(half >> 1) * 4u);
    }
    const uint32_t b_lane = (uint32_t)(quad * 1024 + c * 16);
    // the scales: 64 rows of A's, or one for each of the tile's panels
    const char* s_base;
    uint32_t s_off, s_dst;
    int64_t s_step;
    if (wave < BM / 64) {
        const int m = wave * 64 + lane;
        s_base = reinterpret_cast<const char*>(g.sA + m0);
        s_off = (uint32_t)(m0 + m < g.M ? m : g.M - 1 - m0) * 4u;
        s_step = g.ld_sA * 4;
        s_dst = T::A_B + T::B_B + wave * 256;
    } else {
        int panel = panel0 + lane % (BN / 32);
        panel = panel < g.npanels ? panel : g.npanels - 1;
        const int row0 = __builtin_amdgcn_readfirstlane(scale_row(g, panel0));  // (the first panel's: gate's, where it is a pair)
        s_base = reinterpret_cast<const char*>(g.sB + (int64_t)row0 * nkb);
        s_off = (uint32_t)(scale_row(g, panel) - row0) * (uint32_t)nkb * 4u;
        s_step = 4;
        s_dst = T::A_B + T::B_B + T::SA_B;
    }
    // Number ic of this wavefront's loads of its group's stage t, the last of which is the scales.
    auto load = [&](auto ic, int t, int slot) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const int kb = group + KG * t;
        const uint32_t st = lds0 + slot * STAGE;
        if constexpr (i < LOADS) {
            const int piece = i * NW + wave;
            const char* const src = i < T::A_LOADS ? a_base + (int64_t)kb * 128 : b_base + (int64_t)kb * 4096;
            const uint32_t to = st + piece * 1024, from = off[i];
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(from), "s"(src) : "memory");
        } else {
            const char* const src = s_base + kb * s_step;
            const uint32_t to = st + s_dst, from = s_off;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(from), "s"(src) : "memory");
        }
    };

    f32x4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 fa[3][2], fb[NJ][2];  // the operands of 16 rows, now and next, and of all columns: two 16-byte halves each
    float sa[3], sb[NJ];

    // where this lane reads in a stage: the two halves of A's operands, A's scales, and B and its scales (what is behind a tile's place are constants)
    uint32_t at_a[2], at_sa, at_b;
    auto places = [&](int slot) __attribute__((always_inline)) {
        const uint32_t st = lds0 + slot * STAGE, a = st + (wm * T::WM + c) * 128;
        at_a[0] = a + ((2 * quad) ^ turn(c)) * 16;
        at_a[1] = a + ((2 * quad + 1) ^ turn(c)) * 16;
        at_sa = st + T::A_B + T::B_B + (wm * T::WM + c) * 4;
        at_b = st + T::A_B + b_lane;
        asm volatile("" : "+v"(at_a[0]), "+v"(at_a[1]), "+v"(at_sa));
    };
    auto read_a = [&](int i, int half) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32x4*>(at_a[half] + i * 2048); };
    auto read_b = [&](int j, int half) __attribute__((always_inline)) { return *reinterpret_cast<lds_u32x4*>(at_b + b_off[j] + half * 512); };
    auto read_sa = [&](int i) __attribute__((always_inline)) { return *reinterpret_cast<lds_float*>(at_sa + i * 64); };
    auto read_sb = [&](int slot, int j) __attribute__((always_inline)) {
        return *reinterpret_cast<lds_float*>(lds0 + slot * STAGE + T::A_B + T::B_B + T::SA_B + sb_off[j]);
    };

    unrolled<0, R - 1>([&](auto rc) __attribute__((always_inline)) {
        constexpr int r = decltype(rc)::value;
        unrolled<0, LOADS + 1>([&](auto ic) __attribute__((always_inline)) { if (r < steps) load(ic, r, r); });
    });
    if (R > 2 && steps >= R - 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((R - 2) * (LOADS + 1)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    places(0);
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int j = 0; j < NJ; j++) fb[j][h] = read_b(j, h);
        fa[0][h] = read_a(0, h);
        fa[1][h] = read_a(1, h);
    }
    sa[0] = read_sa(0);
    sa[1] = read_sa(1);
#pragma unroll
    for (int j = 0; j < NJ; j++) sb[j] = read_sb(0, j);
    __builtin_amdgcn_sched_barrier(0);

    // One slot per MFMA, in this order and no other (the compiler would gather the multiply-adds behind the last of them): the MFMA; the multiply-adds of
    // the one LAG slots before, whose result is there by now; an LDS read for the rows or the stage to come; a load.
    // The loads are spread over the slots in front of the barrier: issued behind one another they hold up the wavefronts, the products and all, until the address unit has taken them.
    constexpr int LAG = 2, SLOTS = MI * NJ, SPAN = MI > 2 ? (MI - 2) * NJ : NJ;
    f32x4 p[LAG + 1];
    float s[LAG + 1];
    int slot = 0;
    auto stage = [&](auto turn_c, int kb) __attribute__((always_inline)) {
        constexpr int F = decltype(turn_c)::value * MI % 3;  // the first rows' operands: the three sets go round
        const int next = slot + 1 < R ? slot + 1 : 0;
        const bool more = kb + R - 1 < steps;
        const int free_slot = slot > 0 ? slot - 1 : R - 1;
        float sb_next[NJ];
        unrolled<0, SLOTS + LAG>([&](auto tc) __attribute__((always_inline)) {
            constexpr int t = decltype(tc)::value, i = t / NJ, j = t % NJ;
            if constexpr (t == SLOTS - NJ) {
                // in front of the last rows: everything of this stage is in registers (their operands arrive now), and the next one has landed
                // (R - 2 younger stages may be on their way; where there are no more to load, all that are)
                if (R > 2 && more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((R - 2) * (LOADS + 1)) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                places(next);
            }
            if constexpr (NW > 4 && t < SLOTS && j == 0) {
                // Of a SIMD's two wavefronts the older one is served first: it was at the barrier 670 of a stage's 3300 cycles before the other,
                // which then had the SIMD to itself and could not fill it.  The younger one is served first for the first half.
                // (256 x 192, 4096 x 8192 x 4096: 186 -> 183 us.)
                if constexpr (i == 0 || i == MI / 2) {
                    if (younger) __builtin_amdgcn_s_setprio(i == 0 ? 1 : 0);
                }
            }
            if constexpr (t < SLOTS) {
                p[t % (LAG + 1)] = mfma_e4m3(join(fb[j][0], fb[j][1]), join(fa[(F + i) % 3][0], fa[(F + i) % 3][1]));
                s[t % (LAG + 1)] = sa[(F + i) % 3] * sb[j];
            }
            if constexpr (t >= LAG) {
                constexpr int d = t - LAG;
                f32x4& a = acc[d / NJ][d % NJ];
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = __builtin_fmaf(p[d % (LAG + 1)][e], s[d % (LAG + 1)], a[e]);
                asm volatile("" : "+v"(a));
            }
            if constexpr (t < SLOTS) {
                unrolled<0, LOADS + 1>([&](auto ic) __attribute__((always_inline)) {
                    if constexpr (decltype(ic)::value * SPAN / (LOADS + 1) == t) {
                        if (more) load(ic, kb + R - 1, free_slot);
                    }
                });
                if constexpr (i < MI - 2) {
                    constexpr int n = (F + i + 2) % 3;
                    if constexpr (j == 0) sa[n] = read_sa(i + 2);
                    if constexpr (j < 2) fa[n][j] = read_a(i + 2, j);
                } else if constexpr (i == MI - 1) {
                    // (past the last stage these read what an earlier one left there: never used)
                    constexpr int n0 = (F + MI) % 3, n1 = (F + MI + 1) % 3;
                    if constexpr (j == 0) {
                        fa[n0][0] = read_a(0, 0);
                        fa[n0][1] = read_a(0, 1);
                        sa[n0] = read_sa(0);
#pragma unroll
                        for (int n = 0; n < NJ; n++) sb_next[n] = read_sb(next, n);
                    }
                    fb[j][0] = read_b(j, 0);
                    fb[j][1] = read_b(j, 1);
                    if constexpr (j == NJ - 1) {
                        fa[n1][0] = read_a(1, 0);
                        fa[n1][1] = read_a(1, 1);
                        sa[n1] = read_sa(1);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int n = 0; n < NJ; n++) sb[n] = sb_next[n];
        slot = next;
    };
    // stages in turn until the sets of registers are where they were
    constexpr int TURN = MI % 3 ? 3 : 1;
    int kb = 0;
    for (; kb + TURN <= steps; kb += TURN) unrolled<0, TURN>([&](auto pc) __attribute__((always_inline)) { stage(pc, kb + decltype(pc)::value); });
    unrolled<0, TURN - 1>([&](auto pc) __attribute__((always_inline)) {
        if (kb + decltype(pc)::value < steps) stage(pc, kb + decltype(pc)::value);
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (KG > 1) {
        if (steps < most) __builtin_amdgcn_s_barrier();  // (the others have one stage more)
        __syncthreads();
        f32x4* const sums = reinterpret_cast<f32x4*>(smem) + threadIdx.x % (NW * 64);
        if (group > 0) {
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++) sums[(((group - 1) * MI + i) * NJ + j) * (NW * 64)] = acc[i][j];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int o = 0; o < KG - 1; o++)
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const f32x4 v = sums[((o * MI + i) * NJ + j) * (NW * 64)];
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] += v[e];
                }
    }

    // ---- post-op: a lane holds columns n + 0..3 of row m of each 16 x 16 tile
#pragma unroll
    for (int i = 0; i < MI; i++) {
        const int m = m0 + wm * T::WM + i * 16 + c;
        if (m >= g.M) continue;
        if (pair) {
            if constexpr (NJ % 2 == 0) {
#pragma unroll
                for (int j = 0; j < NJ / 2; j++) {
                    float r[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) r[e] = silu32(acc[i][j][e]) * acc[i][j + NJ / 2][e];
                    const int n = panel0 * 16 + (wn * (NJ / 2) + j) * 16 + quad * 4;
                    if (n < g.N / 2) store4(g.ep, m, n, g.N / 2, r);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int n = panel0 * 32 + (wn * NJ + j) * 16 + quad * 4;
                if (n >= g.N) continue;
                float r[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                post4(g.ep, n, g.N, r);
                store4(g.ep, m, n, g.N, r);
            }
        }
    }
}

template <int BM, int BN, int NW, int WGM, int R, int KG = 1>
static int launch_tile(const Fp8Gemm& g, hipStream_t st, const char* name) {
    using T = Fp8Tile<BM, BN, NW, WGM, R, KG>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = fp8_tile_kernel<BM, BN, NW, WGM, R, KG>;
    const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), T::BYTES, done);
    if (rc) return rc;
    const int64_t tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.npanels * 32 + BN - 1) / BN, total = tiles_m * tiles_n, per_xcd = (total + 7) / 8;
    if (per_xcd * 8 * (NW * KG * 64) > 0xffffffffll) return set_error(MMX_E_INVALID, "mmx_gemm_fp8: too many tiles for one launch");
    note_kernel(name);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(per_xcd * 8)), dim3(NW * KG * 64), T::BYTES, st, g, (int)tiles_m, (int)tiles_n, (int)total, (int)per_xcd);
    return check_hip(hipGetLastError(), "fp8_tile_kernel launch");
}

static size_t quantized_in_lds(int M, int K) {
    const size_t nkb = ((size_t)K + BLOCK - 1) / BLOCK;
    return (size_t)M * (nkb * 128 + 16) + (size_t)M * nkb * 4;
}
template <int MT, int NT, bool PAIR, bool QUANTIZE = false>
static int launch_rows(const Fp8Gemm& g, hipStream_t st, const char* name) {
    note_kernel(name);
    const unsigned cols = PAIR ? (unsigned)g.npanels : (unsigned)((g.N + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((fp8_rows_kernel<MT, NT, PAIR, QUANTIZE>), dim3(cols, (unsigned)((g.M + 16 * MT - 1) / (16 * MT))), dim3(512),
                       QUANTIZE ? quantized_in_lds(g.M, g.K) : 0, st, g);
    return check_hip(hipGetLastError(), "fp8_rows_kernel launch");
}

// Which tile: the least of rounds * (fixed + blocks of k * stage), a round being as many tiles as fit on the chip; one that is not full leaves each of its tiles more of the chip, down to
// `least` of the time.  The constants are fitted to these measurements, us at 2048 x 4096 x 11008 / 4096 x 8192 x 4096 / 8192 x 8192 x 8192 / 1024 x 11008 x 4096 / 512 x 4096 x 4096 /
// 256 x 11008 x 4096 / 391 x 1000 x 3001 / 128 x 4096 x 4096 ("fixed" holds the first loads and the post-op):
//     256 x 192           108 / 194 /  596 / 103 / 43 / 100 / 18.9 / 40
//     128 x 256           115 / 152 /  553 /  80 / 33 /  75 / 14.7 / 32
//      64 x 128           144 / 198 /   -  /  66 / 18 /  35 /  7.2 / 15
//      64 x 64            199 / 305 /   -  /  85 / 18 /  30 /  7.0 / 13
//      64 x 64, K shared  248 / 322 /   -  /  93 / 21 /  24 /  9.4 / 11
// Over 60 products of 33 to 6000 rows, 200 to 11008 k and 200 to 16000 columns the tile chosen was 1.4 % behind the fastest on average, 12 % at most; over 66 gate/up pairs of 40 to 2048 rows, 300 to
// 11008 k and 1408 to 22016 packed columns 0.5 %, 10 % at most (64 x 4096 x 22016 21.0 us, 19.1 in 64 x 128).
struct TileCost {
    int bm, bn, per_cu;
    float fixed_us, stage_us, least;
};
enum { T_256_192, T_128_256, T_64_128, T_64_64, T_64_64_SHARED, TILES };
static constexpr TileCost COSTS[TILES] = {{256, 192, 1, 9.0f, 1.45f, 0.7f}, {128, 256, 1, 6.0f, 1.03f, 0.78f}, {64, 128, 2, 5.5f, 0.66f, 0.55f}, {64, 64, 2, 2.9f, 0.46f, 0.55f}, {64, 64, 1, 2.5f, 0.26f, 0.85f}};

static int choose_tile(const Fp8Gemm& g) {
    int best = 0;
    double fastest = 0;
    for (int i = 0; i < TILES; i++) {
        const TileCost& t = COSTS[i];
        const int64_t tiles = (int64_t)((g.M + t.bm - 1) / t.bm) * ((g.npanels * 32 + t.bn - 1) / t.bn), at_once = (int64_t)num_cus() * t.per_cu;
        const double full = (double)(tiles / at_once), rest = (double)(tiles % at_once) / at_once;
        const double us = (full + (rest > 0 ? t.least + (1 - t.least) * rest : 0)) * (t.fixed_us + g.nkb * t.stage_us);
        if (i == 0 || us < fastest) {
            best = i;
            fastest = us;
        }
    }
    return best;
}

// Whether the kernel for few rows quantises bf16 rows on the way
// (us, with a launch of its own / on the way: 1 x 4096 x 11008 11.0 / 9.3, 1 x 11008 x 4096 11.4 / 10.5, 4 x 4096 x 11008 11.3 / 11.2, 8 x 2048 x 2048 4.8 / 4.3,
// 8 x 4096 x 11008 11.5 / 14.6, 2 x 11008 x 4096 11.5 / 11.4)
bool fp8_takes_bf16(int M, int K) { return M <= 8 && (int64_t)M * K <= 16384; }

int launch_gemm_fp8(const Fp8Gemm& g, hipStream_t st) {
    const bool pair = g.pair_up != 0;
    if (!g.sA) return pair ? launch_rows<1, 2, true, true>(g, st, "fp8_rows_16_pair_bf16") : launch_rows<1, 1, false, true>(g, st, "fp8_rows_16_bf16");
    if (g.M <= 16) return pair ? launch_rows<1, 2, true>(g, st, "fp8_rows_16_pair") : launch_rows<1, 1, false>(g, st, "fp8_rows_16");
    // (16 columns a workgroup where 32 would leave half of the CUs without one: 24 x 8192 x 1024 10.5 -> 9.7 us, 20 x 2048 x 2048 4.3 -> 3.9; 32 x 4096 x 11008 13.2 -> 15.9)
    if (g.M <= 32 && !pair && 2 * g.npanels <= num_cus()) return launch_rows<2, 1, false>(g, st, "fp8_rows_32");
    if (g.M <= 32) return pair ? launch_rows<2, 2, true>(g, st, "fp8_rows_32_pair") : launch_rows<2, 2, false>(g, st, "fp8_rows_32");
    switch (choose_tile(g)) {
    case T_256_192:  // (a wavefront of a pair needs as many gate columns as up's: 64 x 96 of the tile instead of 128 x 48)
        return pair ? launch_tile<256, 192, 8, 4, 2>(g, st, "fp8_256x192_pair") : launch_tile<256, 192, 8, 2, 2>(g, st, "fp8_256x192");
    case T_128_256: return launch_tile<128, 256, 8, 2, 3>(g, st, pair ? "fp8_128x256_pair" : "fp8_128x256");
    case T_64_128: return launch_tile<64, 128, 4, 1, 3>(g, st, "fp8_64x128");
    case T_64_64: return launch_tile<64, 64, 4, 2, 4>(g, st, "fp8_64x64");
    default: return launch_tile<64, 64, 4, 2, 3, 2>(g, st, "fp8_64x64_shared_k");
    }
}

}  // namespace mmx
