// Products in e4m3 with a scale for each block of 128: C = PP( sum over kb of sA[kb][m] sB[n / 128][kb] * (A_kb . B_kb) ).
//
// v_mfma_f32_16x16x128_f8f6f4 multiplies one block of 128 k in one instruction, so its result, started from zero, is what the
// two scales are applied to; the sums over the blocks are kept in 32 bits by vector instructions, 4 fused multiply-adds per MFMA
// of 32 cycles.  The weights are the first operand: a lane then holds four neighbouring columns of one row of C, and its row's
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
template <int MT, int NT, bool PAIR>
__global__ __launch_bounds__(512) void fp8_rows_kernel(const Fp8Gemm g) {
    static_assert(!PAIR || NT == 2, "a gate and an up tile");
    constexpr int NW = 8;
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, quad = lane >> 4;
    const int m0 = blockIdx.y * (16 * MT);

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
        x_at[i] = g.A + (int64_t)m * g.lda + quad * 32;
        sx_at[i] = g.sA + m;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto blocks = [&](auto u_c, int kb) __attribute__((always_inline)) {  // U blocks of k: kb, kb + NW, ...
        constexpr int U = decltype(u_c)::value;
        i32x8 w[U][NT], x[U][MT];
        float sw[U][NT], sx[U][MT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = kb + u * NW;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const u32x4* p = reinterpret_cast<const u32x4*>(w_at[j] + (int64_t)k * 4096);
                w[u][j] = join(p[0], p[32]);
                sw[u][j] = s_at[j][k];
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const u32x4* p = reinterpret_cast<const u32x4*>(x_at[i] + (int64_t)k * 128);
                x[u][i] = join(p[0], p[1]);
                sx[u][i] = sx_at[i][k * g.ld_sA];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const f32x4 p = mfma_e4m3(w[u][j], x[u][i]);
                    const float s = sx[u][i] * sw[u][j];
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(p[e], s, acc[i][j][e]);
                }
    };
    constexpr int U = MT * NT <= 2 ? 4 : 2;
    int kb = wave;
    for (; kb + (U - 1) * NW < g.nkb; kb += U * NW) blocks(std::integral_constant<int, U>{}, kb);
    for (; kb < g.nkb; kb += NW) blocks(std::integral_constant<int, 1>{}, kb);

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

// ---- many rows: tiles through LDS --------------------------------------------------------------------------------------
// A workgroup computes BM rows x BN columns, its NW wavefronts a grid of WGM x (NW / WGM).  Stages of 128 k (one block: A rows of
// 128 bytes, B whole fragments, and the stage's scales) go from memory straight into a ring of R LDS slots.  A wavefront walks
// its rows 16 at a time against all its columns' fragments, which it holds in registers.  The one barrier per stage stands
// in front of the last 16 rows: all of this stage has been read into registers then, so its slot is free for the loads of
// stage kb + R, and the next stage has landed, so its first fragments are fetched beside the last rows' products.
template <int BM, int BN, int NW, int WGM, int R>
struct Fp8Tile {
    static constexpr int WGN = NW / WGM, WM = BM / WGM, WN = BN / WGN;
    static constexpr int MI = WM / 16, NJ = WN / 16;
    static constexpr int A_B = BM * 128, B_B = BN * 128, SA_B = BM * 4, SB_B = 256;
    static constexpr int STAGE = A_B + B_B + SA_B + SB_B;
    static constexpr int BYTES = R * STAGE;
    static constexpr int LOADS = (BM + BN) / 8 / NW;  // of 1 KiB per wavefront and stage
    static_assert((BM + BN) / 8 % NW == 0 && BM % 64 == 0, "every wavefront issues the same number of loads");
    // wavefront w < BM / 64 brings 64 rows' scales, the others B's (again): one load each
    static_assert(BM / 64 < NW, "a wavefront is left for B's scales");
};

template <int BM, int BN, int NW, int WGM, int R>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) void fp8_tile_kernel(const Fp8Gemm g, int tiles_m, int total,
                                                                                                          int per_xcd) {
    using T = Fp8Tile<BM, BN, NW, WGM, R>;
    constexpr int MI = T::MI, NJ = T::NJ, STAGE = T::STAGE, LOADS = T::LOADS;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // neighbouring workgroups go to different XCDs: each XCD gets a run of tiles, rows fastest, which share their columns' weights
    const int L = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (L >= total) return;
    const int tn = L / tiles_m, tm = L - tn * tiles_m;
    const int m0 = tm * BM, panel0 = tn * (BN / 32);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / T::WGN, wn = wave % T::WGN;
    const int c = lane & 15, quad = lane >> 4;
    const int nkb = g.nkb;

    // ---- loads: this wavefront's pieces of 1 KiB of a stage, as offsets from the stage's place in A and B
    const char* const a_base = g.A + (int64_t)m0 * g.lda;
    const char* const b_base = g.Bp + (int64_t)panel0 * g.panel_stride;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem);
    uint32_t off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int piece = i * NW + wave;
        if (piece < BM / 8) {
            // 8 rows x 128 bytes: the 16-byte chunk c of row r lies at position c ^ (r & 7), so that the 16 rows which an MFMA
            // operand is read from fall into different banks
            const int row = piece * 8 + (lane >> 3);
            int m = m0 + row;
            m = m < g.M ? m : g.M - 1;
            off[i] = (uint32_t)(m - m0) * (uint32_t)g.lda + (uint32_t)(((lane & 7) ^ (row & 7)) * 16);
        } else {
            const int frag = piece - BM / 8;
            int panel = panel0 + (frag >> 2);
            panel = panel < g.npanels ? panel : g.npanels - 1;
            off[i] = (uint32_t)(panel - panel0) * (uint32_t)g.panel_stride + (uint32_t)((frag & 3) * 1024 + lane * 16);
        }
    }
    // the scales: 64 rows of A's, or one for each of the tile's panels
    const char* s_src;
    int64_t s_step;
    uint32_t s_dst;
    if (wave < BM / 64) {
        int m = m0 + wave * 64 + lane;
        m = m < g.M ? m : g.M - 1;
        s_src = reinterpret_cast<const char*>(g.sA + m);
        s_step = g.ld_sA * 4;
        s_dst = T::A_B + T::B_B + wave * 256;
    } else {
        int panel = panel0 + lane % (BN / 32);
        panel = panel < g.npanels ? panel : g.npanels - 1;
        s_src = reinterpret_cast<const char*>(g.sB + (int64_t)scale_row(g, panel) * nkb);
        s_step = 4;
        s_dst = T::A_B + T::B_B + T::SA_B;
    }
    auto load_stage = [&](int kb, int slot) __attribute__((always_inline)) {
        const uint32_t at = lds0 + slot * STAGE;
        const char* const a = a_base + (int64_t)kb * 128;
        const char* const b = b_base + (int64_t)kb * 4096;
        unrolled<0, LOADS>([&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value;
            const int piece = i * NW + wave;
            const char* const src = piece < BM / 8 ? a : b;
            const uint32_t to = at + piece * 1024, from = off[i];
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(from), "s"(src) : "memory");
        });
        const char* const s = s_src + kb * s_step;
        const uint32_t to = at + s_dst;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(s) : "memory");
    };

    f32x4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    i32x8 fa[2], fb[NJ];
    float sa[MI], sb[(NJ + 1) / 2];

    const int a_row = (wm * T::WM + c) * 128, a_x0 = ((2 * quad) ^ (c & 7)) * 16, a_x1 = ((2 * quad + 1) ^ (c & 7)) * 16;
    auto read_a = [&](const char* st, int i) __attribute__((always_inline)) {
        const char* const p = st + a_row + i * 2048;
        return join(*reinterpret_cast<const u32x4*>(p + a_x0), *reinterpret_cast<const u32x4*>(p + a_x1));
    };
    auto read_b = [&](const char* st, int j) __attribute__((always_inline)) {
        const int tile = wn * NJ + j;  // of 16 columns
        const char* const p = st + T::A_B + (tile >> 1) * 4096 + quad * 1024 + ((tile & 1) * 16 + c) * 16;
        return join(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 512));
    };
    auto read_scales = [&](const char* st) __attribute__((always_inline)) {
        const float* const pa = reinterpret_cast<const float*>(st + T::A_B + T::B_B) + wm * T::WM + c;
#pragma unroll
        for (int i = 0; i < MI; i++) sa[i] = pa[i * 16];
        const float* const pb = reinterpret_cast<const float*>(st + T::A_B + T::B_B + T::SA_B) + ((wn * NJ) >> 1);
#pragma unroll
        for (int j = 0; j < (NJ + 1) / 2; j++) sb[j] = pb[j];
    };

    unrolled<0, R>([&](auto rc) __attribute__((always_inline)) {
        constexpr int r = decltype(rc)::value;
        if (r < nkb) load_stage(r, r);
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    {
#pragma unroll
        for (int j = 0; j < NJ; j++) fb[j] = read_b(smem, j);
        fa[0] = read_a(smem, 0);
        read_scales(smem);
    }
    int slot = 0;
    for (int kb = 0; kb < nkb; kb++) {
        const char* const st = smem + slot * STAGE;
        const int next = slot + 1 < R ? slot + 1 : 0;
        const char* const st_next = smem + next * STAGE;
        unrolled<0, MI>([&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value;
            constexpr bool LAST = i == MI - 1;
            if constexpr (!LAST) {
                fa[(i + 1) & 1] = read_a(st, i + 1);
            } else {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __syncthreads();
                if (kb + R < nkb) load_stage(kb + R, slot);
            }
            unrolled<0, NJ>([&](auto jc) __attribute__((always_inline)) {
                constexpr int j = decltype(jc)::value;
                const f32x4 p = mfma_e4m3(fb[j], fa[i & 1]);
                const float s = sa[i] * sb[j >> 1];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(p[e], s, acc[i][j][e]);
            });
        });
        // (past the last stage these read what an earlier one left there: never used)
#pragma unroll
        for (int j = 0; j < NJ; j++) fb[j] = read_b(st_next, j);
        fa[0] = read_a(st_next, 0);
        read_scales(st_next);
        slot = next;
    }

    // ---- post-op: a lane holds columns n + 0..3 of row m of each 16 x 16 tile
#pragma unroll
    for (int i = 0; i < MI; i++) {
        const int m = m0 + wm * T::WM + i * 16 + c;
        if (m >= g.M) continue;
        if (g.pair_up) {
            if constexpr (NJ % 4 == 0) {
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    if (j & 2) continue;  // panels alternate: two gate tiles, two up tiles
                    const int pair = ((panel0 * 2 + wn * NJ + j) >> 2);
                    float r[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) r[e] = silu32(acc[i][j][e]) * acc[i][j + 2][e];
                    const int n = pair * 32 + (j & 1) * 16 + quad * 4;
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

template <int BM, int BN, int NW, int WGM, int R>
static int launch_tile(const Fp8Gemm& g, hipStream_t st, const char* name) {
    using T = Fp8Tile<BM, BN, NW, WGM, R>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = fp8_tile_kernel<BM, BN, NW, WGM, R>;
    const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), T::BYTES, done);
    if (rc) return rc;
    const int64_t tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.npanels * 32 + BN - 1) / BN, total = tiles_m * tiles_n, per_xcd = (total + 7) / 8;
    if (per_xcd * 8 > 0x7fffffff) return set_error(MMX_E_INVALID, "mmx_gemm_fp8: too many tiles for one launch");
    note_kernel(name);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(per_xcd * 8)), dim3(NW * 64), T::BYTES, st, g, (int)tiles_m, (int)total, (int)per_xcd);
    return check_hip(hipGetLastError(), "fp8_tile_kernel launch");
}

template <int MT, int NT, bool PAIR>
static int launch_rows(const Fp8Gemm& g, hipStream_t st, const char* name) {
    note_kernel(name);
    const unsigned cols = PAIR ? (unsigned)g.npanels : (unsigned)((g.N + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((fp8_rows_kernel<MT, NT, PAIR>), dim3(cols, (unsigned)((g.M + 16 * MT - 1) / (16 * MT))), dim3(512), 0, st, g);
    return check_hip(hipGetLastError(), "fp8_rows_kernel launch");
}

int launch_gemm_fp8(const Fp8Gemm& g, hipStream_t st) {
    const bool pair = g.pair_up != 0;
    if (g.M <= 16) return pair ? launch_rows<1, 2, true>(g, st, "fp8_rows_16_pair") : launch_rows<1, 1, false>(g, st, "fp8_rows_16");
    if (g.M <= 32) return pair ? launch_rows<2, 2, true>(g, st, "fp8_rows_32_pair") : launch_rows<2, 2, false>(g, st, "fp8_rows_32");
    if (g.M <= 128) return pair ? launch_rows<4, 2, true>(g, st, "fp8_rows_64_pair") : launch_rows<4, 2, false>(g, st, "fp8_rows_64");
    return launch_tile<256, 256, 8, 2, 2>(g, st, "fp8_256x256");
}

}  // namespace mmx
