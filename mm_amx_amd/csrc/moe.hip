// A mixture-of-experts layer for a few tokens: routing, then the chosen experts' gate/up products, then their down products.
//
//   route    l = x . Wr^T; p = softmax(l) or sigmoid(l); the k experts of the largest p + bias (the lowest index of equal ones);
//            w = scale * p, divided by the sum of the chosen p if asked for
//   experts  y[t] = sum over j of w[t][j] * Wd_e ( silu(Wg_e x[t]) * (Wu_e x[t]) ),  e = ids[t][j]
//
// Bound: HBM - with few tokens every chosen expert's weights are read once and multiplied with one to a few rows.  So the
// products run on 16 x 16 MFMA tiles whose second side is tokens, most of them empty at T = 1, which costs nothing beside the reads.
#include "ffn.hpp"

namespace mmx {

constexpr int MOE_GROUP = 32;   // tokens that one pass over an expert's weights serves
constexpr int MOE_TOP_K = 16;   // experts of a token at most
constexpr int MOE_EXPERTS = 1024;
constexpr int MOE_SLOTS = MOE_GROUP * MOE_TOP_K;
constexpr int MOE_SPLITS = 4;
constexpr int MOST_GRID_Y = 65535;

int num_cus();

// ---- routing ----------------------------------------------------------------------------------------------------------
// A wavefront takes one expert and TB tokens.  Which expert is chosen hangs on the order of near-equal logits, so they are
// summed more exactly than 32 bits: products of bf16 are exact in 32 bits, eight of them are added there, the rest in 64.
// What bounds it is latency: few tokens per wavefront, so that there are many, and all loads of a step before its products (8 tokens x 128 experts x 4096 with all
// eight tokens in a wavefront, each load behind a test: 37 us).
template <int TB>
__global__ __launch_bounds__(256) void moe_logits_kernel(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ Wr, int64_t ldr, int T,
                                                         int H, int E, double* __restrict__ logits) {
    const int lane = threadIdx.x & 63, e = blockIdx.x * 4 + (threadIdx.x >> 6), t0 = blockIdx.y * TB;
    if (e >= E) return;
    const uint16_t* const w_row = Wr + e * ldr;
    const uint16_t* x_row[TB];
    double sum[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) {
        x_row[t] = x + (int64_t)(t0 + t < T ? t0 + t : T - 1) * ldx;
        sum[t] = 0.0;
    }
    auto add = [&](const float (&w)[8], const float (&v)[8], double& to) __attribute__((always_inline)) {
        float s = v[0] * w[0];
#pragma unroll
        for (int i = 1; i < 8; i++) s = __builtin_fmaf(v[i], w[i], s);
        to += (double)s;
    };
    constexpr int U = TB == 1 ? 4 : 2;
    int h = lane * 8;
    for (; h - lane * 8 + U * 512 <= H; h += U * 512) {  // (uniform: whole steps)
        u32x4 wv[U], xv[U][TB];
#pragma unroll
        for (int u = 0; u < U; u++) {
            __builtin_memcpy(&wv[u], __builtin_assume_aligned(w_row + h + u * 512, 2), 16);
#pragma unroll
            for (int t = 0; t < TB; t++) __builtin_memcpy(&xv[u][t], __builtin_assume_aligned(x_row[t] + h + u * 512, 2), 16);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float w[8], v[8];
            widen8(wv[u], w);
#pragma unroll
            for (int t = 0; t < TB; t++) {
                widen8(xv[u][t], v);
                add(w, v, sum[t]);
            }
        }
    }
    for (; h < H; h += 512) {
        float w[8], v[8];
        load_row_f32(w_row, h, H, w);
#pragma unroll
        for (int t = 0; t < TB; t++) {
            load_row_f32(x_row[t], h, H, v);
            add(w, v, sum[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < TB; t++) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) sum[t] += __shfl_xor(sum[t], d);
        if (lane == 0 && t0 + t < T) logits[(int64_t)(t0 + t) * E + e] = sum[t];
    }
}

// A workgroup per token, a thread per expert: its place among all of them is the number of those in front of it, counted against every key in LDS (chosen one after
// another by a maximum over the wavefront, 8 of 64 took 7.5 us).  A NaN counts as less than any number, so that there are always k different experts.
__global__ void moe_topk_kernel(const double* __restrict__ logits, int E, int k, int sigmoid, int renormalize, float scale, const float* __restrict__ bias,
                                int* __restrict__ ids, float* __restrict__ weights) {
    __shared__ double keys[MOE_EXPERTS];
    __shared__ double tops[MOE_EXPERTS / 64];
    __shared__ double totals[MOE_EXPERTS / 64];
    __shared__ double chosen[MOE_TOP_K], chosen_l[MOE_TOP_K];  // their p (of softmax less the division) and their logits
    const int e = threadIdx.x, lane = e & 63, wave = e >> 6, waves = blockDim.x >> 6;
    const int64_t t = blockIdx.x;
    const double l = e < E ? logits[t * E + e] : -__builtin_inf();
    double top = l, total = 1.0, u;
    if (sigmoid) {
        const double far = exp(-__builtin_fabs(l));  // (1 / (1 + e^-l) would be zero below -709)
        u = (l < 0.0 ? far : 1.0) / (1.0 + far);
    } else {  // softmax's terms against the largest logit
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) top = __builtin_fmax(top, __shfl_xor(top, d));
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        for (int w = 0; w < waves; w++) top = __builtin_fmax(top, tops[w]);
        u = total = e < E ? exp(l - top) : 0.0;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d);
        if (lane == 0) totals[wave] = total;
        __syncthreads();
        total = totals[0];
        for (int w = 1; w < waves; w++) total += totals[w];
    }
    // (without a bias the logits have the order of the p, and no two of them meet in rounding)
    double key = l;
    if (bias && e < E) key = u / total + (double)bias[e];
    if (!(key == key)) key = -__builtin_inf();
    keys[e] = key;
    __syncthreads();
    // (equal ones go by their index: those of the wavefronts before this one are in front, of the later ones behind)
    const int low = wave * 64, high = low + 64 < E ? low + 64 : E;
    int before = 0;
#pragma unroll 8
    for (int o = 0; o < low; o++) before += keys[o] >= key;
#pragma unroll 8
    for (int o = low; o < high; o++) {
        const double other = keys[o];
        before += other > key || (other == key && o < e);
    }
#pragma unroll 8
    for (int o = high; o < E; o++) before += keys[o] > key;
    const bool mine = e < E && before < k;
    if (mine) {
        chosen[before] = u;
        chosen_l[before] = l;
    }
    __syncthreads();
    if (mine) {
        if (renormalize) {
            // Shares are ratios, and a bias can choose experts whose p 32 bits cannot hold (from e^-104 on), nor 64 (e^-745).  Where even their sum is below 2^-700 every p is
            // e^l times what all experts of the token share, to far more than 64 bits, and the terms are formed against the largest chosen logit.  Above that, a term
            // that is no longer exact (below 2^-1022) is less than 2^-322 of the sum.
            total = 0.0;
            for (int j = 0; j < k; j++) total += chosen[j];
            if (total < 0x1p-700) {
                double largest = chosen_l[0];
                for (int j = 1; j < k; j++) largest = __builtin_fmax(largest, chosen_l[j]);
                u = exp(l - largest);
                total = 0.0;
                for (int j = 0; j < k; j++) total += exp(chosen_l[j] - largest);
            }
        }
        ids[t * k + before] = e;
        weights[t * k + before] = (float)(scale * u / total);
    }
}

int launch_moe_route(const void* x, int64_t ldx, const void* Wr, int64_t ldr, int T, int H, int E, int k, int sigmoid, int renormalize, float scale,
                     const float* bias, double* logits, int* ids, float* weights, hipStream_t st) {
    const auto xp = static_cast<const uint16_t*>(x), wp = static_cast<const uint16_t*>(Wr);
    const unsigned gx = (unsigned)((E + 3) / 4);
    const int tb = (int64_t)T * E <= 2048 ? 1 : 4;  // (wavefronts for all CUs first, then less of the router read again)
    for (int t0 = 0; t0 < T; t0 += MOST_GRID_Y * tb) {  // (one launch up to 262140 tokens)
        const int n = T - t0 < MOST_GRID_Y * tb ? T - t0 : MOST_GRID_Y * tb;
        const uint16_t* const from = xp + t0 * (ldx / 2);
        double* const to = logits + (int64_t)t0 * E;
        const dim3 grid(gx, (unsigned)((n + tb - 1) / tb));
        if (tb == 1) hipLaunchKernelGGL(moe_logits_kernel<1>, grid, dim3(256), 0, st, from, ldx / 2, wp, ldr / 2, n, H, E, to);
        else hipLaunchKernelGGL(moe_logits_kernel<4>, grid, dim3(256), 0, st, from, ldx / 2, wp, ldr / 2, n, H, E, to);
        const int rc = check_hip(hipGetLastError(), "moe_logits_kernel launch");
        if (rc) return rc;
    }
    hipLaunchKernelGGL(moe_topk_kernel, dim3((unsigned)T), dim3((unsigned)((E + 63) / 64 * 64)), 0, st, logits, E, k, sigmoid, renormalize, scale, bias, ids, weights);
    return check_hip(hipGetLastError(), "moe_topk_kernel launch");
}

// ---- experts ----------------------------------------------------------------------------------------------------------
struct MoeArgs {
    const uint16_t* x;
    int64_t ldx;  // elements
    const int* ids;
    const float* weights;
    int T, H, I, E, k;
    const char* W;        // packed, expert after expert
    int64_t expert_bytes, panel_stride;
    const float* scales;  // of e4m3 weights: [expert][scale_rows][kunits]
    int scale_rows;
    uint16_t* h;          // [T * k][2][I]: w * silu(gate) * up as a bf16 and what that leaves, also as bf16
    char* y;
    int64_t ldy;
    int y_f32;
    int splits;           // workgroups that share 16 columns of y
    float* parts;         // splits > 1: their sums, [splits][T][H]
    int* arrived;         //             and how many of them are there, for each group of tokens and 16 columns; zeroed by the gate/up kernel
};

// The experts that the tokens [t0, t0 + n / k) chose, in ascending order.  flags: LDS, E bytes.
__device__ __forceinline__ void mark_experts(const MoeArgs& g, int first, int n, uint8_t* flags) {
    for (int e = threadIdx.x; e < g.E; e += blockDim.x) flags[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int e = g.ids[first + i];
        if ((unsigned)e < (unsigned)g.E) flags[e] = 1;  // (-1 or anything else out of range: no expert)
    }
    __syncthreads();
}

// Whether slot i (its token's j-th choice) is the first of its token with that expert: a later one only adds its weight.
__device__ __forceinline__ bool first_of_token(const int* ids, int i, int k) {
    const int e = ids[i], begin = i - i % k;
    bool first = true;
#pragma unroll 4
    for (int o = 0; o < k; o++) first &= ids[begin + o] != e || begin + o >= i;  // (no way out before the end: the loads do not wait for one another)
    return first;
}

// How a wavefront reads 16 columns x KU of k of packed weights, and the tokens' values beside them: each step is one
// v_mfma_f32_16x16x32_bf16, for which a lane holds eight k of its column, and of its token.
struct W_bf16 {
    static constexpr bool F8 = false;
    static constexpr int KU = 64;       // k of a 4 KiB unit of a panel
    static constexpr int LOADS = 2;     // 16-byte loads per lane and unit
    static constexpr int STEPS = 2;     // MFMAs per unit
    // packed bf16: [k / 16][lane = n % 32 + 32 * ((k % 16) / 8)][8 of k]
    static __device__ __forceinline__ int offset(int l, int quad, int col) { return (2 * l + (quad >> 1)) * 1024 + (col + 32 * (quad & 1)) * 16; }
    static __device__ __forceinline__ int k_of(int step, int quad) { return step * 32 + quad * 8; }
    static __device__ __forceinline__ bf16x8 operand(const u32x4 (&w)[LOADS], int step) { return __builtin_bit_cast(bf16x8, w[step]); }
};
struct W_fp8 {
    static constexpr bool F8 = true;
    static constexpr int KU = 128;
    static constexpr int LOADS = 2;
    static constexpr int STEPS = 4;
    // packed bytes: [k / 32][lane = n % 32 + 32 * ((k % 32) / 16)][16 of k]; a lane's 16 k serve two steps
    static __device__ __forceinline__ int offset(int l, int quad, int col) { return (2 * l + (quad >> 1)) * 1024 + (col + 32 * (quad & 1)) * 16; }
    static __device__ __forceinline__ int k_of(int step, int quad) { return (step >> 1) * 64 + quad * 16 + (step & 1) * 8; }
    static __device__ __forceinline__ bf16x8 operand(const u32x4 (&w)[LOADS], int step) {  // (every e4m3 is a bf16)
        bf16x8 r;
#pragma unroll
        for (int d = 0; d < 2; d++) {
            const uint32_t q = w[step >> 1][2 * (step & 1) + d];
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
            r[4 * d] = (__bf16)lo[0];
            r[4 * d + 1] = (__bf16)lo[1];
            r[4 * d + 2] = (__bf16)hi[0];
            r[4 * d + 3] = (__bf16)hi[1];
        }
        return r;
    }
};

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ bf16x8 load8(const uint16_t* row, int at, int len) {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (at + 8 <= len) {
        __builtin_memcpy(&w, __builtin_assume_aligned(row + at, 2), 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (at + e < len) w[e >> 1] |= (uint32_t)row[at + e] << (16 * (e & 1));
    }
    return __builtin_bit_cast(bf16x8, w);
}

// STEPS operands of a unit of k of a token's row; zero from len on
template <typename W>
__device__ __forceinline__ void load_steps(const uint16_t* row, int k0, int quad, int len, bool whole, bf16x8 (&x)[W::STEPS]) {
    if (whole) {  // (uniform)
#pragma unroll
        for (int s = 0; s < W::STEPS; s++) __builtin_memcpy(&x[s], __builtin_assume_aligned(row + k0 + W::k_of(s, quad), 2), 16);
    } else {
#pragma unroll
        for (int s = 0; s < W::STEPS; s++) x[s] = load8(row, k0 + W::k_of(s, quad), len);
    }
}

// Gate and up: a workgroup takes one chosen expert and 16 columns of each, its eight wavefronts units of k in turn, U of them at a time so that many loads are
// in flight.
template <typename W, int MT>
__global__ __launch_bounds__(512) void moe_up_kernel(const MoeArgs g, int col_units) {
    constexpr int NW = 8, U = W::F8 || MT > 1 ? 2 : 4;  // (more, and fewer wavefronts fit: e4m3, 8 tokens, 128 experts of 4096 x 1536, 120 us with 4 wavefronts on a SIMD, 177 with 3)
    __shared__ uint8_t flags[MOE_EXPERTS];
    __shared__ uint16_t list[MOE_SLOTS];
    __shared__ int found[2];  // the expert, and how many slots chose it
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][2 * MT][64];
    const int t0 = blockIdx.y * MOE_GROUP, tokens = g.T - t0 < MOE_GROUP ? g.T - t0 : MOE_GROUP;
    const int first = t0 * g.k, n = tokens * g.k;
    const int a = blockIdx.x / col_units, u = blockIdx.x - a * col_units;
    if (g.splits > 1 && blockIdx.x == 0) {
        const int tiles = (g.H + 15) / 16;
        for (int i = threadIdx.x; i < tiles; i += NW * 64) g.arrived[blockIdx.y * tiles + i] = 0;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int expert, count;
    if (tokens == 1) {  // its slots are the chosen experts themselves (there are places for all of them)
        const int mine = lane < n ? g.ids[first + lane] : -1;
        expert = a < n ? __builtin_amdgcn_readlane(mine, a) : -1;
        if ((unsigned)expert >= (unsigned)g.E || __builtin_amdgcn_ballot_w64(lane < a && mine == expert)) expert = -1;
        count = 1;
        if (threadIdx.x == 0) list[0] = (uint16_t)a;
    } else {
        mark_experts(g, first, n, flags);
        if (wave == 0) {
            int left = a, is = -1;
            for (int e0 = 0; e0 < g.E && is < 0; e0 += 64) {
                const uint64_t has = __builtin_amdgcn_ballot_w64(e0 + lane < g.E && flags[e0 + lane]);
                const int here = __builtin_popcountll(has);
                if (left < here) {
                    uint64_t rest = has;
                    for (int i = 0; i < left; i++) rest &= rest - 1;
                    is = e0 + __builtin_ctzll(rest);
                }
                left -= here;
            }
            int slots = 0;
            if (is >= 0) {
                for (int i0 = 0; i0 < n; i0 += 64) {
                    const int i = i0 + lane;
                    const bool mine = i < n && g.ids[first + i] == is && first_of_token(g.ids + first, i, g.k);
                    const uint64_t all = __builtin_amdgcn_ballot_w64(mine);
                    if (mine) list[slots + __builtin_popcountll(all & ((1ull << lane) - 1))] = (uint16_t)i;
                    slots += __builtin_popcountll(all);
                }
            }
            if (lane == 0) {
                found[0] = is;
                found[1] = slots;
            }
        }
    }
    __syncthreads();
    if (tokens > 1) {
        expert = found[0];
        count = found[1];
    }
    if (expert < 0) return;  // (fewer experts were chosen than there are places for)
    expert = __builtin_amdgcn_readfirstlane(expert);

    const int c = lane & 15, quad = lane >> 4, half = u & 1;
    const int kunits = (g.H + W::KU - 1) / W::KU;
    const char* w_at[2];
    const float* s_at[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        w_at[j] = g.W + expert * g.expert_bytes + (int64_t)((u >> 1) * 2 + j) * g.panel_stride;
        s_at[j] = W::F8 ? g.scales + ((int64_t)expert * g.scale_rows + j * (g.scale_rows >> 1) + (u >> 3)) * kunits : nullptr;
    }
    for (int i0 = 0; i0 < count; i0 += 16 * MT) {
        const uint16_t* x_at[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int s = i0 + i * 16 + c;
            x_at[i] = g.x + (int64_t)(t0 + list[s < count ? s : count - 1] / g.k) * g.ldx;
        }
        {
            f32x4 acc[MT][2];
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            auto units = [&](auto u_c, int ku0) __attribute__((always_inline)) {
                constexpr int N = decltype(u_c)::value;
                u32x4 w[N][2][W::LOADS];
                float sc[N][2];
#pragma unroll
                for (int v = 0; v < N; v++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
#pragma unroll
                        for (int l = 0; l < W::LOADS; l++)
                            w[v][j][l] = *reinterpret_cast<const u32x4*>(w_at[j] + (int64_t)(ku0 + v * NW) * 4096 + W::offset(l, quad, half * 16 + c));
                        sc[v][j] = W::F8 ? s_at[j][ku0 + v * NW] : 1.0f;
                    }
#pragma unroll
                for (int v = 0; v < N; v++) {
                    const int k0 = (ku0 + v * NW) * W::KU;
                    bf16x8 x[MT][W::STEPS];
#pragma unroll
                    for (int i = 0; i < MT; i++) load_steps<W>(x_at[i], k0, quad, g.H, k0 + W::KU <= g.H, x[i]);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        f32x4 p[MT];
#pragma unroll
                        for (int i = 0; i < MT; i++) p[i] = W::F8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i][j];
#pragma unroll
                        for (int s = 0; s < W::STEPS; s++) {
                            const bf16x8 b = W::operand(w[v][j], s);
#pragma unroll
                            for (int i = 0; i < MT; i++) p[i] = mfma_bf16(b, x[i][s], p[i]);
                        }
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            if constexpr (W::F8) {
#pragma unroll
                                for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(p[i][e], sc[v][j], acc[i][j][e]);
                            } else {
                                acc[i][j] = p[i];
                            }
                        }
                    }
                }
            };
            int ku = wave;
            for (; ku + (U - 1) * NW < kunits; ku += U * NW) units(std::integral_constant<int, U>{}, ku);
            for (; ku < kunits; ku += NW) units(std::integral_constant<int, 1>{}, ku);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                red[wave][2 * i][lane] = acc[i][0];
                red[wave][2 * i + 1][lane] = acc[i][1];
            }
        }
        // (fetched while the other wavefronts finish)
        float weight = 0.0f;
        if (threadIdx.x < 64 * MT && i0 + (int)(threadIdx.x >> 6) * 16 + c < count) {
            const int slot = list[i0 + (threadIdx.x >> 6) * 16 + c], begin = first + slot - slot % g.k;
#pragma unroll 4
            for (int j = 0; j < g.k; j++) {
                const float w = g.weights[begin + j];
                weight += g.ids[begin + j] == expert ? w : 0.0f;
            }
        }
        __syncthreads();
        // 64 lanes per 16 tokens: tile i, lane l holds columns 4 (l / 16) + 0..3 of its token l % 16
        if (threadIdx.x < 64 * MT) {
            const int i = threadIdx.x >> 6, s = i0 + i * 16 + c;
            if (s < count) {
                float gate[4] = {0, 0, 0, 0}, up[4] = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const f32x4 a0 = red[w][2 * i][lane], a1 = red[w][2 * i + 1][lane];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        gate[e] += a0[e];
                        up[e] += a1[e];
                    }
                }
                const int slot = list[s];
                uint16_t* const h = g.h + (int64_t)(first + slot) * 2 * g.I + u * 16 + quad * 4;
                uint16_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = weight * (silu32(gate[e]) * up[e]);
                    hi[e] = to_bf16(v);
                    const float rest = v - from_bf16(hi[e]);
                    lo[e] = abs_bits(rest) < 0x7f800000u ? to_bf16(rest) : 0;  // (an infinity, or a NaN, is all in the first)
                }
                __builtin_memcpy(__builtin_assume_aligned(h, 8), hi, 8);
                __builtin_memcpy(__builtin_assume_aligned(h + g.I, 8), lo, 8);
            }
        }
        __syncthreads();
    }
}

// Down: a workgroup takes 16 columns of the result for the group's tokens.  A wavefront takes a part of an expert's k at a time, multiplies it with the rows of h of the slots that
// chose the expert, and adds what comes out to its own copy of the tokens' 16 columns in LDS; at the end the copies are added in the order of the wavefronts, so the result
// does not depend on who was first.  (With the second side of the MFMA the tokens themselves, those that did not choose the expert as rows of zeros, all experts add up in the
// same registers, but the zeros have to be loaded: 32 tokens, 2 of 16 experts, 1000 x 1376, 39 us.)
// h enters as the sum of two bf16: rounded to one, its error would be as large as that of the result's own rounding.  Sixteen wavefronts, each with the weights of U units on their way:
// a narrow layer has columns for a part of the CUs only.
template <typename W, int MT>  // MT: 16 tokens each
__global__ __launch_bounds__(1024) void moe_down_kernel(const MoeArgs g) {
    constexpr int NW = 16, TOKENS = 16 * MT, SLOTS = TOKENS * MOE_TOP_K, U = W::F8 ? 2 : 4;
    constexpr uint16_t NONE = 0xffff;
    __shared__ uint16_t named[SLOTS], expert_at[SLOTS];  // a slot's expert as it is named, and NONE for a slot that does not count
    __shared__ uint16_t sorted[SLOTS], start[SLOTS + 1]; // the slots by expert, and where each expert's begin
    __shared__ uint8_t begins[SLOTS];
    __shared__ int chosen, last;
    __shared__ __attribute__((aligned(16))) float part[NW][TOKENS][16];
    const int t0 = blockIdx.y * MOE_GROUP, tokens = g.T - t0 < MOE_GROUP ? g.T - t0 : MOE_GROUP;
    const int first = t0 * g.k, n = tokens * g.k;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int i = lane; i < TOKENS * 16; i += 64) (&part[wave][0][0])[i] = 0.0f;
    int experts;
    if (tokens == 1) {  // every wavefront finds and writes all of it, the same, and waits for nobody
        const int e = lane < n ? g.ids[first + lane] : -1;
        bool counts = (unsigned)e < (unsigned)g.E;
        for (int o = 0; o < n; o++) counts &= __builtin_amdgcn_readlane(e, o) != e || o >= lane;
        const uint64_t all = __builtin_amdgcn_ballot_w64(counts);
        const int place = __builtin_popcountll(all & ((1ull << lane) - 1));
        experts = __builtin_popcountll(all);
        if (counts) {
            sorted[place] = (uint16_t)lane;
            expert_at[lane] = (uint16_t)e;
        }
        if (lane <= experts) start[lane] = (uint16_t)lane;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        for (int i = threadIdx.x; i < n; i += NW * 64) {
            const int e = g.ids[first + i];
            named[i] = (unsigned)e < (unsigned)g.E ? (uint16_t)e : NONE;  // (-1 or anything else out of range: no expert)
            begins[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NW * 64) {
            uint16_t e = named[i];
            for (int o = i - i % g.k; o < i; o++)
                if (named[o] == e) e = NONE;  // (its token has named it before: that slot has both weights)
            expert_at[i] = e;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NW * 64) {
            const uint16_t e = expert_at[i];
            if (e != NONE) {
                int before = 0, same = 0;
#pragma unroll 16
                for (int o = 0; o < n; o++) {
                    const uint16_t other = expert_at[o];
                    before += other < e;
                    same += other == e && o < i;
                }
                sorted[before + same] = (uint16_t)i;
                if (same == 0) begins[before] = 1;
            }
        }
        __syncthreads();
        if (wave == 0) {
            int count = 0, valid = 0;
            for (int i0 = 0; i0 < n; i0 += 64) {
                const bool is = i0 + lane < n && begins[i0 + lane];
                const uint64_t has = __builtin_amdgcn_ballot_w64(is);
                if (is) start[count + __builtin_popcountll(has & ((1ull << lane) - 1))] = (uint16_t)(i0 + lane);
                count += __builtin_popcountll(has);
                valid += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i0 + lane < n && expert_at[i0 + lane] != NONE));
            }
            if (lane == 0) {
                start[count] = (uint16_t)valid;
                chosen = count;
            }
        }
        __syncthreads();
        experts = chosen;
    }

    const int c = lane & 15, quad = lane >> 4, u = blockIdx.x, half = u & 1;
    const int kunits = (g.I + W::KU - 1) / W::KU;
    // parts of an expert's k: as many as give every wavefront four or more, of U units or more
    int parts = experts > 0 ? (4 * NW * g.splits + experts - 1) / experts : 1;
    if (parts > (kunits + U - 1) / U) parts = (kunits + U - 1) / U;
    for (int item = blockIdx.z * NW + wave; item < experts * parts; item += NW * g.splits) {
        const int a = item / parts, piece = item - a * parts;
        const int begin = __builtin_amdgcn_readfirstlane((int)start[a]), end = __builtin_amdgcn_readfirstlane((int)start[a + 1]);
        const int expert = __builtin_amdgcn_readfirstlane((int)expert_at[sorted[begin]]);
        const char* const w_at = g.W + expert * g.expert_bytes + (int64_t)(u >> 1) * g.panel_stride;
        const float* const s_at = W::F8 ? g.scales + ((int64_t)expert * g.scale_rows + (u >> 3)) * kunits : nullptr;
        const int ku_end = (piece + 1) * kunits / parts;
        for (int b = begin; b < end; b += 16) {
            const bool live = b + c < end;
            const int slot = sorted[live ? b + c : begin];
            const uint16_t* const h = g.h + (int64_t)(first + slot) * 2 * g.I;
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            auto units = [&](auto u_c, int ku0) __attribute__((always_inline)) {
                constexpr int N = decltype(u_c)::value;
                u32x4 w[N][W::LOADS];
                float sc[N];
                bf16x8 hi[N][W::STEPS], lo[N][W::STEPS];
#pragma unroll
                for (int v = 0; v < N; v++) {
#pragma unroll
                    for (int l = 0; l < W::LOADS; l++)
                        w[v][l] = *reinterpret_cast<const u32x4*>(w_at + (int64_t)(ku0 + v) * 4096 + W::offset(l, quad, half * 16 + c));
                    sc[v] = W::F8 ? s_at[ku0 + v] : 1.0f;
                }
#pragma unroll
                for (int v = 0; v < N; v++)
#pragma unroll
                    for (int s = 0; s < W::STEPS; s++) {
                        const int at = (ku0 + v) * W::KU + W::k_of(s, quad);
                        hi[v][s] = lo[v][s] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
                        if (live && at < g.I) {  // (I is a multiple of 32: eight values are there or not)
                            hi[v][s] = *reinterpret_cast<const bf16x8*>(h + at);
                            lo[v][s] = *reinterpret_cast<const bf16x8*>(h + g.I + at);
                        }
                    }
#pragma unroll
                for (int v = 0; v < N; v++) {
                    f32x4 p = W::F8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc;
#pragma unroll
                    for (int s = 0; s < W::STEPS; s++) {
                        const bf16x8 o = W::operand(w[v], s);
                        p = mfma_bf16(o, hi[v][s], p);
                        p = mfma_bf16(o, lo[v][s], p);
                    }
                    if constexpr (W::F8) {
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(p[e], sc[v], acc[e]);
                    } else {
                        acc = p;
                    }
                }
            };
            int ku = piece * kunits / parts;
            for (; ku + U <= ku_end; ku += U) units(std::integral_constant<int, U>{}, ku);
            for (; ku < ku_end; ku++) units(std::integral_constant<int, 1>{}, ku);
            if (live) {
                f32x4* const to = reinterpret_cast<f32x4*>(&part[wave][slot / g.k][quad * 4]);
                f32x4 sum = *to;
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] += acc[e];
                *to = sum;
            }
        }
    }
    __syncthreads();
    auto store_y = [&](int t, int n0, const float (&r)[4]) __attribute__((always_inline)) {
        char* const row = g.y + (int64_t)(t0 + t) * g.ldy;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (n0 + e >= g.H) break;
            if (g.y_f32) reinterpret_cast<float*>(row)[n0 + e] = r[e];
            else reinterpret_cast<uint16_t*>(row)[n0 + e] = to_bf16(r[e]);
        }
    };
    if (threadIdx.x < TOKENS * 4) {
        const int t = threadIdx.x >> 2, n0 = u * 16 + (threadIdx.x & 3) * 4;
        if (t < tokens) {
            float r[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&part[w][t][(threadIdx.x & 3) * 4]);
#pragma unroll
                for (int e = 0; e < 4; e++) r[e] += v[e];
            }
            if (g.splits == 1) {
                store_y(t, n0, r);
            } else {
                float* const to = g.parts + ((int64_t)blockIdx.z * g.T + t0 + t) * g.H;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n0 + e < g.H) __hip_atomic_store(to + n0 + e, r[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    if (g.splits == 1) return;
    // Whoever comes last adds all sums, in the order of the workgroups; nobody waits.  The sums are written and read past the L2, which another XCD does not see, and have arrived before
    // this workgroup counts itself.  (With ordinary stores and __threadfence(), which writes back all of the L2, in each wavefront: 1 x 2048 x 1024, 8 of 64 experts, 115 us instead of 27.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(g.arrived + blockIdx.y * gridDim.x + u, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == g.splits - 1;
    __syncthreads();
    if (!last) return;
    const int t = threadIdx.x >> 2, n0 = u * 16 + (threadIdx.x & 3) * 4;
    if (t < tokens) {
        float v[MOE_SPLITS][4], r[4];
#pragma unroll
        for (int z = 0; z < MOE_SPLITS; z++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[z][e] = z < g.splits && n0 + e < g.H ? __hip_atomic_load(g.parts + ((int64_t)z * g.T + t0 + t) * g.H + n0 + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            r[e] = v[0][e];
#pragma unroll
            for (int z = 1; z < MOE_SPLITS; z++) r[e] += v[z][e];
        }
        store_y(t, n0, r);
    }
}

// Into how many workgroups the down products of 16 columns are split: a narrow layer's columns are a workgroup each for a part of the CUs only.  The sums then go through memory, some 2 us,
// for which there have to be CUs without work (us whole / split, experts' calls: in two 4 x 2048 x 768, 8 of 128, 72 / 68; 32 x 2048 x 1024, 8 of 64, 219 / 190;
// 1 x 2048 x 1024, 8 of 64, 27 / 27; the down products alone in four 32 x 1000 x 1376, 2 of 16, 30.5 / 19).
static int moe_splits(int T, int H) {
    const int64_t tiles = (int64_t)((H + 15) / 16) * ((T + MOE_GROUP - 1) / MOE_GROUP), cus = num_cus();
    return tiles * MOE_SPLITS <= cus ? MOE_SPLITS : tiles * 2 <= cus ? 2 : 1;
}
static size_t moe_h_bytes(int T, int I, int k) { return ((size_t)T * k * 2 * I * 2 + 255) & ~(size_t)255; }
size_t moe_scratch_bytes(int T, int H, int I, int k) {
    const int splits = moe_splits(T, H);
    return moe_h_bytes(T, I, k) + (splits > 1 ? (size_t)splits * T * H * 4 + (size_t)((T + MOE_GROUP - 1) / MOE_GROUP) * ((H + 15) / 16) * 4 : 0);
}

static int launch_experts(bool f8, const void* x, int64_t ldx_bytes, const int* ids, const float* weights, int T, int H, int I, int E, int k,
                          const void* w_gate_up, const float* s_gate_up, const void* w_down, const float* s_down, void* h, void* y, int64_t ldy, int y_f32,
                          hipStream_t st) {
    MoeArgs g;
    g.x = static_cast<const uint16_t*>(x);
    g.ldx = ldx_bytes / 2;
    g.ids = ids;
    g.weights = weights;
    g.T = T, g.H = H, g.I = I, g.E = E, g.k = k;
    g.h = static_cast<uint16_t*>(h);
    g.y = static_cast<char*>(y);
    g.ldy = ldy;
    g.y_f32 = y_f32;
    g.splits = moe_splits(T, H);
    g.parts = reinterpret_cast<float*>(static_cast<char*>(h) + moe_h_bytes(T, I, k));
    g.arrived = reinterpret_cast<int*>(g.parts + (int64_t)g.splits * T * H);
    const int64_t ku_h = f8 ? (H + 127) / 128 : (H + 63) / 64, ku_i = f8 ? (I + 127) / 128 : (I + 63) / 64;
    const unsigned groups = (unsigned)((T + MOE_GROUP - 1) / MOE_GROUP);
    // a place for each expert that a group's tokens can choose, and for each slot of a token alone in its group, which names experts more than once, or none, where k > E
    const int most = (T < MOE_GROUP ? T : MOE_GROUP) * k, distinct = most < E ? most : E, units = I / 16;
    const int64_t grid = (int64_t)(distinct > k ? distinct : k) * units;
    if (grid * 512 > 0xffffffffll) return set_error(MMX_E_UNSUPPORTED, "mmx_moe_experts: %d experts at a time of I = %d columns are too many for one launch", (int)(grid / units), I);
    g.W = static_cast<const char*>(w_gate_up);
    g.panel_stride = ku_h * 4096;
    g.expert_bytes = g.panel_stride * (I / 32 * 2);
    g.scales = s_gate_up;
    g.scale_rows = 2 * ((I + 127) / 128);
    const auto up = T <= 16 ? (f8 ? moe_up_kernel<W_fp8, 1> : moe_up_kernel<W_bf16, 1>) : f8 ? moe_up_kernel<W_fp8, 2> : moe_up_kernel<W_bf16, 2>;
    hipLaunchKernelGGL(up, dim3((unsigned)grid, groups), dim3(512), 0, st, g, units);
    int rc = check_hip(hipGetLastError(), "moe_up_kernel launch");
    if (rc) return rc;
    g.W = static_cast<const char*>(w_down);
    g.panel_stride = ku_i * 4096;
    g.expert_bytes = g.panel_stride * ((H + 31) / 32);
    g.scales = s_down;
    g.scale_rows = (H + 127) / 128;
    const auto down = T <= 16 ? (f8 ? moe_down_kernel<W_fp8, 1> : moe_down_kernel<W_bf16, 1>) : f8 ? moe_down_kernel<W_fp8, 2> : moe_down_kernel<W_bf16, 2>;
    hipLaunchKernelGGL(down, dim3((unsigned)((H + 15) / 16), groups, (unsigned)g.splits), dim3(1024), 0, st, g);
    return check_hip(hipGetLastError(), "moe_down_kernel launch");
}

// One pair of launches up to 2097120 tokens.  The pairs take the scratch from its start, one behind the other on the stream; sums of split down products, which only the last
// of them can have, are a megabyte at most behind its own rows of h, and there the scratch has the rows of the pairs before it.
int launch_moe_experts(bool f8, const void* x, int64_t ldx_bytes, const int* ids, const float* weights, int T, int H, int I, int E, int k,
                       const void* w_gate_up, const float* s_gate_up, const void* w_down, const float* s_down, void* h, void* y, int64_t ldy, int y_f32,
                       hipStream_t st) {
    constexpr int MOST = MOST_GRID_Y * MOE_GROUP;
    int rc = MMX_OK;
    for (int t0 = 0; t0 < T && !rc; t0 += MOST)
        rc = launch_experts(f8, static_cast<const char*>(x) + t0 * ldx_bytes, ldx_bytes, ids + (int64_t)t0 * k, weights + (int64_t)t0 * k, T - t0 < MOST ? T - t0 : MOST, H, I, E, k,
                            w_gate_up, s_gate_up, w_down, s_down, h, static_cast<char*>(y) + t0 * ldy, ldy, y_f32, st);
    return rc;
}

}  // namespace mmx
