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

// ---- routing ----------------------------------------------------------------------------------------------------------
// A wavefront takes one expert and up to 8 tokens.  Which expert is chosen hangs on the order of near-equal logits, so they are
// summed more exactly than 32 bits: products of bf16 are exact in 32 bits, eight of them are added there, the rest in 64.
template <int TB>
__global__ __launch_bounds__(256) void moe_logits_kernel(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ Wr, int64_t ldr, int T,
                                                         int H, int E, double* __restrict__ logits) {
    const int lane = threadIdx.x & 63, e = blockIdx.x * 4 + (threadIdx.x >> 6), t0 = blockIdx.y * TB;
    if (e >= E) return;
    double sum[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) sum[t] = 0.0;
    for (int h = lane * 8; h < H; h += 512) {
        float w[8];
        load_row_f32(Wr + e * ldr, h, H, w);
#pragma unroll
        for (int t = 0; t < TB; t++) {
            if (t0 + t >= T) break;
            float v[8];
            load_row_f32(x + (t0 + t) * ldx, h, H, v);
            float s = v[0] * w[0];
#pragma unroll
            for (int i = 1; i < 8; i++) s = __builtin_fmaf(v[i], w[i], s);
            sum[t] += (double)s;
        }
    }
#pragma unroll
    for (int t = 0; t < TB; t++) {
        if (t0 + t >= T) break;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) sum[t] += __shfl_xor(sum[t], d);
        if (lane == 0) logits[(int64_t)(t0 + t) * E + e] = sum[t];
    }
}

// A wavefront per token.  A NaN counts as less than any number, so that there are always k different experts.
template <int PER>  // experts per lane
__global__ __launch_bounds__(64) void moe_topk_kernel(const double* __restrict__ logits, int E, int k, int sigmoid, int renormalize, float scale,
                                                      const float* __restrict__ bias, int* __restrict__ ids, float* __restrict__ weights) {
    const int lane = threadIdx.x;
    const int64_t t = blockIdx.x;
    double l[PER], key[PER];
    double top = -__builtin_inf();
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 64 + lane;
        l[i] = e < E ? logits[t * E + e] : 0.0;
        if (e < E) top = __builtin_fmax(top, l[i]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = __builtin_fmax(top, __shfl_xor(top, d));
    // p = u / total: softmax's terms against the largest logit, or the sigmoid itself
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 64 + lane;
        double p = l[i];  // (without a bias the logits have the order of the p, and no two of them meet in rounding)
        if (e < E && bias) p = (sigmoid ? 1.0 / (1.0 + exp(-l[i])) : exp(l[i] - top));
        key[i] = p;
        if (e < E && !sigmoid) total += expf((float)(l[i] - top));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d);
    if (bias) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = i * 64 + lane;
            if (e < E) key[i] = (sigmoid ? key[i] : key[i] / (double)total) + (double)bias[e];
        }
    }
    uint32_t open = 0;  // this lane's experts that can be chosen still
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i * 64 + lane < E) open |= 1u << i;
        if (!(key[i] == key[i])) key[i] = -__builtin_inf();
    }
    int my_id = 0;
    float my_u = 0.0f, chosen = 0.0f;
    for (int j = 0; j < k; j++) {
        double best = 0.0;
        int at = -1;
        double l_best = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if ((open >> i & 1) && (at < 0 || key[i] > best)) {
                best = key[i];
                l_best = l[i];
                at = i * 64 + lane;
            }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const double o = __shfl_xor(best, d), ol = __shfl_xor(l_best, d);
            const int oa = __shfl_xor(at, d);
            if (oa >= 0 && (at < 0 || o > best || (o == best && oa < at))) {
                best = o;
                l_best = ol;
                at = oa;
            }
        }
        if ((at & 63) == lane) open &= ~(1u << (at >> 6));
        const float u = sigmoid ? (float)(1.0 / (1.0 + exp(-l_best))) : expf((float)(l_best - top));
        chosen += u;
        if (j == lane) {
            my_id = at;
            my_u = u;
        }
    }
    if (lane < k) {
        ids[t * k + lane] = my_id;
        weights[t * k + lane] = scale * my_u / (renormalize ? chosen : sigmoid ? 1.0f : total);
    }
}

int launch_moe_route(const void* x, int64_t ldx, const void* Wr, int64_t ldr, int T, int H, int E, int k, int sigmoid, int renormalize, float scale,
                     const float* bias, double* logits, int* ids, float* weights, hipStream_t st) {
    const auto xp = static_cast<const uint16_t*>(x), wp = static_cast<const uint16_t*>(Wr);
    const unsigned gx = (unsigned)((E + 3) / 4);
    if (T == 1) hipLaunchKernelGGL(moe_logits_kernel<1>, dim3(gx), dim3(256), 0, st, xp, ldx / 2, wp, ldr / 2, T, H, E, logits);
    else hipLaunchKernelGGL(moe_logits_kernel<8>, dim3(gx, (unsigned)((T + 7) / 8)), dim3(256), 0, st, xp, ldx / 2, wp, ldr / 2, T, H, E, logits);
    int rc = check_hip(hipGetLastError(), "moe_logits_kernel launch");
    if (rc) return rc;
#define MMX_TOPK(PER) hipLaunchKernelGGL(moe_topk_kernel<PER>, dim3((unsigned)T), dim3(64), 0, st, logits, E, k, sigmoid, renormalize, scale, bias, ids, weights)
    if (E <= 64) MMX_TOPK(1);
    else if (E <= 128) MMX_TOPK(2);
    else if (E <= 256) MMX_TOPK(4);
    else MMX_TOPK(16);
#undef MMX_TOPK
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
    for (int o = begin; o < i; o++)
        if (ids[o] == e) return false;
    return true;
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

// Gate and up: a workgroup takes one chosen expert and 16 columns of each, its eight wavefronts units of k in turn.
template <typename W>
__global__ __launch_bounds__(512) void moe_up_kernel(const MoeArgs g, int col_units) {
    constexpr int NW = 8;
    __shared__ uint8_t flags[MOE_EXPERTS];
    __shared__ uint16_t list[MOE_SLOTS];
    __shared__ int found[2];  // the expert, and how many slots chose it
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][4][64];
    const int t0 = blockIdx.y * MOE_GROUP, tokens = g.T - t0 < MOE_GROUP ? g.T - t0 : MOE_GROUP;
    const int first = t0 * g.k, n = tokens * g.k;
    const int a = blockIdx.x / col_units, u = blockIdx.x - a * col_units;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    mark_experts(g, first, n, flags);
    if (wave == 0) {
        int left = a, expert = -1;
        for (int e0 = 0; e0 < g.E && expert < 0; e0 += 64) {
            const uint64_t has = __builtin_amdgcn_ballot_w64(e0 + lane < g.E && flags[e0 + lane]);
            const int here = __builtin_popcountll(has);
            if (left < here) {
                uint64_t rest = has;
                for (int i = 0; i < left; i++) rest &= rest - 1;
                expert = e0 + __builtin_ctzll(rest);
            }
            left -= here;
        }
        int count = 0;
        if (expert >= 0) {
            for (int i0 = 0; i0 < n; i0 += 64) {
                const int i = i0 + lane;
                const bool mine = i < n && g.ids[first + i] == expert && first_of_token(g.ids + first, i, g.k);
                const uint64_t all = __builtin_amdgcn_ballot_w64(mine);
                if (mine) list[count + __builtin_popcountll(all & ((1ull << lane) - 1))] = (uint16_t)i;
                count += __builtin_popcountll(all);
            }
        }
        if (lane == 0) {
            found[0] = expert;
            found[1] = count;
        }
    }
    __syncthreads();
    const int expert = found[0], count = found[1];
    if (expert < 0) return;  // (fewer experts were chosen than there are workgroups for)

    const int c = lane & 15, quad = lane >> 4, half = u & 1;
    const int kunits = (g.H + W::KU - 1) / W::KU;
    const char* w_at[2];
    const float* s_at[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        w_at[j] = g.W + expert * g.expert_bytes + (int64_t)((u >> 1) * 2 + j) * g.panel_stride;
        s_at[j] = W::F8 ? g.scales + ((int64_t)expert * g.scale_rows + j * (g.scale_rows >> 1) + (u >> 3)) * kunits : nullptr;
    }
    for (int i0 = 0; i0 < count; i0 += 32) {
        const uint16_t* x_at[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int s = i0 + i * 16 + c;
            x_at[i] = g.x + (int64_t)(t0 + list[s < count ? s : count - 1] / g.k) * g.ldx;
        }
        auto pass = [&](auto mt_c) __attribute__((always_inline)) {
            constexpr int MT = decltype(mt_c)::value;
            f32x4 acc[MT][2];
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int ku = wave; ku < kunits; ku += NW) {
                u32x4 w[2][W::LOADS];
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int l = 0; l < W::LOADS; l++)
                        w[j][l] = *reinterpret_cast<const u32x4*>(w_at[j] + (int64_t)ku * 4096 + W::offset(l, quad, half * 16 + c));
                bf16x8 x[MT][W::STEPS];
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int s = 0; s < W::STEPS; s++) x[i][s] = load8(x_at[i], ku * W::KU + W::k_of(s, quad), g.H);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    f32x4 p[MT];
#pragma unroll
                    for (int i = 0; i < MT; i++) p[i] = W::F8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i][j];
#pragma unroll
                    for (int s = 0; s < W::STEPS; s++) {
                        const bf16x8 b = W::operand(w[j], s);
#pragma unroll
                        for (int i = 0; i < MT; i++) p[i] = mfma_bf16(b, x[i][s], p[i]);
                    }
                    if constexpr (W::F8) {
                        const float sc = s_at[j][ku];
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(p[i][e], sc, acc[i][j][e]);
                    } else {
#pragma unroll
                        for (int i = 0; i < MT; i++) acc[i][j] = p[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
                red[wave][2 * i][lane] = acc[i][0];
                red[wave][2 * i + 1][lane] = acc[i][1];
            }
        };
        if (count - i0 > 16) pass(std::integral_constant<int, 2>{});
        else pass(std::integral_constant<int, 1>{});
        __syncthreads();
        // 64 lanes per 16 tokens: tile i, lane l holds columns 4 (l / 16) + 0..3 of its token l % 16
        if (threadIdx.x < 128) {
            const int i = threadIdx.x >> 6, s = i0 + i * 16 + c;
            if (s < count) {
                float gate[4] = {0, 0, 0, 0}, up[4] = {0, 0, 0, 0};
                for (int w = 0; w < NW; w++) {
                    const f32x4 a0 = red[w][2 * i][lane], a1 = red[w][2 * i + 1][lane];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        gate[e] += a0[e];
                        up[e] += a1[e];
                    }
                }
                const int slot = list[s];
                float weight = 0.0f;
                for (int o = slot - slot % g.k, j = 0; j < g.k; j++)
                    if (g.ids[first + o + j] == expert) weight += g.weights[first + o + j];
                uint16_t* const h = g.h + (int64_t)(first + slot) * 2 * g.I + u * 16 + quad * 4;
                uint16_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = weight * (silu32(gate[e]) * up[e]);
                    hi[e] = to_bf16(v);
                    lo[e] = to_bf16(v - from_bf16(hi[e]));
                }
                __builtin_memcpy(__builtin_assume_aligned(h, 8), hi, 8);
                __builtin_memcpy(__builtin_assume_aligned(h + g.I, 8), lo, 8);
            }
        }
        __syncthreads();
    }
}

// Down: a workgroup takes 16 columns of the result for the group's tokens and walks all their experts, (expert, unit of k) in
// turn per wavefront.  The MFMA's second side is the tokens themselves: one that did not choose the expert has zeros there, so all
// experts' products add up in the same registers.  h enters as the sum of two bf16: rounded to one, its error would be as large
// as that of the result's own rounding.
template <typename W>
__global__ __launch_bounds__(512) void moe_down_kernel(const MoeArgs g) {
    constexpr int NW = 8, MT = 2;
    __shared__ uint8_t flags[MOE_EXPERTS];
    __shared__ uint16_t rank[MOE_EXPERTS];            // position of an expert among the chosen ones
    __shared__ uint16_t expert_of[MOE_SLOTS];
    __shared__ int16_t slot_of[MOE_SLOTS * MOE_GROUP];  // [chosen expert][token]: the token's slot, -1 for none
    __shared__ int chosen;
    __shared__ __attribute__((aligned(16))) f32x4 red[NW][MT][64];
    const int t0 = blockIdx.y * MOE_GROUP, tokens = g.T - t0 < MOE_GROUP ? g.T - t0 : MOE_GROUP;
    const int first = t0 * g.k, n = tokens * g.k;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    mark_experts(g, first, n, flags);
    if (wave == 0) {
        int before = 0;
        for (int e0 = 0; e0 < g.E; e0 += 64) {
            const bool is = e0 + lane < g.E && flags[e0 + lane];
            const uint64_t has = __builtin_amdgcn_ballot_w64(is);
            if (is) {
                const int at = before + __builtin_popcountll(has & ((1ull << lane) - 1));
                rank[e0 + lane] = (uint16_t)at;
                expert_of[at] = (uint16_t)(e0 + lane);
            }
            before += __builtin_popcountll(has);
        }
        if (lane == 0) chosen = before;
    }
    __syncthreads();
    const int experts = chosen;
    for (int i = threadIdx.x; i < experts * MOE_GROUP; i += NW * 64) slot_of[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NW * 64) {
        const int e = g.ids[first + i];
        if ((unsigned)e < (unsigned)g.E && first_of_token(g.ids + first, i, g.k)) slot_of[rank[e] * MOE_GROUP + i / g.k] = (int16_t)i;
    }
    __syncthreads();

    const int c = lane & 15, quad = lane >> 4, u = blockIdx.x, half = u & 1;
    const int kunits = (g.I + W::KU - 1) / W::KU;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int it = wave; it < experts * kunits; it += NW) {
        const int a = it / kunits, ku = it - a * kunits, expert = expert_of[a];
        const char* const w_at = g.W + expert * g.expert_bytes + (int64_t)(u >> 1) * g.panel_stride + (int64_t)ku * 4096;
        u32x4 w[W::LOADS];
#pragma unroll
        for (int l = 0; l < W::LOADS; l++) w[l] = *reinterpret_cast<const u32x4*>(w_at + W::offset(l, quad, half * 16 + c));
        const float sc = W::F8 ? g.scales[((int64_t)expert * g.scale_rows + (u >> 3)) * kunits + ku] : 1.0f;
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if (i * 16 >= tokens) break;
            const int slot = slot_of[a * MOE_GROUP + i * 16 + c];
            const uint16_t* const h = g.h + (int64_t)(first + (slot < 0 ? 0 : slot)) * 2 * g.I;
            f32x4 p = W::F8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i];
#pragma unroll
            for (int s = 0; s < W::STEPS; s++) {
                const int at = ku * W::KU + W::k_of(s, quad);
                bf16x8 hi = {0, 0, 0, 0, 0, 0, 0, 0}, lo = hi;
                if (slot >= 0 && at < g.I) {  // (I is a multiple of 32: eight values are there or not)
                    hi = load8(h, at, g.I);
                    lo = load8(h + g.I, at, g.I);
                }
                const bf16x8 b = W::operand(w, s);
                p = mfma_bf16(b, hi, p);
                p = mfma_bf16(b, lo, p);
            }
            if constexpr (W::F8) {
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = __builtin_fmaf(p[e], sc, acc[i][e]);
            } else {
                acc[i] = p;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) red[wave][i][lane] = acc[i];
    __syncthreads();
    if (threadIdx.x < 128) {
        const int t = (threadIdx.x >> 6) * 16 + c, n0 = u * 16 + quad * 4;
        if (t < tokens) {
            float r[4] = {0, 0, 0, 0};
            for (int w = 0; w < NW; w++) {
                const f32x4 v = red[w][threadIdx.x >> 6][lane];
#pragma unroll
                for (int e = 0; e < 4; e++) r[e] += v[e];
            }
            char* const row = g.y + (int64_t)(t0 + t) * g.ldy;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (n0 + e >= g.H) break;
                if (g.y_f32) reinterpret_cast<float*>(row)[n0 + e] = r[e];
                else reinterpret_cast<uint16_t*>(row)[n0 + e] = to_bf16(r[e]);
            }
        }
    }
}

int launch_moe_experts(bool f8, const void* x, int64_t ldx_bytes, const int* ids, const float* weights, int T, int H, int I, int E, int k,
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
    const int64_t ku_h = f8 ? (H + 127) / 128 : (H + 63) / 64, ku_i = f8 ? (I + 127) / 128 : (I + 63) / 64;
    const unsigned groups = (unsigned)((T + MOE_GROUP - 1) / MOE_GROUP);
    const int most = (T < MOE_GROUP ? T : MOE_GROUP) * k, units = I / 16;
    const int64_t grid = (int64_t)(most < E ? most : E) * units;
    if (grid > 0x7fffffff || groups > 65535) return set_error(MMX_E_INVALID, "mmx_moe_experts: too many experts, columns or tokens for one launch");
    g.W = static_cast<const char*>(w_gate_up);
    g.panel_stride = ku_h * 4096;
    g.expert_bytes = g.panel_stride * (I / 32 * 2);
    g.scales = s_gate_up;
    g.scale_rows = 2 * ((I + 127) / 128);
    hipLaunchKernelGGL((f8 ? moe_up_kernel<W_fp8> : moe_up_kernel<W_bf16>), dim3((unsigned)grid, groups), dim3(512), 0, st, g, units);
    int rc = check_hip(hipGetLastError(), "moe_up_kernel launch");
    if (rc) return rc;
    g.W = static_cast<const char*>(w_down);
    g.panel_stride = ku_i * 4096;
    g.expert_bytes = g.panel_stride * ((H + 31) / 32);
    g.scales = s_down;
    g.scale_rows = (H + 127) / 128;
    hipLaunchKernelGGL((f8 ? moe_down_kernel<W_fp8> : moe_down_kernel<W_bf16>), dim3((unsigned)((H + 15) / 16), groups), dim3(512), 0, st, g);
    return check_hip(hipGetLastError(), "moe_down_kernel launch");
}

}  // namespace mmx
