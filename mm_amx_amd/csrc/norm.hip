// The seam between two blocks of a transformer, in one pass over the rows:
//
//   u = f,  or  f / sqrt(mean(f^2) + eps) * (offset + post)          the norm behind the block that made f
//   r = residual + scale * gate * u                                  its gate and the residual stream
//   z = r / sqrt(mean(r^2) + eps) * (offset + pre)                   the norm in front of the next block, bf16 or e4m3 with scales
//
// Bound: HBM - f, residual and a gate per row are read once, r and z are written once.  A row stays in registers between its two
// sums of squares; r goes on into the second norm as it is in 32 bits, not as it is stored.
#include "ffn.hpp"

namespace mmx {

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    if constexpr (TPR > 64) {
        __syncthreads();  // (what an earlier sum left has been read)
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; w++) v += part[w];
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store8(T* row, int at, int len, const float (&v)[8]) {
    T w[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (sizeof(T) == 2) w[e] = to_bf16(v[e]);
        else w[e] = v[e];
    }
    if (at + 8 <= len) {
        __builtin_memcpy(__builtin_assume_aligned(row + at, sizeof(T)), w, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (at + e < len) row[at + e] = w[e];
    }
}

// Eight values of a row as they are in memory, so that they can be on their way long before they are needed; zero past the row's len.
template <typename T>
struct Raw8 {
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int at, int len) {
        constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; q++) {
            const int from = at + q * PER;
            if (from + PER <= len) {
                __builtin_memcpy(&w[q], __builtin_assume_aligned(row + from, sizeof(T)), 16);  // (the hardware takes any address)
            } else {
                w[q] = u32x4{0u, 0u, 0u, 0u};
                if (from < len) {
#pragma unroll
                    for (int e = 0; e < PER; e++)
                        if (from + e < len) {
                            if constexpr (sizeof(T) == 2) w[q][e >> 1] |= (uint32_t)row[from + e] << (16 * (e & 1));
                            else w[q][e] = f2u(row[from + e]);
                        }
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(T) == 2) {
            widen8(w[0], v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = u2f(w[e >> 2][e & 3]);
        }
    }
};

// TPR threads per row, each NC chunks of 8 neighbouring values: chunk threadIdx + TPR * i.  A block of 128 is 16 neighbouring threads.
// Everything is asked for before the first sum: behind it, and the barrier in it, each of them would be one more trip to memory (one row of 4096 1.2 times as long,
// 8192 rows 1.15 times; now 3.2 and 47 us in a kernel trace, the latter 5.7 TB/s).
template <typename TR, int TPR, int NC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_kernel(const NormArgs g) {
    constexpr int ROWS = TPR >= 256 ? 1 : 256 / TPR;
    constexpr bool AHEAD = NC <= 2;  // (registers)
    __shared__ float part[TPR / 64 > 1 ? TPR / 64 : 1];
    const int tid = threadIdx.x % TPR;
    const int m = blockIdx.x * ROWS + threadIdx.x / TPR;
    if (m >= g.M) return;  // (a row's threads are a workgroup or whole wavefronts)
    const float inv_h = 1.0f / (float)g.H;
    float v[NC][8];
    Raw8<uint16_t> post_w[NC], gate[NC], pre_w[NC];
    Raw8<TR> old[NC];
    auto at_of = [&](int i) __attribute__((always_inline)) { return (tid + TPR * i) * 8; };
    auto load_old = [&]() __attribute__((always_inline)) {
        if (g.residual) {
#pragma unroll
            for (int i = 0; i < NC; i++) old[i].load(static_cast<const TR*>(g.residual) + m * g.ld_residual, at_of(i), g.H);
        }
    };
    auto load_weights = [&](const uint16_t* row, Raw8<uint16_t> (&w)[NC]) __attribute__((always_inline)) {
        if (row) {
#pragma unroll
            for (int i = 0; i < NC; i++) w[i].load(row, at_of(i), g.H);
        }
    };
    {
        Raw8<uint16_t> f[NC];
#pragma unroll
        for (int i = 0; i < NC; i++) f[i].load(g.f + m * g.ld_f, at_of(i), g.H);
        load_old();
        if constexpr (AHEAD) {
            load_weights(g.post_weight, post_w);
            load_weights(g.gate ? g.gate + m * g.ld_gate : nullptr, gate);
            load_weights(g.pre_weight, pre_w);
        }
#pragma unroll
        for (int i = 0; i < NC; i++) f[i].get(v[i]);
    }
    if (g.post) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) sq = __builtin_fmaf(v[i][e], v[i][e], sq);
        const float inv = rsqrtf(row_sum<TPR>(sq, part) * inv_h + g.eps);
        if constexpr (!AHEAD) load_weights(g.post_weight, post_w);
#pragma unroll
        for (int i = 0; i < NC; i++) {
            float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
            if (g.post_weight) {
                post_w[i].get(w);
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = w[e] + g.offset;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = v[i][e] * inv * w[e];
        }
    }
    if constexpr (!AHEAD) load_weights(g.gate ? g.gate + m * g.ld_gate : nullptr, gate);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        float s[8] = {1, 1, 1, 1, 1, 1, 1, 1}, r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (g.gate) gate[i].get(s);
        if (g.residual) old[i].get(r);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // (past the end of the row everything loaded is zero)
            v[i][e] = __builtin_fmaf(v[i][e], s[e] * g.scale, r[e]);
            sq = __builtin_fmaf(v[i][e], v[i][e], sq);
        }
        if (g.r) store8(static_cast<TR*>(g.r) + m * g.ld_r, at_of(i), g.H, v[i]);
    }
    if (!g.z) return;
    if constexpr (!AHEAD) load_weights(g.pre_weight, pre_w);
    const float inv = g.pre ? rsqrtf(row_sum<TPR>(sq, part) * inv_h + g.eps) : 1.0f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int at = at_of(i);
        float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (g.pre_weight) {
            pre_w[i].get(w);
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = w[e] + g.offset;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = at + e < g.H ? v[i][e] * inv * w[e] : 0.0f;
        if (!g.z_f8) {
            store8(reinterpret_cast<uint16_t*>(g.z + m * g.ld_z), at, g.H, v[i]);
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) top = umax(top, abs_bits(v[i][e]));
#pragma unroll
            for (int d = 1; d < 16; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
            const float s = fp8_scale_of(top), is = fp8_inverse(s);
            const int kb = at / BLOCK;
            if (kb * BLOCK < g.H) {  // (the last block is written whole, zero behind the end of the row)
                const uint32_t q[2] = {to_fp8x4(v[i][0] * is, v[i][1] * is, v[i][2] * is, v[i][3] * is),
                                       to_fp8x4(v[i][4] * is, v[i][5] * is, v[i][6] * is, v[i][7] * is)};
                __builtin_memcpy(__builtin_assume_aligned(g.z + m * g.ld_z + at, 8), q, 8);
                if ((at & (BLOCK - 1)) == 0) g.z_scales[kb * g.ld_scales + m] = s;
            }
        }
    }
}

// (us with and without: 1 x 4096 3.5 / 3.9, 200 x 8192 5.4 / 6.5, 391 x 1000 4.1 / 4.6; 512 threads at 2048 x 4096 14.6 / 13.6)
constexpr int FEW = 256, MANY = 512;
template <typename TR>
static int launch_norm(const NormArgs& g, hipStream_t st) {
#define MMX_NORM(TPR, NC)                                                                                                                              \
    hipLaunchKernelGGL((block_norm_kernel<TR, TPR, NC>), dim3((unsigned)((g.M + (TPR >= 256 ? 1 : 256 / TPR) - 1) / (TPR >= 256 ? 1 : 256 / TPR))), \
                       dim3(TPR > 256 ? TPR : 256), 0, st, g)
    // few rows: more threads for each, since they wait for memory and for each other only
    if (g.H <= 512) MMX_NORM(64, 1);
    else if (g.H <= 1024 && g.M > MANY) MMX_NORM(64, 2);
    else if (g.H <= 2048) MMX_NORM(256, 1);
    else if (g.H <= 4096 && g.M <= FEW) MMX_NORM(512, 1);
    else if (g.H <= 4096) MMX_NORM(256, 2);
    else if (g.H <= 8192 && g.M <= FEW) MMX_NORM(1024, 1);
    else if (g.H <= 8192) MMX_NORM(256, 4);
    else if (g.H <= 16384) MMX_NORM(1024, 2);
    else MMX_NORM(1024, 4);
#undef MMX_NORM
    return check_hip(hipGetLastError(), "block_norm_kernel launch");
}

int launch_block_norm(const NormArgs& g, bool residual_f32, hipStream_t st) {
    return residual_f32 ? launch_norm<float>(g, st) : launch_norm<uint16_t>(g, st);
}

}  // namespace mmx
