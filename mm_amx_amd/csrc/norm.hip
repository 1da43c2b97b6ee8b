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

// TPR threads per row, each NC chunks of 8 neighbouring values: chunk threadIdx + TPR * i.  A block of 128 is 16 neighbouring threads.
template <typename TR, int TPR, int NC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_kernel(const NormArgs g) {
    constexpr int ROWS = TPR >= 256 ? 1 : 256 / TPR;
    __shared__ float part[TPR / 64 > 1 ? TPR / 64 : 1];
    const int tid = threadIdx.x % TPR;
    const int m = blockIdx.x * ROWS + threadIdx.x / TPR;
    if (m >= g.M) return;  // (a row's threads are a workgroup or whole wavefronts)
    const float inv_h = 1.0f / (float)g.H;
    float v[NC][8];
    const uint16_t* const f = g.f + m * g.ld_f;
#pragma unroll
    for (int i = 0; i < NC; i++) load_row_f32(f, (tid + TPR * i) * 8, g.H, v[i]);
    if (g.post) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) sq = __builtin_fmaf(v[i][e], v[i][e], sq);
        const float inv = rsqrtf(row_sum<TPR>(sq, part) * inv_h + g.eps);
#pragma unroll
        for (int i = 0; i < NC; i++) {
            float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
            if (g.post_weight) {
                load_row_f32(g.post_weight, (tid + TPR * i) * 8, g.H, w);
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = w[e] + g.offset;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = v[i][e] * inv * w[e];
        }
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int at = (tid + TPR * i) * 8;
        float s[8];
        if (g.gate) {
            load_row_f32(g.gate + m * g.ld_gate, at, g.H, s);
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = s[e] * g.scale;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = g.scale;
        }
        float old[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (g.residual) load_row_f32(static_cast<const TR*>(g.residual) + m * g.ld_residual, at, g.H, old);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // (past the end of the row everything loaded is zero)
            v[i][e] = __builtin_fmaf(v[i][e], s[e], old[e]);
            sq = __builtin_fmaf(v[i][e], v[i][e], sq);
        }
        if (g.r) store8(static_cast<TR*>(g.r) + m * g.ld_r, at, g.H, v[i]);
    }
    if (!g.z) return;
    const float inv = g.pre ? rsqrtf(row_sum<TPR>(sq, part) * inv_h + g.eps) : 1.0f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int at = (tid + TPR * i) * 8;
        float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (g.pre_weight) {
            load_row_f32(g.pre_weight, at, g.H, w);
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

template <typename TR>
static int launch_norm(const NormArgs& g, hipStream_t st) {
#define MMX_NORM(TPR, NC)                                                                                                                              \
    hipLaunchKernelGGL((block_norm_kernel<TR, TPR, NC>), dim3((unsigned)((g.M + (TPR >= 256 ? 1 : 256 / TPR) - 1) / (TPR >= 256 ? 1 : 256 / TPR))), \
                       dim3(TPR > 256 ? TPR : 256), 0, st, g)
    if (g.H <= 512) MMX_NORM(64, 1);
    else if (g.H <= 1024) MMX_NORM(64, 2);
    else if (g.H <= 2048) MMX_NORM(256, 1);
    else if (g.H <= 4096) MMX_NORM(256, 2);
    else if (g.H <= 8192) MMX_NORM(256, 4);
    else if (g.H <= 16384) MMX_NORM(1024, 2);
    else if (g.H <= 32768) MMX_NORM(1024, 4);
    else MMX_NORM(1024, 8);
#undef MMX_NORM
    return check_hip(hipGetLastError(), "block_norm_kernel launch");
}

int launch_block_norm(const NormArgs& g, bool residual_f32, hipStream_t st) {
    return residual_f32 ? launch_norm<float>(g, st) : launch_norm<uint16_t>(g, st);
}

}  // namespace mmx
