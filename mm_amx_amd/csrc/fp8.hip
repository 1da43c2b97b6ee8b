// Quantisation to e4m3 with a scale for each block of 128: rows of activations, and weights into the packed order.  Bound: HBM.
#include "ffn.hpp"

namespace mmx {

// ---- activations ------------------------------------------------------------------------------------------------------
// q[m][k] = e4m3(x[m][k] / s), s = scales[k / 128][m] the least power of two with which the block's largest magnitude is at most 448.
// Eight lanes take a block of 128, 16 values each; neighbouring groups of lanes take neighbouring rows, so that a wavefront's eight scales are neighbours in memory too.  Past
// the end of a row the bytes are zero up to the next multiple of 128: the products read whole blocks.  (Medians of a kernel trace: 2048 x 4096 bf16 8.3 us, or 10.0 from memory behind a
// product that fills the caches; 1024 x 11008 fp32 11.1 us just after it was written, 5.1 TB/s, and 15.4 from memory; one row 2.6.  Four blocks of a row per group of lanes, to have more on
// its way, were no faster.)
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const T* __restrict__ x, int64_t ldx, int M, int K, char* __restrict__ q, int64_t ldq,
                                                                float* __restrict__ scales, int64_t ld_s) {
    const int m = blockIdx.x * 32 + (threadIdx.x >> 3), kb = blockIdx.y, c = threadIdx.x & 7;
    if (m >= M) return;  // (whole groups of eight lanes)
    float v[16];
    load_row_f32(x + (int64_t)m * ldx, kb * BLOCK + c * 16, K, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) top = umax(top, abs_bits(v[e]));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
    const float s = fp8_scale_of(top);
    *reinterpret_cast<u32x4*>(q + (int64_t)m * ldq + (int64_t)kb * BLOCK + c * 16) = to_fp8x16(v, fp8_inverse(s));
    if (c == 0) scales[kb * ld_s + m] = s;
}

template <typename T>
static int launch_quantize_rows(const T* x, int64_t ldx, int M, int K, void* q, int64_t ldq, float* scales, int64_t ld_s, hipStream_t st) {
    // (K up to 2^22: at most 32768 blocks in a row)
    hipLaunchKernelGGL(quantize_rows_fp8_kernel<T>, dim3((unsigned)(((int64_t)M + 31) / 32), (unsigned)((K + BLOCK - 1) / BLOCK)), dim3(256), 0, st, x, ldx, M, K,
                       static_cast<char*>(q), ldq, scales, ld_s);
    return check_hip(hipGetLastError(), "quantize_rows_fp8_kernel launch");
}
int launch_quantize_rows_fp8(bool f32, const void* x, int64_t ldx_bytes, int M, int K, void* q, int64_t ldq, float* scales, int64_t ld_s,
                             hipStream_t st) {
    return f32 ? launch_quantize_rows(static_cast<const float*>(x), ldx_bytes / 4, M, K, q, ldq, scales, ld_s, st)
               : launch_quantize_rows(static_cast<const uint16_t*>(x), ldx_bytes / 2, M, K, q, ldq, scales, ld_s, st);
}

// ---- weights ----------------------------------------------------------------------------------------------------------
// A workgroup takes a block of 128 columns x 128 of k: its largest magnitude, then the bytes straight into the packed order,
//     packed[panel][kb][f = (k % 128) / 32][lane = n % 32 + 32 * ((k % 32) / 16)][k % 16].
// From [N, K] a thread's 16 values of a row are the 16 bytes of one such lane; from [K, N] the bytes are turned in LDS.
// PAIR: 0 alone, 1 / 2 the gate / up half of a pair (panel p of it is panel 2 p / 2 p + 1).
template <bool TRANS>
__global__ __launch_bounds__(256) void quantize_pack_fp8_kernel(const uint16_t* __restrict__ W, int64_t ldw, int K, int N, int nkb, int pair,
                                                                char* __restrict__ packed, float* __restrict__ scales) {
    __shared__ uint32_t tops[4];
    __shared__ __attribute__((aligned(16))) char turned[TRANS ? 16 : 128 * 144];
    const int kb = blockIdx.x % nkb, nb = blockIdx.x / nkb;
    const int t = threadIdx.x, c = t & 7;
    float v[4][16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = (t >> 3) + 32 * i;  // TRANS: column n of the block; else: k of the block
        const int row = (TRANS ? nb : kb) * BLOCK + r, rows = TRANS ? N : K;
        if (row < rows) {
            load_row_f32(W + row * ldw, (TRANS ? kb : nb) * BLOCK + c * 16, TRANS ? K : N, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) v[i][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) top = umax(top, abs_bits(v[i][e]));
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
    if ((t & 63) == 0) tops[t >> 6] = top;
    __syncthreads();
    const float s = fp8_scale_of(umax(umax(tops[0], tops[1]), umax(tops[2], tops[3]))), inv = fp8_inverse(s);
    if (t == 0) scales[(int64_t)nb * nkb + kb] = s;
    if constexpr (!TRANS) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const u32x4 w = to_fp8x16(v[i], inv);
#pragma unroll
            for (int e = 0; e < 16; e++) turned[(c * 16 + e) * 144 + (t >> 3) + 32 * i] = (char)(w[e >> 2] >> (8 * (e & 3)));
        }
        __syncthreads();
    }
    const int panels = (N + 31) / 32;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = (t >> 3) + 32 * i, panel = nb * 4 + i;
        if (panel >= panels) break;
        u32x4 w;
        if constexpr (TRANS) w = to_fp8x16(v[i], inv);
        else w = *reinterpret_cast<const u32x4*>(turned + r * 144 + c * 16);
        const int64_t at = pair ? 2 * panel + pair - 1 : panel;
        *reinterpret_cast<u32x4*>(packed + (at * nkb + kb) * 4096 + (c >> 1) * 1024 + ((c & 1) * 32 + (r & 31)) * 16) = w;
    }
}

int launch_quantize_pack_fp8(const void* W, int64_t ldw_bytes, int K, int N, int transpose, int pair, void* packed, float* scales, hipStream_t st) {
    const int nkb = (K + BLOCK - 1) / BLOCK;
    const int64_t grid = (int64_t)nkb * ((N + BLOCK - 1) / BLOCK);
    if (grid > 0x7fffffff) return set_error(MMX_E_INVALID, "weight matrix too large to pack in one launch");
    hipLaunchKernelGGL((transpose ? quantize_pack_fp8_kernel<true> : quantize_pack_fp8_kernel<false>), dim3((unsigned)grid), dim3(256), 0, st,
                       static_cast<const uint16_t*>(W), ldw_bytes / 2, K, N, nkb, pair, static_cast<char*>(packed), scales);
    return check_hip(hipGetLastError(), "quantize_pack_fp8_kernel launch");
}

}  // namespace mmx
