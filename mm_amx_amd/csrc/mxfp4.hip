// Rows to microscaled 4-bit floating point and back.  Bound: HBM (where a device copy moves 4.9 TB/s), one row and a few by the launch, 3 us.
#include "mxfp4.hpp"

namespace mmx {

// A workgroup takes a panel of 32 rows x a chunk of 256 k, eight lanes to a row: in each of four steps a lane has eight neighbouring values, four lanes a block.  Reads are 128 bytes of a row
// (256 of fp32), writes 512 in order: 2048 x 11008 fp32 21.7 us, 4.7 TB/s read and written; 2048 x 4096 bf16 7.9 us.  What lies past K is zero up to the end of the chunk; rows from M up are left as they were.
// Panel p of x goes to panel p * step + first (1, 0; or of a gate/up pair 2, 0 and 2, 1).
template <typename T>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const T* __restrict__ x, int64_t ldx, int M, int K, int chunks, int step, int first, char* __restrict__ out) {
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int m = blockIdx.x * 32 + r, chunk = blockIdx.y;
    if (m >= M) return;  // (whole groups of eight lanes)
    float v[4][8];
#pragma unroll
    for (int u = 0; u < 4; u++) load_row_f32(x + (int64_t)m * ldx, chunk * MX_CHUNK + u * 64 + c * 8, K, v[u]);
    char* const at = out + (((int64_t)blockIdx.x * step + first) * chunks + chunk) * MX_CHUNK_BYTES;
    uint32_t scales = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) top = umax(top, abs_bits(v[u][e]));
#pragma unroll
        for (int d = 1; d < 4; d *= 2) top = umax(top, (uint32_t)__shfl_xor((int)top, d));
        const uint32_t b = mx_scale_of(top);
        scales |= b << 8 * u;
        *reinterpret_cast<uint32_t*>(at + u * 1024 + ((c >> 2) * 32 + r) * 16 + (c & 3) * 4) = to_fp4x8(v[u], mx_value_of(b));
    }
    if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(at + MX_SCALES_AT + ((c >> 2) * 32 + r) * 4) = scales;
}

int launch_quantize_mxfp4(bool f32, const void* x, int64_t ldx_bytes, int M, int K, int pair, void* out, hipStream_t st) {
    const int chunks = (int)mx_chunks(K), step = pair ? 2 : 1, first = pair == 2;
    const dim3 grid((unsigned)(((int64_t)M + 31) / 32), (unsigned)chunks);  // (K up to 2^22: at most 16384 chunks)
    if (f32)
        hipLaunchKernelGGL(quantize_mxfp4_kernel<float>, grid, dim3(256), 0, st, static_cast<const float*>(x), ldx_bytes / 4, M, K, chunks, step, first, static_cast<char*>(out));
    else
        hipLaunchKernelGGL(quantize_mxfp4_kernel<uint16_t>, grid, dim3(256), 0, st, static_cast<const uint16_t*>(x), ldx_bytes / 2, M, K, chunks, step, first, static_cast<char*>(out));
    return check_hip(hipGetLastError(), "quantize_mxfp4_kernel launch");
}

// ---- back -----------------------------------------------------------------------------------------------------------------
// Eight values of 4 bits in 32: magnitudes are 0.5 * {0, 1, 2, 3, 4, 6, 8, 12}.  The workgroups of the kernel above, the other way: 2048 x 11008 to bf16 11.2 us, 5.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const char* __restrict__ in, int M, int K, int chunks, T* __restrict__ y, int64_t ldy) {
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int m = blockIdx.x * 32 + r, chunk = blockIdx.y;
    if (m >= M) return;
    const char* const at = in + ((int64_t)blockIdx.x * chunks + chunk) * MX_CHUNK_BYTES;
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; u++) w[u] = *reinterpret_cast<const uint32_t*>(at + u * 1024 + ((c >> 2) * 32 + r) * 16 + (c & 3) * 4);
    const uint32_t scales = *reinterpret_cast<const uint32_t*>(at + MX_SCALES_AT + ((c >> 2) * 32 + r) * 4);
    T* const row = y + (int64_t)m * ldy;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const uint32_t b = scales >> 8 * u & 255;
        // 2^(b - 127) is subnormal for b = 0; 255 is NaN
        const float s = b == 255u ? u2f(0x7fc00000u) : b ? u2f(b << 23) : u2f(0x400000u);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t code = w[u] >> 4 * e & 15;
            const uint32_t mag = 0xc8643210u >> 4 * (code & 7) & 15;
            const float a = (float)mag * 0.5f * s;
            v[e] = code & 8 ? -a : a;
        }
        const int k = chunk * MX_CHUNK + u * 64 + c * 8;
        T o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (sizeof(T) == 2) o[e] = to_bf16(v[e]);  // (two bits of mantissa: exact but for what bf16 cannot hold, past its largest value and below 2^-133)
            else o[e] = v[e];
        }
        if (k + 8 <= K) {
            __builtin_memcpy(__builtin_assume_aligned(row + k, sizeof(T)), o, 8 * sizeof(T));
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k + e < K) row[k + e] = o[e];
        }
    }
}

int launch_dequantize_mxfp4(const void* in, int M, int K, bool f32, void* y, int64_t ldy_bytes, hipStream_t st) {
    const int chunks = (int)mx_chunks(K);
    const dim3 grid((unsigned)(((int64_t)M + 31) / 32), (unsigned)chunks);
    if (f32) hipLaunchKernelGGL(dequantize_mxfp4_kernel<float>, grid, dim3(256), 0, st, static_cast<const char*>(in), M, K, chunks, static_cast<float*>(y), ldy_bytes / 4);
    else hipLaunchKernelGGL(dequantize_mxfp4_kernel<uint16_t>, grid, dim3(256), 0, st, static_cast<const char*>(in), M, K, chunks, static_cast<uint16_t*>(y), ldy_bytes / 2);
    return check_hip(hipGetLastError(), "dequantize_mxfp4_kernel launch");
}

// ---- rows of codes and scales as checkpoints hold them, to and from the layout ------------------------------------------------
// q [M][ceil(K / 2)] bytes, the value of the lower k in a byte's low half, and scales [M][ceil(K / 32)] bytes, each with rows of any pitch.  A thread takes a block of a row; an odd K's last
// half byte, and a last block's bytes that are not there, are zero.  Byte by byte, since rows lie anywhere: 11008 x 4096 29 us, once for a weight.  TO_LAYOUT also fills the blocks between K and the end of the chunk (zeros at scale one).
template <bool TO_LAYOUT>
__global__ __launch_bounds__(256) void repack_mxfp4_kernel(char* __restrict__ q, int64_t ldq, char* __restrict__ scales, int64_t lds, int M, int K, int chunks, int step, int first,
                                                           char* __restrict__ packed) {
    const int r = threadIdx.x >> 3;
    const int m = blockIdx.x * 32 + r, kb = blockIdx.y * 8 + (threadIdx.x & 7);
    if (m >= M) return;
    char* const panel = packed + ((int64_t)blockIdx.x * step + first) * chunks * MX_CHUNK_BYTES;
    char* const piece = panel + mx_piece(r, kb);
    const int64_t row = (int64_t)m * ldq + (int64_t)kb * 16;
    const int bytes = (K + 1) / 2 - kb * 16;  // of the row from here on (may be negative)
    const bool last_half = (K & 1) && bytes >= 1 && bytes <= 16;
    uint32_t w[4] = {0, 0, 0, 0};
    if constexpr (TO_LAYOUT) {
#pragma unroll
        for (int b = 0; b < 16; b++)
            if (b < bytes) w[b >> 2] |= (uint32_t)(uint8_t)q[row + b] << 8 * (b & 3);
        if (last_half) {
#pragma unroll
            for (int b = 0; b < 16; b++)
                if (b == bytes - 1) w[b >> 2] &= ~(0xf0u << 8 * (b & 3));
        }
        *reinterpret_cast<u32x4*>(piece) = u32x4{w[0], w[1], w[2], w[3]};
        panel[mx_scale_at(r, kb)] = bytes > 0 ? scales[(int64_t)m * lds + kb] : 127;
    } else {
        if (bytes <= 0) return;
        const u32x4 v = *reinterpret_cast<const u32x4*>(piece);
#pragma unroll
        for (int b = 0; b < 16; b++)
            if (b < bytes) q[row + b] = (char)(v[b >> 2] >> 8 * (b & 3));
        scales[(int64_t)m * lds + kb] = panel[mx_scale_at(r, kb)];
    }
}

int launch_repack_mxfp4(bool to_layout, void* q, int64_t ldq, void* scales, int64_t lds, int M, int K, int pair, void* packed, hipStream_t st) {
    const int chunks = (int)mx_chunks(K), step = pair ? 2 : 1, first = pair == 2;
    const dim3 grid((unsigned)(((int64_t)M + 31) / 32), (unsigned)chunks);
    const auto kernel = to_layout ? repack_mxfp4_kernel<true> : repack_mxfp4_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, static_cast<char*>(q), ldq, static_cast<char*>(scales), lds, M, K, chunks, step, first, static_cast<char*>(packed));
    return check_hip(hipGetLastError(), "repack_mxfp4_kernel launch");
}

}  // namespace mmx
