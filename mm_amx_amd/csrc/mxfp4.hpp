// Microscaled 4-bit floating point: e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a scale 2^(b - 127), b in 8 bits, for each row and 32 of k.
//
// Activations and weights are laid out alike, in the order in which v_mfma_scale_f32_32x32x64_f8f6f4 takes them: a panel of 32 rows after the other, in it a
// chunk of 256 k after the other, a chunk being
//     4 x 64 x 16 bytes: step u = (k % 256) / 64, lane = row % 32 + 32 ((k % 64) / 32), the lane's 32 values two a byte, the first in the low half
//     64 x 4 bytes:      lane as above, byte u the scale's b
// so that a step of the matrix cores reads one KiB in order, from memory or LDS, and a lane's four scales are one register.
#pragma once

#include "ffn.hpp"

namespace mmx {

constexpr int MX_BLOCK = 32, MX_CHUNK = 256, MX_SCALES_AT = 4096, MX_CHUNK_BYTES = 4352;

inline __host__ __device__ int64_t mx_chunks(int64_t K) { return (K + MX_CHUNK - 1) / MX_CHUNK; }
inline __host__ __device__ int64_t mx_bytes(int64_t rows, int64_t K) { return (rows + 31) / 32 * mx_chunks(K) * MX_CHUNK_BYTES; }

// b of a block whose largest magnitude has these bits: the least power of two s, 2^-126 at least, with amax < 7 s, so that nothing rounds past 6; 255 (NaN) for a block that holds an
// infinity or a NaN.  7 is 1.75 * 2^2.  With a power of two x / s is exact: one rounding, the same however it is computed.
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t amax_bits) {
    const int b = (int)(amax_bits >> 23) - ((amax_bits & 0x7fffffu) < 0x600000u ? 2 : 1);
    return amax_bits >= 0x7f800000u ? 255u : (uint32_t)(b < 1 ? 1 : b);
}
// the scale as a number, for b from 1 on (a NaN block's: any, its values are never seen)
__device__ __forceinline__ float mx_value_of(uint32_t b) { return u2f((b == 255u ? 127u : b) << 23); }

// eight values to 4 bytes, to nearest even; s as above
__device__ __forceinline__ uint32_t to_fp4x8(const float* v, float s) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
}
// four values to 2 bytes
__device__ __forceinline__ uint32_t to_fp4x4(float a, float b, float c, float d, float s) {
    const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, s, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c, d, s, 1);
}

// where block kb (of 32 k) of a row lies, from the start of the row's panel: its 16 bytes and its scale
__device__ __forceinline__ int64_t mx_piece(int row, int64_t kb) {
    return (kb >> 3) * MX_CHUNK_BYTES + (((int)kb & 7) >> 1) * 1024 + (((int)kb & 1) * 32 + (row & 31)) * 16;
}
__device__ __forceinline__ int64_t mx_scale_at(int row, int64_t kb) {
    return (kb >> 3) * MX_CHUNK_BYTES + MX_SCALES_AT + (((int)kb & 1) * 32 + (row & 31)) * 4 + (((int)kb & 7) >> 1);
}

// What a product is made of.  A and B in the layout above; or, where mx_takes_bf16(), A rows of K bf16 that lie anywhere, lda bytes apart.
struct Mxfp4Gemm {
    const char* A;
    int64_t lda;       // bytes of a 32-row panel of A, or of a row of bf16
    const char* B;
    int64_t ldb;       // bytes of a 32-column panel of B
    int M, N;          // N: packed columns (both of a gate/up pair, whose panels alternate)
    int K, chunks;
    int npanels;
    int pair, a_bf16;
    char* packed_out;  // a pair's result quantised into this layout, in place of ep.C; or NULL
    int64_t ld_out;    // bytes of a 32-row panel of it
    Epilogue ep;
};

bool mx_takes_bf16(int M, int K, int N, bool pair);

}  // namespace mmx
