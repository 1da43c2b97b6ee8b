// Shared by the operators of the feed-forward block: helpers in 8-bit floating point (e4m3, the OCP form: largest value 448, NaN but no infinities).
#pragma once

#include <type_traits>

#include "common.hpp"

namespace mmx {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// compile-time loop: f(integral_constant<int, B>) ... f(integral_constant<int, E - 1>), for arrays that have to stay in registers
template <int B, int E, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
    if constexpr (B < E) {
        f(std::integral_constant<int, B>{});
        unrolled<B + 1, E>(f);
    }
}

constexpr int BLOCK = 128;  // values of k (and, of weights, columns) that share a scale

// The scale of a block whose largest magnitude has these bits: the least power of two s with amax <= 448 s, 2^-126 at least, and
// NaN for a block that holds an infinity or a NaN (their bits are the largest).  448 is 1.75 * 2^8, so the exponent follows from
// amax's own by one comparison of significands.  With a power of two x / s is exact, so a value is rounded once, to e4m3, and
// the result is the same however it is computed; a scale of amax / 448 itself would be rounded, and values on the border
// between two of e4m3 would go by that rounding.
__device__ __forceinline__ float fp8_scale_of(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - ((amax_bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    return amax_bits >= 0x7f800000u ? u2f(0x7fc00000u) : u2f((uint32_t)(e < 1 ? 1 : e) << 23);
}
// 1 / s of such a scale, exactly (2^-120 ... 2^126)
__device__ __forceinline__ float fp8_inverse(float s) {
    return s == s ? u2f(0x7f000000u - f2u(s)) : s;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return f2u(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// four values of magnitude 448 at most (or NaN) to e4m3, to nearest even
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// x / (1 + e^-x) to a few units in the last place of 32 bits: what it feeds is rounded to e4m3 or bf16, and a value near the
// border between two of e4m3 should fall on its own side.  (The bf16 MLP's sigmoid has a reciprocal of 14 bits.)
__device__ __forceinline__ float silu32(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// eight bf16 in 32 bits
__device__ __forceinline__ void widen8(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[2 * e] = u2f(w[e] << 16);
        v[2 * e + 1] = u2f(w[e] & 0xffff0000u);
    }
}

// 8 or 16 values of a row in 32 bits, from element `at` on; what lies past the row's len elements is zero and not touched
template <int N>
__device__ __forceinline__ void load_row_f32(const uint16_t* row, int at, int len, float (&v)[N]) {
    static_assert(N % 8 == 0, "whole 16 bytes");
#pragma unroll
    for (int c = 0; c < N; c += 8) {
        if (at + c + 8 <= len) {
            u32x4 w;
            __builtin_memcpy(&w, __builtin_assume_aligned(row + at + c, 2), 16);  // (the hardware takes any address)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[c + 2 * e] = u2f(w[e] << 16);
                v[c + 2 * e + 1] = u2f(w[e] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[c + e] = at + c + e < len ? from_bf16(row[at + c + e]) : 0.0f;
        }
    }
}
template <int N>
__device__ __forceinline__ void load_row_f32(const float* row, int at, int len, float (&v)[N]) {
    static_assert(N % 4 == 0, "whole 16 bytes");
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        if (at + c + 4 <= len) {
            u32x4 w;
            __builtin_memcpy(&w, __builtin_assume_aligned(row + at + c, 4), 16);
#pragma unroll
            for (int e = 0; e < 4; e++) v[c + e] = u2f(w[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[c + e] = at + c + e < len ? row[at + c + e] : 0.0f;
        }
    }
}

// 16 values to 16 bytes of e4m3, given 1 / scale
__device__ __forceinline__ u32x4 to_fp8x16(const float (&v)[16], float inv) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = to_fp8x4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
    return w;
}

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

// What the products in 8-bit floating point are made of.  A: rows of e4m3, lda bytes apart, 16-byte aligned, zero from K up to the
// next multiple of 128; sA[kb * ld_sA + m].  Or, where fp8_takes_bf16(M, K), rows of K bf16 that lie anywhere, and sA = NULL.  B: packed as mmx_repack_b packs bytes; sB[row of B's scales][kb].
struct Fp8Gemm {
    const char* A;
    int64_t lda;
    const float* sA;
    int64_t ld_sA;
    const char* Bp;
    int64_t panel_stride;  // bytes of a 32-column panel
    const float* sB;
    int M, N;     // N: packed columns (both of a gate/up pair)
    int K, nkb;   // nkb: blocks of 128 k
    int npanels;
    int pair_up;  // gate/up pair: rows of gate's scales before up's; 0: plain columns
    Epilogue ep;
};

// which row of B's scales a 32-column panel goes by
__device__ __forceinline__ int scale_row(const Fp8Gemm& g, int panel) {
    return g.pair_up ? (panel & 1 ? g.pair_up : 0) + (panel >> 3) : panel >> 2;
}

// A seam between two blocks (norm.hip); strides in elements unless they say bytes.
struct NormArgs {
    const uint16_t* f;
    int64_t ld_f;
    const void* residual;  // or NULL
    int64_t ld_residual;
    const uint16_t *post_weight, *gate, *pre_weight;  // or NULL
    int64_t ld_gate;
    void* r;
    int64_t ld_r;
    char* z;
    int64_t ld_z;  // bytes
    float* z_scales;
    int64_t ld_scales;
    float scale, eps, offset;
    int M, H;
    int post, pre, z_type;  // of z: MMX_BF16, MMX_F8 or MMX_F4 (packed)
};

bool fp8_takes_bf16(int M, int K);

}  // namespace mmx
