// C ABI of the feed-forward block's operators: argument validation, scratch layout, dispatch.
#include <string.h>

#include "ffn.hpp"

namespace mmx {

int make_epilogue(const mmx_epilogue* in, int a_dtype, int b_dtype, int M, int n0, int n1, Epilogue* out);
int launch_quantize_rows_fp8(bool f32, const void* x, int64_t ldx_bytes, int M, int K, void* q, int64_t ldq, float* scales, int64_t ld_s,
                             hipStream_t st);
int launch_quantize_pack_fp8(const void* W, int64_t ldw_bytes, int K, int N, int transpose, int pair, void* packed, float* scales, hipStream_t st);
int launch_repack_gate_up_bytes(const void* wg, const void* wu, int64_t ldw, int K, int N, void* out, hipStream_t st);
int launch_gemm_fp8(const Fp8Gemm& g, hipStream_t st);
int launch_moe_route(const void* x, int64_t ldx, const void* Wr, int64_t ldr, int T, int H, int E, int k, int sigmoid, int renormalize, float scale,
                     const float* bias, double* logits, int* ids, float* weights, hipStream_t st);
int launch_moe_experts(bool f8, const void* x, int64_t ldx_bytes, const int* ids, const float* weights, int T, int H, int I, int E, int k,
                       const void* w_gate_up, const float* s_gate_up, const void* w_down, const float* s_down, void* h, void* y, int64_t ldy, int y_f32,
                       hipStream_t st);
size_t moe_scratch_bytes(int T, int H, int I, int k);
int launch_block_norm(const NormArgs& g, bool residual_f32, hipStream_t st);

static bool misaligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(to - 1)) != 0; }
static int64_t padded_k(int K) { return ((int64_t)K + BLOCK - 1) / BLOCK * BLOCK; }
static int blocks_of(int n) { return (int)(((int64_t)n + BLOCK - 1) / BLOCK); }
static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// rows [M, cols] of `size` bytes a value
static int check_rows(const char* who, const char* what, const void* p, int64_t ld_bytes, int M, int64_t cols, int size) {
    if (!p) return set_error(MMX_E_INVALID, "%s: %s is NULL", who, what);
    if (misaligned(p, size) || ld_bytes % size) return set_error(MMX_E_INVALID, "%s: %s is not aligned to its element size", who, what);
    if ((M > 1 && ld_bytes < cols * size) || ld_bytes < 0)
        return set_error(MMX_E_INVALID, "%s: rows of %s are %lld bytes apart, a row has %lld", who, what, (long long)ld_bytes, (long long)(cols * size));
    return MMX_OK;
}
// quantised rows, as the products read them and the quantisers write them
static int check_rows_fp8(const char* who, const char* what, const void* q, int64_t ld_bytes, const float* scales, int64_t ld_scales, int M, int K) {
    if (!q || !scales) return set_error(MMX_E_INVALID, "%s: %s or its scales are NULL", who, what);
    if (misaligned(q, 16) || ld_bytes % 16) return set_error(MMX_E_INVALID, "%s: rows of %s are not 16-byte aligned", who, what);
    if (ld_bytes < 0 || (M > 1 && ld_bytes < padded_k(K)))
        return set_error(MMX_E_INVALID, "%s: rows of %s are %lld bytes apart, a padded row has %lld", who, what, (long long)ld_bytes, (long long)padded_k(K));
    if (ld_bytes > (8 << 20)) return set_error(MMX_E_UNSUPPORTED, "%s: rows of %s more than 8 MiB apart", who, what);
    if (misaligned(scales, 4)) return set_error(MMX_E_INVALID, "%s: scales are not aligned to their element size", who);
    if (ld_scales < M) return set_error(MMX_E_INVALID, "%s: rows of %s's scales are %lld apart, M = %d", who, what, (long long)ld_scales, M);
    return MMX_OK;
}
static int check_weights(const char* who, const void* packed, const float* scales) {
    if (!packed || !scales) return set_error(MMX_E_INVALID, "%s: packed weights or their scales are NULL", who);
    if (misaligned(packed, 16)) return set_error(MMX_E_INVALID, "%s: packed weights must be 16-byte aligned", who);
    if (misaligned(scales, 4)) return set_error(MMX_E_INVALID, "%s: scales are not aligned to their element size", who);
    return MMX_OK;
}
static int check_scratch(const char* who, const void* scratch, size_t have, size_t need) {
    if (need == 0) return MMX_OK;
    if (!scratch || have < need) return set_error(MMX_E_INVALID, "%s: %zu bytes of scratch, %zu are needed", who, scratch ? have : (size_t)0, need);
    if (misaligned(scratch, 256)) return set_error(MMX_E_INVALID, "%s: the scratch must be 256-byte aligned", who);
    return MMX_OK;
}

// K and N within what the kernels address with 32 bits; M such that a launch of up to 1024 threads for each row has fewer than 2^32 of them
constexpr int MOST_K = 1 << 22, MOST_N = 1 << 26, MOST_M = (1 << 22) - 1;
static int check_sizes(const char* who, int M, int K, int N) {
    if (M < 0 || K <= 0 || N <= 0) return set_error(MMX_E_INVALID, "%s: K and N must be positive and M not negative (got %d, %d, %d)", who, M, K, N);
    if (K > MOST_K || N > MOST_N || M > MOST_M)
        return set_error(MMX_E_UNSUPPORTED, "%s: M up to %d, N up to %d and K up to %d (got %d, %d, %d)", who, MOST_M, MOST_N, MOST_K, M, K, N);
    return MMX_OK;
}

// quantised rows in scratch: the bytes, then the scales
// (rows a multiple of 2 KiB apart meet in few channels of the L2)
static int64_t pitch_of(int K) { return padded_k(K) % 2048 ? padded_k(K) : padded_k(K) + 128; }
static size_t rows_bytes(int M, int K) { return round256((size_t)M * pitch_of(K)) + round256((size_t)blocks_of(K) * M * 4); }
struct Rows {
    const char* q;
    int64_t ld;
    const float* scales;
    int64_t ld_scales;
};
// A as quantised rows: as given, or made in scratch; or as bf16 rows that the product quantises itself
static int quantised(int dtype, const void* A, int64_t lda, const float* scales, int64_t ld_scales, int M, int K, char* scratch, Rows* out,
                     hipStream_t st) {
    if (dtype == MMX_F8 || (dtype == MMX_BF16 && fp8_takes_bf16(M, K))) {
        *out = {static_cast<const char*>(A), lda, scales, ld_scales};
        return MMX_OK;
    }
    float* const s = reinterpret_cast<float*>(scratch + round256((size_t)M * pitch_of(K)));
    *out = {scratch, pitch_of(K), s, M};
    return launch_quantize_rows_fp8(dtype == MMX_F32, A, lda, M, K, scratch, pitch_of(K), s, M, st);
}

static Fp8Gemm product(const Rows& a, const void* Bp, const float* b_scales, int M, int K, int N, bool pair, const Epilogue& ep) {
    Fp8Gemm g;
    g.A = a.q;
    g.lda = a.ld;
    g.sA = a.scales;
    g.ld_sA = a.ld_scales;
    g.Bp = static_cast<const char*>(Bp);
    g.K = K;
    g.nkb = blocks_of(K);
    g.panel_stride = (int64_t)g.nkb * 4096;
    g.sB = b_scales;
    g.M = M;
    g.N = N;
    g.npanels = (N + 31) / 32;
    g.pair_up = pair ? blocks_of(N / 2) : 0;
    g.ep = ep;
    return g;
}

static int check_a(const char* who, int dtype, const void* A, int64_t lda, const float* scales, int64_t ld_scales, int M, int K) {
    if (dtype == MMX_F8) return check_rows_fp8(who, "A", A, lda, scales, ld_scales, M, K);
    if (dtype != MMX_BF16 && dtype != MMX_F32) return set_error(MMX_E_INVALID, "%s: activations of dtype %d (bf16, fp32 and e4m3 exist)", who, dtype);
    if (scales) return set_error(MMX_E_INVALID, "%s: scales come with e4m3 activations only", who);
    return check_rows(who, "A", A, lda, M, K, dtype == MMX_F32 ? 4 : 2);
}

}  // namespace mmx

using namespace mmx;

extern "C" {

int mmx_quantize_rows_fp8(int x_dtype, const void* x, int64_t ldx_bytes, int M, int K, void* q, int64_t ldq_bytes, float* scales, int64_t ld_scales,
                          void* stream) {
    const char* const who = "mmx_quantize_rows_fp8";
    if (x_dtype != MMX_BF16 && x_dtype != MMX_F32) return set_error(MMX_E_INVALID, "%s: x of dtype %d (bf16 and fp32 exist)", who, x_dtype);
    int rc = check_sizes(who, M, K, 1);
    if (rc || M == 0) return rc;
    if ((rc = check_rows(who, "x", x, ldx_bytes, M, K, x_dtype == MMX_F32 ? 4 : 2))) return rc;
    if ((rc = check_rows_fp8(who, "q", q, ldq_bytes, scales, ld_scales, M, K))) return rc;
    return launch_quantize_rows_fp8(x_dtype == MMX_F32, x, ldx_bytes, M, K, q, ldq_bytes, scales, ld_scales, static_cast<hipStream_t>(stream));
}

int mmx_quantize_pack_fp8(const void* W, int64_t ldw_bytes, int K, int N, int transpose, int pair, void* packed, float* scales, void* stream) {
    const char* const who = "mmx_quantize_pack_fp8";
    int rc = check_sizes(who, 0, K, N);
    if (rc) return rc;
    if (pair < 0 || pair > 2 || (pair && N % 32)) return set_error(MMX_E_INVALID, "%s: pair = %d, N = %d (a half of a pair has a multiple of 32 columns)", who, pair, N);
    if ((rc = check_rows(who, "W", W, ldw_bytes, transpose ? N : K, transpose ? K : N, 2))) return rc;
    if ((rc = check_weights(who, packed, scales))) return rc;
    return launch_quantize_pack_fp8(W, ldw_bytes, K, N, transpose, pair, packed, pair == 2 ? scales + (int64_t)blocks_of(N) * blocks_of(K) : scales,
                                    static_cast<hipStream_t>(stream));
}

int mmx_repack_gate_up_fp8(const void* w_gate, const void* w_up, int64_t ldw_bytes, int K, int N, void* packed, void* stream) {
    const char* const who = "mmx_repack_gate_up_fp8";
    if (!w_gate || !w_up || !packed) return set_error(MMX_E_INVALID, "%s: NULL pointer", who);
    int rc = check_sizes(who, 0, K, N);
    if (rc) return rc;
    if (N % 32) return set_error(MMX_E_INVALID, "%s: N = %d must be a multiple of 32", who, N);
    if (ldw_bytes < K) return set_error(MMX_E_INVALID, "%s: ldw_bytes %lld smaller than a row", who, (long long)ldw_bytes);
    if (misaligned(packed, 16)) return set_error(MMX_E_INVALID, "%s: packed buffer must be 16-byte aligned", who);
    return launch_repack_gate_up_bytes(w_gate, w_up, ldw_bytes, K, N, packed, static_cast<hipStream_t>(stream));
}

size_t mmx_gemm_fp8_scratch_bytes(int a_dtype, int M, int K, int N) {
    if (M <= 0 || K <= 0 || N <= 0 || (a_dtype != MMX_BF16 && a_dtype != MMX_F32) || (a_dtype == MMX_BF16 && fp8_takes_bf16(M, K))) return 0;
    return rows_bytes(M, K);
}

int mmx_gemm_fp8(int a_dtype, const void* A, int64_t lda_bytes, const float* a_scales, int64_t ld_a_scales, const void* Bpacked, const float* b_scales,
                 int M, int K, int N, const mmx_epilogue* ep_in, void* scratch, size_t scratch_bytes, void* stream) {
    const char* const who = "mmx_gemm_fp8";
    int rc = check_sizes(who, M, K, N);
    if (rc || M == 0) return rc;
    if ((rc = check_a(who, a_dtype, A, lda_bytes, a_scales, ld_a_scales, M, K))) return rc;
    if ((rc = check_weights(who, Bpacked, b_scales))) return rc;
    Epilogue ep;
    if ((rc = make_epilogue(ep_in, MMX_BF16, MMX_F8, M, 0, N, &ep))) return rc;
    if (ep.steps & (MMX_PP_DEQUANT | MMX_PP_QUANT)) return set_error(MMX_E_INVALID, "%s: the scales of the blocks take the place of DEQUANT, and there is no QUANT", who);
    if (ep.out_dtype != MMX_F32 && ep.out_dtype != MMX_BF16) return set_error(MMX_E_INVALID, "%s: output dtype %d (bf16 and fp32 exist)", who, ep.out_dtype);
    const bool pair = ep.steps & MMX_PP_SILU_GATE;
    if (pair && (N % 64 || ep.steps != MMX_PP_SILU_GATE)) return set_error(MMX_E_INVALID, "%s: SILU_GATE stands alone and needs N %% 64 == 0 (got %d)", who, N);
    if ((rc = check_scratch(who, scratch, scratch_bytes, mmx_gemm_fp8_scratch_bytes(a_dtype, M, K, N)))) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    Rows a;
    if ((rc = quantised(a_dtype, A, lda_bytes, a_scales, ld_a_scales, M, K, static_cast<char*>(scratch), &a, st))) return rc;
    return launch_gemm_fp8(product(a, Bpacked, b_scales, M, K, N, pair, ep), st);
}

size_t mmx_mlp_fp8_scratch_bytes(int x_dtype, int M, int K, int N) {
    if (M <= 0 || K <= 0 || N <= 0) return 0;
    return mmx_gemm_fp8_scratch_bytes(x_dtype, M, K, N) + round256((size_t)M * N * 4) + rows_bytes(M, N);
}

int mmx_mlp_fp8(int x_dtype, const void* x, int64_t ldx_bytes, const float* x_scales, int64_t ld_x_scales, const void* w_gate_up,
                const float* gate_up_scales, const void* w_down, const float* down_scales, int y_dtype, void* y, int64_t ldy_bytes, int M, int K, int N,
                void* scratch, size_t scratch_bytes, void* stream) {
    const char* const who = "mmx_mlp_fp8";
    int rc = check_sizes(who, M, K, N);
    if (rc || M == 0) return rc;
    if (N % 32 || N > MOST_N / 2 || N > MOST_K) return set_error(MMX_E_INVALID, "%s: N = %d must be a multiple of 32, %d at most", who, N, MOST_K);
    if ((rc = check_a(who, x_dtype, x, ldx_bytes, x_scales, ld_x_scales, M, K))) return rc;
    if ((rc = check_weights(who, w_gate_up, gate_up_scales)) || (rc = check_weights(who, w_down, down_scales))) return rc;
    if (y_dtype != MMX_F32 && y_dtype != MMX_BF16) return set_error(MMX_E_INVALID, "%s: output dtype %d (bf16 and fp32 exist)", who, y_dtype);
    if ((rc = check_scratch(who, scratch, scratch_bytes, mmx_mlp_fp8_scratch_bytes(x_dtype, M, K, N)))) return rc;
    mmx_epilogue e;
    memset(&e, 0, sizeof e);
    e.out_dtype = y_dtype;
    e.C = y;
    e.ldc_bytes = ldy_bytes;
    Epilogue out;
    if ((rc = make_epilogue(&e, MMX_BF16, MMX_F8, M, 0, K, &out))) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* at = static_cast<char*>(scratch);
    Rows a, hq;
    if ((rc = quantised(x_dtype, x, ldx_bytes, x_scales, ld_x_scales, M, K, at, &a, st))) return rc;
    at += mmx_gemm_fp8_scratch_bytes(x_dtype, M, K, N);
    char* const h = at;
    at += round256((size_t)M * N * 4);
    Epilogue mid;
    memset(&mid, 0, sizeof mid);
    mid.steps = MMX_PP_SILU_GATE;
    mid.out_dtype = MMX_F32;
    mid.C = h;
    mid.ldc = (int64_t)N * 4;
    if ((rc = launch_gemm_fp8(product(a, w_gate_up, gate_up_scales, M, K, 2 * N, true, mid), st))) return rc;
    if ((rc = quantised(MMX_F32, h, (int64_t)N * 4, nullptr, 0, M, N, at, &hq, st))) return rc;
    return launch_gemm_fp8(product(hq, w_down, down_scales, M, N, K, false, out), st);
}

int mmx_moe_route(const void* x, int64_t ldx_bytes, const void* router, int64_t ldr_bytes, int T, int H, int E, int top_k, int flags, float scale,
                  const float* bias, double* logits, int32_t* ids, float* weights, void* stream) {
    const char* const who = "mmx_moe_route";
    int rc = check_sizes(who, T, H, 1);
    if (rc) return rc;
    if (E < 1 || E > 1024 || top_k < 1 || top_k > 16 || top_k > E)
        return set_error(MMX_E_INVALID, "%s: top_k = %d of E = %d experts (up to 16 of up to 1024)", who, top_k, E);
    if (flags & ~(MMX_MOE_SIGMOID | MMX_MOE_RENORMALIZE)) return set_error(MMX_E_INVALID, "%s: unknown flags 0x%x", who, flags);
    if (T == 0) return MMX_OK;
    if ((rc = check_rows(who, "x", x, ldx_bytes, T, H, 2)) || (rc = check_rows(who, "router", router, ldr_bytes, E, H, 2))) return rc;
    if (!logits || !ids || !weights) return set_error(MMX_E_INVALID, "%s: NULL pointer", who);
    if (misaligned(logits, 8) || misaligned(ids, 4) || misaligned(weights, 4) || misaligned(bias, 4))
        return set_error(MMX_E_INVALID, "%s: an operand is not aligned to its element size", who);
    return launch_moe_route(x, ldx_bytes, router, ldr_bytes, T, H, E, top_k, flags & MMX_MOE_SIGMOID, flags & MMX_MOE_RENORMALIZE, scale, bias, logits, ids,
                            weights, static_cast<hipStream_t>(stream));
}

size_t mmx_moe_experts_scratch_bytes(int T, int H, int I, int top_k) {
    return T <= 0 || H <= 0 || I <= 0 || top_k <= 0 ? 0 : moe_scratch_bytes(T, H, I, top_k);
}

int mmx_moe_experts(int w_dtype, const void* x, int64_t ldx_bytes, const int32_t* ids, const float* weights, int T, int H, int I, int E, int top_k,
                    const void* w_gate_up, const float* gate_up_scales, const void* w_down, const float* down_scales, int y_dtype, void* y,
                    int64_t ldy_bytes, void* scratch, size_t scratch_bytes, void* stream) {
    const char* const who = "mmx_moe_experts";
    int rc = check_sizes(who, T, H, I);
    if (rc) return rc;
    if (w_dtype != MMX_BF16 && w_dtype != MMX_F8) return set_error(MMX_E_INVALID, "%s: weights of dtype %d (bf16 and e4m3 exist)", who, w_dtype);
    if (I % 32 || I > MOST_K) return set_error(MMX_E_INVALID, "%s: I = %d must be a multiple of 32, %d at most", who, I, MOST_K);
    if (E < 1 || E > 1024 || top_k < 1 || top_k > 16) return set_error(MMX_E_INVALID, "%s: top_k = %d of E = %d experts (up to 16 of up to 1024)", who, top_k, E);
    if (y_dtype != MMX_F32 && y_dtype != MMX_BF16) return set_error(MMX_E_INVALID, "%s: output dtype %d (bf16 and fp32 exist)", who, y_dtype);
    if (T == 0) return MMX_OK;
    if ((rc = check_rows(who, "x", x, ldx_bytes, T, H, 2)) || (rc = check_rows(who, "y", y, ldy_bytes, T, H, y_dtype == MMX_F32 ? 4 : 2))) return rc;
    if (!ids || !weights || !w_gate_up || !w_down) return set_error(MMX_E_INVALID, "%s: NULL pointer", who);
    if (misaligned(ids, 4) || misaligned(weights, 4) || misaligned(w_gate_up, 16) || misaligned(w_down, 16))
        return set_error(MMX_E_INVALID, "%s: ids and weights are not aligned to their element size, or packed weights not to 16 bytes", who);
    if ((rc = check_scratch(who, scratch, scratch_bytes, moe_scratch_bytes(T, H, I, top_k)))) return rc;
    const bool f8 = w_dtype == MMX_F8;
    if (f8 ? !gate_up_scales || !down_scales : gate_up_scales || down_scales)
        return set_error(MMX_E_INVALID, "%s: e4m3 weights come with scales, bf16 weights without", who);
    if (misaligned(gate_up_scales, 4) || misaligned(down_scales, 4)) return set_error(MMX_E_INVALID, "%s: scales are not aligned to their element size", who);
    return launch_moe_experts(f8, x, ldx_bytes, ids, weights, T, H, I, E, top_k, w_gate_up, gate_up_scales, w_down, down_scales, scratch, y, ldy_bytes,
                              y_dtype == MMX_F32, static_cast<hipStream_t>(stream));
}

int mmx_block_norm(const mmx_block_norm_args* a, int M, int H, void* stream) {
    const char* const who = "mmx_block_norm";
    if (!a) return set_error(MMX_E_INVALID, "%s: NULL arguments", who);
    int rc = check_sizes(who, M, H, 1);
    if (rc) return rc;
    if (H > 32768) return set_error(MMX_E_UNSUPPORTED, "%s: H = %d, 32768 at most", who, H);
    if (a->residual_dtype != MMX_BF16 && a->residual_dtype != MMX_F32) return set_error(MMX_E_INVALID, "%s: residual of dtype %d (bf16 and fp32 exist)", who, a->residual_dtype);
    if (a->z && a->z_dtype != MMX_BF16 && a->z_dtype != MMX_F8) return set_error(MMX_E_INVALID, "%s: z of dtype %d (bf16 and e4m3 exist)", who, a->z_dtype);
    if (!a->r && !a->z) return set_error(MMX_E_INVALID, "%s: neither r nor z is wanted", who);
    if ((a->post_weight && !a->post) || (a->pre_weight && !a->pre)) return set_error(MMX_E_INVALID, "%s: weights of a norm that is off", who);
    if (M == 0) return MMX_OK;
    const int rs = a->residual_dtype == MMX_F32 ? 4 : 2;
    if ((rc = check_rows(who, "f", a->f, a->ldf_bytes, M, H, 2))) return rc;
    if (a->residual && (rc = check_rows(who, "residual", a->residual, a->ld_residual_bytes, M, H, rs))) return rc;
    if (a->r && (rc = check_rows(who, "r", a->r, a->ldr_bytes, M, H, rs))) return rc;
    if (a->gate && (rc = check_rows(who, "gate", a->gate, a->ld_gate_bytes, a->ld_gate_bytes == 0 ? 1 : M, H, 2))) return rc;
    if (misaligned(a->post_weight, 2) || misaligned(a->pre_weight, 2)) return set_error(MMX_E_INVALID, "%s: weights are not aligned to their element size", who);
    if (a->z && a->z_dtype == MMX_BF16 && (rc = check_rows(who, "z", a->z, a->ldz_bytes, M, H, 2))) return rc;
    if (a->z && a->z_dtype == MMX_F8 && (rc = check_rows_fp8(who, "z", a->z, a->ldz_bytes, a->z_scales, a->ld_z_scales, M, H))) return rc;
    NormArgs g;
    g.f = static_cast<const uint16_t*>(a->f);
    g.ld_f = a->ldf_bytes / 2;
    g.residual = a->residual;
    g.ld_residual = a->ld_residual_bytes / rs;
    g.post_weight = static_cast<const uint16_t*>(a->post_weight);
    g.gate = static_cast<const uint16_t*>(a->gate);
    g.pre_weight = static_cast<const uint16_t*>(a->pre_weight);
    g.ld_gate = a->ld_gate_bytes / 2;
    g.r = a->r;
    g.ld_r = a->ldr_bytes / rs;
    g.z = static_cast<char*>(a->z);
    g.ld_z = a->ldz_bytes;
    g.z_scales = a->z_scales;
    g.ld_scales = a->ld_z_scales;
    g.scale = a->scale, g.eps = a->eps, g.offset = a->weight_offset;
    g.M = M, g.H = H;
    g.post = a->post, g.pre = a->pre;
    g.z_f8 = a->z && a->z_dtype == MMX_F8;
    return launch_block_norm(g, a->residual_dtype == MMX_F32, static_cast<hipStream_t>(stream));
}

}  // extern "C"
