// fp8_api.cpp -- C ABI of the linear layer in 8-bit floating point and of the
// root-mean-square norm in front of it: checks of the arguments and the kernels'
// launches. No call allocates, waits or keeps anything for the next.
#include <algorithm>

#include "api_util.hpp"
#include "fp8.hpp"
#include "linear.hpp"
#include "moe_internal.hpp"

using namespace tmt;

namespace {

constexpr int32_t kMaxRows = 1 << 30;
constexpr int64_t kMaxScales = int64_t(1) << 31;   // stride of scales
constexpr int64_t kMaxOutputs = int64_t(1) << 40;  // of a product, so that 32 bits count the tiles
constexpr int64_t kMaxGrid = int64_t(1) << 23;     // workgroups of 512: a launch holds less than 2^32 threads

int64_t blocks_of(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

int check_dtype(int32_t dtype) {
    if (dtype != TMT_MOE_BF16 && dtype != TMT_MOE_F32)
        return fail(TMT_MOE_EINVAL, "dtype=%d is neither TMT_MOE_BF16 nor TMT_MOE_F32", dtype);
    return TMT_MOE_OK;
}
int check_blocks(int32_t blocks) {
    if (blocks != TMT_MOE_FP8_ROWS && blocks != TMT_MOE_FP8_TILES)
        return fail(TMT_MOE_EINVAL, "blocks=%d is neither TMT_MOE_FP8_ROWS nor TMT_MOE_FP8_TILES", blocks);
    return TMT_MOE_OK;
}
// Rows of `width` elements, `piece` of which are 16 bytes.
int check_rows(const char* what, const void* p, int64_t ld, int64_t width, int piece) {
    if (!p) return fail(TMT_MOE_EINVAL, "%s must be non-NULL", what);
    if (!aligned16(p)) return fail(TMT_MOE_EINVAL, "%s must be 16-byte aligned", what);
    if (ld < width || ld % piece != 0)
        return fail(TMT_MOE_EINVAL, "the row stride %lld of %s must be a multiple of %d, at least %lld", (long long)ld,
                    what, piece, (long long)width);
    if (ld > kMaxStride) return fail(TMT_MOE_EINVAL, "the row stride %lld of %s is over %lld", (long long)ld, what, (long long)kMaxStride);
    return TMT_MOE_OK;
}
int check_scales(const char* what, const float* p, int64_t ld, int64_t width) {
    if (!p) return fail(TMT_MOE_EINVAL, "%s must be non-NULL", what);
    if (!aligned_to(p, 4)) return fail(TMT_MOE_EINVAL, "%s must be 4-byte aligned", what);
    if (ld < width || ld > kMaxScales)
        return fail(TMT_MOE_EINVAL, "the stride %lld of %s must be at least %lld and at most %lld", (long long)ld, what,
                    (long long)width, (long long)kMaxScales);
    return TMT_MOE_OK;
}
int check_floats(const char* what, const float* p, unsigned align) {
    if (!p) return fail(TMT_MOE_EINVAL, "%s must be non-NULL", what);
    if (!aligned_to(p, align)) return fail(TMT_MOE_EINVAL, "%s must be %u-byte aligned", what, align);
    return TMT_MOE_OK;
}
int check_norm_shape(int32_t T, int32_t d) {
    if (T < 0 || T > kMaxRows) return fail(TMT_MOE_EINVAL, "T=%d must be from 0 to %d", T, kMaxRows);
    if (d < 1 || d > kRmsMaxWidth) return fail(TMT_MOE_EINVAL, "d=%d must be from 1 to %d", d, kRmsMaxWidth);
    return TMT_MOE_OK;
}
int check_workspace(const void* workspace, size_t bytes, size_t need) {
    if (need == 0) return TMT_MOE_OK;
    if (!workspace || !aligned_to(workspace, 256))
        return fail(TMT_MOE_EINVAL, "workspace must be a 256-byte aligned device pointer");
    if (bytes < need) return fail(TMT_MOE_EINVAL, "workspace of %zu bytes is smaller than the %zu bytes needed", bytes, need);
    return TMT_MOE_OK;
}
// A workspace for T serves every call of fewer rows: the partial rows of the
// backward do not outnumber the workgroups that the chip holds.
size_t norm_workspace(int32_t T, int32_t d) {
    return (size_t)std::min<int64_t>(rms_partials_max(d, cu_count()), T) * ln_width4(d) * sizeof(float);
}

int check_product_shape(int32_t M, int32_t N, int32_t K) {
    if (M < 0 || M > kMaxRows) return fail(TMT_MOE_EINVAL, "M=%d must be from 0 to %d", M, kMaxRows);
    if (N < 0 || N % 8 != 0 || N > kMaxStride) return fail(TMT_MOE_EINVAL, "N=%d must be a multiple of 8 from 0 to %lld", N, (long long)kMaxStride);
    if (K < 0 || K > kMaxStride) return fail(TMT_MOE_EINVAL, "K=%d must be from 0 to %lld", K, (long long)kMaxStride);
    if ((int64_t)M * N > kMaxOutputs) return fail(TMT_MOE_EINVAL, "M=%d, N=%d: M*N must be at most 2^40", M, N);
    return TMT_MOE_OK;
}

}  // namespace

extern "C" {

int tmt_moe_rmsnorm_forward(void* stream, int32_t T, int32_t d, int32_t dtype, const uint16_t* X, int64_t ldx,
                            const void* R, int64_t ldr, const float* gamma, float eps, void* S, int64_t lds, uint16_t* Y,
                            int64_t ldy, uint8_t* codes, int64_t ldc, float* scales, int64_t ldsc, float* rstd) {
    int rc = check_norm_shape(T, d);
    if (rc || (rc = check_dtype(dtype))) return rc;
    if (!(eps >= 0.0f)) return fail(TMT_MOE_EINVAL, "eps=%g must not be negative", (double)eps);
    if (T == 0) return TMT_MOE_OK;
    if (!X && !R) return fail(TMT_MOE_EINVAL, "X and R are both NULL");
    if (!R && dtype != TMT_MOE_BF16) return fail(TMT_MOE_EINVAL, "without R the stream is X's: dtype must be TMT_MOE_BF16");
    if (!S && !Y && !codes && !rstd) return fail(TMT_MOE_EINVAL, "S, Y, codes and rstd are all NULL");
    const int piece = dtype == TMT_MOE_BF16 ? 8 : 4;
    if ((X && (rc = check_rows("X", X, ldx, d, 8))) || (R && (rc = check_rows("R", R, ldr, d, piece))) ||
        (rc = check_floats("gamma", gamma, 16)) || (S && (rc = check_rows("S", S, lds, d, piece))) ||
        (Y && (rc = check_rows("Y", Y, ldy, d, 8))) || (rstd && (rc = check_floats("rstd", rstd, 4))))
        return rc;
    if (codes && ((rc = check_rows("codes", codes, ldc, d, 16)) || (rc = check_scales("scales", scales, ldsc, T)))) return rc;
    RmsParams p{};
    p.T = T; p.d = d; p.f32 = dtype == TMT_MOE_F32; p.X = X; p.ldx = ldx; p.R = R; p.ldr = ldr; p.gamma = gamma; p.eps = eps;
    p.S = S; p.lds = lds; p.Y = Y; p.ldy = ldy; p.codes = codes; p.ldc = ldc; p.scales = scales; p.ldsc = ldsc; p.rstd = rstd;
    HIP_TRY(launch_rms_fwd(p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_rmsnorm_workspace_size(int32_t T, int32_t d, size_t* bytes) {
    int rc = check_norm_shape(T, d);
    if (rc) return rc;
    if (!bytes) return fail(TMT_MOE_EINVAL, "bytes is NULL");
    *bytes = norm_workspace(T, d);
    return TMT_MOE_OK;
}

int tmt_moe_rmsnorm_backward(void* stream, int32_t T, int32_t d, int32_t dtype, const uint16_t* dY, int64_t lddy,
                             const void* S, int64_t lds, const float* gamma, const float* rstd, const void* dR,
                             int64_t lddr, void* dS, int64_t ldds, float* dgamma, void* workspace, size_t workspace_bytes) {
    int rc = check_norm_shape(T, d);
    if (rc || (rc = check_dtype(dtype)) || (rc = check_floats("dgamma", dgamma, 16))) return rc;
    const int piece = dtype == TMT_MOE_BF16 ? 8 : 4;
    if (T > 0 && ((rc = check_rows("dY", dY, lddy, d, 8)) || (rc = check_rows("S", S, lds, d, piece)) ||
                  (rc = check_floats("gamma", gamma, 16)) || (rc = check_floats("rstd", rstd, 4)) ||
                  (dR && (rc = check_rows("dR", dR, lddr, d, piece))) || (rc = check_rows("dS", dS, ldds, d, piece)) ||
                  (rc = check_workspace(workspace, workspace_bytes, norm_workspace(T, d)))))
        return rc;
    RmsParams p{};
    p.T = T; p.d = d; p.f32 = dtype == TMT_MOE_F32; p.dY = dY; p.lddy = lddy; p.S = const_cast<void*>(S); p.lds = lds;
    p.gamma = gamma; p.rstd = const_cast<float*>(rstd); p.dR = dR; p.lddr = lddr; p.dS = dS; p.ldds = ldds;
    p.dgamma = dgamma; p.partial = static_cast<float*>(workspace);
    HIP_TRY(launch_rms_bwd(p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_fp8_quantize(void* stream, int32_t blocks, int32_t dtype, const void* X, int64_t ldx, int32_t rows,
                         int32_t K, uint8_t* codes, int64_t ldc, float* scales, int64_t lds, uint8_t* codes_t,
                         int64_t ldct, float* scales_t, int64_t ldst) {
    int rc = check_blocks(blocks);
    if (rc || (rc = check_dtype(dtype))) return rc;
    if (rows < 0 || K < 0) return fail(TMT_MOE_EINVAL, "rows=%d and K=%d must not be negative", rows, K);
    if (rows == 0 || K == 0) return TMT_MOE_OK;
    if (!codes && !codes_t) return fail(TMT_MOE_EINVAL, "codes and codes_t are both NULL");
    const bool tiles = blocks == TMT_MOE_FP8_TILES;
    if (blocks_of(rows) * blocks_of(K) >= kMaxGrid)
        return fail(TMT_MOE_EINVAL, "rows=%d of K=%d are 2^23 tiles of 128 x 128 or more", rows, K);
    if ((rc = check_rows("X", X, ldx, K, dtype == TMT_MOE_BF16 ? 8 : 4))) return rc;
    if (codes && ((rc = check_rows("codes", codes, ldc, K, 16)) ||
                  (rc = check_scales("scales", scales, lds, tiles ? blocks_of(K) : rows))))
        return rc;
    if (codes_t && ((rc = check_rows("codes_t", codes_t, ldct, rows, 16)) ||
                    (rc = check_scales("scales_t", scales_t, ldst, tiles ? blocks_of(rows) : K))))
        return rc;
    Fp8QuantParams p{};
    p.x = X; p.ldx = ldx; p.rows = rows; p.K = K; p.codes = codes; p.ldc = ldc; p.scales = scales; p.lds = lds;
    p.codes_t = codes_t; p.ldct = ldct; p.scales_t = scales_t; p.ldst = ldst;
    HIP_TRY(launch_fp8_quantize(tiles, dtype == TMT_MOE_F32, p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_fp8_transpose(void* stream, const uint8_t* codes, int64_t ldc, int32_t rows, int32_t K, uint8_t* codes_t,
                          int64_t ldct) {
    if (rows < 0 || K < 0) return fail(TMT_MOE_EINVAL, "rows=%d and K=%d must not be negative", rows, K);
    if (rows == 0 || K == 0) return TMT_MOE_OK;
    if (blocks_of(rows) * blocks_of(K) >= kMaxGrid)
        return fail(TMT_MOE_EINVAL, "rows=%d of K=%d are 2^23 tiles of 128 x 128 or more", rows, K);
    if (!codes) return fail(TMT_MOE_EINVAL, "codes must be non-NULL");
    if (ldc < K || ldc > kMaxStride)
        return fail(TMT_MOE_EINVAL, "the row stride %lld of codes must be at least %d and at most %lld", (long long)ldc, K, (long long)kMaxStride);
    int rc = check_rows("codes_t", codes_t, ldct, rows, 16);
    if (rc) return rc;
    HIP_TRY(launch_fp8_transpose(codes, ldc, rows, K, codes_t, ldct, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_fp8_workspace_size(int32_t b_blocks, int32_t M, int32_t N, int32_t K, size_t* bytes) {
    int rc = check_blocks(b_blocks);
    if (rc || (rc = check_product_shape(M, N, K))) return rc;
    if (!bytes) return fail(TMT_MOE_EINVAL, "bytes is NULL");
    *bytes = M == 0 || N == 0 ? 0 : fp8_workspace(M, N, K);
    return TMT_MOE_OK;
}

int tmt_moe_fp8_matmul(void* stream, int32_t b_blocks, int32_t dtype, int32_t M, int32_t N, int32_t K, const uint8_t* A,
                       int64_t lda, const float* A_scale, int64_t ldas, const uint8_t* B, int64_t ldb,
                       const float* B_scale, int64_t ldbs, void* Y, int64_t ldy, float beta, void* workspace,
                       size_t workspace_bytes) {
    int rc = check_blocks(b_blocks);
    if (rc || (rc = check_dtype(dtype)) || (rc = check_product_shape(M, N, K))) return rc;
    if (M == 0 || N == 0) return TMT_MOE_OK;
    const bool tiles = b_blocks == TMT_MOE_FP8_TILES;
    if (K > 0 && ((rc = check_rows("A", A, lda, K, 16)) || (rc = check_scales("A_scale", A_scale, ldas, M)) ||
                  (rc = check_rows("B", B, ldb, K, 16)) ||
                  (rc = check_scales("B_scale", B_scale, ldbs, tiles ? blocks_of(K) : N))))
        return rc;
    if ((rc = check_rows("Y", Y, ldy, N, dtype == TMT_MOE_BF16 ? 8 : 4))) return rc;
    if ((rc = check_workspace(workspace, workspace_bytes, fp8_workspace(M, N, K)))) return rc;
    Fp8Params p{};
    p.M = M; p.N = N; p.K = K; p.a = A; p.lda = lda; p.as = A_scale; p.ldas = ldas; p.b = B; p.ldb = ldb;
    p.bs = B_scale; p.ldbs = ldbs; p.y = Y; p.ldy = ldy; p.beta = beta; p.part = static_cast<float*>(workspace);
    HIP_TRY(launch_fp8_matmul(tiles, dtype == TMT_MOE_F32, p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

}  // extern "C"
