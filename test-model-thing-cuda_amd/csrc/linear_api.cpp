// linear_api.cpp -- C ABI of the linear layer on microscaled numbers: checks
// of the arguments and the kernels' launches. No call allocates, waits or
// keeps anything for the next.
#include "api_util.hpp"
#include "linear.hpp"

using namespace tmt;

static_assert((int)TMT_MOE_LINEAR_FORWARD == LINEAR_FORWARD && (int)TMT_MOE_LINEAR_MATMUL == LINEAR_MATMUL &&
                  (int)TMT_MOE_LINEAR_DX == LINEAR_DX && (int)TMT_MOE_LINEAR_DW == LINEAR_DW,
              "the header's operators are the kernels'");

namespace {

// Values quantised by one call: a launch holds less than 2^32 threads, 2^24
// workgroups of a tile each. Matrices that round up to as many are refused too.
constexpr int64_t kMaxValues = int64_t(1) << 36;

int check_rows(int32_t format, int32_t dtype, int32_t rows, int32_t K, const void* X, int64_t ldx,
               const uint8_t* codes, const uint8_t* scales, int64_t lds) {
    if (format != TMT_MOE_MX_FP4 && format != TMT_MOE_MX_FP8)
        return fail(TMT_MOE_EINVAL, "format=%d is neither TMT_MOE_MX_FP4 nor TMT_MOE_MX_FP8", format);
    if (dtype != TMT_MOE_BF16 && dtype != TMT_MOE_F32)
        return fail(TMT_MOE_EINVAL, "dtype=%d is neither TMT_MOE_BF16 nor TMT_MOE_F32", dtype);
    if (rows < 0) return fail(TMT_MOE_EINVAL, "rows=%d < 0", rows);
    if (K <= 0 || K % 32 != 0) return fail(TMT_MOE_EINVAL, "K=%d must be a positive multiple of 32", K);
    if (rows == 0) return TMT_MOE_OK;
    if ((int64_t)rows * ((K + 255LL) / 256 * 256) >= kMaxValues || mx_tiles(rows, K) >= kMaxValues / kMxTile)
        return fail(TMT_MOE_EINVAL, "rows=%d of K=%d, rounded up to whole tiles, are 2^36 values or more", rows, K);
    const int piece = dtype == TMT_MOE_BF16 ? 8 : 4;  // elements of 16 bytes
    if (ldx < K || ldx % piece != 0)
        return fail(TMT_MOE_EINVAL, "ldx=%lld must be a multiple of %d, at least K=%d", (long long)ldx, piece, K);
    if (lds < rows) return fail(TMT_MOE_EINVAL, "lds=%lld is less than rows=%d", (long long)lds, rows);
    if (!X || !codes || !scales) return fail(TMT_MOE_EINVAL, "X, codes and scales must be non-NULL");
    if (!aligned16(X) || !aligned16(codes)) return fail(TMT_MOE_EINVAL, "X and codes must be 16-byte aligned");
    return TMT_MOE_OK;
}

constexpr int32_t kMaxWidth = 1 << 22;             // N and K
constexpr int32_t kMaxTokens = 1 << 30;
constexpr int64_t kMaxOutputs = int64_t(1) << 40;  // of a product, so that 32 bits count the tiles

int check_shape(int32_t T, int32_t N, int32_t K) {
    if (T < 0) return fail(TMT_MOE_EINVAL, "T=%d < 0", T);
    if (N <= 0 || N % 16 != 0) return fail(TMT_MOE_EINVAL, "N=%d must be a positive multiple of 16", N);
    if (K <= 0 || K % 64 != 0) return fail(TMT_MOE_EINVAL, "K=%d must be a positive multiple of 64", K);
    if (N > kMaxWidth || K > kMaxWidth) return fail(TMT_MOE_EINVAL, "N=%d and K=%d must be at most %d", N, K, kMaxWidth);
    if ((int64_t)T * N > kMaxOutputs || (int64_t)T * K > kMaxOutputs || (int64_t)N * K > kMaxOutputs)
        return fail(TMT_MOE_EINVAL, "T=%d, N=%d, K=%d: T*N, T*K and N*K must be at most 2^40", T, N, K);
    if (T > kMaxTokens) return fail(TMT_MOE_EINVAL, "T=%d is over %d", T, kMaxTokens);
    return TMT_MOE_OK;
}

int check_matrix(const char* what, const void* p, int64_t ld, int width, int piece) {
    if (!p) return fail(TMT_MOE_EINVAL, "%s must be non-NULL", what);
    if (!aligned16(p)) return fail(TMT_MOE_EINVAL, "%s must be 16-byte aligned", what);
    if (ld < width || ld % piece != 0)
        return fail(TMT_MOE_EINVAL, "the row stride %lld of %s must be a multiple of %d, at least %d", (long long)ld,
                    what, piece, width);
    if (ld > kMaxStride) return fail(TMT_MOE_EINVAL, "the row stride %lld of %s is over %lld", (long long)ld, what, (long long)kMaxStride);
    return TMT_MOE_OK;
}

// Codes [rows][...] and scales [K/32][lds] of a product's operand.
int check_mx(const char* what, const uint8_t* codes, const uint8_t* scales, int64_t lds, int rows) {
    if (!codes || !scales) return fail(TMT_MOE_EINVAL, "codes and scales of %s must be non-NULL", what);
    if (!aligned16(codes) || !aligned16(scales))
        return fail(TMT_MOE_EINVAL, "codes and scales of %s must be 16-byte aligned", what);
    if (lds < rows || lds % 16 != 0)
        return fail(TMT_MOE_EINVAL, "the scale stride %lld of %s must be a multiple of 16, at least %d", (long long)lds,
                    what, rows);
    if (lds > kMaxScaleStride)
        return fail(TMT_MOE_EINVAL, "the scale stride %lld of %s is over %lld", (long long)lds, what, (long long)kMaxScaleStride);
    return TMT_MOE_OK;
}

int run(LinearOp op, LinearParams& p, void* workspace, size_t workspace_bytes, void* stream) {
    const size_t need = linear_workspace(op, p.T, p.N, p.K);
    if (need > 0) {
        if (!workspace || !aligned_to(workspace, 256))
            return fail(TMT_MOE_EINVAL, "workspace must be a 256-byte aligned device pointer");
        if (workspace_bytes < need)
            return fail(TMT_MOE_EINVAL, "workspace of %zu bytes is smaller than the %zu bytes needed", workspace_bytes, need);
    }
    p.part = static_cast<float*>(workspace);
    HIP_TRY(launch_linear(op, p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

}  // namespace

extern "C" {

int tmt_moe_mx_quantize(void* stream, int32_t format, int32_t dtype, const void* X, int64_t ldx, int32_t rows,
                        int32_t K, uint8_t* codes, uint8_t* scales, int64_t lds) {
    int rc = check_rows(format, dtype, rows, K, X, ldx, codes, scales, lds);
    if (rc || rows == 0) return rc;
    MxRowsParams p{};
    p.x = X; p.ldx = ldx; p.rows = rows; p.K = K; p.codes = codes; p.scales = scales; p.lds = lds;
    HIP_TRY(launch_mx_rows(true, format, dtype == TMT_MOE_F32, p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_mx_dequantize(void* stream, int32_t format, const uint8_t* codes, const uint8_t* scales, int64_t lds,
                          int32_t rows, int32_t K, int32_t dtype, void* X, int64_t ldx) {
    int rc = check_rows(format, dtype, rows, K, X, ldx, codes, scales, lds);
    if (rc || rows == 0) return rc;
    MxRowsParams p{};
    p.y = X; p.ldx = ldx; p.rows = rows; p.K = K; p.lds = lds;
    p.codes = const_cast<uint8_t*>(codes);
    p.scales = const_cast<uint8_t*>(scales);
    HIP_TRY(launch_mx_rows(false, format, dtype == TMT_MOE_F32, p, (hipStream_t)stream));
    return TMT_MOE_OK;
}

int tmt_moe_linear_workspace_size(int32_t op, int32_t T, int32_t N, int32_t K, size_t* bytes) {
    if (op < TMT_MOE_LINEAR_FORWARD || op > TMT_MOE_LINEAR_DW) return fail(TMT_MOE_EINVAL, "op=%d is no TMT_MOE_LINEAR_* operator", op);
    int rc = check_shape(T, N, K);
    if (rc) return rc;
    if (!bytes) return fail(TMT_MOE_EINVAL, "bytes is NULL");
    *bytes = linear_workspace((LinearOp)op, T, N, K);
    return TMT_MOE_OK;
}

int tmt_moe_mxfp4_linear(void* stream, int32_t T, int32_t N, int32_t K, const uint16_t* X, int64_t ldx,
                         const uint8_t* W, const uint8_t* W_scale, int64_t ldws, uint16_t* Y, int64_t ldy,
                         float beta, void* workspace, size_t workspace_bytes) {
    int rc = check_shape(T, N, K);
    if (rc || T == 0) return rc;
    if ((rc = check_matrix("X", X, ldx, K, 8)) || (rc = check_mx("W", W, W_scale, ldws, N)) ||
        (rc = check_matrix("Y", Y, ldy, N, 8)))
        return rc;
    LinearParams p{};
    p.T = T; p.N = N; p.K = K; p.x = X; p.ldx = ldx; p.w = W; p.ws = W_scale; p.wlds = ldws;
    p.y = Y; p.ldy = ldy; p.beta = beta;
    return run(LINEAR_FORWARD, p, workspace, workspace_bytes, stream);
}

int tmt_moe_mxfp4_matmul(void* stream, int32_t T, int32_t N, int32_t K, const uint8_t* X, const uint8_t* X_scale,
                         int64_t ldxs, const uint8_t* W, const uint8_t* W_scale, int64_t ldws, uint16_t* Y,
                         int64_t ldy, float beta, void* workspace, size_t workspace_bytes) {
    int rc = check_shape(T, N, K);
    if (rc || T == 0) return rc;
    if ((rc = check_mx("X", X, X_scale, ldxs, T)) || (rc = check_mx("W", W, W_scale, ldws, N)) ||
        (rc = check_matrix("Y", Y, ldy, N, 8)))
        return rc;
    LinearParams p{};
    p.T = T; p.N = N; p.K = K; p.xq = X; p.xs = X_scale; p.xlds = ldxs; p.w = W; p.ws = W_scale; p.wlds = ldws;
    p.y = Y; p.ldy = ldy; p.beta = beta;
    return run(LINEAR_MATMUL, p, workspace, workspace_bytes, stream);
}

int tmt_moe_mxfp4_linear_dx(void* stream, int32_t T, int32_t N, int32_t K, const uint16_t* dY, int64_t lddy,
                            const uint8_t* W, const uint8_t* W_scale, int64_t ldws, uint16_t* dX, int64_t lddx,
                            float beta, void* workspace, size_t workspace_bytes) {
    int rc = check_shape(T, N, K);
    if (rc || T == 0) return rc;
    if ((rc = check_matrix("dY", dY, lddy, N, 8)) || (rc = check_mx("W", W, W_scale, ldws, N)) ||
        (rc = check_matrix("dX", dX, lddx, K, 8)))
        return rc;
    LinearParams p{};
    p.T = T; p.N = N; p.K = K; p.x = dY; p.ldx = lddy; p.w = W; p.ws = W_scale; p.wlds = ldws;
    p.y = dX; p.ldy = lddx; p.beta = beta;
    return run(LINEAR_DX, p, workspace, workspace_bytes, stream);
}

int tmt_moe_mxfp8_linear_dw(void* stream, int32_t T, int32_t N, int32_t K, const uint16_t* dY, int64_t lddy,
                            const uint8_t* X, const uint8_t* X_scale, int64_t ldxs, float* dW, int64_t lddw,
                            float beta, void* workspace, size_t workspace_bytes) {
    int rc = check_shape(T, N, K);
    if (rc) return rc;
    if (T > 0 && ((rc = check_matrix("dY", dY, lddy, N, 8)) || (rc = check_mx("X", X, X_scale, ldxs, T)))) return rc;
    if ((rc = check_matrix("dW", dW, lddw, K, 4))) return rc;
    LinearParams p{};
    p.T = T; p.N = N; p.K = K; p.x = dY; p.ldx = lddy; p.w = X; p.ws = X_scale; p.wlds = ldxs;
    p.y = dW; p.ldy = lddw; p.beta = beta;
    return run(LINEAR_DW, p, workspace, workspace_bytes, stream);
}

}  // extern "C"
