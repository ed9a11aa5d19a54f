// fp8.hpp -- declarations of the 8-bit linear layer's kernels (fp8_quant.hip,
// fp8_gemm.hip) and of the norm in front of it (rmsnorm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmt {

constexpr int kFp8Block = 128;  // values that share one scale (a side of a tile)

// ---- norm ------------------------------------------------------------------
constexpr int kRmsMaxWidth = 16384;
struct RmsParams {
    int T, d;
    bool f32;             // R, S, dR and dS are fp32 (else bf16)
    const uint16_t* X;    // [T][ldx] bf16, or nullptr
    int64_t ldx;
    const void* R;        // [T][ldr], or nullptr
    int64_t ldr;
    const float* gamma;   // [d]
    float eps;
    void* S;              // [T][lds]: forward's output or nullptr; backward's input
    int64_t lds;
    uint16_t* Y;          // [T][ldy] bf16, or nullptr
    int64_t ldy;
    uint8_t* codes;       // [T][ldc], or nullptr
    int64_t ldc;
    float* scales;        // [ceil(d / 128)][ldsc]
    int64_t ldsc;
    float* rstd;          // [T]: forward's output or nullptr; backward's input
    // backward
    const uint16_t* dY;   // [T][lddy] bf16
    int64_t lddy;
    const void* dR;       // [T][lddr], or nullptr
    int64_t lddr;
    void* dS;             // [T][ldds]
    int64_t ldds;
    float* dgamma;        // [d]
    float* partial;       // workspace: [rms_partials][d rounded up to 4]
};
// The most workgroups of the backward, each of which leaves one row of partial dgamma.
int rms_partials_max(int d, int cus);
// Arguments as the C ABI has checked them, T > 0.
hipError_t launch_rms_fwd(const RmsParams& p, hipStream_t s);
hipError_t launch_rms_bwd(const RmsParams& p, hipStream_t s);

// ---- quantisation -------------------------------------------------------------
struct Fp8QuantParams {
    const void* x;        // [rows][ldx] bf16 or fp32
    int64_t ldx;
    int rows, K;
    uint8_t* codes;       // [rows][ldc], or nullptr
    int64_t ldc;
    float* scales;        // rows: [ceil(K / 128)][lds]; tiles: [ceil(rows / 128)][lds]
    int64_t lds;
    uint8_t* codes_t;     // [K][ldct], or nullptr
    int64_t ldct;
    float* scales_t;      // rows: [ceil(rows / 128)][ldst]; tiles: [ceil(K / 128)][ldst]
    int64_t ldst;
};
// Arguments as the C ABI has checked them, rows and K > 0.
hipError_t launch_fp8_quantize(bool tiles, bool f32, const Fp8QuantParams& p, hipStream_t s);

// codes [rows][ldc], of any alignment, to codes_t [K][ldct], zeros up to a multiple of 16.
hipError_t launch_fp8_transpose(const uint8_t* codes, int64_t ldc, int rows, int K, uint8_t* codes_t, int64_t ldct, hipStream_t s);

// ---- products --------------------------------------------------------------------
// y[m][n] = beta y + sum over blocks b of a_scale[b][m] b_scale(b, n) sum_{k in b} a[m][k] b[n][k]
struct Fp8Params {
    int M, N, K;
    const uint8_t* a;     // codes [M][lda]
    int64_t lda;
    const float* as;      // [ceil(K / 128)][ldas]
    int64_t ldas;
    const uint8_t* b;     // codes [N][ldb]
    int64_t ldb;
    const float* bs;      // rows: [ceil(K / 128)][ldbs]; tiles: [ceil(N / 128)][ldbs]
    int64_t ldbs;
    void* y;              // [M][ldy] bf16 or fp32
    int64_t ldy;
    float beta;
    float* part;          // workspace: split reductions' partial sums
};
size_t fp8_workspace(int M, int N, int K);
// Arguments as the C ABI has checked them, M and N > 0, K >= 0.
hipError_t launch_fp8_matmul(bool tiles, bool f32, const Fp8Params& p, hipStream_t s);

}  // namespace tmt
