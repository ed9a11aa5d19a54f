// linear.hpp -- declarations of the microscaled linear layer's kernels
// (mx_quant.hip, linear.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmt {

struct MxRowsParams {
    const void* x;    // quantisation: bf16 or fp32 rows
    void* y;          // dequantisation: bf16 or fp32 rows
    int64_t ldx;      // their stride in elements
    int rows, K;      // K a multiple of 32
    uint8_t* codes;   // [rows][K/2] or [rows][K]
    uint8_t* scales;  // [K/32][lds]
    int64_t lds;
};
// Their launch: tiles of kMxTile values, as wide as K fills, a workgroup each.
constexpr int kMxTile = 4096;
__host__ __device__ inline int mx_tile_log2_cols(int K) { return K >= 256 ? 8 : K >= 128 ? 7 : 6; }
__host__ __device__ inline int mx_tiles_per_row(int K) {
    const int lg = mx_tile_log2_cols(K);
    return (int)(((uint32_t)K + (1u << lg) - 1) >> lg);  // K + 255 may pass 31 bits
}
inline int64_t mx_tiles(int rows, int K) {
    const int rt = kMxTile >> mx_tile_log2_cols(K);
    return ((int64_t)rows + rt - 1) / rt * mx_tiles_per_row(K);
}
// Arguments as the C ABI has checked them, rows > 0.
hipError_t launch_mx_rows(bool quantize, int format, bool f32, const MxRowsParams& p, hipStream_t s);

// The products. M output rows, C output columns, R the reduction length:
//   FORWARD  y[t][n] = x[t] . w[n]          M = T, C = N, R = K
//   MATMUL   the same with x in MXFP4
//   DX       y[t][k] = sum_n x[t][n] w[n][k]   M = T, C = K, R = N
//   DW       y[n][k] = sum_t x[t][n] w[t][k]   M = N, C = K, R = T; w in MXFP8, y fp32
// The kernels' offsets inside a tile are 32-bit.
constexpr int64_t kMaxStride = int64_t(1) << 22;   // elements between rows
constexpr int64_t kMaxScaleStride = int64_t(1) << 27;
enum LinearOp { LINEAR_FORWARD = 0, LINEAR_MATMUL = 1, LINEAR_DX = 2, LINEAR_DW = 3 };
struct LinearParams {
    int T, N, K;
    const uint16_t* x;    // bf16 operand: X [T][ldx], or dY [T][ldx]
    int64_t ldx;
    const uint8_t* xq;    // MATMUL: codes [T][K/2] and scales [K/32][xlds] of X
    const uint8_t* xs;
    int64_t xlds;
    const uint8_t* w;     // codes [N][K/2], or [T][K] (DW)
    const uint8_t* ws;    // scales [K/32][wlds]
    int64_t wlds;
    void* y;              // bf16 [T][ldy], fp32 [N][ldy] (DW)
    int64_t ldy;
    float beta;
    float* part;          // workspace: split reductions' partial sums
};
size_t linear_workspace(LinearOp op, int T, int N, int K);
// Arguments as the C ABI has checked them; T == 0 for DW only.
hipError_t launch_linear(LinearOp op, const LinearParams& p, hipStream_t s);

}  // namespace tmt
