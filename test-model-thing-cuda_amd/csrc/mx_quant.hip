// mx_quant.hip -- rows of bf16 or fp32 to microscaled codes and back.
//
// codes [rows][K/2] (MXFP4, low nibble = even column) or [rows][K] (MXFP8);
// scales [K/32][lds], block-major, as the expert GEMMs read them. Per block b
// of row r: s = mx_scale(max |x|), code = RNE(x / 2^(s - 127)). The division
// is a product with a power of two and the rounding one conversion
// instruction, so codes are exact: no statistics, no other rounding.
//
// Bound by memory: 2 or 4 bytes a value read, 1/2 or 1 written, and the
// scales. Eight values per lane make 16-byte (bf16) loads, four lanes own a
// block and find its maximum in two DPP steps. A workgroup takes 4096 values as
// a tile of 256, 128 or 64 columns (the widest that K fills), so the scales of a
// tile leave as runs of 16 bytes or more through LDS instead of one scattered
// byte a block. Small tiles keep every CU busy (quantisation and back, us with
// 2048 / 4096 / 8192 / 16384 values a workgroup: 4096 x 1024 fp32 to MXFP4 12.1 /
// 11.9 / 11.6 / 15.8; 32768 x 1024 bf16 to MXFP8 43.5 / 41.7 / 44.8 / 46.5, which
// moves 204 MB, 4.9 TB/s). fp32 values come back slower than they go: a lane's
// eight leave as two 16-byte stores, so that a wave's store writes every second
// 16 bytes (32768 x 1024, MXFP4: quantised in 29 us, 5.3 TB/s, back in 38, 4.0).
#include "linear.hpp"
#include "moe_internal.hpp"
#include "mx_format.hpp"

namespace tmt {
namespace {

constexpr int kPieces = 2;                        // pieces of 8 values per lane
constexpr int kTile = kPieces * 8 * kThreads;     // values per workgroup
static_assert(kTile == kMxTile, "the launch's tiles are the kernels'");

__device__ __forceinline__ void load8(const void* x, bool f32, int64_t at, float* f) {
    if (f32) {
        const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = a[i], f[i + 4] = b[i];
    } else {
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at), f);
    }
}

template <int FMT, bool F32>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(MxRowsParams p) {
    __shared__ uint8_t sc[kTile / 32];  // [column block][row]
    const int lg = mx_tile_log2_cols(p.K), rt = kTile >> lg, lanes = 1 << (lg - 3);  // pieces per row
    const int tc = mx_tiles_per_row(p.K);
    const int64_t r0 = (int64_t)(blockIdx.x / tc) * rt;
    const int c0 = (int)(blockIdx.x % tc) << lg;
    const int pc = threadIdx.x & (lanes - 1), pr = threadIdx.x >> (lg - 3);
    const int col = c0 + pc * 8;
    float f[kPieces][8];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int64_t r = r0 + pr + i * (kThreads >> (lg - 3));
        if (r < p.rows && col < p.K) load8(p.x, F32, r * p.ldx + col, f[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int row = pr + i * (kThreads >> (lg - 3));
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[i][j]) & 0x7fffffffu);
        m = max(m, xor_lane_u32<1>(m));
        m = max(m, xor_lane_u32<2>(m));
        const uint32_t s = mx_scale<FMT>(m);
        if ((threadIdx.x & 3) == 0) sc[(pc >> 2) * rt + row] = (uint8_t)s;
        const float inv = mx_inverse(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = s == 255 ? 0.0f : f[i][j] * inv;  // a block that is NaN: codes of 0
        const int64_t r = r0 + row;
        if (r < p.rows && col < p.K) {
            if constexpr (FMT == MX_FP4)
                *reinterpret_cast<uint32_t*>(p.codes + r * (p.K / 2) + col / 2) = to_e2m1(f[i]);
            else
                *reinterpret_cast<uint2*>(p.codes + r * p.K + col) = make_uint2(to_e4m3(f[i]), to_e4m3(f[i] + 4));
        }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < kTile / 32; q += kThreads) {
        const int b = q / rt, row = q % rt;
        const int64_t r = r0 + row;
        if (r < p.rows && c0 / 32 + b < p.K / 32) p.scales[(int64_t)(c0 / 32 + b) * p.lds + r] = sc[q];
    }
}

template <int FMT, bool F32>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(MxRowsParams p) {
    __shared__ uint8_t sc[kTile / 32];
    const int lg = mx_tile_log2_cols(p.K), rt = kTile >> lg, lanes = 1 << (lg - 3);
    const int tc = mx_tiles_per_row(p.K);
    const int64_t r0 = (int64_t)(blockIdx.x / tc) * rt;
    const int c0 = (int)(blockIdx.x % tc) << lg;
    const int pc = threadIdx.x & (lanes - 1), pr = threadIdx.x >> (lg - 3);
    const int col = c0 + pc * 8;
    uint2 q[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int64_t r = r0 + pr + i * (kThreads >> (lg - 3));
        q[i] = make_uint2(0, 0);
        if (r < p.rows && col < p.K) {
            if constexpr (FMT == MX_FP4) q[i].x = *reinterpret_cast<const uint32_t*>(p.codes + r * (p.K / 2) + col / 2);
            else q[i] = *reinterpret_cast<const uint2*>(p.codes + r * p.K + col);
        }
    }
    for (int k = threadIdx.x; k < kTile / 32; k += kThreads) {
        const int b = k / rt, row = k % rt;
        const int64_t r = r0 + row;
        sc[k] = r < p.rows && c0 / 32 + b < p.K / 32 ? p.scales[(int64_t)(c0 / 32 + b) * p.lds + r] : 127;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int row = pr + i * (kThreads >> (lg - 3));
        const int64_t r = r0 + row;
        if (r >= p.rows || col >= p.K) continue;
        const float unit = e8m0_value(sc[(pc >> 2) * rt + row]);
        float v[8];
        if constexpr (FMT == MX_FP4) {
            from_e2m1(q[i].x, v);
        } else {
            from_e4m3(q[i].x, v);
            from_e4m3(q[i].y, v + 4);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= unit;
        if constexpr (F32) {
            f32x4* o = reinterpret_cast<f32x4*>(static_cast<float*>(p.y) + r * p.ldx + col);
            o[0] = f32x4{v[0], v[1], v[2], v[3]};
            o[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + r * p.ldx + col) = pack8(v);
        }
    }
}

}  // namespace

hipError_t launch_mx_rows(bool quantize, int format, bool f32, const MxRowsParams& p, hipStream_t s) {
    const unsigned g = (unsigned)mx_tiles(p.rows, p.K);
#define TMT_MX(FMT_, F32_)                                                        \
    (quantize ? mx_quantize_kernel<FMT_, F32_><<<g, kThreads, 0, s>>>(p)          \
              : mx_dequantize_kernel<FMT_, F32_><<<g, kThreads, 0, s>>>(p))
    if (format == MX_FP4) f32 ? TMT_MX(MX_FP4, true) : TMT_MX(MX_FP4, false);
    else f32 ? TMT_MX(MX_FP8, true) : TMT_MX(MX_FP8, false);
#undef TMT_MX
    return hipGetLastError();
}

}  // namespace tmt
