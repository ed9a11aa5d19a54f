// linear.hip -- products of the linear layer on microscaled numbers.
//
// Every operand value is exact in bf16 (an e2m1 code has two significant
// bits, an e4m3 code four, and scales are powers of two), so each product is
// one bf16 matrix product with fp32 sums of exact terms.
#include "linear.hpp"
#include "moe_internal.hpp"
#include "mx_format.hpp"

namespace tmt {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint16_t fp4_at(const uint8_t* codes, const uint8_t* scales, int64_t lds, int K, int64_t row, int k) {
    const uint32_t q = (codes[row * (K / 2) + k / 2] >> (4 * (k & 1))) & 15;
    float v[8];
    from_e2m1(q, v);
    return f2bf(v[0] * e8m0_value(scales[(k / 32) * lds + row]));
}

constexpr int BT = 64, BK = 32, LD = BK + 8;

// 64 x 64 outputs per workgroup, a wave each 32 x 32; both operands staged
// K-contiguous in LDS, element by element.
template <int OP>
__global__ __launch_bounds__(256) void linear_simple_kernel(LinearParams p, int M, int C, int R, int tiles_c) {
    __shared__ __align__(16) uint16_t as[BT * LD], bs[BT * LD];
    const int m0 = (int)(blockIdx.x / tiles_c) * BT, c0 = (int)(blockIdx.x % tiles_c) * BT;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * 32, wc = (wave & 1) * 32;
    f32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    for (int k0 = 0; k0 < R; k0 += BK) {
#pragma unroll
        for (int i = 0; i < BT * BK / 256; ++i) {
            const int q = tid + 256 * i;
            // neighbouring lanes along the operand's contiguous direction
            const bool kc = OP != LINEAR_DW;
            const int r = kc ? q / BK : q % BT, k = kc ? q % BK : q / BT;
            const int m = m0 + r, kk = k0 + k;
            uint16_t v = 0;
            if (m < M && kk < R) {
                if constexpr (OP == LINEAR_MATMUL) v = fp4_at(p.xq, p.xs, p.xlds, p.K, m, kk);
                else if constexpr (OP == LINEAR_DW) v = p.x[(int64_t)kk * p.ldx + m];
                else v = p.x[(int64_t)m * p.ldx + kk];
            }
            as[r * LD + k] = v;
            const bool bkc = OP == LINEAR_FORWARD || OP == LINEAR_MATMUL;
            const int br = bkc ? q / BK : q % BT, bk = bkc ? q % BK : q / BT;
            const int c = c0 + br, kb = k0 + bk;
            v = 0;
            if (c < C && kb < R) {
                if constexpr (OP == LINEAR_DW) {
                    float f[4];
                    from_e4m3(p.w[(int64_t)kb * p.K + c], f);
                    v = f2bf(f[0] * e8m0_value(p.ws[(c / 32) * p.wlds + kb]));
                } else if constexpr (OP == LINEAR_DX) {
                    v = fp4_at(p.w, p.ws, p.wlds, p.K, kb, c);
                } else {
                    v = fp4_at(p.w, p.ws, p.wlds, p.K, c, kb);
                }
            }
            bs[br * LD + bk] = v;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            const int k = 16 * s + 8 * (lane >> 5);
            const uint4 a = *reinterpret_cast<const uint4*>(as + (wm + (lane & 31)) * LD + k);
            const uint4 b = *reinterpret_cast<const uint4*>(bs + (wc + (lane & 31)) * LD + k);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
        }
        __syncthreads();
    }
    const int m = m0 + wm + (lane & 31);
    if (m >= M) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int c = c0 + wc + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (c >= C) continue;
        const int64_t at = (int64_t)m * p.ldy + c;
        if constexpr (OP == LINEAR_DW) {
            float* y = static_cast<float*>(p.y) + at;
            *y = p.beta != 0.0f ? p.beta * *y + acc[r] : acc[r];
        } else {
            uint16_t* y = static_cast<uint16_t*>(p.y) + at;
            *y = f2bf(p.beta != 0.0f ? p.beta * bf1(*y) + acc[r] : acc[r]);
        }
    }
}

}  // namespace

size_t linear_workspace(LinearOp, int, int, int) { return 0; }

hipError_t launch_linear(LinearOp op, const LinearParams& p, hipStream_t s) {
    const int M = op == LINEAR_DW ? p.N : p.T, C = op == LINEAR_FORWARD || op == LINEAR_MATMUL ? p.N : p.K;
    const int R = op == LINEAR_DW ? p.T : op == LINEAR_DX ? p.N : p.K;
    if (M <= 0 || C <= 0) return hipSuccess;
    const int tc = (C + BT - 1) / BT;
    const int64_t grid = (int64_t)((M + BT - 1) / BT) * tc;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    const unsigned g = (unsigned)grid;
    switch (op) {
        case LINEAR_FORWARD: linear_simple_kernel<LINEAR_FORWARD><<<g, 256, 0, s>>>(p, M, C, R, tc); break;
        case LINEAR_MATMUL: linear_simple_kernel<LINEAR_MATMUL><<<g, 256, 0, s>>>(p, M, C, R, tc); break;
        case LINEAR_DX: linear_simple_kernel<LINEAR_DX><<<g, 256, 0, s>>>(p, M, C, R, tc); break;
        case LINEAR_DW: linear_simple_kernel<LINEAR_DW><<<g, 256, 0, s>>>(p, M, C, R, tc); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace tmt
