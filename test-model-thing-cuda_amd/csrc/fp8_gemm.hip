// fp8_gemm.hip -- products of the 8-bit linear layer.
//
//   y[m][n] = beta y + sum_b sa[b][m] sb(b, n) sum_{k in b} a[m][k] b[n][k]
//
// over blocks b of 128 of the reduction: a[m] in rows (a scale for each row and
// block), b[n] in rows or in tiles (a scale for 128 rows and a block). A block's
// sum is formed by the matrix instructions, multiplied by its fp32 scales and added
// to the fp32 result in the vector unit.
//
// The 8-bit matrix instructions align the products of 8 neighbouring codes to the
// largest of them and keep 13 bits below its exponent; sums of such groups are in
// fp32 (measured with single products next to large ones that cancel; the same in
// all four forms of the instruction). On normal data a block's sum is 1.5e-5 off in
// norm, 2^-16, nothing next to a bf16 result's rounding (2^-9), but 20 times what
// fp32 sums lose. So
//   bf16 results  take v_mfma_f32_32x32x64_f8f6f4 (16x16x128 for few rows) on the
//                 codes as they are, and
//   fp32 results  take the bf16 instructions, in which every code is exact and
//                 the sums are fp32's, at half the rate: the codes are converted
//                 in registers.
//
// b is the first operand of the matrix instruction and a the second, so that a
// lane's values belong to one row m, whose scale it holds, and to neighbouring
// columns n. The instruction's order of the reduction does not matter as long as
// both operands are laid out alike.
#include "fp8.hpp"
#include "fp8_format.hpp"
#include "moe_internal.hpp"
#include "tile_stream.hpp"

namespace tmt {
namespace {

__device__ __forceinline__ i32x8 join(uint4 a, uint4 b) {
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// 8 codes as bf16, exact.
__device__ __forceinline__ bf16x8 widen(int lo, int hi) {
    return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))));
}
// 16 x 16 sums over a block of 128.
template <bool WIDE>
__device__ __forceinline__ f32x4 mma16(i32x8 b, i32x8 a) {
    f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (WIDE) {
#pragma unroll
        for (int q = 0; q < 8; q += 2)
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(b[q], b[q + 1]), widen(a[q], a[q + 1]), d, 0, 0, 0);
        return d;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, d, 0, 0, 0, 0, 0, 0);
    }
}

// ---- few rows ----------------------------------------------------------------------
// A workgroup takes 16 NB columns and 16 RB rows of y; its NW waves deal out the
// reduction in blocks of 128. Lane l loads chunks l / 16 and l / 16 + 4 (16 codes
// each) of row l % 16 of a block straight into registers, of both operands. The
// waves' sums meet in LDS and are added in wave order.
template <bool TILES, bool F32, int RB, int NB, int NW>
__global__ __launch_bounds__(64 * NW) void fp8_rows_kernel(Fp8Params p) {
    constexpr int OUT = 256 * RB * NB;
    __shared__ float red[NW * OUT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, g = lane >> 4;
    const int nb = (p.N + 16 * NB - 1) / (16 * NB);  // blocks of columns, which run fastest
    const int n0 = (int)(blockIdx.x % nb) * 16 * NB, m0 = (int)(blockIdx.x / nb) * 16 * RB;
    const int blocks = (p.K + kFp8Block - 1) / kFp8Block;
    f32x4 acc[RB][NB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[r][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto chunk = [&](const uint8_t* codes, int k) {
        return k < p.K ? *reinterpret_cast<const uint4*>(codes + k) : make_uint4(0, 0, 0, 0);
    };
    for (int kb = wave; kb < blocks; kb += NW) {
        const int k = kb * kFp8Block + 16 * g;
        i32x8 b[NB], a[RB];
        f32x4 sb[NB];
        float sa[RB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint8_t* q = p.b + (int64_t)min(n0 + 16 * i + row, p.N - 1) * p.ldb;
            b[i] = join(chunk(q, k), chunk(q, k + 64));
            if constexpr (TILES) {
                const float s = p.bs[(int64_t)(min(n0 + 16 * i, p.N - 1) / kFp8Block) * p.ldbs + kb];
                sb[i] = f32x4{s, s, s, s};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) sb[i][e] = p.bs[(int64_t)kb * p.ldbs + min(n0 + 16 * i + 4 * g + e, p.N - 1)];
            }
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const int m = min(m0 + 16 * r + row, p.M - 1);
            const uint8_t* q = p.a + (int64_t)m * p.lda;
            a[r] = join(chunk(q, k), chunk(q, k + 64));
            sa[r] = p.as[(int64_t)kb * p.ldas + m];
        }
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int i = 0; i < NB; ++i) acc[r][i] += mma16<F32>(b[i], a[r]) * (sb[i] * sa[r]);
    }
    // acc[r][i][e]: row 16 r + lane % 16, column 16 i + 4 (lane / 16) + e
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < NB; ++i)
            *reinterpret_cast<f32x4*>(red + wave * OUT + (16 * r + row) * (16 * NB) + 16 * i + 4 * g) = acc[r][i];
    __syncthreads();
    for (int o = threadIdx.x * 2; o < OUT; o += 128 * NW) {
        const int m = m0 + o / (16 * NB), n = n0 + o % (16 * NB);
        if (m >= p.M || n >= p.N) continue;
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            v[0] += red[w * OUT + o];
            v[1] += red[w * OUT + o + 1];
        }
        if constexpr (F32) {
            float2* y = reinterpret_cast<float2*>(static_cast<float*>(p.y) + (int64_t)m * p.ldy + n);
            if (p.beta != 0.0f) {
                const float2 old = *y;
                v[0] += p.beta * old.x;
                v[1] += p.beta * old.y;
            }
            *y = make_float2(v[0], v[1]);
        } else {
            uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.y) + (int64_t)m * p.ldy + n);
            if (p.beta != 0.0f) {
                const uint32_t old = *y;
                v[0] += p.beta * bf_lo(old);
                v[1] += p.beta * bf_hi(old);
            }
            *y = pack_bf2(v[0], v[1]);
        }
    }
}

template <bool TILES, bool F32>
void launch_rows(const Fp8Params& p, hipStream_t s) {
    const int64_t grid = (int64_t)((p.N + 31) / 32) * ((p.M + 31) / 32);
    fp8_rows_kernel<TILES, F32, 2, 2, 4><<<(unsigned)grid, 256, 0, s>>>(p);
}

}  // namespace

size_t fp8_workspace(bool tiles, int M, int N, int K) { return 0; }

hipError_t launch_fp8_matmul(bool tiles, bool f32, const Fp8Params& p, hipStream_t s) {
    if (tiles) f32 ? launch_rows<true, true>(p, s) : launch_rows<true, false>(p, s);
    else f32 ? launch_rows<false, true>(p, s) : launch_rows<false, false>(p, s);
    return hipGetLastError();
}

}  // namespace tmt
