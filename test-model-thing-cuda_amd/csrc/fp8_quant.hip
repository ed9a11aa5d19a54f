// fp8_quant.hip -- a matrix of bf16 or fp32 to e4m3 codes with one fp32 scale
// for every 128 values, in its own order, transposed, or both in one pass.
//
//   rows   blocks of 1 x 128: scales of X's rows, and of the rows of X^T
//          (columns of X in blocks of 128 rows);
//   tiles  blocks of 128 x 128, the same both ways.
//
// Bound by memory: 2 or 4 bytes a value read, one written a side. A workgroup
// owns a tile of 128 x 128 values, held in registers, 8 columns a piece, so that
// the input is read once for both sides. A row's block is found in 16 lanes by
// DPP, a column's through the waves' maxima in LDS. Codes of X leave straight from
// the registers (128 bytes a row and tile). Codes of X^T go through LDS: a thread
// holds the same columns of 4 neighbouring rows, so that a dword holds 4 codes of
// a column, and the dwords of a column are XOR-swizzled.
#include "fp8.hpp"
#include "fp8_format.hpp"
#include "moe_internal.hpp"

namespace tmt {
namespace {

constexpr int kTile = kFp8Block;
// 512 threads of 4 pieces, whose loads are all in flight at once (32768 x 4096 bf16, rows
// both ways: 117 us; 256 threads of 8 127).
constexpr int kThreads8 = 512;

// Pieces of 8 columns a thread: of rows 4 (t / 16) .. + 3 of each 64.
template <int THREADS>
struct Quant {
    static constexpr int P = kTile * 16 / THREADS;    // pieces
    static constexpr int SPAN = THREADS / 4;          // rows of 4 pieces
    static constexpr int WAVES = THREADS / 64;
};

template <bool TILES, bool F32, int PASS>
__global__ __launch_bounds__(kThreads8) void fp8_quantize_kernel(Fp8QuantParams p, int tiles_k) {
    constexpr int THREADS = kThreads8;
    using Q = Quant<THREADS>;
    __shared__ uint32_t most[Q::WAVES][kTile];        // largest magnitudes: a wave's columns, or [wave][0]
    __shared__ float row_scale[kTile];
    __shared__ uint4 codes_t[kTile * kTile / 16];     // [column][row]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int a = tid & 15, c0 = (int)(blockIdx.x % tiles_k) * kTile;
    const int64_t r0 = (int64_t)(blockIdx.x / tiles_k) * kTile;
    const int rows = (int)min((int64_t)kTile, p.rows - r0), cols = min(kTile, p.K - c0);
    auto row_of = [&](int i) { return (i >> 2) * Q::SPAN + (tid >> 4) * 4 + (i & 3); };

    float v[Q::P][8];
#pragma unroll
    for (int i = 0; i < Q::P; ++i) {
        const int row = row_of(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row >= rows || 8 * a >= cols) continue;
        const int64_t at = (r0 + row) * p.ldx + c0 + 8 * a;
        if (8 * a + 8 <= cols) {
            if constexpr (F32) {
                const float* x = static_cast<const float*>(p.x) + at;
                const f32x4 lo = get<PASS, f32x4>(x), hi = get<PASS, f32x4>(x + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = lo[j], v[i][j + 4] = hi[j];
            } else {
                unpack8(__builtin_bit_cast(uint4, get<PASS, u32x4_t>(static_cast<const uint16_t*>(p.x) + at)), v[i]);
            }
        } else {  // a row's last columns, one by one
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * a + j < cols) v[i][j] = F32 ? static_cast<const float*>(p.x)[at + j] : bf1(static_cast<const uint16_t*>(p.x)[at + j]);
        }
    }

    // largest magnitudes
    if constexpr (TILES) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < Q::P; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
        m = max(m, xor_lane_u32<1>(m));
        m = max(m, xor_lane_u32<2>(m));
        m = max(m, xor_lane_u32<4>(m));
        m = max(m, xor_lane_u32<8>(m));
        m = max(m, xor_lane_u32<16>(m));
        m = max(m, xor_lane_u32<32>(m));
        if (lane == 0) most[wave][0] = m;
    } else if (p.codes_t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < Q::P; ++i) m = max(m, abs_bits(v[i][j]));
            m = max(m, xor_lane_u32<16>(m));
            m = max(m, xor_lane_u32<32>(m));
            if (lane < 16) most[wave][8 * a + j] = m;
        }
    }
    if (TILES || p.codes_t) __syncthreads();
    Fp8Scale tile{};
    if constexpr (TILES) {
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < Q::WAVES; ++w) m = max(m, most[w][0]);
        tile = fp8_scale(m);
        if (tid == 0) {
            const int64_t rb = r0 / kTile, kb = c0 / kTile;
            if (p.codes) p.scales[rb * p.lds + kb] = tile.scale;
            if (p.codes_t) p.scales_t[kb * p.ldst + rb] = tile.scale;
        }
    }

    // in X's order
    if (p.codes) {
        const int width = min(kTile, ((p.K + 15) & ~15) - c0);  // up to the 16 bytes' end: zeros
#pragma unroll
        for (int i = 0; i < Q::P; ++i) {
            const int row = row_of(i);
            Fp8Scale q = tile;
            if constexpr (!TILES) {
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
                m = max(m, xor_lane_u32<1>(m));
                m = max(m, xor_lane_u32<2>(m));
                m = max(m, xor_lane_u32<4>(m));
                m = max(m, xor_lane_u32<8>(m));
                q = fp8_scale(m);
                if (a == 0) row_scale[row] = q.scale;
            }
            if (row < rows && 8 * a < width)
                put<PASS>(p.codes + (r0 + row) * p.ldc + c0 + 8 * a, u32x2_t{fp8_codes(v[i], q.inv), fp8_codes(v[i] + 4, q.inv)});
        }
    }

    // transposed
    if (p.codes_t) {
        uint8_t* ct = reinterpret_cast<uint8_t*>(codes_t);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            Fp8Scale q = tile;
            const int col = 8 * a + j;
            if constexpr (!TILES) {
                uint32_t m = 0;
#pragma unroll
                for (int w = 0; w < Q::WAVES; ++w) m = max(m, most[w][col]);
                q = fp8_scale(m);
                if (tid < 16 && col < cols) p.scales_t[r0 / kTile * p.ldst + c0 + col] = q.scale;
            }
#pragma unroll
            for (int h = 0; h < Q::P; h += 4) {
                const float f[4] = {v[h][j], v[h + 1][j], v[h + 2][j], v[h + 3][j]};
                const int dword = (h >> 2) * (Q::SPAN / 4) + (tid >> 4);
                *reinterpret_cast<uint32_t*>(ct + col * kTile + ((dword ^ ((a & 7) * 4)) * 4)) = fp8_codes(f, q.inv);
            }
        }
    }
    __syncthreads();
    if (!TILES && p.codes)
        for (int i = tid; i < rows; i += THREADS) p.scales[(int64_t)(c0 / kTile) * p.lds + r0 + i] = row_scale[i];
    if (p.codes_t) {
        const uint8_t* ct = reinterpret_cast<const uint8_t*>(codes_t);
        const int height = (int)min((int64_t)kTile, ((p.rows + 15LL) & ~15LL) - r0);
#pragma unroll
        for (int i = 0; i < kTile * 8 / THREADS; ++i) {
            const int col = i * (THREADS / 8) + tid / 8, chunk = tid & 7;
            if (col < cols && 16 * chunk < height)
                put<PASS>(p.codes_t + (int64_t)(c0 + col) * p.ldct + r0 + 16 * chunk,
                        *reinterpret_cast<const u32x4_t*>(ct + col * kTile + ((chunk ^ ((col >> 3) & 7)) * 16)));
        }
    }
}

// Codes of X to those of X^T: 8 x 8 codes a thread, turned in registers; a column's 8 rows
// go through LDS, swizzled as above. Bound by memory, one byte read and one written a code:
// 32768 x 4096 57 us, 4.75 TB/s, 2048 x 1280 2.9. WIDE: rows start at multiples of 8 bytes.
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_transpose_kernel(const uint8_t* x, int64_t ldx, int rows_all, int K, uint8_t* y, int64_t ldy,
                                                            int tiles_k) {
    __shared__ uint4 turned[kTile * kTile / 16];  // [column][row]
    uint8_t* t = reinterpret_cast<uint8_t*>(turned);
    const int tid = threadIdx.x, a = tid & 15, b = tid >> 4;
    const int c0 = (int)(blockIdx.x % tiles_k) * kTile;
    const int64_t r0 = (int64_t)(blockIdx.x / tiles_k) * kTile;
    const int rows = (int)min((int64_t)kTile, rows_all - r0), cols = min(kTile, K - c0);
    uint32_t v[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i][0] = v[i][1] = 0;
        if (8 * b + i >= rows) continue;
        const uint8_t* at = x + (r0 + 8 * b + i) * ldx + c0 + 8 * a;
        if (WIDE && 8 * a + 8 <= cols) {
            const uint2 q = *reinterpret_cast<const uint2*>(at);
            v[i][0] = q.x, v[i][1] = q.y;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * a + j < cols) v[i][j >> 2] |= (uint32_t)at[j] << (8 * (j & 3));
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // columns 4 h .. 4 h + 3
        uint32_t o[4][2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {  // rows 4 q .. 4 q + 3
            const uint32_t w0 = v[4 * q][h], w1 = v[4 * q + 1][h], w2 = v[4 * q + 2][h], w3 = v[4 * q + 3][h];
            const uint32_t l01 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), h01 = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
            const uint32_t l23 = __builtin_amdgcn_perm(w3, w2, 0x05010400u), h23 = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
            o[0][q] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
            o[1][q] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
            o[2][q] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
            o[3][q] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint2*>(t + (8 * a + 4 * h + j) * kTile + (((b >> 1) ^ (a & 7)) * 16) + (b & 1) * 8) = make_uint2(o[j][0], o[j][1]);
    }
    __syncthreads();
    const int height = (int)min((int64_t)kTile, ((rows_all + 15LL) & ~15LL) - r0);  // up to the 16 bytes' end: zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int col = i * 32 + tid / 8, chunk = tid & 7;
        if (col < cols && 16 * chunk < height)
            *reinterpret_cast<uint4*>(y + (int64_t)(c0 + col) * ldy + r0 + 16 * chunk) =
                *reinterpret_cast<const uint4*>(t + col * kTile + ((chunk ^ ((col >> 3) & 7)) * 16));
    }
}

}  // namespace

hipError_t launch_fp8_transpose(const uint8_t* codes, int64_t ldc, int rows, int K, uint8_t* codes_t, int64_t ldct, hipStream_t s) {
    const int tiles_k = (K + kTile - 1) / kTile;
    const unsigned grid = (unsigned)((((int64_t)rows + kTile - 1) / kTile) * tiles_k);
    if (reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldc % 8 == 0) fp8_transpose_kernel<true><<<grid, 256, 0, s>>>(codes, ldc, rows, K, codes_t, ldct, tiles_k);
    else fp8_transpose_kernel<false><<<grid, 256, 0, s>>>(codes, ldc, rows, K, codes_t, ldct, tiles_k);
    return hipGetLastError();
}

hipError_t launch_fp8_quantize(bool tiles, bool f32, const Fp8QuantParams& p, hipStream_t s) {
    const int tiles_k = (p.K + kTile - 1) / kTile;
    const unsigned grid = (unsigned)((((int64_t)p.rows + kTile - 1) / kTile) * tiles_k);
    // Codes larger than the L2s hold together are stored non-temporally: 117 -> 115 us in
    // the case above, tiles 107 -> 105.
    const bool nt = (int64_t)p.rows * p.K * ((p.codes ? 1 : 0) + (p.codes_t ? 1 : 0)) > (int64_t)16 << 20;
#define TMT_Q(TILES_, F32_)                                                                              \
    (nt ? fp8_quantize_kernel<TILES_, F32_, kStoreOnce><<<grid, kThreads8, 0, s>>>(p, tiles_k)                 \
        : fp8_quantize_kernel<TILES_, F32_, kCached><<<grid, kThreads8, 0, s>>>(p, tiles_k))
    if (tiles) f32 ? TMT_Q(true, true) : TMT_Q(true, false);
    else f32 ? TMT_Q(false, true) : TMT_Q(false, false);
#undef TMT_Q
    return hipGetLastError();
}

}  // namespace tmt
