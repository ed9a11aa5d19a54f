// rmsnorm.hip -- root-mean-square norm with the residual's addition, out in
// bf16 and in 8 bits, and its backward.
//
//   forward   s = x + r, rounded to the stream's type; rstd = 1 / sqrt(mean(s^2) + eps);
//             y = (s * rstd) * gamma, to bf16 and to e4m3 codes with a scale for
//             every 128 columns (the codes not from y in bf16 but as from 64 bits)
//   backward  g = dy gamma, xh = s rstd, c = mean(g xh);
//             ds = dr + rstd (g - xh c); dgamma = sum over rows of dy xh
//
// Bound by memory. A row belongs to 16 lanes (d <= 128) or 32 (d <= 256), a wave (d <=
// 1024), or a workgroup of four waves (d <= 4096) or of sixteen, and is held in
// registers between its statistics and its outputs, so each value is read once and
// written once. A lane has V = 8 or 16 values (4 of the narrowest fp32 rows) in pieces
// of 16 bytes of the stream: 8 bf16 or 4 fp32 values (with 8 fp32 values a wave's store
// would cover every second 16 bytes). A row's pieces are consecutive, so 16 (32)
// neighbouring lanes own a block of 128 columns and find its maximum by DPP. us, and
// TB/s of what has to pass: forward 32768 x 1024 fp32 to stream and codes 61, 6.0; 16384 x
// 4096 125, 5.9; 777 x 1280 bf16 to bf16 and codes 5.0; one row 3.5; backward 32768 x 1024 fp32 84, 5.6; 16384 x
// 4096 bf16 113, 4.8; 5003 x 1000 13.0. A copy of 1 GiB reaches 5.0 TB/s.
//
// The forward's squares are added in 64 bits, a lane's values, the lanes (a butterfly)
// and the waves (in order): rstd moves a whole row, and with it which way its codes
// round. The backward's
// lanes keep dgamma of their columns in registers over the rows that they walk; a
// workgroup's sums are added in the order of its rows into one row of the workspace, and
// those rows by launch_colsum: no atomics, the same bits every time.
#include <algorithm>

#include "fp8.hpp"
#include "fp8_format.hpp"
#include "moe_internal.hpp"

namespace tmt {
namespace {

// N consecutive elements of a row from k0 on (16-byte aligned where a piece is
// whole); TAIL: d is not a multiple of N, and elements from d on are zeros.
template <int N, bool TAIL, int PASS>
__device__ __forceinline__ void load_piece(const float* row, int k0, int d, float* v) {
    if (!TAIL || k0 + N <= d) {
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            const f32x4 a = get<PASS, f32x4>(row + k0 + q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[q + i] = a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = k0 + i < d ? row[k0 + i] : 0.0f;
    }
}
template <int N, bool TAIL, int PASS>
__device__ __forceinline__ void load_piece(const uint16_t* row, int k0, int d, float* v) {
    if (!TAIL || k0 + N <= d) {
        if constexpr (N == 8) {
            unpack8(__builtin_bit_cast(uint4, get<PASS, u32x4_t>(row + k0)), v);
        } else {
            const u32x2_t a = get<PASS, u32x2_t>(row + k0);
            v[0] = bf_lo(a[0]), v[1] = bf_hi(a[0]), v[2] = bf_lo(a[1]), v[3] = bf_hi(a[1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = k0 + i < d ? bf1(row[k0 + i]) : 0.0f;
    }
}
template <int N, bool TAIL, int PASS>
__device__ __forceinline__ void store_piece(float* row, int k0, int d, const float* v) {
    if (!TAIL || k0 + N <= d) {
#pragma unroll
        for (int q = 0; q < N; q += 4) put<PASS>(row + k0 + q, f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]});
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k0 + i < d) row[k0 + i] = v[i];
    }
}
template <int N, bool TAIL, int PASS>
__device__ __forceinline__ void store_piece(uint16_t* row, int k0, int d, const float* v) {
    if (!TAIL || k0 + N <= d) {
        if constexpr (N == 8) put<PASS>(row + k0, __builtin_bit_cast(u32x4_t, pack8(v)));
        else put<PASS>(row + k0, u32x2_t{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])});
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k0 + i < d) row[k0 + i] = f2bf(v[i]);
    }
}

template <bool F32>
struct StreamType {
    using T = uint16_t;
};
template <>
struct StreamType<true> {
    using T = float;
};

// The shape of a launch: LANES per row, V values a lane, rows per workgroup.
template <bool F32, int LANES, int V>
struct Shape {
    static constexpr int N = F32 ? 4 : 8;             // values of a piece
    static constexpr int C = V / N;                   // pieces a lane
    static constexpr int WAVES = LANES < 64 ? 1 : LANES / 64;
    static constexpr int THREADS = LANES < 256 ? 256 : LANES;
    static constexpr int ROWS = THREADS / LANES;
    static constexpr int STRIDE = LANES * N;          // columns between a lane's pieces
    static_assert(STRIDE % kFp8Block == 0, "a block lies in one piece of neighbouring lanes");
};

// gamma of a lane's columns; zeros past the last one.
template <class S, bool TAIL, int C, int N>
__device__ __forceinline__ void load_gamma(const float* gamma, int lane, int d, float (&g)[C][N]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k0 = c * S::STRIDE + lane * N;
        if (k0 < d) load_piece<N, TAIL, kCached>(gamma, k0, d, g[c]);
        else
#pragma unroll
            for (int i = 0; i < N; ++i) g[c][i] = 0.0f;
    }
}

template <int OFF>
__device__ __forceinline__ double xor_lane_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, ((uint64_t)xor_lane_u32<OFF>((uint32_t)(b >> 32)) << 32) | xor_lane_u32<OFF>((uint32_t)b));
}
template <int OFF>
__device__ __forceinline__ double add_xor_lane(double v) {
    return v + xor_lane_f64<OFF>(v);
}
template <int OFF>
__device__ __forceinline__ float add_xor_lane(float v) {
    return v + xor_lane<OFF>(v);
}
// Sum over the row's lanes and waves; `red` is the workgroup's, one of two in turn, so
// that one barrier a row is enough.
template <int LANES, class F>
__device__ __forceinline__ F row_sum(F v, F* red) {
    if constexpr (LANES >= 64) v = add_xor_lane<32>(v);
    if constexpr (LANES >= 32) v = add_xor_lane<16>(v);
    v = add_xor_lane<8>(v);
    v = add_xor_lane<4>(v);
    v = add_xor_lane<2>(v);
    v = add_xor_lane<1>(v);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) v += red[w];
    }
    return v;
}

// Cut off after 20 bits of the mantissa, the last of which is set if anything was lost:
// rounded to e4m3 that is the value's own rounding, where fp32's nearest may be the middle
// between two codes.
__device__ __forceinline__ float odd_float(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t hi = (uint32_t)(b >> 32) | min((uint32_t)b, 1u);
    return (float)__builtin_bit_cast(double, (uint64_t)hi << 32);
}
// A code goes one way or the other by the last bits where its value lies near the middle
// between two. In fp32 rstd, the two products, the same three in the block's maximum, its
// quotient and the last product leave it at most 4 units of the last place off, 8 where
// those of the maximum's binade are twice as large; where a value of a wave lies that near
// (one piece of a hundred), its codes are found in 64 bits. Codes of 2^25 values that are
// not those of 64 bits: 25, now none; in 64 bits throughout, 32768 x 1024 bf16 takes 54 us,
// so 48. e4m3's subnormals lie 2^-9 apart, as the codes of [2^-6, 2^-5) do: moved there, they
// have their middles at the same bit. Their values are at most 4 of that binade's units off,
// the sum half of one more.
constexpr uint32_t kNear = 8;
__device__ __forceinline__ float middle_bits(float q) {
    const float a = fabsf(q);
    return a < 0x1p-6f ? a + 0x1p-6f : a;
}
template <int N>
__device__ void exact_scaled(const float* v, const float* g, double rstd, float inv, float* q) {
    double y[N], m = 0x1p-100;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        y[i] = (double)v[i] * rstd * (double)g[i];
        m = fmax(m, fabs(y[i]));
    }
    m = fmax(m, xor_lane_f64<1>(m));
    m = fmax(m, xor_lane_f64<2>(m));
    m = fmax(m, xor_lane_f64<4>(m));
    m = fmax(m, xor_lane_f64<8>(m));
    if constexpr (N == 4) m = fmax(m, xor_lane_f64<16>(m));
    const double inv64 = 448.0 / m;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (inv != 0.0f) q[i] = odd_float(y[i] * inv64);
}

template <bool F32, bool TAIL, int LANES, int V, int PASS>
__global__ __launch_bounds__((Shape<F32, LANES, V>::THREADS)) void rms_fwd_kernel(RmsParams p) {
    using S = Shape<F32, LANES, V>;
    using E = typename StreamType<F32>::T;
    constexpr int N = S::N, C = S::C;
    __shared__ double red[S::WAVES];
    const int d = p.d, lane = threadIdx.x % LANES;
    const int64_t r = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * S::ROWS + threadIdx.x / LANES;
    if (r >= p.T) return;  // whole rows
    float v[C][N], g[C][N];
    load_gamma<S, TAIL>(p.gamma, lane, d, g);
    double sq = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k0 = c * S::STRIDE + lane * N;
#pragma unroll
        for (int i = 0; i < N; ++i) v[c][i] = 0.0f;
        if (k0 < d) {
            float x[N];
            if (p.R) load_piece<N, TAIL, PASS>(static_cast<const E*>(p.R) + r * p.ldr, k0, d, v[c]);
            if (p.X) {
                load_piece<N, TAIL, kCached>(p.X + r * p.ldx, k0, d, x);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    v[c][i] += x[i];
                    if constexpr (!F32) v[c][i] = bf1(f2bf(v[c][i]));
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) sq = __builtin_fma((double)v[c][i], (double)v[c][i], sq);
    const double rstd64 = 1.0 / sqrt(row_sum<LANES>(sq, red) / d + p.eps);
    const float rstd = (float)rstd64;
    if (p.rstd && lane == 0) p.rstd[r] = rstd;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k0 = c * S::STRIDE + lane * N;
        if (k0 < d && p.S) store_piece<N, TAIL, PASS>(static_cast<E*>(p.S) + r * p.lds, k0, d, v[c]);
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = v[c][i] * rstd * g[c][i];
        if (k0 < d && p.Y) store_piece<N, TAIL, PASS>(p.Y + r * p.ldy, k0, d, y);
        if (p.codes) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m = max(m, k0 < d ? abs_bits(y[i]) : 0u);
            m = max(m, xor_lane_u32<1>(m));
            m = max(m, xor_lane_u32<2>(m));
            m = max(m, xor_lane_u32<4>(m));
            m = max(m, xor_lane_u32<8>(m));
            if constexpr (N == 4) m = max(m, xor_lane_u32<16>(m));
            const Fp8Scale f = fp8_scale(m);
            if (lane % (kFp8Block / N) == 0 && k0 < d) p.scales[(int64_t)(k0 / kFp8Block) * p.ldsc + r] = f.scale;
            float q[N];
            uint32_t near = ~0u;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                q[i] = fp8_scaled(y[i], f.inv);
                near = min(near, (__float_as_uint(middle_bits(q[i])) - (0x80000u - kNear)) & 0xfffffu);
            }
            if (__any(near <= 2 * kNear)) exact_scaled<N>(v[c], g[c], rstd64, f.inv, q);
            if (k0 < ((d + 15) & ~15)) {  // up to the 16 bytes' end: zeros
                uint8_t* o = p.codes + r * p.ldc + k0;
                if constexpr (N == 8) put<PASS>(o, u32x2_t{to_e4m3(q), to_e4m3(q + 4)});
                else put<PASS>(o, to_e4m3(q));
            }
        }
    }
}

template <bool F32, bool TAIL, int LANES, int V, int PASS>
__global__ __launch_bounds__((Shape<F32, LANES, V>::THREADS)) void rms_bwd_kernel(RmsParams p, int rows_per_block) {
    using S = Shape<F32, LANES, V>;
    using E = typename StreamType<F32>::T;
    constexpr int N = S::N, C = S::C;
    // dr's loads go out with the others, but for the widest rows, whose registers they overrun
    constexpr bool EARLY = V * LANES < kRmsMaxWidth;
    __shared__ float red[2][S::WAVES];
    const int d = p.d, sub = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int first = blockIdx.x * rows_per_block, last = min(p.T, first + rows_per_block);
    const float over = 1.0f / (float)d;
    float dg[C][N], g[C][N];
    load_gamma<S, TAIL>(p.gamma, lane, d, g);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) dg[c][i] = 0.0f;
    int turn = 0;
    for (int r = first + sub; r < last; r += S::ROWS) {
        float dy[C][N], xh[C][N], o[C][N] = {};
        float dot = 0.0f;
        const float rstd = p.rstd[r];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int k0 = c * S::STRIDE + lane * N;
            if (k0 < d) {
                load_piece<N, TAIL, kCached>(p.dY + (int64_t)r * p.lddy, k0, d, dy[c]);
                load_piece<N, TAIL, PASS>(static_cast<const E*>(p.S) + (int64_t)r * p.lds, k0, d, xh[c]);
                if (EARLY && p.dR) load_piece<N, TAIL, PASS>(static_cast<const E*>(p.dR) + (int64_t)r * p.lddr, k0, d, o[c]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) dy[c][i] = xh[c][i] = 0.0f;
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                xh[c][i] *= rstd;
                dg[c][i] = __builtin_fmaf(dy[c][i], xh[c][i], dg[c][i]);
                dy[c][i] *= g[c][i];
                dot = __builtin_fmaf(dy[c][i], xh[c][i], dot);
            }
        }
        const float mean = row_sum<LANES>(dot, red[turn]) * over;
        turn ^= 1;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int k0 = c * S::STRIDE + lane * N;
            if (k0 < d) {
                if (!EARLY && p.dR) load_piece<N, TAIL, PASS>(static_cast<const E*>(p.dR) + (int64_t)r * p.lddr, k0, d, o[c]);
#pragma unroll
                for (int i = 0; i < N; ++i) o[c][i] += rstd * __builtin_fmaf(-xh[c][i], mean, dy[c][i]);
                store_piece<N, TAIL, PASS>(static_cast<E*>(p.dS) + (int64_t)r * p.ldds, k0, d, o[c]);
            }
        }
    }
    // the workgroup's rows of sums, in wave order
    const int w4 = ln_width4(d);
    float* out = p.partial + (int64_t)blockIdx.x * w4;
    if constexpr (S::ROWS == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int k0 = c * S::STRIDE + lane * N;
#pragma unroll
            for (int q = 0; q < N; q += 4)
                if (k0 + q < w4) *reinterpret_cast<f32x4*>(out + k0 + q) = f32x4{dg[c][q], dg[c][q + 1], dg[c][q + 2], dg[c][q + 3]};
        }
    } else {
        __shared__ float sum[S::ROWS][V * LANES];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < N; q += 4)
                *reinterpret_cast<f32x4*>(&sum[sub][c * S::STRIDE + lane * N + q]) = f32x4{dg[c][q], dg[c][q + 1], dg[c][q + 2], dg[c][q + 3]};
        __syncthreads();
        for (int k = threadIdx.x * 4; k < w4; k += S::THREADS * 4) {
            f32x4 t = *reinterpret_cast<f32x4*>(&sum[0][k]);
#pragma unroll
            for (int w = 1; w < S::ROWS; ++w) t += *reinterpret_cast<f32x4*>(&sum[w][k]);
            *reinterpret_cast<f32x4*>(out + k) = t;
        }
    }
}

// Lanes per row for a width: so many that a lane has 8 or 16 values (4 of a narrow
// fp32 row).
int lanes_of(bool f32, int d) {
    return d <= 128 ? (f32 ? 32 : 16) : d <= 256 ? 32 : d <= 1024 ? 64 : d <= 4096 ? 256 : 1024;
}
// Rows of a workgroup of the backward, so that the launch is about one round of
// kBwdThreads threads a CU (rows kept by a wave save partial sums). us with 512 / 1024 /
// 2048: 32768 x 1024 bf16 66.9 / 64.7 / 62.5, fp32 112 / 105 / 107; 5003 x 1000 13.8 /
// 13.2 / 15.9.
constexpr int kBwdThreads = 1024;
int bwd_blocks(bool f32, int d, int cus) { return cus * kBwdThreads / std::max(256, lanes_of(f32, d)); }
int rows_per_block(bool f32, int T, int d, int cus) {
    const int rows = std::max(1, 256 / lanes_of(f32, d)), blocks = bwd_blocks(f32, d, cus);
    const int each = (int)(((int64_t)T + blocks - 1) / blocks);
    return (each + rows - 1) / rows * rows;
}
// Outputs larger than the L2s hold together are stored non-temporally: 32768 x 1024
// forward fp32 75 -> 68 us, bf16 51 -> 44, backward fp32 112 -> 105. A call that passes
// over 250 MB, about what the memory-side cache (256 MiB) holds, also loads s, r and dr like
// that, but not x and dy, which the products before it have just written: backward of
// that shape fp32 105 -> 84, bf16 62 -> 48, forward fp32 68 -> 61; x and dy too: 98, 57, 65.
// What decides is whether the inputs are still there, as they may be below the bound: widths
// 256 to 8192 after other calls, 260 MB forward 3 to 9% faster and backward 9 to 20%, 200 MB
// 0 to 4 and 9 to 20, 150 MB forward 3 to 15% slower; on the same buffers again, 150 to 300
// MB, all 3 to 22% slower.
int pass_of(int64_t in, int64_t out) { return in + out > 250'000'000 ? kOnce : out > 16 << 20 ? kStoreOnce : kCached; }

template <bool F32, bool TAIL, int LANES, int V, int PASS>
void launch(bool fwd, const RmsParams& p, int grid, int rpb, hipStream_t s) {
    using S = Shape<F32, LANES, V>;
    if (fwd) {  // in two dimensions, for one's threads are counted in 32 bits
        const int64_t blocks = ((int64_t)p.T + S::ROWS - 1) / S::ROWS, x = std::min<int64_t>(blocks, 1 << 20);
        rms_fwd_kernel<F32, TAIL, LANES, V, PASS><<<dim3(x, (blocks + x - 1) / x), S::THREADS, 0, s>>>(p);
    } else rms_bwd_kernel<F32, TAIL, LANES, V, PASS><<<grid, S::THREADS, 0, s>>>(p, rpb);
}
template <bool F32, bool TAIL, int PASS>
void launch_width(bool fwd, const RmsParams& p, int grid, int rpb, hipStream_t s) {
    const int d = p.d;
    if (d <= 128) launch<F32, TAIL, F32 ? 32 : 16, F32 ? 4 : 8, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 256) launch<F32, TAIL, 32, 8, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 512) launch<F32, TAIL, 64, 8, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 1024) launch<F32, TAIL, 64, 16, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 2048) launch<F32, TAIL, 256, 8, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 4096) launch<F32, TAIL, 256, 16, PASS>(fwd, p, grid, rpb, s);
    else if (d <= 8192) launch<F32, TAIL, 1024, 8, PASS>(fwd, p, grid, rpb, s);
    else launch<F32, TAIL, 1024, 16, PASS>(fwd, p, grid, rpb, s);
}
template <bool F32>
void launch_pass(bool fwd, const RmsParams& p, int grid, int rpb, hipStream_t s) {
    const int stream = F32 ? 4 : 2;
    const int64_t n = (int64_t)p.T * p.d;
    const int in = fwd ? (p.X ? 2 : 0) + (p.R ? stream : 0) : 2 + stream + (p.dR ? stream : 0);
    const int out = fwd ? (p.S ? stream : 0) + (p.Y ? 2 : 0) + (p.codes ? 1 : 0) : stream;
    const int pass = pass_of(n * in, n * out);
    if (p.d % (F32 ? 4 : 8) != 0) launch_width<F32, true, kCached>(fwd, p, grid, rpb, s);
    else if (pass == kOnce) launch_width<F32, false, kOnce>(fwd, p, grid, rpb, s);
    else if (pass == kStoreOnce) launch_width<F32, false, kStoreOnce>(fwd, p, grid, rpb, s);
    else launch_width<F32, false, kCached>(fwd, p, grid, rpb, s);
}
void launch_rms(bool fwd, const RmsParams& p, int grid, int rpb, hipStream_t s) {
    p.f32 ? launch_pass<true>(fwd, p, grid, rpb, s) : launch_pass<false>(fwd, p, grid, rpb, s);
}

}  // namespace

int rms_partials_max(int d, int cus) { return std::max(bwd_blocks(false, d, cus), bwd_blocks(true, d, cus)); }

hipError_t launch_rms_fwd(const RmsParams& p, hipStream_t s) {
    launch_rms(true, p, 0, 0, s);
    return hipGetLastError();
}

hipError_t launch_rms_bwd(const RmsParams& p, hipStream_t s) {
    const int rpb = rows_per_block(p.f32, p.T, p.d, cu_count());
    const int grid = p.T > 0 ? (p.T + rpb - 1) / rpb : 0, w4 = ln_width4(p.d);
    if (grid > 0) launch_rms(false, p, grid, rpb, s);
    return launch_colsum(p.partial, grid, w4, w4, p.d, p.dgamma, nullptr, s);
}

}  // namespace tmt
