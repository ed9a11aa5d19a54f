// tile_stream.hpp -- what the tiled products' kernels share (linear.hip,
// fp8_gemm.hip): loads from windows on global memory into LDS, the waits behind
// them, and the epilogue that writes a unit's outputs.
#pragma once
#include <type_traits>

#include "device_util.hpp"
#include "linear_plan.hpp"

namespace tmt {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ i32x4 descriptor(const Window& w) {
    return i32x4{(int)(uint32_t)w.at, (int)(uint32_t)(w.at >> 32), (int)w.bytes, 0x00020000};  // raw buffer
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 (4) bytes per lane from a window into LDS at lds_base + 16 (4) * lane
// (lds_base wave-uniform); M0 is written, one wait state ahead of the load.
__device__ __forceinline__ void dma16(const Window& w, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(descriptor(w)), "s"(lds_base) : "m0");
}
__device__ __forceinline__ void dma4(const Window& w, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(descriptor(w)), "s"(lds_base) : "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Workgroup barrier behind the LDS accesses only: a compiler's barrier would
// also wait for the last unit's output stores.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- epilogue ----------------------------------------------------------------
// acc[i][j][r] = C[m][c] with m = 32 i + lane % 32 and c = 32 j + 8 (r / 4) +
// 4 (lane / 32) + r % 4 in the wave's outputs. 32 rows by 32 JS columns
// at a time go through the wave's own LDS, so that a row's columns leave as one
// run of 16-byte stores; no barrier.
template <bool F32, int JS>
struct Stage {
    static constexpr int ROWB = 32 * JS * (F32 ? 4 : 2);  // bytes per staged row
    static constexpr int BYTES = 32 * ROWB;
};

template <int MI, int NJ>
__device__ __forceinline__ void clear(f32x16 (&acc)[MI][NJ]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
}

__device__ __forceinline__ void wave_lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// Keeps the compiler from moving a wave's LDS accesses across.
__device__ __forceinline__ void wave_lds_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// out: the wave's first output element, ld its row stride; rows, cols: valid
// ones. The outputs are a window: rows past its end are dropped by the hardware,
// columns past the end get an offset past it. BETA: beta times what is there is
// added in fp32. NT: results are written once and leave the caches to the
// operands; partial tiles are read again at once.
//
// With one wave per SIMD this is bound by its instructions, so it has few: one
// addition and one store per 1 KiB, no branch (MXFP4 x MXFP4, T 65536, N 4096, K
// 1024: 222 us with addresses, branches and a sum with beta = 0, 210 without). A
// slice is converted while the one
// before comes back from LDS, and its own way through LDS needs no wait: a wave's
// LDS accesses run in order.
// AGPR: the sums are the matrix instructions' own, else the vector unit's.
template <bool F32, int JS, bool NT, bool BETA, bool AGPR, int MI, int NJ>
__device__ __forceinline__ void store_wave(f32x16 (&acc)[MI][NJ], uint8_t* st, void* out, int64_t ld, int rows,
                                           int cols, float beta) {
    using S = Stage<F32, JS>;
    constexpr int CH = S::ROWB / 16, RPI = 64 / CH;  // 16-byte chunks per staged row, rows per store
    constexpr int JG = NJ / JS, SLICES = MI * JG, SIZE = F32 ? 4 : 2;
    constexpr uint32_t FAR = 0x80000000u;
    // a value of this unit's own: the addresses below are not kept in registers
    // through the main loop
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int lr = lane & 31, cl = lane % CH;
    const uint32_t row = (uint32_t)(ld * SIZE);
    rows = min(rows, 32 * MI);
    cols = min(cols, 32 * NJ);
    const __amdgpu_buffer_rsrc_t win =
        __builtin_amdgcn_make_buffer_rsrc(out, 0, (int)output_window(rows, row, cols, SIZE), 0x00020000);
    uint4 v[32 / RPI];  // rows of a slice
    auto store = [&](int n) {
        const int c = 32 * JS * (n % JG) + cl * (16 / SIZE);
        uint32_t at = c < cols ? (uint32_t)(32 * (n / JG) + lane / CH) * row + (uint32_t)c * SIZE : FAR;
        if constexpr (F32 && BETA) {
            u32x4 was[32 / RPI];
#pragma unroll
            for (int k = 0; k < 32 / RPI; ++k) was[k] = __builtin_amdgcn_raw_buffer_load_b128(win, (int)(at + k * RPI * row), 0, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 32 / RPI; ++k)
                v[k] = __builtin_bit_cast(uint4, __builtin_bit_cast(f32x4, v[k]) + beta * __builtin_bit_cast(f32x4, was[k]));
        }
#pragma unroll
        for (int k = 0; k < 32 / RPI; ++k) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[k]), win, (int)at, 0, NT ? 2 : 0);
            at += RPI * row;
        }
    };
    // bf16 outputs that are added to: a slice's are loaded while the one before is
    // converted, ahead of the stores, which a later load would wait for
    u32x2 old[2][JS][4];
    auto load_old = [&](int n) {
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 32 * (n % JG * JS + j) + 8 * q + 4 * (lane >> 5);
                old[n & 1][j][q] = __builtin_amdgcn_raw_buffer_load_b64(
                    win, c < cols ? (int)((uint32_t)(32 * (n / JG) + lr) * row + (uint32_t)c * SIZE) : (int)FAR, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (!F32 && BETA) load_old(0);
#pragma unroll
    for (int n = 0; n < SLICES; ++n) {
        const int i = n / JG, jg = n % JG * JS;
        if constexpr (!F32 && BETA)
            if (n + 1 < SLICES) load_old(n + 1);
        // the outputs not yet staged stay in the accumulator registers
        if constexpr (AGPR) {
#pragma unroll
            for (int i2 = i; i2 < MI; ++i2)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (i2 > i || j >= jg) asm volatile("" : "+a"(acc[i2][j]));
        }
        uint2 half[JS][4];
        if constexpr (!F32) {
#pragma unroll
            for (int j = 0; j < JS; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x16& a = acc[i][jg + j];
                    f32x4 f = {a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                    if constexpr (BETA) {
                        const u32x2 o = old[n & 1][j][q];
                        f = f + beta * f32x4{bf_lo(o[0]), bf_hi(o[0]), bf_lo(o[1]), bf_hi(o[1])};
                    }
                    half[j][q] = make_uint2(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]));
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (n > 0) store(n - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (F32) {
                    const f32x16& a = acc[i][jg + j];
                    const int ch = j * 8 + 2 * q + (lane >> 5);
                    *reinterpret_cast<f32x4*>(st + lr * S::ROWB + ((ch ^ (lr & (CH - 1))) * 16)) =
                        f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                } else {
                    const int ch = j * 4 + q;
                    *reinterpret_cast<uint2*>(st + lr * S::ROWB + ((ch ^ (lr & (CH - 1))) * 16) + (lane >> 5) * 8) = half[j][q];
                }
            }
        wave_lds_order();
#pragma unroll
        for (int k = 0; k < 32 / RPI; ++k) {
            const int rr = lane / CH + RPI * k;
            v[k] = *reinterpret_cast<const uint4*>(st + rr * S::ROWB + ((cl ^ (rr & (CH - 1))) * 16));
        }
        wave_lds_order();
    }
    store(SLICES - 1);
}

constexpr auto workgroups = [] __device__() { return (int)gridDim.x; };

// Writes a unit's wave outputs: to the result (p.y, p.ldy, p.beta) or, SPLIT, as a partial tile
// (fp32; bf16 results' partial tiles leave from the registers, whose LDS holds
// no fp32 rows).
template <int TILE, bool F32, int JS, bool SPLIT, bool BETA, bool AGPR = true, class Params>
__device__ __forceinline__ void finish_unit(f32x16 (&acc)[TILE / 64][TILE / 64], uint8_t* st, const Params& p,
                                            const Unit& u, int M, int C, int wrow, int wcol) {
    constexpr int WT = TILE / 2;
    const int rows = M - u.m0 - wrow, cols = C - u.c0 - wcol;
    if (rows <= 0 || cols <= 0) return;
    if constexpr (SPLIT) {
        float* o = p.part + (int64_t)u.part * TILE * TILE + wrow * TILE + wcol;
        if constexpr (F32) {
            store_wave<true, JS, false, false, AGPR>(acc, st, o, TILE, rows, cols, 0.0f);
        } else {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int i = 0; i < WT / 32; ++i) {
                const int m = 32 * i + (lane & 31);
#pragma unroll
                for (int j = 0; j < WT / 32; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int c = 32 * j + 8 * q + 4 * (lane >> 5);
                        if (m < rows && c < cols)
                            *reinterpret_cast<f32x4*>(o + m * TILE + c) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                                                               acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    }
            }
        }
    } else {
        using Out = std::conditional_t<F32, float, uint16_t>;
        Out* o = static_cast<Out*>(p.y) + (int64_t)(u.m0 + wrow) * p.ldy + u.c0 + wcol;
        store_wave<F32, JS, true, BETA, AGPR>(acc, st, o, p.ldy, rows, cols, p.beta);
    }
}

// ---- the last round's sums ------------------------------------------------------
// Tail tile j is the sum of its partial tiles in part order, plus beta times
// what is there, rounded once. A thread takes 4 columns of a row.
template <int TILE, bool F32, class Params>
__global__ __launch_bounds__(256) void linear_fixup_kernel(Params p, LinearPlan pl, int M, int C) {
    constexpr int TPR = TILE / 4, RPW = 256 / TPR, SLABS = TILE / RPW;
    const int j = blockIdx.x / SLABS, slab = blockIdx.x % SLABS;
    int mt, ct;
    tile_at(pl, pl.whole + j, mt, ct);
    const int r = slab * RPW + threadIdx.x / TPR, c = (threadIdx.x % TPR) * 4;
    const int m = mt * TILE + r, col = ct * TILE + c;
    if (m >= M || col >= C) return;
    const float* src = p.part + (int64_t)j * pl.parts * TILE * TILE + r * TILE + c;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int q0 = 0; q0 < pl.parts; q0 += 8) {  // up to 8 loads in flight
        f32x4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const f32x4*>(src + (int64_t)min(q0 + q, pl.parts - 1) * TILE * TILE);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q0 + q < pl.parts) sum = sum + v[q];
    }
    const int64_t at = (int64_t)m * p.ldy + col;
    if constexpr (F32) {
        f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(p.y) + at);
        if (p.beta != 0.0f) sum = sum + p.beta * *y;
        *y = sum;
    } else {
        uint2* y = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at);
        if (p.beta != 0.0f) {
            const uint2 old = *y;
            sum = sum + p.beta * f32x4{bf_lo(old.x), bf_hi(old.x), bf_lo(old.y), bf_hi(old.y)};
        }
        *y = make_uint2(pack_bf2(sum[0], sum[1]), pack_bf2(sum[2], sum[3]));
    }
}

}  // namespace
}  // namespace tmt
