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
#include "fp8_format.hpp"
#include "fp8_plan.hpp"
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

// Operand rows of 16, from LDS rows of 128 bytes whose chunks of 16 are
// XOR-swizzled by row / 2: lane l holds chunks g and g + 4 of row l % 16, g = l / 16.
__device__ __forceinline__ i32x8 read_codes16(const uint8_t* t, int r, int g) {
    const int sw = (r >> 1) & 7;
    return join(*reinterpret_cast<const uint4*>(t + r * 128 + ((g ^ sw) * 16)),
                *reinterpret_cast<const uint4*>(t + r * 128 + (((g + 4) ^ sw) * 16)));
}

// ---- few rows ----------------------------------------------------------------------
// A workgroup takes 16 NB columns and 16 RB rows of y; its 8 waves deal out the
// reduction in blocks of 128. A wave loads its blocks into LDS of its own, 8 rows of
// 128 bytes a load, DEPTH blocks ahead (1 where it has no more: ONE, whose LDS leaves
// room for more workgroups on a CU), and no wave waits for another until their sums
// meet in LDS and are added in wave order. Bound by a launch and a trip to memory: M 1,
// N 4096, K 1024 2.9 us, M 64, N 1024, K 4096 4.4 (6.2 with loads straight into
// registers, where neighbouring lanes hold different rows and four of them take four
// cache lines).
template <bool TILES, bool F32, int RB, int NB, bool ONE>
__global__ __launch_bounds__(512) void fp8_rows_kernel(Fp8Params p) {
    using S = RowSlot<RB, NB, ONE>;
    constexpr int OUT = 256 * RB * NB, NW = 8, DEPTH = S::DEPTH;
    __shared__ uint4 lds_raw[NW * S::WAVE / 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, g = lane >> 4;
    uint8_t* own = reinterpret_cast<uint8_t*>(lds_raw) + wave * S::WAVE;
    const uint32_t lds0 = lds_u32(own);
    RowBlock<TILES, RB, NB> at;
    at.set(p, blockIdx.x);
    const int blocks = (p.K + kFp8Block - 1) / kFp8Block, steps = (blocks - wave + NW - 1) / NW;
    const int chunk = row_chunk(lane);
    const uint32_t a_row = (uint32_t)(lane >> 3) * (uint32_t)p.lda, b_row = (uint32_t)(lane >> 3) * (uint32_t)p.ldb;
    auto load = [&](int n) {
        const int kb = wave + n * NW, k = kb * kFp8Block;
        const uint32_t slot = lds0 + (uint32_t)(n % DEPTH) * S::BYTES;
        uint32_t from[2];
#pragma unroll
        for (int o = 0; o < 2; ++o) from[o] = row_chunk_at(p.K, k, chunk ^ (4 * o));
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) dma16(at.wb, from[i & 1] + b_row + (uint32_t)(8 * i) * (uint32_t)p.ldb, slot + 2048 * RB + 1024 * i);
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i) dma16(at.wa, from[i & 1] + a_row + (uint32_t)(8 * i) * (uint32_t)p.lda, slot + 1024 * i);
        dma4(at.a_scales(p, kb), 4u * lane, slot + S::SA);
        dma4(at.b_scales(p, kb), 4u * lane, slot + S::SB);
    };
    f32x4 acc[RB][NB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < DEPTH; ++n)
        if (n < steps) load(n);
    for (int n = 0; n < steps; ++n) {
        const int behind = min(DEPTH - 1, steps - 1 - n);  // blocks that are still to come
        if (DEPTH > 3 && behind == 3) wait_vm<(DEPTH > 3 ? 3 : 0) * S::ND>();
        else if (DEPTH > 2 && behind == 2) wait_vm<(DEPTH > 2 ? 2 : 0) * S::ND>();
        else if (DEPTH > 1 && behind == 1) wait_vm<(DEPTH > 1 ? 1 : 0) * S::ND>();
        else wait_vm<0>();
        const uint8_t* t = own + (n % DEPTH) * S::BYTES;
        const float* psa = reinterpret_cast<const float*>(t + S::SA);
        const float* psb = reinterpret_cast<const float*>(t + S::SB);
        i32x8 a[RB], b[NB];
        float sa[RB];
        f32x4 sb[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            b[i] = read_codes16(t + 2048 * (RB + i), row, g);
            if constexpr (!TILES) sb[i] = *reinterpret_cast<const f32x4*>(psb + 16 * i + 4 * g);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            a[r] = read_codes16(t + 2048 * r, row, g);
            sa[r] = psa[16 * r + row];
            if constexpr (TILES) sa[r] *= psb[0];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is read
        if (n + DEPTH < steps) load(n + DEPTH);
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const f32x4 d = mma16<F32>(b[i], a[r]);
                if constexpr (TILES) acc[r][i] += d * sa[r];
                else acc[r][i] += d * (sb[i] * sa[r]);
            }
    }
    // acc[r][i][e]: row 16 r + lane % 16, column 16 i + 4 (lane / 16) + e
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < NB; ++i)
            *reinterpret_cast<f32x4*>(own + 4 * ((16 * r + row) * (16 * NB) + 16 * i + 4 * g)) = acc[r][i];
    __syncthreads();
    const float* red = reinterpret_cast<const float*>(lds_raw);
    for (int o = threadIdx.x * 2; o < OUT; o += 128 * NW) {
        const int m = at.m0 + o / (16 * NB), n = at.n0 + o % (16 * NB);
        if (m >= p.M || n >= p.N) continue;
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            v[0] += red[w * (S::WAVE / 4) + o];
            v[1] += red[w * (S::WAVE / 4) + o + 1];
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

// ---- tiles -------------------------------------------------------------------------
// The 32 x 32 sums of a block of 128 from LDS rows of 128 bytes, whose chunks of 16
// are XOR-swizzled by row / 2: lane l holds 64 codes of row l % 32, chunks 2 h, 2 h
// + 1, 4 + 2 h and 5 + 2 h with h = l / 32.
struct Codes {
    i32x8 q[2];
};
__device__ __forceinline__ Codes read_codes(const uint8_t* t, int r, int h) {
    auto at = [&](int c) { return *reinterpret_cast<const uint4*>(t + r * 128 + ((c ^ ((r >> 1) & 7)) * 16)); };
    return {{join(at(2 * h), at(2 * h + 1)), join(at(4 + 2 * h), at(5 + 2 * h))}};
}
__device__ __forceinline__ f32x16 zero16() {
    return f32x16{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
}
struct Wide {
    bf16x8 v[8];
};
__device__ __forceinline__ Wide widen(const Codes& c) {
    Wide w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.v[i] = widen(c.q[i >> 2][2 * (i & 3)], c.q[i >> 2][2 * (i & 3) + 1]);
    return w;
}
__device__ __forceinline__ f32x16 mma32(const Codes& b, const Codes& a) {
    const f32x16 d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b.q[0], a.q[0], zero16(), 0, 0, 0, 0, 0, 0);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b.q[1], a.q[1], d, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const Wide& b, const Wide& a) {
    f32x16 d = zero16();
#pragma unroll
    for (int i = 0; i < 8; ++i) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b.v[i], a.v[i], d, 0, 0, 0);
    return d;
}

// A step's place in LDS: codes of a and b, the scales of a's rows and of b's (tiles:
// one for each 128 columns, 256 bytes apart).
template <int TILE, int WAVES>
struct Slot {
    static constexpr int CODES = TILE * 128, LOADS = CODES / (1024 * WAVES);  // per operand; 1 KiB loads per wave
    static constexpr int SA = 2 * CODES, SB = SA + TILE * 4, BYTES = SB + TILE * 4;
    static constexpr int ND = 2 * LOADS + 2;                        // loads per wave and step
};

// The loads of a tiled kernel's wave: load(d) issues load d of the next step; those
// of b's codes come first, then the scales', then those of a's codes.
// FULL: K is a multiple of 128, and no chunk lies behind a row's end.
template <int TILE, int WAVES, bool TILES, bool SPLIT, bool FULL>
struct Loader {
    using S = Slot<TILE, WAVES>;
    Fp8Cursor<TILE, TILES, SPLIT> at;
    uint32_t a_off[S::LOADS], b_off[S::LOADS], sc_off;
    int wave, chunk, lim = 0;
    __device__ int chunk_of(int i) const { return chunk ^ (4 * ((wave * S::LOADS + i) & 1)); }
    __device__ void init(const Fp8Params& p, int wave_, int lane, int nb) {
        wave = wave_;
        at.nb = nb;
        chunk = (lane & 7) ^ (lane >> 4);  // of the even loads
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) {
            const int r = 8 * (wave * S::LOADS + i) + (lane >> 3), c = chunk_of(i);
            a_off[i] = (uint32_t)r * (uint32_t)p.lda + c * 16;
            b_off[i] = (uint32_t)r * (uint32_t)p.ldb + c * 16;
        }
        sc_off = 4 * (uint32_t)(64 * (wave & (TILE / 64 - 1)) + lane);
    }
    __device__ void load(const Fp8Params& p, int d, uint32_t slot) {
        constexpr uint32_t FAR = 0x80000000u;  // past any window
        if (!FULL && d == 0) lim = at.chunks(p);
        if (d < S::LOADS) {
            dma16(at.wb, FULL || chunk_of(d) < lim ? b_off[d] : FAR, slot + S::CODES + (wave * S::LOADS + d) * 1024);
        } else if (d >= S::LOADS + 2) {
            const int i = d - S::LOADS - 2;
            dma16(at.wa, FULL || chunk_of(i) < lim ? a_off[i] : FAR, slot + (wave * S::LOADS + i) * 1024);
        } else if (d == S::LOADS) {
            dma4(at.wsa, sc_off, slot + S::SA + 256 * (wave & (TILE / 64 - 1)));
        } else if constexpr (TILES) {
            dma4(at.wsb, sc_off & 255, slot + S::SB + 256 * at.nb);
        } else {
            dma4(at.wsb, sc_off, slot + S::SB + 256 * (wave & (TILE / 64 - 1)));
        }
    }
};

// fp32 results, many units: 128 x 128 outputs of 4 waves, a wave 64 x 64; ring of 2, two
// workgroups per CU, which cover each other's waits. A unit's first step is loaded
// before the previous unit's epilogue, which stages through the other slot. Bound by
// the issue port: a matrix instruction takes 20 clocks of it and 32 of the matrix
// cores, and each of the 8 vector instructions that widen and scale for it 4. T 32768,
// 4096 x 1024 290 to 300 us, 0.93 PFLOP/s, with 9 of them for the split sums; a plain bf16
// product would take 198.
template <bool TILES, bool SPLIT, bool BETA>
__global__ __launch_bounds__(256, 2) void fp8_wide_kernel(Fp8Params p, LinearPlan pl) {
    constexpr int TILE = 128, WT = 64, MI = 2;
    using S = Slot<TILE, 4>;
    static_assert(4 * Stage<true, MI>::BYTES <= S::BYTES, "the epilogue stages in a slot");
    __shared__ uint4 lds_raw[2 * S::BYTES / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT, row = lane & 31, h = lane >> 5;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) return;
    Loader<TILE, 4, TILES, SPLIT, false> ld;
    ld.init(p, wave, lane, 0);
    ld.at.vl = vb;
    ld.at.set(p, u);
    int sl = 0, slot = 0;
    auto load_step = [&]() {
#pragma unroll
        for (int d = 0; d < S::ND; ++d) ld.load(p, d, lds0 + sl * S::BYTES);
        sl ^= 1;
        ld.at.next(p, pl, workgroups);
    };
    auto operand = [&](const uint8_t* t, int r) { return widen(read_codes(t, r, h)); };
    f32x16 acc[MI][MI];
    clear(acc);
    load_step();
    for (;;) {
        for (int k = u.kbeg; k < u.kend; k += kFp8Block) {
            wait_vm<0>();
            lds_barrier();  // step k is whole in LDS, and the slot before is read
            load_step();    // past the last unit: zeros
            const uint8_t* t = lds + slot * S::BYTES;
            const float* sa = reinterpret_cast<const float*>(t + S::SA);
            const float* sb = reinterpret_cast<const float*>(t + S::SB);
            Wide a[MI];
            float s[MI];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                a[i] = operand(t, wrow + 32 * i + row);
                s[i] = sa[wrow + 32 * i + row];
                if constexpr (TILES) s[i] *= sb[0];
            }
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                const Wide b = operand(t + S::CODES, wcol + 32 * j + row);
                f32x4 sn[4];
                if constexpr (!TILES)
#pragma unroll
                    for (int q = 0; q < 4; ++q) sn[q] = *reinterpret_cast<const f32x4*>(sb + wcol + 32 * j + 8 * q + 4 * h);
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const f32x16 d = mma32(b, a[i]);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        acc[i][j][r] = __builtin_fmaf(d[r], TILES ? s[i] : s[i] * sn[r >> 2][r & 3], acc[i][j][r]);
                }
            }
            slot ^= 1;
        }
        lds_barrier();  // the last step's slot is read: the epilogue stages there
        finish_unit<TILE, true, MI, SPLIT, BETA, false>(acc, lds + (slot ^ 1) * S::BYTES + wave * Stage<true, MI>::BYTES, p, u, p.M, p.N,
                                                wrow, wcol);
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) break;
        clear(acc);
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// fp32 results, few units, and bf16 results on 64 x 64 tiles: TILE x TILE outputs of 4
// waves, a wave a quarter of them; a ring of 4, filled ahead, whose steps' operands
// are read one step ahead too. A step of 64 x 64 is bound by its instructions, of
// which one 32 x 32 sum a wave has the fewest (T 777, N 1024, K 4096 in one group 15.1 us;
// with 16 x 16 sums, four in flight, 17.4 on 4 waves and 16.3 on 8). The stream does not
// stop between units; the epilogue stages through the slot whose step is in registers
// already.
// GROUPS 2, where there is a CU for every unit: two such groups of waves, each with its
// ring and half of the reduction; the first adds the second's sums to its own.
template <int TILE, bool TILES, bool F32, bool SPLIT, bool BETA, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, (TILE == 128 ? 1 : 2)) void fp8_quarter_kernel(Fp8Params p, LinearPlan pl) {
    constexpr int WT = TILE / 2, MI = WT / 32, RING = 4;
    using S = Slot<TILE, 4>;
    static_assert(4 * Stage<F32, MI>::BYTES <= S::BYTES, "the epilogue stages in a slot");
    static_assert(GROUPS == 1 || (!SPLIT && MI == 1 && 4 * 4096 <= S::BYTES), "a group's sums pass through a slot");
    __shared__ uint4 lds_raw[GROUPS * RING * S::BYTES / 16];
    const int lane = threadIdx.x & 63;
    const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw) + group * RING * S::BYTES;
    const uint32_t lds0 = lds_u32(lds);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT, row = lane & 31, h = lane >> 5;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) return;
    Loader<TILE, 4, TILES, SPLIT, false> ld;
    ld.init(p, wave, lane, 0);
    ld.at.vl = vb;
    ld.at.set(p, GROUPS == 1 ? u : half_of(u, group));
    int sl = 0, slot = 0;  // of the next loads, of the step in registers
    auto load_step = [&]() {
#pragma unroll
        for (int d = 0; d < S::ND; ++d) ld.load(p, d, lds0 + sl * S::BYTES);
        sl = (sl + 1) & (RING - 1);
        ld.at.next(p, pl, workgroups);
    };
    struct Step {
        Codes a[MI], b[MI];
        float s[MI];
        f32x4 sn[MI][4];
    } f[2];
    auto read_step = [&](Step& t, int slot) {
        const uint8_t* at = lds + slot * S::BYTES;
        const float* sa = reinterpret_cast<const float*>(at + S::SA);
        const float* sb = reinterpret_cast<const float*>(at + S::SB);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            t.a[i] = read_codes(at, wrow + 32 * i + row, h);
            t.b[i] = read_codes(at + S::CODES, wcol + 32 * i + row, h);
            t.s[i] = sa[wrow + 32 * i + row];
            if constexpr (TILES) {
                t.s[i] *= sb[0];
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) t.sn[i][q] = *reinterpret_cast<const f32x4*>(sb + wcol + 32 * i + 8 * q + 4 * h);
            }
        }
    };
    f32x16 acc[MI][MI];
    clear(acc);
    // multiplies the step in t and reads the next one into t2
    auto step = [&](const Step& t, Step& t2) {
        wait_vm<(RING - 2) * S::ND>();
        lds_barrier();  // the next step is whole in LDS, and this one's slot is read
        load_step();    // past the last unit: zeros
        slot = (slot + 1) & (RING - 1);
        read_step(t2, slot);
        __builtin_amdgcn_sched_barrier(0);
        using Operand = std::conditional_t<F32, Wide, Codes>;
        auto operand = [](const Codes& c) {
            if constexpr (F32) return widen(c);
            else return c;
        };
        Operand a[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = operand(t.a[i]);
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            const Operand b = operand(t.b[j]);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const f32x16 d = mma32(b, a[i]);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[i][j][r] = __builtin_fmaf(d[r], TILES ? t.s[i] : t.s[i] * t.sn[j][r >> 2][r & 3], acc[i][j][r]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int n = 0; n < RING; ++n) load_step();
    wait_vm<(RING - 1) * S::ND>();
    lds_barrier();
    read_step(f[0], 0);
    for (;;) {
        int left = (u.kend - u.kbeg + kFp8Block - 1) / kFp8Block;
        if constexpr (GROUPS == 2) left = (left + 1) / 2;  // the second's last step may be one of zeros
        for (; left >= 2; left -= 2) {
            step(f[0], f[1]);
            step(f[1], f[0]);
        }
        if (left > 0) {
            step(f[0], f[1]);
            f[0] = f[1];
        }
        lds_barrier();  // the slot of the step in registers is read: the epilogue stages there
        if constexpr (GROUPS == 2) {
            f32x4* sums = reinterpret_cast<f32x4*>(reinterpret_cast<uint8_t*>(lds_raw) + (RING + slot) * S::BYTES + wave * 4096) + lane;
            if (group == 1) {
#pragma unroll
                for (int q = 0; q < 4; ++q) sums[64 * q] = f32x4{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
            }
            lds_barrier();
            if (group == 1) break;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 o = sums[64 * q];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[0][0][4 * q + e] += o[e];
            }
        }
        finish_unit<TILE, F32, MI, SPLIT, BETA, false>(acc, lds + slot * S::BYTES + wave * Stage<F32, MI>::BYTES, p, u, p.M, p.N, wrow, wcol);
        if constexpr (GROUPS == 2) break;  // a unit a workgroup
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) break;
        clear(acc);
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// ---- sums of 16 x 16 ---------------------------------------------------------------
// acc[i][j][e] = C[m][c] with m = 16 i + lane % 16 and c = 16 j + 4 (lane / 16) + e
// in a wave's outputs.

// Outputs to memory: 16 rows at a time go through the wave's own LDS (NJ * 512
// bytes), so that a row's 16 NJ columns leave as one run of 16-byte stores; no
// barrier. `out` is the wave's first output; rows and columns past the last ones are
// dropped by the hardware's bounds.
template <bool BETA, int MI, int NJ>
__device__ __forceinline__ void store_wave16(f32x4 (&acc)[MI][NJ], uint8_t* st, uint16_t* out, int64_t ld, int rows, int cols,
                                             float beta) {
    constexpr uint32_t FAR = 0x80000000u;
    constexpr int CH = 2 * NJ, RPI = 64 / CH, K = 16 / RPI;  // chunks of a staged row, rows per store, stores
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // the addresses below are not kept through the main loop
    const int lr = lane & 15, g = lane >> 4, cl = lane % CH;
    const uint32_t row = (uint32_t)(ld * 2);
    rows = min(rows, 16 * MI);
    cols = min(cols, 16 * NJ);
    const __amdgpu_buffer_rsrc_t win = __builtin_amdgcn_make_buffer_rsrc(out, 0, (int)output_window(rows, row, cols, 2), 0x00020000);
    u32x2 old[2][NJ];
    auto load_old = [&](int i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int c = 16 * j + 4 * g;
            old[i & 1][j] = __builtin_amdgcn_raw_buffer_load_b64(win, c < cols ? (int)((uint32_t)(16 * i + lr) * row + 2 * c) : (int)FAR, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (BETA) load_old(0);
    uint4 v[K];
    auto store = [&](int i) {
        uint32_t at = 8 * cl < cols ? (uint32_t)(16 * i + lane / CH) * row + 16 * cl : FAR;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[k]), win, (int)at, 0, 2);
            at += RPI * row;
        }
    };
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        if constexpr (BETA)
            if (i + 1 < MI) load_old(i + 1);
        uint2 half[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            f32x4 f = acc[i][j];
            if constexpr (BETA) {
                const u32x2 o = old[i & 1][j];
                f = f + beta * f32x4{bf_lo(o[0]), bf_hi(o[0]), bf_lo(o[1]), bf_hi(o[1])};
            }
            half[j] = make_uint2(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]));
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i > 0) store(i - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            *reinterpret_cast<uint2*>(st + lr * (16 * CH) + (((2 * j + (g >> 1)) ^ (lr & (CH - 1))) * 16) + (g & 1) * 8) = half[j];
        wave_lds_order();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int r = lane / CH + RPI * k;
            v[k] = *reinterpret_cast<const uint4*>(st + r * (16 * CH) + ((cl ^ (r & (CH - 1))) * 16));
        }
        wave_lds_order();
    }
    store(MI - 1);
}

// bf16 results, not many units: 128 x 128 outputs of 8 waves, a wave 64 x 32; a ring of
// 4 steps, filled ahead, whose operands are read one step ahead too, so that a step
// waits for neither. Sums of 16 x 16, four of them in flight as in the kernel for
// large products. A step takes 0.6 us (0.85 on 4 waves, with 32 x 32 sums or 16 x 16,
// whatever its loads did: a lone wave per SIMD is bound by its instructions). The
// stream does not stop between units; the epilogue stages through the slot whose step
// is in registers already.
template <bool TILES, bool SPLIT, bool BETA>
__global__ __launch_bounds__(512, 2) void fp8_deep_kernel(Fp8Params p, LinearPlan pl) {
    constexpr int TILE = 128, RING = 4, MI = 4, NJ = 2, NQ = MI * NJ, DEPTH = 3;
    using S = Slot<TILE, 8>;
    static_assert(8 * NJ * 512 <= S::BYTES && (RING - 1) * S::ND < 64, "the epilogue stages in a slot; what a wait counts");
    __shared__ uint4 lds_raw[RING * S::BYTES / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 2) * 64, wcol = (wave & 3) * 32, row = lane & 15, g = lane >> 4;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) return;
    Loader<TILE, 8, TILES, SPLIT, false> ld;
    ld.init(p, wave, lane, 0);
    ld.at.vl = vb;
    ld.at.set(p, u);
    int sl = 0, slot = 0;  // of the next loads, of the step in registers
    auto load_step = [&]() {
#pragma unroll
        for (int d = 0; d < S::ND; ++d) ld.load(p, d, lds0 + sl * S::BYTES);
        sl = (sl + 1) & (RING - 1);
        ld.at.next(p, pl, workgroups);
    };
    struct Scales {
        float m[MI];   // of a's rows (tiles: times b's)
        f32x4 n[NJ];   // rows: of b's
    };
    struct Step {
        i32x8 a[MI], b[NJ];
        Scales s;
    } f[2];
    Scales before;  // of the step whose last sums are still in flight
    auto read_step = [&](Step& t, int slot) {
        const uint8_t* at = lds + slot * S::BYTES;
        const float* sa = reinterpret_cast<const float*>(at + S::SA);
        const float* sb = reinterpret_cast<const float*>(at + S::SB);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            t.a[i] = read_codes16(at, wrow + 16 * i + row, g);
            t.s.m[i] = sa[wrow + 16 * i + row];
            if constexpr (TILES) t.s.m[i] *= sb[0];
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            t.b[j] = read_codes16(at + S::CODES, wcol + 16 * j + row, g);
            if constexpr (!TILES) t.s.n[j] = *reinterpret_cast<const f32x4*>(sb + wcol + 16 * j + 4 * g);
        }
    };
    f32x4 acc[MI][NJ], d[DEPTH + 1];
    auto start = [&]() {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            before.m[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) before.n[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q <= DEPTH; ++q) d[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    // sums q are scaled and added
    auto add = [&](const Scales& s, int q) {
        const int i = q / NJ, j = q % NJ;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(d[q & DEPTH][e], TILES ? s.m[i] : s.m[i] * s.n[j][e], acc[i][j][e]);
        asm volatile("" : "+v"(acc[i][j]));  // here, not later: the sums in flight are few
    };
    // multiplies the step in t and reads the next one into t2
    auto step = [&](const Step& t, Step& t2) {
        wait_vm<(RING - 2) * S::ND>();
        lds_barrier();  // the next step is whole in LDS, and this one's slot is read
        load_step();    // past the last unit: zeros
        slot = (slot + 1) & (RING - 1);
        read_step(t2, slot);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            d[q & DEPTH] = mma16<false>(t.b[q % NJ], t.a[q / NJ]);
            __builtin_amdgcn_sched_barrier(0);
            if (q < DEPTH) add(before, NQ - DEPTH + q);
            else add(t.s, q - DEPTH);
            __builtin_amdgcn_sched_barrier(0);
        }
        before = t.s;
    };
#pragma unroll
    for (int n = 0; n < RING; ++n) load_step();
    wait_vm<(RING - 1) * S::ND>();
    lds_barrier();
    read_step(f[0], 0);
    for (;;) {
        start();
        int left = (u.kend - u.kbeg + kFp8Block - 1) / kFp8Block;
        for (; left >= 2; left -= 2) {
            step(f[0], f[1]);
            step(f[1], f[0]);
        }
        if (left > 0) {
            step(f[0], f[1]);
            f[0] = f[1];
        }
#pragma unroll
        for (int q = NQ - DEPTH; q < NQ; ++q) add(before, q);
        lds_barrier();  // the slot of the step in registers is read: the epilogue stages there
        const int rows = p.M - u.m0 - wrow, cols = p.N - u.c0 - wcol;
        if (rows > 0 && cols > 0) {
            if constexpr (SPLIT) {
                float* o = p.part + (int64_t)u.part * TILE * TILE + (wrow + row) * TILE + wcol + 4 * g;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        if (16 * i + row < rows && 16 * j + 4 * g < cols) *reinterpret_cast<f32x4*>(o + 16 * i * TILE + 16 * j) = acc[i][j];
            } else {
                store_wave16<BETA>(acc, lds + slot * S::BYTES + wave * NJ * 512,
                                   static_cast<uint16_t*>(p.y) + (int64_t)(u.m0 + wrow) * p.ldy + u.c0 + wcol, p.ldy, rows, cols, p.beta);
            }
        }
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) break;
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// ---- large products ------------------------------------------------------------------
// 256 x 256 outputs of 8 waves, a wave 128 x 64; one workgroup, two waves per SIMD.
// Half the reads from L2 of 128 x 128. The sums have to be vector registers, since
// the vector unit scales and adds: 128 a wave.
// 16 x 16 sums, whose instruction takes a whole block of 128: four of them are in
// flight, and the vector unit adds the one issued three before while the next run,
// so that neither waits for the other. T 32768, N 4096, K 1024 138 to 148 us, 1.9
// PFLOP/s (32 x 32 sums, two instructions a block, with one in flight: 162); T = N = K =
// 8192 442 to 459, 2.45, at the power limit.
// Ring of 2. A wave holds a step's b and streams its a. Behind the last but one
// read the whole slot is in registers: the barrier stands there; the last sums cover
// the next slot's first reads, and the freed slot's loads begin. The stream does not
// stop between units: their outputs go through LDS of its own, behind the next
// unit's loads.
struct Large {
    static constexpr int TILE = 256, WAVES = 8, MI = 8, NJ = 4, DEPTH = 3;
    using S = Slot<TILE, WAVES>;
    static constexpr int ST0 = 2 * S::BYTES, STB = 16 * 128, LDS = ST0 + WAVES * STB;
    static constexpr int STORES = 2 * MI;      // of a wave's outputs
    static constexpr int EARLY = S::LOADS + 2; // a step's loads ahead of its a
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <bool FULL, bool BETA>
__global__ __launch_bounds__(512, 2) void fp8_large_kernel(Fp8Params p, LinearPlan pl) {
    using G = Large;
    using S = G::S;
    constexpr int MI = G::MI, NJ = G::NJ, TILE = G::TILE, DEPTH = G::DEPTH, NQ = MI * NJ;
    __shared__ uint4 lds_raw[G::LDS / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 2) * 128, wcol = (wave & 3) * 64, row = lane & 15, g = lane >> 4;
    const int nb = (wave & 3) >> 1;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, false>(pl, p.K, vb, u)) return;
    Loader<TILE, G::WAVES, true, false, FULL> ld;
    ld.init(p, wave, lane, nb);
    ld.at.vl = vb;
    ld.at.set(p, u);
    int sll = 0;  // slot of the next loads
    auto load = [&](int d) { ld.load(p, d, lds0 + sll * S::BYTES); };
    auto next_loads = [&]() {
        sll ^= 1;
        ld.at.next(p, pl, workgroups);
    };

    i32x8 a[2], b[NJ];
    float s[MI], next[2];
    auto read_a = [&](int i, int sl) { a[i & 1] = read_codes16(lds + sl * S::BYTES, wrow + 16 * i + row, g); };
    auto read_b = [&](int j, int sl) { b[j] = read_codes16(lds + sl * S::BYTES + S::CODES, wcol + 16 * j + row, g); };
    // the next step's scales, while the last two rows' are still in use
    auto read_scales = [&](int sl) {
        const uint8_t* t = lds + sl * S::BYTES;
        const float sb = *reinterpret_cast<const float*>(t + S::SB + 256 * nb);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            float& to = i < MI - 2 ? s[i] : next[i - MI + 2];
            to = sb * reinterpret_cast<const float*>(t + S::SA)[wrow + 16 * i + row];
        }
    };
    f32x4 acc[MI][NJ], d[DEPTH + 1];
    float last = 0.0f;  // the scale of the sums still in flight from the step before
    // sums q of this step (q < 0: the step before) are scaled and added
    auto add = [&](int q) {
        f32x4& t = acc[(q + NQ) % NQ / NJ][(q + NQ) % NQ % NJ];
        const float by = q < 0 ? last : s[q / NJ];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __builtin_fmaf(d[(q + NQ) & DEPTH][e], by, t[e]);
        asm volatile("" : "+v"(t));  // here, not later: the sums in flight are few
    };

    // ---- stream
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < S::ND; ++n) load(n);
        next_loads();
    }
    wait_vm<S::ND>();
    lds_barrier();
    int sl = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) read_b(j, sl);
    read_a(0, sl);
    read_scales(sl);
    bool stored = false;  // the last unit's outputs are STORES stores behind the loads
    uint8_t* st = lds + G::ST0 + wave * G::STB;
    for (;;) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                asm volatile("" : "+v"(acc[i][j]));  // no first step of its own
            }
        last = 0.0f;  // and no sums in flight: times zero, a NaN of the unit before would stay one
#pragma unroll
        for (int q = 0; q <= DEPTH; ++q) d[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < p.K; k += kFp8Block) {
            s[MI - 2] = next[0];
            s[MI - 1] = next[1];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const int i = q / NJ, j = q % NJ;
                if (q == NJ) lds_barrier();  // this slot's b and scales are read
                if (q == NQ - NJ) {
                    if (stored) wait_vm<G::STORES + G::EARLY>();
                    else wait_vm<G::EARLY>();
                    stored = false;
                    lds_barrier();  // all of this slot is read, the other one is whole
                    sl ^= 1;
                }
                d[q & DEPTH] = mma16<false>(b[j], a[i & 1]);
                __builtin_amdgcn_sched_barrier(0);
                if (j == 0) read_a((i + 1) % MI, sl);
                if (q == NQ - NJ + 1) read_scales(sl);
                if (i == MI - 1) read_b(j, sl);
                if (i > 0 && i <= G::EARLY && j == 1) load(i - 1);
                if (i == MI - 1) load(G::EARLY + j);
                add(q - DEPTH);
                __builtin_amdgcn_sched_barrier(0);
            }
            next_loads();
            last = s[MI - 1];
        }
#pragma unroll
        for (int q = -DEPTH; q < 0; ++q) add(q);
        const int rows = p.M - u.m0 - wrow, cols = p.N - u.c0 - wcol;
        stored = rows > 0 && cols > 0;
        if (stored)
            store_wave16<BETA>(acc, st, static_cast<uint16_t*>(p.y) + (int64_t)(u.m0 + wrow) * p.ldy + u.c0 + wcol, p.ldy, rows, cols,
                               p.beta);
        vb += gridDim.x;
        if (!unit_at<TILE, false>(pl, p.K, vb, u)) break;
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// y = beta y, where the reduction is empty: 16 bytes a thread, by strides.
template <bool F32>
__global__ __launch_bounds__(256) void fp8_scale_kernel(Fp8Params p) {
    constexpr int PER = F32 ? 4 : 8;
    const int pieces = p.N / PER;
    const int64_t all = (int64_t)p.M * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i / pieces * p.ldy + i % pieces * PER;
        if constexpr (F32) {
            f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(p.y) + at);
            *y = p.beta != 0.0f ? p.beta * *y : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        } else {
            uint4* y = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + at);
            float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (p.beta != 0.0f) {
                unpack8(*y, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= p.beta;
            }
            *y = pack8(v);
        }
    }
}

// Blocks of outputs are the largest of which there are enough for 3/4 of the CUs,
// and 16 x 16 otherwise: a larger block reads its operands less often, but a CU
// without one is idle. us with 16 x 16 / 16 x 32 (columns) / 32 x 32 / 64 x 64:
// M 1, N 4096, K 1024 2.9 / 3.3 / 3.9 / 7.3; M 64, N 1024, K 4096 4.4 / 5.1 / 5.8 /
// 11.5; M 128, N 1024, K 4096 7.1 / 5.5 / 5.8 / 11.5; M 128, N 4096, K 1024 6.6 / 7.2
// / 5.7 / 7.8; M 256, N 4096, K 1024 11.3 / 11.1 / 9.3 / 8.5.
template <bool TILES, bool F32, int RB, int NB>
void launch_rows_as(const Fp8Params& p, hipStream_t s) {
    const int64_t grid = (int64_t)((p.N + 16 * NB - 1) / (16 * NB)) * ((p.M + 16 * RB - 1) / (16 * RB));
    if (RB == 4 || p.K <= 8 * kFp8Block) fp8_rows_kernel<TILES, F32, RB, NB, true><<<(unsigned)grid, 512, 0, s>>>(p);
    else fp8_rows_kernel<TILES, F32, RB, NB, RB == 4><<<(unsigned)grid, 512, 0, s>>>(p);
}
template <bool TILES, bool F32>
void launch_rows(const Fp8Params& p, int cus, hipStream_t s) {
    switch (fp8_rows_block(p.M, p.N, cus)) {
        case 64: launch_rows_as<TILES, F32, 4, 4>(p, s); break;
        case 32: launch_rows_as<TILES, F32, 2, 2>(p, s); break;
        case 24: launch_rows_as<TILES, F32, 1, 2>(p, s); break;
        default: launch_rows_as<TILES, F32, 1, 1>(p, s); break;
    }
}

template <int TILE, bool TILES, bool F32, bool SPLIT, bool BETA>
void launch_units(const Fp8Params& p, const LinearPlan& pl, int units, int cus, hipStream_t s) {
    const int grid = fp8_grid(TILE, F32, units, cus);
    if constexpr (F32 && TILE == 128) {
        if (units > cus) {
            fp8_wide_kernel<TILES, SPLIT, BETA><<<grid, 256, 0, s>>>(p, pl);
            return;
        }
    }
    if constexpr (TILE == 64 && !SPLIT) {
        if (fp8_paired(TILE, units, p.K, cus)) {
            fp8_quarter_kernel<TILE, TILES, F32, SPLIT, BETA, 2><<<grid, 512, 0, s>>>(p, pl);
            return;
        }
    }
    if constexpr (F32 || TILE == 64) fp8_quarter_kernel<TILE, TILES, F32, SPLIT, BETA, 1><<<grid, 256, 0, s>>>(p, pl);
    else fp8_deep_kernel<TILES, SPLIT, BETA><<<grid, 512, 0, s>>>(p, pl);
}
template <int TILE, bool TILES, bool F32>
void launch_tiles(const Fp8Params& p, const LinearPlan& pl, int cus, hipStream_t s) {
    if (pl.whole > 0) {
        if (p.beta == 0.0f) launch_units<TILE, TILES, F32, false, false>(p, pl, pl.whole, cus, s);
        else launch_units<TILE, TILES, F32, false, true>(p, pl, pl.whole, cus, s);
    }
    if (pl.tail > 0) {
        launch_units<TILE, TILES, F32, true, false>(p, pl, pl.tail * pl.parts, cus, s);  // the sums add what is there
        constexpr int SLABS = TILE / (256 / (TILE / 4));
        linear_fixup_kernel<TILE, F32><<<pl.tail * SLABS, 256, 0, s>>>(p, pl, p.M, p.N);
    }
}

void launch_large(const Fp8Params& p, const LinearPlan& pl, int cus, hipStream_t s) {
    const int grid = fp8_grid(256, false, pl.whole, cus);
    const bool full = p.K % kFp8Block == 0;
    if (p.beta == 0.0f) full ? fp8_large_kernel<true, false><<<grid, 512, 0, s>>>(p, pl) : fp8_large_kernel<false, false><<<grid, 512, 0, s>>>(p, pl);
    else full ? fp8_large_kernel<true, true><<<grid, 512, 0, s>>>(p, pl) : fp8_large_kernel<false, true><<<grid, 512, 0, s>>>(p, pl);
}

template <bool TILES, bool F32>
void launch(const Fp8Params& p, hipStream_t s) {
    const int cus = cu_count();
    if (p.K == 0) {
        const int64_t blocks = std::min<int64_t>(((int64_t)p.M * (p.N / 4) + 255) / 256, 16 * (int64_t)cus);
        fp8_scale_kernel<F32><<<(unsigned)blocks, 256, 0, s>>>(p);
        return;
    }
    const Fp8Plan pl = fp8_plan(TILES, F32, p.M, p.N, p.K, cus);
    if (pl.kernel == FP8_ROWS_KERNEL) launch_rows<TILES, F32>(p, cus, s);
    else if (pl.kernel == FP8_LARGE_KERNEL) launch_large(p, pl.tiles, cus, s);
    else if (pl.tiles.tile == 64) launch_tiles<64, TILES, F32>(p, pl.tiles, cus, s);
    else launch_tiles<128, TILES, F32>(p, pl.tiles, cus, s);
}

}  // namespace

size_t fp8_workspace(int M, int N, int K) { return fp8_workspace_bound(M, N, K, cu_count()); }

hipError_t launch_fp8_matmul(bool tiles, bool f32, const Fp8Params& p, hipStream_t s) {
    if (tiles) f32 ? launch<true, true>(p, s) : launch<true, false>(p, s);
    else f32 ? launch<false, true>(p, s) : launch<false, false>(p, s);
    return hipGetLastError();
}

}  // namespace tmt
