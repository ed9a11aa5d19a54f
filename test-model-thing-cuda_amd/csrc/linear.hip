// linear.hip -- products of the linear layer on microscaled numbers.
//
// Every operand value inside bf16's range is exact in bf16 (an e2m1 code has
// two significant bits, an e4m3 code four, and scales are powers of two), so a
// product with bf16 rows is one bf16 matrix product with fp32 sums of exact
// terms.
//
//   FORWARD  Y[t][n] = sum_k X[t][k] W[n][k]     X and the codes along k
//   MATMUL   the same with X in MXFP4, on the scaled matrix instructions
//   DX       dX[t][k] = sum_n dY[t][n] W[n][k]   codes across the reduction
//   DW       dW[n][k] = sum_t dY[t][n] X[t][k]   both operands across it
//
// Tiles of 256 x 256 outputs (one workgroup of 4 waves per CU, a wave 128 x
// 128 = 4 x 4 v_mfma_f32_32x32x16_bf16 tiles) or 128 x 128 (two workgroups
// per CU, a wave 64 x 64); linear_plan chooses. Workgroups are persistent and
// walk units (a tile, or a part of one along the reduction). All operands
// stream from global memory into LDS rings by direct loads, and the stream
// does not stop between units: a unit's last steps already load the next
// one's first, and its epilogue stages outputs in LDS of its own, so the
// matrix cores wait for neither a first load nor a drained ring.
//
// FORWARD expands the codes where a fragment is read (8 codes, 4 bytes of
// LDS, a lane: four conversion instructions under the MFMAs). In DX and DW
// the reduction runs across the codes' rows, every element of a fragment
// with a scale of its own, so each code is expanded once per workgroup: raw
// codes land in LDS, 32 reduction rows a sub-step, are converted one sub-step
// ahead into a row-contiguous bf16 tile, and fragments are read from that with
// the transposing ds_read_b64_tr_b16.
#include <algorithm>
#include <type_traits>

#include "moe_internal.hpp"
#include "mx_format.hpp"
#include "tile_stream.hpp"

namespace tmt {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// What is read past the end of a reduction.
__device__ __align__(16) const uint32_t zero_piece[4] = {0, 0, 0, 0};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes per lane from the lane's 64-bit address into LDS at lds_base + 16 * lane
// (lds_base wave-uniform); M0 is written, one wait state ahead of the load.
__device__ __forceinline__ void dma16v(const void* g, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds_base) : "m0");
}
#pragma clang diagnostic pop

// 8 e2m1 codes and their scale operand as 8 bf16.
__device__ __forceinline__ uint4 expand_fp4(uint32_t w, float sc) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3)));
}
// 8 e4m3 codes.
__device__ __forceinline__ uint4 expand_fp8(uint2 w, float sc) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, sc, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, sc, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, sc, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, sc, true)));
}

// ---- forward -------------------------------------------------------------------
// Per K = 64 step: activations [TILE rows][64] bf16 (rows of 128 bytes, 16-byte
// chunks XOR-swizzled by row / 2), codes [TILE rows][32 bytes] and scales [2
// blocks][TILE]. Rings of 3: step s loads step s + 2.
template <int TILE>
struct Fwd {
    static constexpr int WT = TILE / 2, MI = WT / 32;
    static constexpr int A_BYTES = TILE * 128, A_LOADS = A_BYTES / 4096;  // 1 KiB loads per wave
    static constexpr int Q_BYTES = TILE * 32, Q_LOADS = Q_BYTES / 4096;
    static constexpr int B_BYTES = Q_BYTES + 1024;  // codes, then scales (2 * TILE bytes of a 1 KiB load)
    static constexpr int A0 = 0, B0 = 3 * A_BYTES, ST0 = B0 + 3 * B_BYTES;
    static constexpr int LDS = ST0 + 4 * Stage<false, MI>::BYTES;
    static constexpr int WGS = TILE == 256 ? 1 : 2;
    static_assert(LDS * WGS <= 160 * 1024, "LDS");
};

template <int TILE, bool SPLIT, bool BETA>
__global__ __launch_bounds__(256, (Fwd<TILE>::WGS)) void linear_fwd_kernel(LinearParams p, LinearPlan pl) {
    using G = Fwd<TILE>;
    constexpr int MI = G::MI, WT = G::WT;
    __shared__ uint4 lds_raw[G::LDS / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT;
    const int K = p.K;

    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, K, vb, u)) return;

    // ---- the next step to load
    FwdCursor<TILE, SPLIT> at;
    at.vl = vb;
    at.set(p, u);
    int sll = 0;
    uint32_t a_off[G::A_LOADS], q_off[G::Q_LOADS];
#pragma unroll
    for (int i = 0; i < G::A_LOADS; ++i) {
        const int r = 8 * (wave * G::A_LOADS + i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        a_off[i] = (uint32_t)r * (uint32_t)(p.ldx * 2) + c * 16;
    }
#pragma unroll
    for (int i = 0; i < G::Q_LOADS; ++i) {
        const int s = (wave * G::Q_LOADS + i) * 64 + lane, m = s >> 1, half = (s & 1) ^ ((m >> 3) & 1);
        q_off[i] = (uint32_t)m * (uint32_t)(K / 2) + half * 16;
    }
    const uint32_t sc_off = (uint32_t)((lane / (TILE / 16)) & 1) * (uint32_t)p.wlds + 16 * (lane % (TILE / 16));
    // load d of the step: the codes, the scales, the activations
    auto load = [&](int d) {
        const uint32_t a = lds0 + G::A0 + sll * G::A_BYTES, b = lds0 + G::B0 + sll * G::B_BYTES;
        if (d < G::Q_LOADS) dma16(at.wq, q_off[d], b + (wave * G::Q_LOADS + d) * 1024);
        else if (d == G::Q_LOADS) dma16(at.wsc, sc_off, b + G::Q_BYTES);
        else dma16(at.wa, a_off[d - G::Q_LOADS - 1], a + (wave * G::A_LOADS + d - G::Q_LOADS - 1) * 1024);
    };
    auto next_loads = [&]() {
        sll = sll == 2 ? 0 : sll + 1;
        at.next(p, pl, workgroups);
    };

    // ---- fragments -----------------------------------------------------------
    struct Frag {
        uint4 a[MI], b[MI];
    };
    struct Raw {  // the lane's codes of a K = 64 step, 8 for each k16 step, and their scales
        uint32_t q[MI][4], s[MI][2];
    };
    // k16 step s of the K = 64 step in ring slot sl
    auto read_a = [&](Frag& f, int i, int sl, int s) {
        const int r = wrow + 32 * i + (lane & 31), c = (2 * s + (lane >> 5)) ^ ((r >> 1) & 7);
        f.a[i] = *reinterpret_cast<const uint4*>(lds + G::A0 + sl * G::A_BYTES + r * 128 + c * 16);
    };
    // lane: codes k = 16 s + 8 (lane / 32) .. + 7 of row lane % 32
    auto read_codes = [&](Raw& w, int j, int sl) {
        const uint8_t* tb = lds + G::B0 + sl * G::B_BYTES;
        const int r = wcol + 32 * j + (lane & 31);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            w.q[j][s] = *reinterpret_cast<const uint32_t*>(tb + r * 32 + (((s >> 1) ^ ((r >> 3) & 1)) * 16) + 8 * (s & 1) + 4 * (lane >> 5));
#pragma unroll
        for (int b = 0; b < 2; ++b) w.s[j][b] = tb[G::Q_BYTES + b * TILE + r];
    };
    auto expand = [&](Frag& f, const Raw& w, int j, int s) { f.b[j] = expand_fp4(w.q[j][s], e8m0_operand(w.s[j][s >> 1])); };
    f32x16 acc[MI][MI];
    constexpr int ND = G::A_LOADS + G::Q_LOADS + 1, NM = MI * MI;
    // MFMAs of one k16 step. Under them, in the slots between two: the reads of
    // the next step's activations (f2: k16 step s of ring slot sl; the first
    // also reads its K = 64 step's codes, which the others find in registers),
    // the conversion of its codes and loads [d0, d0 + dn). A wave's
    // instructions issue in order and an MFMA takes 32 cycles, so what stands
    // in one slot is free up to about seven instructions; in a bunch it stalls
    // the matrix core (T = N = K = 4096: 1.72 us a step with the conversions
    // bunched, 1.43 spread).
    Raw w;
    auto mma = [&](const Frag& f, Frag& f2, int sl, int s, int d0, int dn) {
        const int c0 = s == 0 ? NM / 2 : 0;  // first slot with conversions
#pragma unroll
        for (int q = 0; q < NM; ++q) {
            const int i = q / MI, j = q % MI;
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f.b[j]),
                                                                __builtin_bit_cast(bf16x8, f.a[i]), acc[i][j], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < MI; ++r)
                if (r * NM / (4 * MI) == q) {
                    if (s == 0) read_codes(w, r, sl);
                    read_a(f2, r, sl, s);
                }
#pragma unroll
            for (int r = 0; r < MI; ++r)
                if (c0 + (2 * r + 1) * (NM - c0) / (2 * MI) == q) expand(f2, w, r, s);
#pragma unroll
            for (int d = 0; d < dn; ++d)
                if ((2 * d + 1) * NM / (2 * dn) == q) load(d0 + d);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // ---- stream ----------------------------------------------------------------
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int d = 0; d < ND; ++d) load(d);
        next_loads();
    }
    wait_vm<ND>();
    lds_barrier();
    int sl = 0;  // ring slot being multiplied
    Frag f[2];
    auto first = [&]() {  // fragments of a unit's first k16 step
#pragma unroll
        for (int r = 0; r < MI; ++r) {
            read_codes(w, r, sl);
            read_a(f[0], r, sl, 0);
        }
#pragma unroll
        for (int r = 0; r < MI; ++r) expand(f[0], w, r, 0);
    };
    first();
    uint8_t* st = lds + G::ST0 + wave * Stage<false, MI>::BYTES;
    for (;;) {
        clear(acc);
        for (int k = u.kbeg; k < u.kend; k += 64) {
            mma(f[0], f[1], sl, 1, 0, ND / 3);
            mma(f[1], f[0], sl, 2, ND / 3, 2 * ND / 3 - ND / 3);
            mma(f[0], f[1], sl, 3, 2 * ND / 3, ND - 2 * ND / 3);
            next_loads();
            wait_vm<ND>();  // all but this step's loads: the next step is whole in LDS
            lds_barrier();
            sl = sl == 2 ? 0 : sl + 1;
            mma(f[1], f[0], sl, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        finish_unit<TILE, false, MI, SPLIT, BETA>(acc, st, p, u, p.T, p.N, wrow, wcol);
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, K, vb, u)) break;
        first();  // again: the fragments' registers served the epilogue
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// ---- gradients -----------------------------------------------------------------
// Sub-steps of 32 reduction rows. DX: dY [TILE rows][64] in a ring of 3 as the
// forward's activations, half of a K = 64 tile loaded per sub-step. DW: dY
// [32 t][TILE n] in a ring of 4, 16-byte chunks XOR-swizzled by 4 (t % 4).
// Raw codes [32][TILE] and scales [TILE / 32][32] in a ring of 3, bf16 tiles
// [32][TILE] (swizzled as DW's dY) in a ring of 2. Sub-step i multiplies tile
// i, expands raw i + 1, and loads raw i + 3 and the activations of sub-steps
// 4 (DX) or 3 (DW) ahead.
template <int OP, int TILE>
struct Grad {
    static constexpr bool DW = OP == LINEAR_DW;
    static constexpr int WT = TILE / 2, MI = WT / 32;
    static constexpr int A_BYTES = DW ? TILE * 64 : TILE * 128, A_SLOTS = DW ? 4 : 3;
    static constexpr int A_LOADS = TILE * 64 / 4096;  // 1 KiB loads per wave and sub-step
    static constexpr int CB = GradCodesCursor<OP, TILE, false>::CB;
    static constexpr int ROWQ = TILE / 8 * CB;        // code bytes per raw row
    static constexpr int Q_BYTES = 32 * ROWQ;
    static constexpr int Q_LOADS = (Q_BYTES + 4095) / 4096;
    static constexpr int R_BYTES = Q_BYTES + 256;     // codes, then scales
    static constexpr int B_BYTES = TILE * 64;
    static constexpr int A0 = 0, B0 = A_SLOTS * A_BYTES, R0 = B0 + 2 * B_BYTES, ST0 = R0 + 3 * R_BYTES;
    static constexpr int STB = Stage<DW, MI / 2>::BYTES;
    static constexpr int LDS = ST0 + 4 * STB;
    static constexpr int WGS = TILE == 256 ? 1 : 2;
    static_assert(LDS * WGS <= 160 * 1024, "LDS");
};


template <int OP, int TILE, bool SPLIT, bool BETA>
__global__ __launch_bounds__(256, (Grad<OP, TILE>::WGS)) void linear_grad_kernel(LinearParams p, LinearPlan pl) {
    using G = Grad<OP, TILE>;
    constexpr bool DW = G::DW;
    constexpr int MI = G::MI, WT = G::WT;
    __shared__ uint4 lds_raw[G::LDS / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT;
    const int M = DW ? p.N : p.T, C = p.K, R = DW ? p.T : p.N;

    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, R, vb, u)) return;

    // ---- the next K = 64 steps to load, of the activations and of the raw codes
    constexpr int AC = TILE / 8;                // 16-byte chunks per row of a tile across the reduction
    constexpr int PPR = G::ROWQ / 16;           // 16-byte pieces per raw row
    constexpr int QL = G::Q_BYTES / 1024;       // wave loads of a raw tile (fewer than the waves: loaded twice)
    constexpr int NA = DW ? G::A_LOADS : 2 * G::A_LOADS;
    using Codes = GradCodesCursor<OP, TILE, SPLIT>;
    const uint32_t ldb = (uint32_t)(p.ldx * 2), rowb = (uint32_t)Codes::row_bytes(p);
    GradRowsCursor<OP, TILE, SPLIT> ca;
    Codes cq;
    ca.vl = cq.vl = vb;
    ca.set(p, u);
    cq.set(p, u);
    int sla = 0, slq = 0;                       // ring slots of the next loads
    // DW and raw codes: [half][load], the lane's piece of a K = 64 step's half
    uint32_t a_off[2 * G::A_LOADS], q_off[2][G::Q_LOADS];
#pragma unroll
    for (int i = 0; i < 2 * G::A_LOADS; ++i) {
        if constexpr (DW) {  // a 32-row tile, row k, chunk c
            const int k = (64 / AC) * (wave * G::A_LOADS + i % G::A_LOADS) + lane / AC, c = (lane % AC) ^ (4 * (k & 3));
            a_off[i] = (uint32_t)(k + 32 * (i / G::A_LOADS)) * ldb + c * 16;
        } else {
            const int r = 8 * (wave * NA + i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
            a_off[i] = (uint32_t)r * ldb + c * 16;
        }
    }
#pragma unroll
    for (int i = 0; i < G::Q_LOADS; ++i) {
        const int s = ((wave * G::Q_LOADS + i) % QL) * 64 + lane;
        q_off[0][i] = (uint32_t)(s / PPR) * rowb + (s % PPR) * 16;
        q_off[1][i] = q_off[0][i] + 32 * rowb;
    }
    const uint32_t sc_off = (uint32_t)(lane >> 3) * (uint32_t)p.wlds + 4 * (lane & 7);
    constexpr int ND = G::Q_LOADS + 1 + G::A_LOADS;  // loads per wave and sub-step, raw codes first
    // Load d of a raw tile (codes, scales) or of a sub-step's activations, which
    // half of their K = 64 steps they are (DX: which half of the rows).
    auto load = [&](int d, int q_half, int a_half) {
        const uint32_t raw = lds0 + G::R0 + slq * G::R_BYTES, act = lds0 + G::A0 + sla * G::A_BYTES;
        if (d < G::Q_LOADS) {
            dma16(cq.wq, q_off[q_half][d], raw + ((wave * G::Q_LOADS + d) % QL) * 1024);
        } else if (d == G::Q_LOADS) {
            dma4(cq.wsc, sc_off + 32 * q_half, raw + G::Q_BYTES);
        } else {
            const int i = d - G::Q_LOADS - 1;
            dma16(ca.wa, a_off[a_half * G::A_LOADS + i], act + (wave * NA + i + (DW ? 0 : a_half * G::A_LOADS)) * 1024);
        }
    };
    // behind a raw tile's loads, and behind a sub-step's activations
    auto next_q = [&](int half) {
        slq = slq == 2 ? 0 : slq + 1;
        if (half == 1) cq.next(p, pl, workgroups);
    };
    auto next_a = [&](int half) {
        if (DW) sla = (sla + 1) & 3;
        else if (half == 1) sla = sla == 2 ? 0 : sla + 1;
        if (half == 1) ca.next(p, pl, workgroups);
    };
    // The lane's share of a raw tile: EP pieces of 8 codes with their scales,
    // in registers from one k16 step to the next.
    constexpr int EP = 32 * AC / 256;
    const int ec = tid % AC, er = tid / AC;
    uint2 eq[EP];
    uint32_t es[EP];
    // DW: reduction rows of the raw tiles in LDS that are not past the end, of
    // the one being multiplied first. (A checkpoint's scales behind its last row
    // are anything. DX leaves out whole k16 steps instead: N is a multiple of 16.)
    int valid[3] = {0, 0, 0};
    auto read_raw = [&](int q, int sr) {
        const uint8_t* raw = lds + G::R0 + sr * G::R_BYTES;
        const int row = er + q * (256 / AC);
        if constexpr (DW) eq[q] = *reinterpret_cast<const uint2*>(raw + row * G::ROWQ + ec * 8);
        else eq[q].x = *reinterpret_cast<const uint32_t*>(raw + row * G::ROWQ + ec * 4);
        es[q] = raw[G::Q_BYTES + (ec >> 2) * 32 + row];
    };
    auto write_piece = [&](int q, int sb, int rows) {  // expanded into bf16 slot sb
        const int row = er + q * (256 / AC);
        const float unit = e8m0_operand(!DW || row < rows ? es[q] : 127);
        uint4 v;
        if constexpr (DW) v = expand_fp8(eq[q], unit);
        else v = expand_fp4(eq[q].x, unit);
        *reinterpret_cast<uint4*>(lds + G::B0 + sb * G::B_BYTES + row * (TILE * 2) + ((ec ^ (4 * (row & 3))) * 16)) = v;
    };

    // ---- fragments -----------------------------------------------------------
    struct Frag {
        uint4 a[MI], b[MI];
    };
    // 8 reduction rows 16 s + 8 (lane / 32) .. of column cbase + lane % 32, from
    // a row-contiguous tile: inside each 16-lane group, lane r points at row
    // k0 + r / 4, columns c0 + 4 (r % 4) .. + 3, and lane i receives column
    // c0 + i of rows k0 .. k0 + 3
    auto read_across = [&](const uint8_t* t, int cbase, int s) {
        const int g = lane >> 4, r = lane & 15;
        const int col = cbase + 16 * (g & 1) + 4 * (r & 3);
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 16 * s + 8 * (g >> 1) + (r >> 2) + 4 * h;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(t + k * (TILE * 2) + (((col >> 3) ^ (4 * (k & 3))) * 16) + (col & 7) * 2));
            w[2 * h] = (uint32_t)(uint16_t)v[0] | ((uint32_t)(uint16_t)v[1] << 16);
            w[2 * h + 1] = (uint32_t)(uint16_t)v[2] | ((uint32_t)(uint16_t)v[3] << 16);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    // k16 step s of the sub-step in activation slot sa (DX: half `half` of it)
    // and bf16 slot sb. Read n of 2 MI, in the order in which the MFMAs need
    // them: a[0], b[0] .., a[1] ..
    auto read_frag = [&](Frag& f, int n, int sa, int half, int sb, int s) {
        const uint8_t* ta = lds + G::A0 + sa * G::A_BYTES;
        const uint8_t* tb = lds + G::B0 + sb * G::B_BYTES;
        if (n >= 1 && n <= MI) {
            f.b[n - 1] = read_across(tb, wcol + 32 * (n - 1), s);
            return;
        }
        const int i = n == 0 ? 0 : n - MI;
        if constexpr (DW) {
            f.a[i] = read_across(ta, wrow + 32 * i, s);
        } else {
            const int r = wrow + 32 * i + (lane & 31), c = (2 * (2 * half + s) + (lane >> 5)) ^ ((r >> 1) & 7);
            f.a[i] = *reinterpret_cast<const uint4*>(ta + r * 128 + c * 16);
        }
    };
    f32x16 acc[MI][MI];
    constexpr int NM = MI * MI;
    // MFMAs of one k16 step; slot(q) stands behind MFMA q (see the forward). A
    // step past the reduction's end (DX) is not `on`.
    auto mma = [&](const Frag& f, bool on, auto slot) {
        if (DW || on) {
#pragma unroll
            for (int q = 0; q < NM; ++q) {
                const int i = q / MI, j = q % MI;
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f.b[j]),
                                                                    __builtin_bit_cast(bf16x8, f.a[i]), acc[i][j], 0, 0, 0);
                slot(q);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int q = 0; q < NM; ++q) slot(q);
        }
    };

    // ---- stream ----------------------------------------------------------------
    // raw tiles 0 .. 2 and the activations of sub-steps 0 .. 2 (DW) or 0 .. 3
#pragma unroll
    for (int t = 0; t < 3; ++t) {
#pragma unroll
        for (int d = 0; d <= G::Q_LOADS; ++d) load(d, t & 1, 0);
        valid[t] = cq.rows - 32 * (t & 1);
        next_q(t & 1);
    }
#pragma unroll
    for (int t = 0; t < (DW ? 3 : 4); ++t) {
#pragma unroll
        for (int d = G::Q_LOADS + 1; d < ND; ++d) load(d, 0, t & 1);
        next_a(t & 1);
    }
    wait_vm<0>();
    lds_barrier();
    int sa = 0, sr = 0;  // activation slot multiplied, raw slot read next
#pragma unroll
    for (int q = 0; q < EP; ++q) read_raw(q, 0);
#pragma unroll
    for (int q = 0; q < EP; ++q) write_piece(q, 0, valid[0]);
#pragma unroll
    for (int q = 0; q < EP; ++q) read_raw(q, 1);
    sr = 2;
    lds_barrier();
    // 256 x 256 tiles read a k16 step's fragments under the MFMAs of the step
    // before. A k16 step of a 128 x 128 tile is four MFMAs, shorter than an LDS
    // read: both steps' fragments are read right behind the barrier, the second
    // step's into f[1] and f[2] in turn (step by step / so: dX T 777, N 1024, K
    // 4096 18.3 / 17.9 us, dW T 2048, N 1280, K 1280 24.7 / 24.1).
    constexpr bool PAIR = MI == 2;
    Frag f[PAIR ? 3 : 2];
    auto first = [&]() {  // fragments of a unit's first sub-step, as far as the loop has them there
#pragma unroll
        for (int n = 0; n < 2 * MI; ++n) {
            read_frag(f[0], n, sa, 0, 0, 0);
            if constexpr (PAIR) read_frag(f[1], n, sa, 0, 0, 1);
        }
    };
    first();
    uint8_t* st = lds + G::ST0 + wave * G::STB;
    for (;;) {
        clear(acc);
        for (int k = u.kbeg; k < u.kend; k += 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag& second = f[PAIR && h == 1 ? 2 : 1];
                // first k16 step: the second's fragments are read, the next
                // sub-step's codes converted, and all loads go out (LDS
                // accesses early, so that the barrier does not wait for them)
                mma(f[0], k + 32 * h < u.kend, [&](int q) {
                    if constexpr (!PAIR) {
#pragma unroll
                        for (int n = 0; n < 2 * MI; ++n)
                            if (n * NM / (4 * MI) == q) read_frag(second, n, sa, h, h, 1);
                    }
#pragma unroll
                    for (int e = 0; e < EP; ++e)
                        if (NM / 8 + e * 5 * NM / (8 * EP) == q) write_piece(e, h ^ 1, valid[1]);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        if (d * NM / ND == q) load(d, h ^ 1, DW ? h ^ 1 : h);
                });
                valid[0] = valid[1];
                valid[1] = valid[2];
                valid[2] = cq.rows - 32 * (h ^ 1);
                next_q(h ^ 1);
                next_a(DW ? h ^ 1 : h);
                // Outstanding at most: the activations of the last sub-step and
                // all loads of this one. The next sub-step's activations and
                // the raw codes read in this one are in LDS.
                wait_vm<2 * G::A_LOADS + G::Q_LOADS + 1>();
                lds_barrier();
                if (DW || h == 1) sa = sa == G::A_SLOTS - 1 ? 0 : sa + 1;
                // second k16 step: the next sub-step's first fragments (PAIR:
                // all) and the raw codes of the one after are read
                mma(second, k + 32 * h + 16 < u.kend, [&](int q) {
#pragma unroll
                    for (int n = 0; n < 2 * MI; ++n)
                        if (n * NM / (4 * MI) == q) read_frag(f[0], n, sa, h ^ 1, h ^ 1, 0);
                    if constexpr (PAIR) {
#pragma unroll
                        for (int n = 0; n < 2 * MI; ++n)
                            if (NM / 2 + n * NM / (4 * MI) == q) read_frag(f[h == 0 ? 2 : 1], n, sa, h ^ 1, h ^ 1, 1);
                    }
#pragma unroll
                    for (int e = 0; e < EP; ++e)
                        if (NM / 8 + e * 5 * NM / (8 * EP) == q) read_raw(e, sr);
                });
                sr = sr == 2 ? 0 : sr + 1;
            }
        }
        finish_unit<TILE, DW, MI / 2, SPLIT, BETA>(acc, st, p, u, M, C, wrow, wcol);
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, R, vb, u)) break;
        first();  // again: the fragments' registers served the epilogue
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// ---- both operands in MXFP4 ------------------------------------------------------
// The scaled matrix instruction takes 32 codes of a row and a scale byte from
// each lane: 32 x 32 outputs over K = 64. Steps of K = 256 make 128-byte row
// segments (a CU takes a 1 KiB load of those in half the time of 64-byte
// ones); codes lie in LDS as [rows][128 bytes], chunks XOR-swizzled by row /
// 2, scales as [16 rows][8 blocks][16 bytes], so that one transposing read
// gives a lane its row's 8 scales.

// Scales of row `base` + lane % 32 (base a multiple of 32, region `sc`): byte g
// is that of block 2 g + lane / 32.
__device__ __forceinline__ int read_scales(const uint8_t* sc, int base, int lane) {
    const i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_i32x2*)(sc + (base + 16 * ((lane >> 4) & 1)) * 8 + (lane & 15) * 8));
    return __builtin_amdgcn_perm(v[1], v[0], lane < 32 ? 0x06040200 : 0x07050301);
}
// 16 code bytes of block blk of row r.
__device__ __forceinline__ i32x4 read_block(const uint8_t* codes, int r, int blk) {
    return *reinterpret_cast<const i32x4*>(codes + r * 128 + ((blk ^ ((r >> 1) & 7)) * 16));
}
template <int G>
__device__ __forceinline__ f32x16 mma_mx(i32x4 w, i32x4 x, f32x16 c, int ws, int xs) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1),
                                                           __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1), c, 4, 4,
                                                           G, ws, G, xs);
}
// Few tokens take a tile's 128 rows too: N 1024, K 4096, split in parts, T 1 / 16
// / 64 6.0 / 6.7 / 8.0 us (bf16 activations, T 16: 5.1).
// FULL: K is a multiple of 256, and no branch stands between a step's reads and
// its MFMAs (T 16384, N 4096, K 4096 185 -> 175 us, T 16384, N 16384, K 8192
// 1319 -> 1201).
//
// 128 x 128 outputs, ring of 2. A unit's first step is loaded before the
// previous unit's epilogue, which stages through the other slot.
struct Mx {
    static constexpr int TILE = 128, WT = 64, MI = 2;
    static constexpr int CODES = TILE * 128, LOADS = CODES / 4096;  // per operand; 1 KiB loads per wave
    static constexpr int SLOT = 2 * CODES + 2048;
    static constexpr int LDS = 2 * SLOT;
};

template <bool SPLIT, bool FULL, bool BETA>
__global__ __launch_bounds__(256, 2) void linear_mx_kernel(LinearParams p, LinearPlan pl) {
    using G = Mx;
    constexpr int MI = G::MI, WT = G::WT, TILE = G::TILE;
    __shared__ uint4 lds_raw[G::LDS / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT;
    const int K = p.K;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, SPLIT>(pl, K, vb, u)) return;

    // ---- the next step to load
    MxCursor<TILE, SPLIT> at;
    at.vl = vb;
    at.of_w = wave & 1;
    at.set(p, u);
    int sl = 0;
    uint32_t off[G::LOADS];
#pragma unroll
    for (int i = 0; i < G::LOADS; ++i) {
        const int r = 8 * (wave * G::LOADS + i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        off[i] = (uint32_t)r * (uint32_t)(K / 2) + c * 16;
    }
    // waves 0 and 1: the scales of X and W; 2 and 3 the same again
    const uint32_t sc_off = (uint32_t)(lane & 7) * (uint32_t)((wave & 1) ? p.wlds : p.xlds) + 16 * (lane >> 3);
    auto load_step = [&]() {
        const uint32_t to = lds0 + sl * G::SLOT;
#pragma unroll
        for (int i = 0; i < G::LOADS; ++i) {
            dma16(at.wx, off[i], to + (wave * G::LOADS + i) * 1024);
            dma16(at.ww, off[i], to + G::CODES + (wave * G::LOADS + i) * 1024);
        }
        dma16(at.wsc, sc_off, to + 2 * G::CODES + (wave & 1) * 1024);
        sl ^= 1;
        at.next(p, pl, workgroups);
    };
    f32x16 acc[MI][MI];
    clear(acc);
    int slot = 0;
    load_step();
    for (;;) {
        for (int k = u.kbeg; k < u.kend; k += 256) {
            wait_vm<0>();
            lds_barrier();  // step k is whole in LDS, and the other slot is read
            if (at.left) load_step();
            const uint8_t* st = lds + slot * G::SLOT;
            const int groups = FULL ? 4 : min(4, (u.kend - k) / 64);
            int as[MI], bs[MI];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                as[i] = read_scales(st + 2 * G::CODES, wrow + 32 * i, lane);
                bs[i] = read_scales(st + 2 * G::CODES + 1024, wcol + 32 * i, lane);
            }
            struct Frag {
                i32x4 a[MI], b[MI];
            } f[2];
            auto read = [&](Frag& f, int g) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    f.a[i] = read_block(st, wrow + 32 * i + (lane & 31), 2 * g + (lane >> 5));
                    f.b[i] = read_block(st + G::CODES, wcol + 32 * i + (lane & 31), 2 * g + (lane >> 5));
                }
            };
            auto mma = [&](auto g_, const Frag& f) {
                constexpr int g = decltype(g_)::value;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < MI; ++j) acc[i][j] = mma_mx<g>(f.b[j], f.a[i], acc[i][j], bs[j], as[i]);
            };
            read(f[0], 0);
            read(f[1], 1);
            __builtin_amdgcn_sched_barrier(0);
            mma(std::integral_constant<int, 0>{}, f[0]);
            read(f[0], 2);
            __builtin_amdgcn_sched_barrier(0);
            if (groups > 1) mma(std::integral_constant<int, 1>{}, f[1]);
            read(f[1], 3);
            __builtin_amdgcn_sched_barrier(0);
            if (groups > 2) mma(std::integral_constant<int, 2>{}, f[0]);
            if (groups > 3) mma(std::integral_constant<int, 3>{}, f[1]);
            slot ^= 1;
        }
        lds_barrier();  // the last step's slot is read: the epilogue stages there
        finish_unit<TILE, false, MI, SPLIT, BETA>(acc, lds + (slot ^ 1) * G::SLOT + wave * Stage<false, MI>::BYTES, p, u, p.T, p.N,
                                            wrow, wcol);
        vb += gridDim.x;
        if (!unit_at<TILE, SPLIT>(pl, K, vb, u)) break;
        clear(acc);
    }
}

// Large products with K a multiple of 256: 256 x 256 outputs, one workgroup per
// CU, which halves what a product reads from LDS and L2. Ring of 2. A K = 64
// group of 16 MFMAs runs on registers; in the slots between them the next
// group's fragments are read and loads are issued. Behind a step's third group
// the whole slot is in registers: the barrier stands there, the fourth group
// reads the next slot's first fragments and the freed slot's loads begin. (us,
// 128 x 128 / 256 x 256, the latter with loads and reads in a bunch ahead of each
// step: T 16384, N 4096, K 4096 162 / 147, 166 bunched; T = N = 16384, K 8192
// 1191 / 1037, 1112 bunched, 4.2 PFLOP/s.)
// At small K the outputs bound it: a unit takes 5.0 us for its 128 KiB of outputs
// (the chip's stores alone: 5.0 to 5.6 us, 6 to 6.7 TB/s) and 1.9 us a step, one behind the
// other, with the CUs' epilogues together or spread over a round.
struct MxLarge {
    static constexpr int TILE = 256, WT = 128, MI = 4;
    static constexpr int CODES = TILE * 128, SCALES = TILE * 8;  // bytes per operand
    static constexpr int LOADS = CODES / 4096, ND = 2 * LOADS + 1, FIRST = 9;
    static constexpr int SLOT = 2 * CODES + 2 * SCALES, ST0 = 2 * SLOT;
    static constexpr int LDS = ST0 + 4 * Stage<false, 2>::BYTES;
    static constexpr int STORES = 32;  // of a wave's full output
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <bool BETA>
__global__ __launch_bounds__(256, 1) void linear_mx_large_kernel(LinearParams p, LinearPlan pl) {
    using G = MxLarge;
    constexpr int MI = G::MI, WT = G::WT, TILE = G::TILE;
    __shared__ uint4 lds_raw[G::LDS / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const uint32_t lds0 = lds_u32(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wrow = (wave >> 1) * WT, wcol = (wave & 1) * WT;
    const int K = p.K;
    Unit u;
    int vb = blockIdx.x;
    if (!unit_at<TILE, false>(pl, K, vb, u)) return;

    // ---- the next step to load
    MxLargeCursor<TILE> at;
    at.vl = vb;
    at.of_w = wave & 1;
    at.set(p, u);
    int sll = 0;
    uint32_t off[G::LOADS];
#pragma unroll
    for (int i = 0; i < G::LOADS; ++i) {
        const int r = 8 * (wave * G::LOADS + i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        off[i] = (uint32_t)r * (uint32_t)(K / 2) + c * 16;
    }
    // even waves: the scales of X, odd waves: of W; 128 rows each
    const uint32_t sc_off = (uint32_t)(lane & 7) * (uint32_t)((wave & 1) ? p.wlds : p.xlds) + 16 * (lane >> 3) + 128 * (wave >> 1);
    auto load = [&](int d) {
        const uint32_t to = lds0 + sll * G::SLOT;
        const int i = d >> 1;
        if (d == 2 * G::LOADS) dma16(at.wsc, sc_off, to + 2 * G::CODES + (wave & 1) * G::SCALES + (wave >> 1) * 1024);
        else if (d & 1) dma16(at.ww, off[i], to + G::CODES + (wave * G::LOADS + i) * 1024);
        else dma16(at.wx, off[i], to + (wave * G::LOADS + i) * 1024);
    };
    auto next_loads = [&]() {
        sll ^= 1;
        at.next(p, pl, workgroups);
    };

    // ---- fragments
    struct Frag {
        i32x4 a[MI], b[MI];
    } f[2];
    int as[MI], bs[MI], as2[MI], bs2[MI];
    auto read = [&](Frag& t, int r, int sl, int g) {  // r: A blocks, then B blocks
        const uint8_t* st = lds + sl * G::SLOT;
        if (r < MI) t.a[r] = read_block(st, wrow + 32 * r + (lane & 31), 2 * g + (lane >> 5));
        else t.b[r - MI] = read_block(st + G::CODES, wcol + 32 * (r - MI) + (lane & 31), 2 * g + (lane >> 5));
    };
    auto scales = [&](int r, int sl) {
        const uint8_t* sc = lds + sl * G::SLOT + 2 * G::CODES;
        if (r < MI) as2[r] = read_scales(sc, wrow + 32 * r, lane);
        else bs2[r - MI] = read_scales(sc + G::SCALES, wcol + 32 * (r - MI), lane);
    };
    f32x16 acc[MI][MI];
    // group g; reads group (g + 1) % 4 of slot sl; issues loads [d0, d0 + dn)
    auto mma = [&](auto g_, const Frag& t, Frag& t2, int sl, int d0, int dn) {
        constexpr int g = decltype(g_)::value;
#pragma unroll
        for (int q = 0; q < MI * MI; ++q) {
            const int i = q / MI, j = q % MI;
            acc[i][j] = mma_mx<g>(t.b[j], t.a[i], acc[i][j], bs[j], as[i]);
            if (q < 2 * MI) read(t2, q, sl, (g + 1) & 3);
            else if (g == 3) scales(q - 2 * MI, sl);
#pragma unroll
            for (int d = 0; d < dn; ++d)
                if ((2 * d + 1) * MI * MI / (2 * dn) == q) load(d0 + d);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int r = 0; r < MI; ++r) as[r] = as2[r], bs[r] = bs2[r];
    };

    // ---- stream
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int d = 0; d < G::ND; ++d) load(d);
        next_loads();
    }
    wait_vm<G::ND>();
    lds_barrier();
    int sl = 0;
    auto first = [&]() {  // a unit's first fragments
#pragma unroll
        for (int r = 0; r < 2 * MI; ++r) {
            read(f[0], r, sl, 0);
            scales(r, sl);
        }
        take_scales();
    };
    first();
    bool stored = false;  // the last unit's outputs fill the wave's part: STORES stores behind the loads
    uint8_t* st = lds + G::ST0 + wave * Stage<false, 2>::BYTES;
    for (;;) {
        clear(acc);
        for (int k = 0; k < K; k += 256) {
            if (k == 0) {
                mma(std::integral_constant<int, 0>{}, f[0], f[1], sl, 0, 0);
            } else {
                mma(std::integral_constant<int, 0>{}, f[0], f[1], sl, G::FIRST, G::ND - G::FIRST);
                next_loads();
            }
            mma(std::integral_constant<int, 1>{}, f[1], f[0], sl, 0, 0);
            mma(std::integral_constant<int, 2>{}, f[0], f[1], sl, 0, 0);
            if (k == 0 && stored) wait_vm<G::STORES>();
            else wait_vm<0>();
            lds_barrier();  // this slot is read, the other one is whole
            sl ^= 1;
            mma(std::integral_constant<int, 3>{}, f[1], f[0], sl, 0, G::FIRST);
            take_scales();
        }
        // the next unit's second step: its loads stand before the stores
#pragma unroll
        for (int d = G::FIRST; d < G::ND; ++d) load(d);
        next_loads();
        __builtin_amdgcn_sched_barrier(0);
        finish_unit<TILE, false, 2, false, BETA>(acc, st, p, u, p.T, p.N, wrow, wcol);
        stored = p.T - u.m0 - wrow >= WT && p.N - u.c0 - wcol >= WT;
        vb += gridDim.x;
        if (!unit_at<TILE, false>(pl, K, vb, u)) break;
        if constexpr (BETA) first();  // again: what is there took the fragments' registers
    }
    wait_vm<0>();  // no load may land in LDS that the next workgroup owns
}

// ---- few tokens -------------------------------------------------------------------
// A workgroup takes 16 NB output columns (rows of W) and 16 RB tokens; its NW
// waves deal out the reduction in pieces of K = 128, U pieces in flight. Lane l
// loads row l % 16's whole block 4 i + l / 16 of a piece straight into
// registers (16 code bytes, one scale) and takes 8 codes of it to each of four
// v_mfma_f32_16x16x32_bf16; the activations follow the same order of the
// reduction. They come through LDS of the wave's own ([16 tokens][256 bytes] a
// piece, chunks XOR-swizzled by token): fragments straight from memory touch 64
// lines a load, which bound the kernel (16 tokens, N 1024, K 4096: 6.5 us).
// The waves' sums meet in LDS and are added in wave order.
template <int RB, int NB, int NW, int U>
__global__ __launch_bounds__(64 * NW) void linear_rows_kernel(LinearParams p) {
    constexpr int OUT = 256 * RB * NB;  // outputs of a workgroup
    constexpr int XB = U * RB * 4096;   // activation bytes of a wave
    __shared__ uint4 lds_raw[(NW * (XB > OUT * 4 ? XB : OUT * 4)) / 16];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds_raw);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, g = lane >> 4;
    const int nb = (p.N + 16 * NB - 1) / (16 * NB);  // blocks of columns, which run fastest
    const int n0 = (int)(blockIdx.x % nb) * 16 * NB, t0 = (int)(blockIdx.x / nb) * 16 * RB;
    const int K = p.K, pieces = (K + 127) / 128;
    const uint8_t* wq[NB];
    const uint8_t* wsc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int n = min(n0 + 16 * b + row, p.N - 1);
        wq[b] = p.w + (int64_t)n * (K / 2) + g * 16;
        wsc[b] = p.ws + (int64_t)g * p.wlds + n;
    }
    const uint8_t* xw = lds + wave * XB;
    const uint32_t xw0 = lds_u32(xw);
    f32x4 acc[RB][NB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[r][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = wave; i0 < pieces; i0 += NW * U) {
        uint4 q[U][NB];
        uint32_t sc[U][NB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NW;
            const bool in = 4 * i + g < K / 32;  // past the end: zero times zero
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                q[u][b] = in ? *reinterpret_cast<const uint4*>(wq[b] + i * 64) : make_uint4(0, 0, 0, 0);
                sc[u][b] = in ? wsc[b][(int64_t)(4 * i) * p.wlds] : 127;
            }
        }
        // load d of a piece: tokens 4 d .. 4 d + 3, lane l chunk l % 16
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    if (t0 + 16 * r + 4 * d >= p.T) break;  // tokens past the last: whatever LDS holds, for no output
                    const int i = i0 + u * NW, t = 4 * d + g, k = i * 128 + 8 * (row ^ t);
                    const uint16_t* src = p.x + (int64_t)min(t0 + 16 * r + t, p.T - 1) * p.ldx + k;
                    dma16v(k < K ? (const void*)src : (const void*)zero_piece, xw0 + (u * RB + r) * 4096 + d * 1024);
                }
        wait_vm<0>();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4 v[RB][4];
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[r][j] = *reinterpret_cast<const uint4*>(xw + (u * RB + r) * 4096 + row * 256 + ((4 * g + j) ^ row) * 16);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float unit = e8m0_operand(sc[u][b]);
                const uint32_t w[4] = {q[u][b].x, q[u][b].y, q[u][b].z, q[u][b].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bf16x8 f = __builtin_bit_cast(bf16x8, expand_fp4(w[j], unit));
#pragma unroll
                    for (int r = 0; r < RB; ++r)
                        acc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, v[r][j]), acc[r][b], 0, 0, 0);
                }
            }
        }
        wave_lds_fence();  // the activations are read: the next loads may land
    }
    __syncthreads();  // the sums take the activations' place
    float* red = reinterpret_cast<float*>(lds);
    // acc[r][b][e]: token 16 r + lane % 16, column 16 b + 4 (lane / 16) + e
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b)
            *reinterpret_cast<f32x4*>(red + wave * OUT + (16 * r + row) * (16 * NB) + 16 * b + 4 * g) = acc[r][b];
    __syncthreads();
    for (int o = threadIdx.x * 2; o < OUT; o += 128 * NW) {
        const int t = t0 + o / (16 * NB), n = n0 + o % (16 * NB);
        if (t >= p.T || n >= p.N) continue;
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            a += red[w * OUT + o];
            b += red[w * OUT + o + 1];
        }
        uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.y) + (int64_t)t * p.ldy + n);
        if (p.beta != 0.0f) {
            const uint32_t old = *y;
            a += p.beta * bf_lo(old);
            b += p.beta * bf_hi(old);
        }
        *y = pack_bf2(a, b);
    }
}

// dW = beta dW: the weight gradient over no tokens. Four values a thread; the
// workgroups stride over the matrix.
__global__ __launch_bounds__(256) void linear_scale_kernel(float* y, int64_t ldy, int rows, int cols, float beta) {
    const int pieces = cols / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * pieces; i += (int64_t)gridDim.x * 256) {
        f32x4* o = reinterpret_cast<f32x4*>(y + i / pieces * ldy + i % pieces * 4);
        *o = beta != 0.0f ? beta * *o : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// BETA: a kernel that adds to what is there. Apart, since two epilogues in one
// kernel spill the accumulators.
template <int OP, int TILE, bool SPLIT, bool BETA>
void launch_units(const LinearParams& p, const LinearPlan& pl, int units, int cus, hipStream_t s) {
    const int grid = unit_grid(TILE, units, cus);
    if constexpr (OP == LINEAR_MATMUL) {
        if (p.K % 256 == 0) linear_mx_kernel<SPLIT, true, BETA><<<grid, 256, 0, s>>>(p, pl);
        else linear_mx_kernel<SPLIT, false, BETA><<<grid, 256, 0, s>>>(p, pl);
    } else if constexpr (OP == LINEAR_FORWARD) linear_fwd_kernel<TILE, SPLIT, BETA><<<grid, 256, 0, s>>>(p, pl);
    else linear_grad_kernel<OP, TILE, SPLIT, BETA><<<grid, 256, 0, s>>>(p, pl);
}
template <int OP, int TILE>
void launch_tiles(const LinearParams& p, const LinearPlan& pl, int cus, hipStream_t s) {
    if (pl.whole > 0) {
        if (p.beta == 0.0f) launch_units<OP, TILE, false, false>(p, pl, pl.whole, cus, s);
        else launch_units<OP, TILE, false, true>(p, pl, pl.whole, cus, s);
    }
    if (pl.tail > 0) {
        launch_units<OP, TILE, true, false>(p, pl, pl.tail * pl.parts, cus, s);  // the sums add what is there
        constexpr int SLABS = TILE / (256 / (TILE / 4));
        const Sizes z = sizes((LinearOp)OP, p.T, p.N, p.K);
        linear_fixup_kernel<TILE, OP == LINEAR_DW><<<pl.tail * SLABS, 256, 0, s>>>(p, pl, z.M, z.C);
    }
}

void launch_mx_large(const LinearParams& p, int cus, hipStream_t s) {
    const LinearPlan pl = plan_tiles(sizes(LINEAR_MATMUL, p.T, p.N, p.K), 256, 1, cus);
    const int grid = unit_grid(256, pl.whole, cus);
    if (p.beta == 0.0f) linear_mx_large_kernel<false><<<grid, 256, 0, s>>>(p, pl);
    else linear_mx_large_kernel<true><<<grid, 256, 0, s>>>(p, pl);
}

template <int RB, int NB, int NW, int U>
void launch_rows_as(const LinearParams& p, hipStream_t s) {
    const int64_t grid = (int64_t)((p.N + 16 * NB - 1) / (16 * NB)) * ((p.T + 16 * RB - 1) / (16 * RB));
    linear_rows_kernel<RB, NB, NW, U><<<(unsigned)grid, 64 * NW, 0, s>>>(p);
}
// Blocks of outputs grow with the grid, which fills the chip twice at most: 16 x
// 16, 16 x 32 (columns), 32 x 32, 64 x 32. Measured (us) 16 x 16 / 16 x 32 / 32 x
// 32 / 64 x 32: T 16, N 1024, K 4096 4.7 / 6.4 / 7.6 / 8.8; T 64, N 4096, K 1024
// 4.8 / 4.6 / 4.7 / 6.4; T 256, N 4096, K 1024 13.8 / 11.4 / 11.2 / 10.0.
// Reductions of more than 8 pieces take 8 waves with two pieces in flight (32 x
// 32: one), shorter ones 4 waves with two (16 x 16: 8 with one).
// Measured to N 4096. Layers so wide that blocks of 32 x 32 fill the chip more
// than twice take blocks of 64 tokens however few there are, and lose by it: one
// token, K 4096: N 16384 10.9 us, N 32768 38, where the codes alone take 14.
void launch_rows(const LinearParams& p, int cus, hipStream_t s) {
    const int64_t most = 2 * (int64_t)cus, n16 = (p.N + 15) / 16, n32 = (p.N + 31) / 32;
    const int64_t t16 = (p.T + 15) / 16, t32 = (p.T + 31) / 32;
    const bool many = p.K > 1024;
    if (n16 * t16 <= most) many ? launch_rows_as<1, 1, 8, 2>(p, s) : launch_rows_as<1, 1, 8, 1>(p, s);
    else if (n32 * t16 <= most) many ? launch_rows_as<1, 2, 8, 2>(p, s) : launch_rows_as<1, 2, 4, 2>(p, s);
    else if (n32 * t32 <= most) many ? launch_rows_as<2, 2, 8, 1>(p, s) : launch_rows_as<2, 2, 4, 2>(p, s);
    else launch_rows_as<4, 2, 4, 1>(p, s);
}

}  // namespace

size_t linear_workspace(LinearOp op, int T, int N, int K) { return workspace_bound(op, T, N, K, cu_count()); }

hipError_t launch_linear(LinearOp op, const LinearParams& p, hipStream_t s) {
    const int cus = cu_count();
    if (op == LINEAR_DW && p.T == 0) {
        if (p.beta == 1.0f) return hipSuccess;
        const int64_t blocks = std::min<int64_t>(((int64_t)p.N * p.K / 4 + 255) / 256, 16 * (int64_t)cus);
        linear_scale_kernel<<<(unsigned)blocks, 256, 0, s>>>(static_cast<float*>(p.y), p.ldy, p.N, p.K, p.beta);
        return hipGetLastError();
    }
    if (op == LINEAR_MATMUL && mx_large(p.T, p.N, p.K, cus)) {
        launch_mx_large(p, cus, s);
        return hipGetLastError();
    }
    double us = 0.0;
    const LinearPlan pl = linear_plan(op, p.T, p.N, p.K, cus, &us);
    if (op == LINEAR_FORWARD && rows_time(p.T, p.N, p.K) <= us) {
        launch_rows(p, cus, s);
        return hipGetLastError();
    }
    const bool big = pl.tile == 256;
    switch (op) {
        case LINEAR_FORWARD: big ? launch_tiles<LINEAR_FORWARD, 256>(p, pl, cus, s) : launch_tiles<LINEAR_FORWARD, 128>(p, pl, cus, s); break;
        case LINEAR_MATMUL: launch_tiles<LINEAR_MATMUL, 128>(p, pl, cus, s); break;
        case LINEAR_DX: big ? launch_tiles<LINEAR_DX, 256>(p, pl, cus, s) : launch_tiles<LINEAR_DX, 128>(p, pl, cus, s); break;
        case LINEAR_DW: big ? launch_tiles<LINEAR_DW, 256>(p, pl, cus, s) : launch_tiles<LINEAR_DW, 128>(p, pl, cus, s); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace tmt
