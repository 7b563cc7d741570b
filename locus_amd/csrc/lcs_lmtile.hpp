// The lm-head's tiled product with the sampler's first statistics in its epilogue
// (gfx950): one kernel template for bf16 and 8-bit operands, with and without
// the rows' low-rank adapters. lcs_lmhead.hip and lcs_lmhead_ex.hip launch it.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"

namespace lcs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a __attribute__((ext_vector_type(4), may_alias));
constexpr float kL2E = 1.4426950408889634f;

// Waits until at most N vector memory operations are outstanding (and every
// LDS operation is done); the compiler moves no memory access across it.
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm_lgkm() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// 16 bytes per lane from a buffer (offsets vo per lane + so) to LDS at
// dst + 16 lane (dst is wave-uniform).
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned char* dst, uint32_t vo, uint32_t so) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, (int)vo, (int)so, 0, 0);
}
// The same from a per-lane address.
__device__ __forceinline__ void dma16_at(const void* src, unsigned char* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
// NaN, by its bits: the build's float comparisons and selects assume that there
// are none (the empty asm keeps the compiler from concluding the same here).
__device__ __forceinline__ bool nan_bits(float v) {
    uint32_t u = __float_as_uint(v);
    asm("" : "+v"(u));
    return (u & 0x7fffffffu) > 0x7f800000u;
}
// The upper 16 bits as bf16: towards zero, so that finite stays finite; NaN stays
// NaN (by its bits, as above).
__device__ __forceinline__ uint32_t bf16_top(float v) {
    uint32_t u = __float_as_uint(v);
    asm("" : "+v"(u));
    return (u >> 16) | ((u & 0x7fffffffu) > 0x7f800000u ? 0x40u : 0u);
}
// Pairs of bf16 with infs and NaNs put to the largest finite value of their sign.
__device__ __forceinline__ u32x4 finite_bf16(u32x4 v) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
    // (as unsigned numbers the negative ones are on top, as signed ones the positive)
    const u16x8 n = __builtin_elementwise_min(__builtin_bit_cast(u16x8, v), (u16x8)(uint16_t)0xff7f);
    return __builtin_bit_cast(u32x4, __builtin_elementwise_min(__builtin_bit_cast(i16x8, n), (i16x8)(int16_t)0x7f7f));
}
// A workgroup barrier that waits for no memory operation.
__device__ __forceinline__ void block_sync() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Whether the step of 16 ranks from k is the last one below `end` of an adapter
// (who: its rank << 16 | its id; below 0 there is no step, and nothing ends).
constexpr bool last_step(int32_t who, uint32_t k, uint32_t end) {
    return who >= 0 && k + 16u >= ((uint32_t)who >> 16 < end ? (uint32_t)who >> 16 : end);
}

template <uint32_t P>
struct Parts { static constexpr uint32_t value = P; };

// A workgroup computes 64 VT columns of BR rows, transposed (columns on the
// MFMA's row side, so that a lane holds many columns of one row and the
// epilogue reduces in registers): NW waves, WN of them over the rows, in
// v_mfma_f32_32x32x16_bf16 tiles (lane l carries 8 consecutive k of row l % 32
// of either operand, k chunk l / 32, and returns rows 8 (e / 4) + 4 (l / 32) +
// e % 4 of column l % 32). The 256 x 256 tile takes eight waves, so that two
// share a SIMD and one's loads, barriers and epilogue leave the matrix cores to
// the other (1024 rows: 990 us with four, 963 with eight).
//
// Both operands go straight from memory into a ring of ST LDS stages of 16 KS k
// with 16-byte DMA loads, so that no register holds data in flight. The loads
// are what holds the matrix cores up (1024 rows: busy 1.03 M of 1.52 M cycles): a
// stage of 64 k reads whole 128-byte lines, half the requests of 32 k, and two
// such stages serve as well as four (1024 rows 963 -> 921 us, 64 rows 209 ->
// 199); narrow and 128-row tiles have too few bytes in flight then (8 x 32000
// 52 -> 69 us, 128 rows 218 -> 229) and keep 32 k. A row's 16-byte chunks are
// permuted by its bits from kSw up: a fragment read's 16 lanes of a phase then
// cover the 64 banks once (0 conflict cycles of 101 M). One barrier per stage, ahead of its last products: each wave has then
// read the stage and its loads of the next one have landed.
//
// The workgroups of a column block are placed on one XCD in consecutive
// dispatch slots (workgroups are dealt to the 8 XCDs in turn): they run
// together, so that the block's weight rows come mostly from that XCD's L2 for
// all but one of the row tiles (four row tiles of 1024 rows x 128256 x 4096 e4m3
// fetch 795 MB where weight and x have 530; two of 512 rows bf16 with
// adapters 1327 of 1186). With one row tile each workgroup starts at its
// own k-step and wraps round, so that those in flight do not all read the same
// offset of their rows (72 rows x 128256 x 4096: 245 -> 225 us); with more the
// row tiles share x through the L2 by running in step (1024 rows: 1013 against
// 1057 us with a start of its own).
//
// F8: e4m3 operands. A 16-byte chunk holds 16 k, which are widened to bf16 (exactly)
// ahead of their two products; the two operands' chunks hold the same k, so which
// ones does not matter. The 8-bit matrix instructions would take half the time
// but sum each 8 consecutive products in units of 2^-13 of the largest of them: 1.5e-5
// of the logits' norm against 9e-8 here (4096 random k), and sums are to be f32.
// The row's and the column's scale multiply the sums once, ahead of the adapters.
// AD: the rows are taken in the order of their adapters (lm_low, which also
// has left each row's low-rank state): see the adapters' part
// below.
template <int VT, int BR, int ST, int NW = 4, int KS = 2, bool BIG = false, bool F8 = false, bool AD = false, int WN = 2>
__global__ __launch_bounds__(NW * kWave, 2) void lmhead_tile(LmArgs a) {
    constexpr uint32_t kTV = 64u * VT;        // columns per workgroup
    constexpr uint32_t EB = F8 ? 1u : 2u;     // bytes of an element
    constexpr uint32_t kTRowB = 32u * KS;     // bytes of a row in a stage
    constexpr int kTK = (int)(kTRowB / EB);   // k per LDS stage
    constexpr uint32_t kStage = (kTV + BR) * kTRowB;
    constexpr int WM = NW / WN;               // waves side by side over the columns, WN over the rows
    constexpr int CT = 2 * VT / WM, RT = BR / (32 * WN);   // 32-column and 32-row tiles per wave
    constexpr uint32_t kCh = 2 * KS, kLog = KS == 4 ? 3 : 2;   // 16-byte chunks of a row
    constexpr uint32_t kSw = KS == 4 ? 1 : 2;   // the row bits that permute them start here
    constexpr int kLR = 64 / (int)kCh * NW;   // rows that one DMA load of every wave covers
    constexpr int LA = kTV / kLR, LB = BR / kLR;   // DMA loads per wave and stage
    constexpr bool SPLIT = KS == 4 && ST == 2;   // half of a stage's loads ahead of the barrier
    static_assert(KS == 2 || KS == 4, "the schedule of the k-loop");
    static_assert(!(BIG && (F8 || AD)), "row offsets");
    static_assert(LA * kLR == (int)kTV && LB * kLR == BR && CT * WM == 2 * VT, "tile shape");
    constexpr int LPS = LA + LB;
    __shared__ __attribute__((aligned(128))) unsigned char lds[ST * kStage];
    const uint32_t tid = tid_x();
    const int lane = lane_id(), wv = __builtin_amdgcn_readfirstlane((int)(tid / kWave));
    uint32_t nb = wg_x();
    const uint32_t slot = nb >> 3;
    const uint32_t r0 = (slot % a.nchunks) * BR;
    nb = 8u * (slot / a.nchunks) + (nb & 7u);
    if (nb >= a.nblocks) return;   // (the grid is a multiple of 8 blocks)
    const uint32_t K = a.hidden, V = a.vocab;
    const uint32_t n0 = nb * kTV;
    const uint32_t vrows = min((uint32_t)BR, a.rows - r0), vcols = min(kTV, V - n0);
    const uint32_t wm = (uint32_t)wv % WM, wn = (uint32_t)wv / WM;   // the wave's columns and rows
    const unsigned char* wbase = reinterpret_cast<const unsigned char*>(a.w) + (uint64_t)n0 * K * EB;
    // (AD: rows from anywhere in x, which is under 4 GiB then)
    const unsigned char* xbase = reinterpret_cast<const unsigned char*>(a.x) + (AD ? 0ull : (uint64_t)r0 * K * EB);
    const __amdgpu_buffer_rsrc_t wrs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(wbase), 0, (int)(vcols * K * EB), 0x00020000);
    const __amdgpu_buffer_rsrc_t xrs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(xbase), 0, (int)((AD ? a.rows : vrows) * K * EB), 0x00020000);
    auto row_of = [&](uint32_t r) -> uint32_t { return AD ? a.perm[r0 + r] : r0 + r; };   // (r < vrows)
    // DMA load i of a wave covers rows kLR i + 16 wv + lane / 4, a 16-byte
    // chunk per lane; rows past the tile read row 0 (masked in the epilogue)
    const uint32_t rr = kWave / kCh * (uint32_t)wv + ((uint32_t)lane >> kLog);
    const uint32_t ch = (((uint32_t)lane & (kCh - 1u)) ^ ((rr >> kSw) & (kCh - 1u))) * 16u;
    uint32_t wo[LA], xo[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i) wo[i] = (kLR * i + rr < vcols ? kLR * i + rr : 0u) * K * EB + ch;
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const uint32_t r = kLR * i + rr < vrows ? kLR * i + rr : 0u;
        xo[i] = (AD ? row_of(r) : r) * K * EB + ch;
    }
    const uint32_t nsteps = K / kTK;
    const uint32_t rot = a.nchunks == 1u && (!F8 || nsteps != 0u) ? nb % nsteps : 0u;
    // (the byte offset of stage t in a row; stages past the end re-read the last)
    auto koff = [&](uint32_t t) -> uint32_t {
        uint32_t q = (t < nsteps ? t : nsteps - 1u) + rot;
        return (q >= nsteps ? q - nsteps : q) * kTRowB;
    };
    auto issue1 = [&](int i, uint32_t ko, uint32_t sl) {   // DMA load i of a stage
        unsigned char* b = lds + sl * kStage + (uint32_t)wv * 1024u + i * (kLR * kTRowB);
        if (BIG) {   // (the row offsets need 64 bits)
            const uint32_t r = kLR * (uint32_t)(i < LA ? i : i - LA) + rr;
            const unsigned char* p = i < LA ? wbase + (uint64_t)(r < vcols ? r : 0u) * K * EB : xbase + (uint64_t)(r < vrows ? r : 0u) * K * EB;
            dma16_at(p + ko + ch, b);
        } else if (i < LA) {
            dma16(wrs, b, wo[i < LA ? i : 0], ko);
        } else {
            dma16(xrs, b, xo[i >= LA ? i - LA : 0], ko);
        }
    };
    auto issue = [&](uint32_t t, uint32_t sl) {
#pragma unroll
        for (int i = 0; i < LPS; ++i) issue1(i, koff(t), sl);
    };
    constexpr uint32_t NSC = F8 ? (kTV + BR + NW * kWave - 1u) / (NW * kWave) : 1u;
    static_assert(!F8 || 16u * WM * BR + 4u * (kTV + BR) <= sizeof(lds), "the scales' place");
    float scales[NSC];
    if constexpr (F8) {
#pragma unroll
        for (uint32_t i = 0; i < NSC; ++i) {
            const uint32_t t = NW * kWave * i + tid, r = t - kTV;
            scales[i] = 1.0f;
            if (t < kTV) {
                if (a.w_scale && t < vcols) scales[i] = a.w_scale[n0 + t];
            } else if (a.x_scale && r < vrows) {
                scales[i] = a.x_scale[row_of(r)];
            }
        }
    }
    f32x16 acc[CT][RT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    // fragment s (16 k) of row r: chunk 2 s + lane / 32
    const uint32_t lr = (uint32_t)lane & 31u, lh = (uint32_t)lane >> 5;
    uint32_t fo[KS];
#pragma unroll
    for (uint32_t s = 0; s < KS; ++s) fo[s] = lr * kTRowB + (((2u * s + lh) ^ ((lr >> kSw) & (kCh - 1u))) * 16u);
    using Chunk = std::conditional_t<F8, u32x4, bf16x8>;
    struct Frag { Chunk w[CT], x[RT]; };
    // read i of a fragment set: x first (every product needs all of it), then w
    constexpr int NR = CT + RT, NP = CT * RT;
    auto read1 = [&](Frag& f, int i, uint32_t sl, int s) {
        const unsigned char* pw = lds + sl * kStage + wm * (kTV / WM * kTRowB) + fo[s];
        const unsigned char* px = lds + sl * kStage + kTV * kTRowB + wn * (BR / WN * kTRowB) + fo[s];
        using At = std::conditional_t<F8, u32x4_a, bf16x8>;
        if (i < RT) f.x[i < RT ? i : 0] = *reinterpret_cast<const At*>(px + i * 32 * kTRowB);
        else f.w[i >= RT ? i - RT : 0] = *reinterpret_cast<const At*>(pw + (i - RT) * 32 * kTRowB);
    };
    // (8 bits) the operands of the products at hand
    bf16x8 cx[RT][2], cw8[2];
    auto widen = [](const u32x4& q, bf16x8 (&o)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            union { bf16x2 p[4]; bf16x8 v; } u;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                u.p[2 * d] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * h + d], 1.0f, false);
                u.p[2 * d + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * h + d], 1.0f, true);
            }
            o[h] = u.v;
        }
    };
    auto mul1 = [&](const Frag& f, int k) {   // product k of NP
        const int i = k / RT, j = k % RT;
        if constexpr (F8) {
            if (j == 0) widen(f.w[i], cw8);
            if (i == 0) widen(f.x[j], cx[j]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cw8[h], cx[j][h], acc[i][j], 0, 0, 0);
        } else {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
        }
    };
    if (!F8 || nsteps != 0u) {
    Frag f0, f1;
#pragma unroll
    for (int t = 0; t < ST; ++t) issue((uint32_t)t, (uint32_t)t);
    wait_vm<(ST - 1) * LPS>();
    block_sync();
#pragma unroll
    for (int i = 0; i < NR; ++i) read1(f0, i, 0u, 0);
    uint32_t sl = 0u;
    // Every LDS read and DMA load is issued behind a product: a wave issues
    // in order, and eight DMA loads in a row hold it for longer than the
    // products queued ahead of them last (1024 rows, four waves: 1022 -> 980 us).
    // (SPLIT: half of a stage's loads go out behind the last products
    // of the stage whose place it takes, half behind the next stage's first)
    uint32_t kn = 0u;   // the offset of the stage whose second half is to be issued
    for (uint32_t t = 0; t < nsteps; ++t) {
        const uint32_t ns = sl + 1u == (uint32_t)ST ? 0u : sl + 1u;
        constexpr int H = LPS / 2;
#pragma unroll
        for (int s = 0; s < KS - 1; ++s) {
            const bool more = SPLIT && s == 0;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                mul1(s % 2 == 0 ? f0 : f1, k);
#pragma unroll
                for (int i = k * (NR + (more ? LPS - H : 0)) / NP; i < (k + 1) * (NR + (more ? LPS - H : 0)) / NP; ++i) {
                    if (i < NR) read1(s % 2 == 0 ? f1 : f0, i, sl, s + 1);
                    else if (t != 0u) issue1(H + i - NR, kn, ns);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // stage t is read, stage t + 1 has landed, in every wave
        wait_vm_lgkm<SPLIT ? 0 : (ST - 2) * LPS>();
        block_sync();
        kn = koff(t + ST);
        constexpr int L = SPLIT ? H : LPS;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            mul1(f1, k);
#pragma unroll
            for (int i = k * (NR + L) / NP; i < (k + 1) * (NR + L) / NP; ++i) {
                if (i < NR) read1(f0, i, ns, 0);
                else issue1(i - NR, kn, sl);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        sl = ns;
    }
    }
    wait_vm_lgkm<0>();
    __syncthreads();   // (the last loads have landed: the ring is free)

    const uint32_t cw = kTV / WM * wm;   // the wave's first column in the tile
    if constexpr (F8) {
        if (K % (uint32_t)kTK != 0u) {   // the last 64 k
#pragma unroll 1
            for (uint32_t h = 0; h < 2u; ++h) {
                const uint32_t ko = K - 64u + 32u * h + 16u * lh;
                Frag f;
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const uint32_t r = wn * (BR / WN) + 32u * j + lr, rs = r < vrows ? r : 0u;
                    f.x[j] = *reinterpret_cast<const u32x4_a*>(xbase + (uint64_t)(AD ? row_of(rs) : rs) * K + ko);
                }
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const uint32_t c = cw + 32u * i + lr;
                    f.w[i] = *reinterpret_cast<const u32x4_a*>(wbase + (uint64_t)(c < vcols ? c : 0u) * K + ko);
                }
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    mul1(f, k);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        // (the scales, which the threads have held since the start, by way of LDS)
        float* sc = reinterpret_cast<float*>(lds + 16u * WM * BR);   // [kTV + BR], past the epilogue's partial results
#pragma unroll
        for (uint32_t i = 0; i < NSC; ++i)
            if (NW * kWave * i + tid < kTV + BR) sc[NW * kWave * i + tid] = scales[i];
        __syncthreads();
        float xs[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) xs[j] = sc[kTV + wn * (BR / WN) + 32u * j + lr];
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 ws = *reinterpret_cast<const float4*>(sc + cw + 32u * i + 8u * q + 4u * lh);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    acc[i][j][4 * q] *= xs[j] * ws.x;
                    acc[i][j][4 * q + 1] *= xs[j] * ws.y;
                    acc[i][j][4 * q + 2] *= xs[j] * ws.z;
                    acc[i][j][4 * q + 3] *= xs[j] * ws.w;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    }
    // ---- the adapters: acc += low b^T for the rows of each adapter that the wave's
    // 32-row tiles hold. The rows are in the order of their adapters, so
    // an adapter's columns are read by one wave of two, as a rule, straight into the
    // fragments (each lane 8 consecutive k of its column, which is how the factor
    // lies in memory), DP steps of 16 ranks ahead; the rows' states, which every wave
    // over the columns needs, go by way of LDS, as many ranks at a time as the free ring
    // holds. A row's state is the sum of three bf16 parts (24 bits of mantissa, as f32:
    // two leave an error of 2.4e-6 of the adapters' part, three 9e-8 with the sums'
    // roundings, 512 k and rank 16), each what the one before leaves, towards zero: they have one sign, and the
    // first is zero with the state only. The first takes the factor as it is and the others
    // take it with infs and NaNs put to finite values, so that an inf times a state is an inf of
    // the product's sign and not the NaN of 0 inf or inf - inf. Each adapter has an
    // accumulator of its own, added to its rows only: a product with zeros instead would
    // carry an inf or NaN of one request's adapter into the others' logits.
    if constexpr (AD) {
        constexpr int DP = CT == 5 || RT == 4 ? 3 : 4;   // (what the registers hold)
        struct Step { u32x4 b[CT]; int32_t who; uint32_t k, j; };
        // (past the epilogue's partial results, the scales and the waves' rows' adapters)
        constexpr uint32_t kPast = 16u * WM * BR + (F8 ? 4u * (kTV + BR) : 0u);
        constexpr uint32_t kLow = (kPast + (RT > 1 ? 4u * WM * BR : 0u) + 127u) / 128u * 128u;
        constexpr uint32_t kFits = ((sizeof(lds) - kLow) / BR - 16u) / 96u * 16u;   // ranks at a time
        static_assert(kFits >= 16u, "the adapters' place");
        const uint32_t wide = a.ad_wide;
        const uint32_t ww = min(wide, kFits), rowb = 6u * ww + 16u;   // (16 bytes more: the rows' banks differ)
        const uint32_t rw = wn * (BR / WN) + lr;   // the lane's row in the wave's first 32-row tile
        int32_t sj[RT];                            // rank << 16 | adapter of its rows, or -1
#pragma unroll
        for (int j = 0; j < RT; ++j) sj[j] = rw + 32u * j < vrows ? a.pslot[r0 + rw + 32u * j] : -1;
        // (the tile at hand changes as the steps go: its rows' adapters by way of the wave's
        // own part of LDS)
        int32_t* ps = reinterpret_cast<int32_t*>(lds + kPast) + (uint32_t)wv * (BR / WN) + lr;
        if (RT > 1) {
#pragma unroll
            for (int j = 0; j < RT; ++j) ps[32 * j] = sj[j];   // (lanes l and l + 32 write the same)
        }
        auto of = [&](uint32_t j) -> int32_t { return RT > 1 ? ps[32u * j] : sj[0]; };
#pragma unroll 1
        for (uint32_t kw = 0u; kw < wide; kw += kFits) {
            const uint32_t kend = kw + kFits;
            if (kw != 0u) __syncthreads();
            // ranks kw to kw + ww - 1 of the rows' states: per row three bf16 parts of ww. What a
            // thread reads at a time is asked for together: the states come from another XCD.
            auto stage = [&](auto np) {
                constexpr uint32_t P = decltype(np)::value, U = P == 4u ? 1u : 2u;
                const uint32_t per = ww / 4u, all = vrows * per;
                for (uint32_t c0 = tid; c0 < all; c0 += U * NW * kWave) {
                    float4 v[U][P];
                    uint32_t row[U], ch[U];
#pragma unroll
                    for (uint32_t u = 0; u < U; ++u) {
                        const uint32_t c = c0 + u * NW * kWave, cc = c < all ? c : c0;
                        row[u] = cc / per, ch[u] = cc - row[u] * per;
                        const float* s = a.low + (uint64_t)(r0 + row[u]) * P * wide + min(kw + 4u * ch[u], wide - 4u);
#pragma unroll
                        for (uint32_t i = 0; i < P; ++i) v[u][i] = *reinterpret_cast<const float4*>(s + i * wide);
                    }
#pragma unroll
                    for (uint32_t u = 0; u < U; ++u) {
                        if (c0 + u * NW * kWave >= all) break;
                        float f[4] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w};
#pragma unroll
                        for (uint32_t i = 1; i < P; ++i) f[0] += v[u][i].x, f[1] += v[u][i].y, f[2] += v[u][i].z, f[3] += v[u][i].w;
#pragma unroll
                        for (uint32_t i = 0; i < 3u; ++i) {
                            uint32_t h[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                h[e] = bf16_top(f[e]);
                                // (an inf or NaN is whole in the first part)
                                f[e] = (h[e] & 0x7f80u) == 0x7f80u ? 0.0f : f[e] - __uint_as_float(h[e] << 16);
                            }
                            *reinterpret_cast<uint2*>(lds + kLow + row[u] * rowb + i * 2u * ww + 8u * ch[u]) =
                                make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
                        }
                    }
                }
            };
            if (a.low_s == 0u) stage(Parts<1>{});
            else if (a.low_s == 1u) stage(Parts<2>{});
            else stage(Parts<4>{});
            __syncthreads();
            uint64_t todo = ballot(sj[0] >= 0);
            uint32_t jn = 0u, kn = kw, end = kw;
            int32_t who = 0;
            const uint16_t* bp = a.ad_b;
            bool more = true;
            // The loads of the next step, tile by tile and adapter by adapter. Past the last
            // one (who -1) they are made all the same, from where the last one's were: the
            // count of loads in flight is then known where a step is used, and the ones
            // after it stay in flight.
            auto fetch = [&](Step& st) {
                while (more && kn >= end) {
                    while (todo == 0u && jn + 1u < (uint32_t)RT) todo = ballot(of(++jn) >= 0);
                    more = todo != 0u;
                    if (!more) break;
                    const int32_t s = of(jn);
                    who = __builtin_amdgcn_readlane(s, __builtin_ctzll(todo));
                    todo &= ~ballot(s == who);
                    kn = kw;
                    end = min((uint32_t)who >> 16, kend);   // (below kw: nothing of it is left)
                    bp = a.ad_b + ((uint64_t)((uint32_t)who & 0xffffu) * V + n0) * wide;
                }
                const uint32_t k = kn + 8u * lh, kk = k < end ? k : 0u;
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const uint32_t c = cw + 32u * i + lr;
                    st.b[i] = *reinterpret_cast<const u32x4_a*>(bp + (c < vcols ? c : 0u) * wide + kk);
                }
                st.who = more ? who : -1;
                st.k = more ? kn : kw;
                st.j = jn;
                kn += more ? 16u : 0u;
            };
            f32x16 t[CT];
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) t[i][e] = 0.0f;
            auto use = [&](Step& st) {
                const uint32_t rank = (uint32_t)st.who >> 16;
                const unsigned char* lp = lds + kLow + (rw + 32u * st.j) * rowb + 2u * (st.k - kw) + 16u * lh;
                u32x4 p[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) p[i] = *reinterpret_cast<const u32x4_a*>(lp + 2u * i * ww);
                if (st.k + 16u > rank) {   // what lies past the rank counts as zero, whatever it holds
                    const uint32_t k = st.k + 8u * lh, left = k < rank ? rank - k : 0u;
                    u32x4 live;
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) live[e] = left > 2u * e + 1u ? 0xffffffffu : left == 2u * e + 1u ? 0xffffu : 0u;
#pragma unroll
                    for (int i = 0; i < CT; ++i) st.b[i] &= live;
#pragma unroll
                    for (int i = 0; i < 3; ++i) p[i] &= live;
                }
                const f32x16 zero = {};
                auto mul = [&](int i, const u32x4& q, bool first) {
                    t[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, st.b[i]), __builtin_bit_cast(bf16x8, q), first ? zero : t[i], 0, 0, 0);
                };
                // (each product of the first part with the clamps of the factor of the one ahead behind it:
                // 151936 x 3584 e4m3 with 64 adapters of rank 16, 179.7 us without clamps, 182.6 so,
                // 184.3 with the clamps first; the 128 x 64 to 256 x 256 tiles are no slower)
                auto top = [&](bool first) {
#pragma unroll
                    for (int i = 0; i <= CT; ++i) {
                        if (i < CT) mul(i < CT ? i : 0, p[0], first);
                        if (i > 0) st.b[i > 0 ? i - 1 : 0] = finite_bf16(st.b[i > 0 ? i - 1 : 0]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                if (st.k == kw) top(true);
                else top(false);
#pragma unroll
                for (int q = 1; q <= 2; ++q)
#pragma unroll
                    for (int i = 0; i < CT; ++i) mul(i, p[q], false);
                if (last_step(st.who, st.k, kend)) {
#pragma unroll
                    for (int j = 0; j < RT; ++j) {
                        if ((RT == 1 || st.j == (uint32_t)j) && sj[j] == st.who) {
#pragma unroll
                            for (int i = 0; i < CT; ++i)
#pragma unroll
                                for (int e = 0; e < 16; ++e) acc[i][j][e] += t[i][e];
                        }
                    }
                }
            };
            Step st[DP];
#pragma unroll
            for (int d = 0; d < DP; ++d) fetch(st[d]);
            // (one way out of the loop, so that the count of loads in flight is the same on every
            // way in: a step past the last one adds to t, which nothing takes any more)
            while (st[0].who >= 0) {
#pragma unroll
                for (int d = 0; d < DP; ++d) {
                    use(st[d]);
                    fetch(st[d]);
                }
            }
        }
    }

    // ---- epilogue: acc[i][j][e] is column n0 + kTV / WM wm + 32 i + 8 (e / 4) +
    // 4 lh + e % 4 of row r0 + BR / WN wn + 32 j + lr ----
    struct Part { float max, sum, draft; uint32_t idx; };
    Part* part = reinterpret_cast<Part*>(lds);   // [WM][BR]: by the wave's columns
    const bool full = vcols == kTV;
    const bool vec = a.logits && (a.ld_logits & 3u) == 0u && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0u;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        const uint32_t rl = wn * (BR / WN) + 32u * j + lr;   // the lane's row in the tile
        const bool rin = rl < vrows;
        const uint32_t cb = kTV / WM * wm + 4u * lh;            // columns cb + 32 i + 8 (e / 4) + e % 4
        if (a.logits && rin) {
            float* out = a.logits + (uint64_t)row_of(rl) * a.ld_logits + n0;
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t c = cb + 32u * i + 8u * q;
                    if (vec && c + 4u <= vcols) {
                        *reinterpret_cast<float4*>(out + c) =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < vcols) out[c + e] = acc[i][j][4 * q + e];
                    }
                }
        }
        const float NEG = -__builtin_huge_valf();
        if (!full) {
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (cb + 32u * i + 8u * (e / 4) + e % 4 >= vcols) acc[i][j][e] = NEG;
        }
        // the lane's max, its first column, the draft's logit
        float m = acc[0][j][0];
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
        const int32_t dr = a.draft && rin ? a.draft[row_of(rl)] : -1;
        const uint32_t dc = (uint32_t)dr < V ? (uint32_t)dr - n0 - cb : 0xffffffffu;   // the draft's column, from cb
        uint32_t ci = kTV;
        float dl = 0.0f;
#pragma unroll
        for (int i = CT - 1; i >= 0; --i)
#pragma unroll
            for (int e = 15; e >= 0; --e) {
                const uint32_t c = 32u * i + 8u * (e / 4) + e % 4;
                ci = acc[i][j][e] == m ? c : ci;
            }
        uint32_t found = 0u;
        if (ballot(dc < kTV / WM && (dc & 4u) == 0u) != 0u) {
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t c = 32u * i + 8u * (e / 4) + e % 4;
                    if (dc == c) { dl = acc[i][j][e]; found = kLmDraftBit; }
                }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float t[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) t[k] = __builtin_amdgcn_exp2f((acc[i][j][e + k] - m) * kL2E);
                s += (t[0] + t[1]) + (t[2] + t[3]);
            }
        if (nan_bits(s)) {
            // a NaN or +inf, or nothing but -inf (columns past the vocabulary
            // too): the max and its first column again, NaNs left out, which
            // keep the sum a NaN; columns of -inf have no term
            bool nan = false;
            m = NEG;
            ci = kTV;
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = acc[i][j][e];
                    const bool n = nan_bits(v), up = !n && (ci == kTV || v > m);
                    nan = nan || n;
                    m = up ? v : m;
                    ci = up ? 32u * i + 8u * (e / 4) + e % 4 : ci;
                }
            s = m == NEG && !nan ? 0.0f : s;
        }
        ci += cb;
        // lanes l and l + 32 share a row
        const float m2 = __shfl_xor(m, 32), s2 = __shfl_xor(s, 32), d2 = __shfl_xor(dl, 32);
        const uint32_t c2 = (uint32_t)__shfl_xor((int)ci, 32), f2 = (uint32_t)__shfl_xor((int)found, 32);
        const float M = fmaxf(m, m2);
        s = (m == NEG ? s : s * __builtin_amdgcn_exp2f((m - M) * kL2E)) +
            (m2 == NEG ? s2 : s2 * __builtin_amdgcn_exp2f((m2 - M) * kL2E));
        ci = m > m2 ? ci : m2 > m ? c2 : min(ci, c2);
        if (lh == 0u) part[wm * BR + rl] = Part{M, s, found ? dl : d2, ci | found | f2};
    }
    __syncthreads();
    if (tid < vrows) {
        const float NEG = -__builtin_huge_valf();
        Part p = part[tid];
#pragma unroll
        for (int w = 1; w < WM; ++w) {
            // (a side of -inf: its sum is 0, or NaN where it holds one)
            const Part q = part[w * BR + tid];
            const float M = fmaxf(p.max, q.max);
            p.sum = (p.max == NEG ? p.sum : p.sum * __builtin_amdgcn_exp2f((p.max - M) * kL2E)) +
                    (q.max == NEG ? q.sum : q.sum * __builtin_amdgcn_exp2f((q.max - M) * kL2E));
            p.draft = (p.idx & kLmDraftBit) ? p.draft : q.draft;
            const uint32_t pc = p.idx & ~kLmDraftBit, qc = q.idx & ~kLmDraftBit;
            p.idx = (p.max > q.max ? pc : q.max > p.max ? qc : min(pc, qc)) | ((p.idx | q.idx) & kLmDraftBit);
            p.max = M;
        }
        LmRec rec;
        rec.max = p.max;
        // (a block of NaNs has no column that equals its max: its first one)
        const uint32_t col = p.idx & ~kLmDraftBit;
        rec.idx = (n0 + (col < vcols ? col : 0u)) | (p.idx & kLmDraftBit);
        rec.sum = p.sum;
        rec.draft = p.draft;
        a.recs[(uint64_t)row_of(tid) * a.nblocks + nb] = rec;
    }
}

}  // namespace lcs
