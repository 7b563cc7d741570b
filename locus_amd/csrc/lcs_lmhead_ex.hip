// The lm-head product in 8 bits and with the rows' low-rank adapters, for MI355X
// (gfx950): logits[i][v] = xs[i] ws[v] sum_k x[i][k] w[v][k]
//   + sum_q low[i][q] b[slot i][v][q],
// low[i][q] = scale[slot i] xs[i] sum_k x[i][k] a[slot i][q][k], with the
// statistics of lcs_lmhead from the epilogue (lcs_lmtile.hpp).
//
// Reference: the output projection matvec(out_w, norm(x))
// (src/locus/model/llama.cpp:512-513, 754-761); it has no adapters.
//
// Two steps before the records' merge: lm_low puts the rows in the order of their
// adapters and computes their low-rank states; lmhead_tile takes the rows in
// that order and adds the adapters' second factor to its sums, so that the
// logits are never read again and an adapter's factors are read once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"
#include "lcs_lmtile.hpp"

namespace lcs {

void lmhead_shape_of(uint32_t rows, uint32_t vocab, uint32_t hidden, uint32_t cus, uint32_t* vt, uint32_t* br);
hipError_t launch_lmhead(const LmArgs& a, uint32_t cus, hipStream_t st);
hipError_t launch_lmhead_fin(const LmArgs& a, hipStream_t st);

namespace {
constexpr int kLowWaves = 16;
constexpr int kLowThreads = kLowWaves * kWave;
constexpr uint32_t kLowRows = 16;   // rows of a group
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 8 elements of a row of x as bf16 (e4m3 values are bf16 values).
template <bool F8>
__device__ __forceinline__ bf16x8 x_frag(const unsigned char* row, uint32_t k) {
    if constexpr (!F8) {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_a*>(row + 2u * k));
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const uint2 q = *reinterpret_cast<const uint2*>(row + k);
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int w = (int)(i == 0 ? q.x : q.y);
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
            r[2 * i] = __float_as_uint(lo.x) >> 16 | (__float_as_uint(lo.y) & 0xffff0000u);
            r[2 * i + 1] = __float_as_uint(hi.x) >> 16 | (__float_as_uint(hi.y) & 0xffff0000u);
        }
        return __builtin_bit_cast(bf16x8, r);
    }
}
__device__ __forceinline__ uint32_t to_bf16(float f) {   // finite: to nearest even
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7f800000u) == 0x7f800000u) return (u >> 16) | ((u & 0x7fffffu) ? 0x40u : 0u);
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
}  // namespace

// Workgroup (i, q): up to 16 rows of one adapter (the i-th such group in the order of
// the adapters), ranks 16 q to 16 q + 15, over all of k: the waves take 64 k in
// turn in v_mfma_f32_16x16x32_bf16 tiles (ranks on its row side; lane l carries
// 8 consecutive k of row l % 16, k chunk l / 16, and returns rows 4 (l / 16) + e of
// column l % 16), and their sums meet in LDS in a fixed order. Latency bounds it:
// small tiles make many workgroups, and up to 256 k a wave are loaded at once.
// Every workgroup finds its group from the rows' slots by itself (a histogram over
// the adapters and its prefix sums), which costs less than a launch for it would.
// The groups' first workgroups also write the order, and workgroup 0 that of
// the rows without an adapter.
template <bool F8>
__global__ __launch_bounds__(kLowThreads) void lm_low(LmArgs a) {
    __shared__ uint32_t hist[kAdMax];
    __shared__ uint2 wsum[kLowWaves];
    __shared__ uint32_t wcnt[kLowWaves];
    __shared__ uint32_t rid[kLowRows];
    __shared__ uint32_t my[4];   // the adapter, its first position, its rows, the group's number in it
    __shared__ float red[kLowWaves][16 * 17];
    const uint32_t tid = tid_x();
    const int lane = lane_id(), wv = __builtin_amdgcn_readfirstlane((int)(tid / kWave));
    const uint32_t item = wg_x(), rt = __builtin_amdgcn_workgroup_id_y();
    const uint32_t K = a.hidden, wide = a.ad_wide;
    // (kAdMax: none; the first kLowThreads rows' slots stay in a register)
    auto slot_at = [&](uint32_t row) -> uint32_t {
        const uint32_t s = row < a.rows ? (uint32_t)a.slot[row] : kAdMax;
        return s < a.ad_n ? s : kAdMax;
    };
    const uint32_t s0 = slot_at(tid);
    hist[tid] = 0u;   // (as many threads as adapters at most)
    if (tid == 0u) my[0] = kAdMax;
    __syncthreads();
    for (uint32_t i = tid; i < a.rows; i += kLowThreads) {
        const uint32_t s = i < kLowThreads ? s0 : slot_at(i);
        if (s < kAdMax) atomicAdd(&hist[s], 1u);
    }
    __syncthreads();
    const uint32_t cnt = hist[tid], its = (cnt + kLowRows - 1u) / kLowRows;
    uint2 inc = make_uint2(cnt, its);   // inclusive sums over the adapters
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t u = (uint32_t)__shfl_up((int)inc.x, d), v = (uint32_t)__shfl_up((int)inc.y, d);
        if (lane >= d) { inc.x += u; inc.y += v; }
    }
    if (lane == kWave - 1) wsum[wv] = inc;
    __syncthreads();
    uint32_t total = 0u;
#pragma unroll
    for (int w = 0; w < kLowWaves; ++w) {
        const uint2 p = wsum[w];
        if (w < wv) { inc.x += p.x; inc.y += p.y; }
        total += p.x;
    }
    if (item >= inc.y - its && item < inc.y) {
        my[0] = tid;
        my[1] = inc.x - cnt;
        my[2] = cnt;
        my[3] = item - (inc.y - its);
    }
    __syncthreads();
    // the rows of adapter s (kAdMax: of none) in their order: fn(number, row)
    auto each = [&](uint32_t s, auto fn) {
        uint32_t seen = 0u;
        for (uint32_t i0 = 0u; i0 < a.rows; i0 += kLowThreads) {
            const uint32_t i = i0 + tid;
            const bool hit = i < a.rows && (i0 == 0u ? s0 : slot_at(i)) == s;
            const uint64_t b = ballot(hit);
            if (lane == 0) wcnt[wv] = (uint32_t)__builtin_popcountll(b);
            __syncthreads();
            uint32_t before = seen, all = 0u;
#pragma unroll
            for (int w = 0; w < kLowWaves; ++w) {
                const uint32_t n = wcnt[w];
                before += w < wv ? n : 0u;
                all += n;
            }
            if (hit) fn(before + (uint32_t)__builtin_popcountll(b & ((1ull << lane) - 1ull)), i);
            seen += all;
            __syncthreads();
        }
    };
    if (item == 0u && rt == 0u && total < a.rows) {
        each(kAdMax, [&](uint32_t n, uint32_t row) {
            a.perm[total + n] = row;
            a.pslot[total + n] = -1;
        });
    }
    const uint32_t ad = my[0];
    if (ad == kAdMax) return;
    const int32_t rk = a.ad_rank ? a.ad_rank[ad] : (int32_t)wide;
    const uint32_t rank = rk <= 0 ? 0u : min((uint32_t)rk, wide);
    if (rt != 0u && rt * 16u >= rank) return;
    const uint32_t g0 = my[3] * kLowRows, pos0 = my[1] + g0, rows = min(kLowRows, my[2] - g0);
    each(ad, [&](uint32_t n, uint32_t row) {
        if (n - g0 < kLowRows) {
            rid[n - g0] = row;
            if (rt == 0u) {
                a.perm[my[1] + n] = row;
                a.pslot[my[1] + n] = rank ? (int32_t)(rank << 16 | ad) : -1;
            }
        }
    });
    if (rank == 0u) return;   // (each ends with a barrier)
    const uint32_t lr = (uint32_t)lane & 15u, lh = (uint32_t)lane >> 4;
    const unsigned char* x = reinterpret_cast<const unsigned char*>(a.x) + (uint64_t)rid[lr < rows ? lr : 0u] * K * (F8 ? 1u : 2u);
    const uint32_t q = rt * 16u + lr;
    const uint16_t* af = a.ad_a + ((uint64_t)ad * wide + (q < rank ? q : 0u)) * K;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k0 = (uint32_t)wv * 64u; k0 < K; k0 += 4u * kLowWaves * 64u) {
        bf16x8 fa[8], fx[8];
#pragma unroll
        for (uint32_t s = 0; s < 8u; ++s) {
            const uint32_t k = k0 + (s / 2u) * (kLowWaves * 64u) + 32u * (s % 2u) + 8u * lh;
            fa[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_a*>(af + (k < K ? k : 8u * lh)));
            fx[s] = x_frag<F8>(x, k < K ? k : 8u * lh);
        }
#pragma unroll
        for (uint32_t s = 0; s < 8u; ++s)
            if (k0 + (s / 2u) * (kLowWaves * 64u) < K) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[s], fx[s], acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wv][(4 * (int)lh + e) * 17 + (int)lr] = acc[e];
    __syncthreads();
    const uint32_t row = tid / 16u, c = tid % 16u, qo = rt * 16u + c;
    if (row < rows && qo < wide) {
        float p = 0.0f;
#pragma unroll
        for (int w = 0; w < kLowWaves; ++w) p += red[w][c * 17u + row];
        // (ranks past the adapter's read rank 0's factor: nothing of theirs is kept)
        p = qo < rank ? p * (a.ad_scale ? a.ad_scale[ad] : 1.0f) * (F8 && a.x_scale ? a.x_scale[rid[row]] : 1.0f) : 0.0f;
        uint16_t* low = a.low + (uint64_t)(pos0 + row) * 3u * wide + qo;
#pragma unroll
        for (uint32_t i = 0; i < 3u; ++i) {
            const uint32_t u = to_bf16(p);
            low[i * wide] = (uint16_t)u;
            p = (u & 0x7f80u) == 0x7f80u ? 0.0f : p - __uint_as_float(u << 16);   // (an inf or NaN is whole in the first part)
        }
    }
}

namespace {

template <int VT, int BR, int ST, int NW, int KS, bool F8, bool AD>
void tile(const LmArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((lmhead_tile<VT, BR, ST, NW, KS, false, F8, AD>), dim3(8u * ((a.nblocks + 7u) / 8u) * a.nchunks),
                       dim3(NW * kWave), 0, st, a);
}

// (the stages: as for bf16 operands, lcs_lmhead.hip)
template <bool AD>
void tiles_f8(const LmArgs& a, uint32_t vt, uint32_t br, hipStream_t st) {
    if (br == 256u && vt == 4u) tile<4, 256, 2, 8, 4, true, AD>(a, st);
    else if (br == 256u) tile<2, 256, 3, 4, 2, true, AD>(a, st);
    else if (br == 128u && vt == 4u) tile<4, 128, 3, 4, 2, true, AD>(a, st);
    else if (br == 128u) tile<2, 128, 2, 4, 4, true, AD>(a, st);
    else if (vt == 5u) tile<5, 64, 3, 4, 2, true, AD>(a, st);
    else if (vt == 4u) tile<4, 64, 2, 4, 4, true, AD>(a, st);
    else if (vt == 2u) tile<2, 64, 2, 4, 4, true, AD>(a, st);
    else tile<1, 64, 2, 4, 4, true, AD>(a, st);
}
void tiles_ad(const LmArgs& a, uint32_t vt, uint32_t br, uint32_t cus, hipStream_t st) {
    if (br == 256u && vt == 4u) tile<4, 256, 2, 8, 4, false, true>(a, st);
    else if (br == 256u) tile<2, 256, 3, 4, 2, false, true>(a, st);
    else if (br == 128u && vt == 4u) tile<4, 128, 3, 4, 2, false, true>(a, st);
    else if (br == 128u) tile<2, 128, 4, 4, 2, false, true>(a, st);
    else if (vt == 5u) tile<5, 64, 3, 4, 2, false, true>(a, st);
    else if (vt == 4u && a.nblocks > cus && a.nblocks <= 2u * cus) tile<4, 64, 2, 4, 4, false, true>(a, st);
    else if (vt == 4u) tile<4, 64, 4, 4, 2, false, true>(a, st);
    else if (vt == 2u) tile<2, 64, 4, 4, 2, false, true>(a, st);
    else tile<1, 64, 6, 4, 2, false, true>(a, st);
}

}  // namespace

hipError_t launch_lmhead_ex(const LmArgs& a0, bool f8, uint32_t cus, hipStream_t st) {
    if (!f8 && a0.ad_n == 0u) return launch_lmhead(a0, cus, st);
    LmArgs a = a0;
    uint32_t vt, br;
    lmhead_shape_of(a.rows, a.vocab, a.hidden, cus, &vt, &br);
    a.nblocks = (a.vocab + 64u * vt - 1u) / (64u * vt);
    a.nchunks = (a.rows + br - 1u) / br;
    if (a.ad_n != 0u) {
        // (groups: at most one that is not full per adapter in use)
        const dim3 grid((a.ad_n < a.rows ? a.ad_n : a.rows) + a.rows / kLowRows, (a.ad_wide + 15u) / 16u);
        if (f8) hipLaunchKernelGGL((lm_low<true>), grid, dim3(kLowThreads), 0, st, a);
        else hipLaunchKernelGGL((lm_low<false>), grid, dim3(kLowThreads), 0, st, a);
        if (f8) tiles_f8<true>(a, vt, br, st);
        else tiles_ad(a, vt, br, cus, st);
    } else {
        tiles_f8<false>(a, vt, br, st);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_lmhead_fin(a, st) : e;
}

}  // namespace lcs
