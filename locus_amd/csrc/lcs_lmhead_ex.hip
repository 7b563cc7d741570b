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
}  // namespace

// Workgroup (i, q, z): adapter i, ranks 16 q to 16 q + 15, one of the parts of k (z's low
// bits) and, from the one that z's other bits name, every low_z-th group of 16 of its
// rows; where there are fewer rows than adapters i is a row, and the workgroup of an
// adapter's first row takes it. The rows' slots give the
// adapter's rows and, by the slots below its own, its place in the order, with one
// exchange between the waves; the workgroups without work end there. A group goes
// over the part of k, the waves taking 64 k in turn in v_mfma_f32_16x16x32_bf16 tiles (ranks
// on its row side; lane l carries 8 consecutive k of row l % 16, k chunk l / 16,
// and returns rows 4 (l / 16) + e of column l % 16), up to 32 N k a wave loaded at
// once, and their sums meet in LDS in a fixed order; lmhead_tile adds up the parts of k.
// Latency bounds it (a launch, the slots, the factor from HBM), and past 128 KB of the
// factor what one CU can have in flight: hence the parts. Us with one part and as it
// is: 1 x 4096 k 8.2 and 5.6, 64 rows with 32 adapters 8.3 and 6.7; the whole call for 33 x
// 67281 x 7808 214 and 203, for 163 x 50257 x 7936 e4m3 181 and 168.
template <bool F8, uint32_t N>
__global__ __launch_bounds__(kLowThreads) void lm_low(LmArgs a) {
    struct Count { uint32_t below, mine, none, ahead; };
    __shared__ Count counts[kLowWaves];
    __shared__ uint32_t rid[kLowRows];
    __shared__ float red[kLowWaves][16 * 17];
    const uint32_t tid = tid_x();
    const int lane = lane_id(), wv = __builtin_amdgcn_readfirstlane((int)(tid / kWave));
    const uint32_t item = wg_x(), rt = __builtin_amdgcn_workgroup_id_y(), z = __builtin_amdgcn_workgroup_id_z(), zs = a.low_z;
    const uint32_t parts = 1u << a.low_s, part = z & (parts - 1u), z0 = z >> a.low_s, kstep = parts * (kLowWaves * 64u);
    const uint32_t K = a.hidden, wide = a.ad_wide;
    auto slot_at = [&](uint32_t row) -> uint32_t {   // (kAdMax: none)
        const uint32_t s = row < a.rows ? (uint32_t)a.slot[row] : kAdMax;
        return s < a.ad_n ? s : kAdMax;
    };
    // wave w holds the rows from w span, 64 at a time
    const uint32_t span = (a.rows + kLowThreads - 1u) / kLowThreads * kWave;
    const uint32_t i0 = (uint32_t)wv * span, i1 = min(i0 + span, a.rows);
    const uint32_t s0 = slot_at(i0 + (uint32_t)lane);
    const uint32_t ad = a.rows < a.ad_n ? slot_at(item) : item;
    const int32_t rk = ad == kAdMax ? 0 : a.ad_rank ? a.ad_rank[ad] : (int32_t)wide;
    const float scale = ad != kAdMax && a.ad_scale ? a.ad_scale[ad] : 1.0f;
    const uint32_t rank = rk <= 0 ? 0u : min((uint32_t)rk, wide);
    const uint32_t lr = (uint32_t)lane & 15u, lh = (uint32_t)lane >> 4;
    const uint32_t kf = (part * kLowWaves + (uint32_t)wv) * 64u, q = rt * 16u + lr;
    const uint16_t* af = a.ad_a + ((uint64_t)(ad == kAdMax ? 0u : ad) * wide + (q < rank ? q : 0u)) * K;
    auto at = [&](uint32_t k0, uint32_t s) -> uint32_t {   // the lane's k of product s
        const uint32_t k = k0 + (s / 2u) * kstep + 32u * (s % 2u) + 8u * lh;
        return k < K ? k : 8u * lh;
    };
    auto a_frag = [&](uint32_t k0, uint32_t s) { return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_a*>(af + at(k0, s))); };
    Count c = {0u, 0u, 0u, 0u};
    for (uint32_t i = i0; i < i1; i += kWave) {
        const uint32_t row = i + (uint32_t)lane, s = i == i0 ? s0 : slot_at(row);
        auto n = [](bool p) { return (uint32_t)__builtin_popcountll(ballot(p)); };
        c.below += n(row < a.rows && s < ad);
        c.mine += n(row < a.rows && s == ad);
        c.none += n(row < a.rows && s == kAdMax);
        c.ahead += n(row < item && s == ad);
    }
    if (lane == 0) counts[wv] = c;
    __syncthreads();
    // (lane w takes wave w's counts; nmine, nnone: those of the waves ahead)
    c = counts[lane < kLowWaves ? lane : 0];
    const bool in = lane < kLowWaves, before = lane < wv;
    const uint32_t pos = wave_sum_u(in ? c.below : 0u), total = wave_sum_u(in ? c.mine : 0u), none = wave_sum_u(in ? c.none : 0u);
    const uint32_t ahead = wave_sum_u(in ? c.ahead : 0u);
    const uint32_t nmine = wave_sum_u(before ? c.mine : 0u), nnone = wave_sum_u(before ? c.none : 0u);
    // this wave's rows of slot s in their order, from number n: fn(number, row)
    auto each = [&](uint32_t s, uint32_t n, auto fn) {
        for (uint32_t i = i0; i < i1; i += kWave) {
            const uint32_t row = i + (uint32_t)lane;
            const bool hit = row < a.rows && (i == i0 ? s0 : slot_at(row)) == s;
            const uint64_t b = ballot(hit);
            if (hit) fn(n + (uint32_t)__builtin_popcountll(b & ((1ull << lane) - 1ull)), row);
            n += (uint32_t)__builtin_popcountll(b);
        }
    };
    if (item == 0u && rt == 0u && z == 0u && none != 0u) {
        each(kAdMax, nnone, [&](uint32_t n, uint32_t row) {
            a.perm[a.rows - none + n] = row;
            a.pslot[a.rows - none + n] = -1;
        });
    }
    if (ad == kAdMax || total <= z0 * kLowRows || (a.rows < a.ad_n && ahead != 0u)) return;
    // the factor's first 32 N k of each wave serve every group; they are on their way
    // while the first group's rows are found
    bf16x8 fa[N];
#pragma unroll
    for (uint32_t s = 0; s < N; ++s) fa[s] = a_frag(kf, s);
    if (rt == 0u && z == 0u) {
        each(ad, nmine, [&](uint32_t n, uint32_t row) {
            a.perm[pos + n] = row;
            a.pslot[pos + n] = rank ? (int32_t)(rank << 16 | ad) : -1;
        });
    }
    if (rt * 16u >= rank) return;
    for (uint32_t g0 = z0 * kLowRows; g0 < total; g0 += zs * kLowRows) {
        const uint32_t rows = min(kLowRows, total - g0);
        each(ad, nmine, [&](uint32_t n, uint32_t row) {
            if (n - g0 < kLowRows) rid[n - g0] = row;
        });
        __syncthreads();
        const unsigned char* x = reinterpret_cast<const unsigned char*>(a.x) + (uint64_t)rid[lr < rows ? lr : 0u] * K * (F8 ? 1u : 2u);
        const uint32_t row = tid / 16u, co = tid % 16u, qo = rt * 16u + co;   // the state that the thread writes
        const float xs = F8 && a.x_scale && row < rows ? a.x_scale[rid[row]] : 1.0f;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        bf16x8 fx[N];
#pragma unroll
        for (uint32_t s = 0; s < N; ++s) fx[s] = x_frag<F8>(x, at(kf, s));
#pragma unroll
        for (uint32_t s = 0; s < N; ++s)
            if (kf + (s / 2u) * kstep < K) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[s], fx[s], acc, 0, 0, 0);
#pragma unroll 1
        for (uint32_t k0 = kf + N / 2u * kstep; k0 < K; k0 += 2u * kstep) {
            bf16x8 fb[4];
#pragma unroll
            for (uint32_t s = 0; s < 4u; ++s) {
                fb[s] = a_frag(k0, s);
                fx[s] = x_frag<F8>(x, at(k0, s));
            }
#pragma unroll
            for (uint32_t s = 0; s < 4u; ++s)
                if (k0 + (s / 2u) * kstep < K) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[s], fx[s], acc, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wv][(4 * (int)lh + e) * 17 + (int)lr] = acc[e];
        __syncthreads();
        if (row < rows && qo < wide) {
            float p = 0.0f;
#pragma unroll
            for (int w = 0; w < kLowWaves; ++w) p += red[w][co * 17u + row];
            // (ranks past the adapter's read rank 0's factor: nothing of theirs is kept)
            a.low[((uint64_t)(pos + g0 + row) * parts + part) * wide + qo] = qo < rank ? p * scale * xs : 0.0f;
        }
        __syncthreads();   // (rid and red are free for the next group)
    }
}

namespace {

template <int VT, int BR, int ST, int NW, int KS, bool F8, bool AD, int WN = 2>
void tile(const LmArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((lmhead_tile<VT, BR, ST, NW, KS, false, F8, AD, WN>), dim3(8u * ((a.nblocks + 7u) / 8u) * a.nchunks),
                       dim3(NW * kWave), 0, st, a);
}

// lm_low's workgroups: adapters or rows, 16 ranks each, z groups of rows side by side by
// 1 << s parts of k. Parts of k, then the rows' groups, side by side as long as all the
// workgroups can run at once and the states' scratch holds the parts. A part costs
// every tile another read of its rows' states: 425 x 32000 x 2688 with two parts 107, four
// 112; with up to 64 rows they pay from 1024 k up (37 x 50257 x 1600 with one 57.3, two 55.3).
struct LowGrid { uint32_t x, y, z, s; };
LowGrid low_grid(uint32_t rows, uint32_t n, uint32_t wide, uint32_t hidden, uint64_t floats, uint32_t cus) {
    LowGrid g{n < rows ? n : rows, (wide + 15u) / 16u, 1u, 0u};
    const uint32_t groups = (rows + kLowRows - 1u) / kLowRows;
    const uint32_t most = 2u * cus / (g.x * g.y), least = kLowWaves * (rows <= 64u ? 64u : 128u);
    while ((2u << g.s) <= kAdParts && (4u << g.s) <= most && least << g.s < hidden && ((uint64_t)rows * wide << g.s) * 2u <= floats) ++g.s;
    const uint32_t nz = most >> g.s;
    g.z = nz == 0u ? 1u : nz < groups ? nz : groups;
    return g;
}

// The tiles: up to 64 rows lmhead_shape's columns, above by the same measure (rounds of
// workgroups over the CUs times what one takes). Rings of 64-k stages (128 k of
// e4m3), three where they fit, and eight waves on the tiles from 256 columns up.
// Us by columns x rows, ST stages, NW waves (rings of four to eight stages are no
// faster):
//   256 x 64: 50257 x 1600 bf16 with adapters, ST 3 NW 8 41.0, NW 4 45.3, ST 2 50;
//     151936 x 3584 e4m3 (594 blocks) 132, 144, 142; 128256 x 4096 e4m3 (501) 116, 126, 116
//   320 x 64, ST 3 NW 4: 151936 x 3584 e4m3 116 (32-k stages 124), bf16 with adapters
//     225 (235), e4m3 with 64 adapters 176 (186; 180 to 183 since the factor's clamps)
//   128 x 64, ST 3 NW 4: 32000 x 2048 e4m3 15.5 (NW 8 16.1)
//   64 x 64: 16000 x 4096 e4m3 18.0 with ST 4, 19.2 with six 32-k stages, bf16 27.0, 26.6
//   256 x 128: 128 x 128256 x 4096 e4m3 ST 3 NW 8 138, NW 4 153, 32-k stages
//     163; bf16 with adapters 230, -, 266
//   256 x 256, ST 2 NW 8: 1024 x 128256 x 4096 e4m3 751 (1433 TFLOP/s); power bounds it: the
//     tile's 1.31 M cycles, of which the matrix cores are busy for 1.03 M, take 745 us on random
//     operands (1.76 GHz); on zeros 1.32 M take 562 (2.36 GHz)
struct LmExShape { uint32_t vt, br; };
LmExShape lmhead_ex_shape(uint32_t rows, uint32_t vocab, uint32_t hidden, bool f8, uint32_t cus) {
    if (rows <= 64u) {
        // 32-row tiles read half as much of x: 5 x 32000 x 2048 e4m3 17.4 -> 15.0, 16 x 128256 x
        // 4096 102.6 -> 98.6; of 64 columns 16000 x 4096 18.0 against 19.5
        LmExShape s{};
        lmhead_shape_of(rows, vocab, hidden, cus, &s.vt, &s.br);
        if (rows <= 32u && (s.vt == 2u || s.vt == 4u)) s.br = 32u;
        return s;
    }
    // (the weights are of 4096 k without adapters; what a tile takes beside its k, which tells at
    // short hidden sizes, and idle CUs at long ones, are not in them)
    // us a round, 4096 k of e4m3 (bf16: / 1.36), from 128 to 1024 rows x 2000 to 128256; one: where
    // no CU gets a second tile. 384 x 128256 e4m3 291 in rows of 192, 308 in 128, 353 in
    // 256; bf16 with adapters 437, 411, 466; 176 x 42468 x 7552 bf16 205, 233, 213; 128 x 32000
    // e4m3 43 in 128 columns, 48 in 256, bf16 66, 81; small vocabularies in 64 x 64, 128 x 64,
    // 128 x 128: 128 x 8000 e4m3 19.5, 23.0, 37.8, bf16 32, 37, 45; 128 x 16000 28.2, 25.9, 39.0 and
    // 59, 43, 49; 512 x 4000 bf16 52, 36, 43; 850 x 6861 x 6144 e4m3 135, 114, 100
    struct { uint32_t vt, br, weight, one, on; } const shapes[] = {   // on: tiles a CU holds
        {4, 256, 86, 86, 1}, {4, 192, f8 ? 72u : 80u, f8 ? 72u : 80u, 1}, {4, 128, 52, 52, 1},
        {2, 128, f8 ? 54u : 46u, f8 ? 42u : 38u, f8 ? 2u : 1u}, {2, 64, 47, f8 ? 24u : 28u, 2}, {1, 64, f8 ? 28u : 40u, f8 ? 20u : 23u, 2}};
    LmExShape best{4u, 256u};
    uint64_t least = ~0ull;
    for (const auto& s : shapes) {
        const uint64_t n = ((uint64_t)vocab + 64u * s.vt - 1u) / (64u * s.vt), all = n * ((rows + s.br - 1u) / s.br);
        if (n > kLmMaxBlocks || (s.vt <= 2u && n > 2u * s.vt * cus)) continue;   // (lmhead_max_blocks)
        const uint64_t cost = all <= cus ? s.one : (all + s.on * cus - 1u) / (s.on * cus) * s.weight;
        if (cost < least) {
            least = cost;
            best = LmExShape{s.vt, s.br};
        }
    }
    return best;
}
template <bool F8, bool AD>
void tiles(const LmArgs& a, uint32_t vt, uint32_t br, hipStream_t st) {
    if (br == 256u) tile<4, 256, 2, 8, 4, F8, AD>(a, st);
    else if (br == 192u) tile<4, 192, 2, 8, 4, F8, AD>(a, st);
    else if (br == 128u && vt == 4u) tile<4, 128, 3, 8, 4, F8, AD>(a, st);
    else if (br == 128u) tile<2, 128, F8 ? 2 : 3, F8 ? 4 : 8, 4, F8, AD>(a, st);
    else if (vt == 5u) tile<5, 64, 3, 4, 4, F8, AD>(a, st);
    else if (br == 32u && vt == 4u) tile<4, 32, 3, 4, 4, F8, AD, 1>(a, st);
    else if (br == 32u) tile<2, 32, 3, 4, 4, F8, AD, 1>(a, st);
    else if (vt == 4u) tile<4, 64, 3, 8, 4, F8, AD>(a, st);
    else if (vt == 2u) tile<2, 64, 3, 4, 4, F8, AD>(a, st);
    else tile<1, 64, F8 ? 4 : 6, 4, F8 ? 4 : 2, F8, AD>(a, st);
}

}  // namespace

hipError_t launch_lmhead_ex(const LmArgs& a0, bool f8, uint32_t cus, hipStream_t st) {
    if (!f8 && a0.ad_n == 0u) return launch_lmhead(a0, cus, st);
    LmArgs a = a0;
    const LmExShape shape = lmhead_ex_shape(a.rows, a.vocab, a.hidden, f8, cus);
    const uint32_t vt = shape.vt, br = shape.br;
    a.nblocks = (a.vocab + 64u * vt - 1u) / (64u * vt);
    a.nchunks = (a.rows + br - 1u) / br;
    if (a.ad_n != 0u) {
        const LowGrid g = low_grid(a.rows, a.ad_n, a.ad_wide, a.hidden, a.low_floats, cus);
        a.low_s = g.s;
        a.low_z = g.z;
        const bool few = a.hidden <= (uint32_t)(kLowWaves * 128) << a.low_s;
        auto low = f8 ? (few ? lm_low<true, 4> : lm_low<true, 8>) : (few ? lm_low<false, 4> : lm_low<false, 8>);
        hipLaunchKernelGGL(low, dim3(g.x, g.y, a.low_z << a.low_s), dim3(kLowThreads), 0, st, a);
        if (f8) tiles<true, true>(a, vt, br, st);
        else tiles<false, true>(a, vt, br, st);
    } else {
        tiles<true, false>(a, vt, br, st);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_lmhead_fin(a, st) : e;
}

}  // namespace lcs
