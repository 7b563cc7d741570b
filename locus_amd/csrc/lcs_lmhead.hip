// The lm-head product with the sampler's first statistics in its epilogue,
// for MI355X (gfx950): logits = X W^T in bf16 on the matrix cores (f32
// accumulation), and per (row, block of vocabulary columns) the block's
// argmax (first index), its sum of exponentials against the block max, and
// the logit of the row's draft token when the block holds it. A per-sequence
// finalize then gives each row's argmax and log-normaliser, the draft's
// log-probability and each sequence's acceptance length, so greedy and
// speculative-verify rows need no second read of the logits (and no logits
// at all when the caller does not ask for them).
//
// Reference: the output projection matvec(out_w, norm(x)) per decode token
// (src/locus/model/llama.cpp:512-513, batched at 754-761; Ops::matvec,
// backend/registry.hpp:14-15), then argmax (llama.cpp:1237-1245) and
// logprobs_from with chosen = draft (sampling.cpp:150-170) per row and the
// acceptance rule of engine.cpp:357-383 per sequence.
//
// Up to 64 rows (decode) the weight stream from HBM is the bound; from 256
// rows up (verify) the matrix cores are.
//
// Measured (us a call; the library bf16 GEMM alone 976 at 1024 rows; "before":
// this kernel's predecessor, 64 rows x 256 columns with the weight fragments
// loaded straight into registers and the shared x behind a barrier per step):
//   rows x columns x hidden       before   now
//   64   x 128256 x 4096 (logits)   218    198
//   8    x 32000  x 4096            124     51
//   128  x 128256 x 4096            448    220
//   1024 x 128256 x 4096           2619    886
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"
#include "lcs_lmtile.hpp"

namespace lcs {

namespace {
constexpr int kLmThreads = 256;
constexpr uint32_t kBigHidden = 1u << 22;     // above: 64-bit row offsets
}  // namespace

// One workgroup per sequence (rows_per_seq rows; a row is its own sequence
// when rows_per_seq is 0): wave w of NW merges rows w, w + NW, ... from their
// blocks' records (the kernel boundary orders them after the product). A row's
// records (at most 64 PER) are requested together and stay in registers: one
// memory round trip a row (1024 rows of 501 records: 13.2 -> 5.6 us).
template <int NW, uint32_t PER>
__global__ __launch_bounds__(NW * kWave) void lmhead_fin(LmArgs a) {
    __shared__ int32_t am[64];
    const uint32_t tid = tid_x();
    const int lane = lane_id(), wv = (int)(tid / kWave);
    const uint32_t R = a.rows_per_seq ? a.rows_per_seq : 1u;
    const uint32_t seq = wg_x();
    for (uint32_t j = (uint32_t)wv; j < R; j += NW) {
        const uint32_t row = seq * R + j;
        const LmRec* rr = a.recs + (uint64_t)row * a.nblocks;
        LmRec rc[PER];
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {   // (past the end: block 0 again)
            const uint32_t b = i * kWave + (uint32_t)lane;
            rc[i] = rr[b < a.nblocks ? b : 0u];
        }
        uint64_t best = ~0ull;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) best = u64_min(best, rank_key(rc[i].max, rc[i].idx & ~kLmDraftBit));
        best = wave_min_u64(best);
        const float M = rank_val(best);
        double z = 0.0;
        float dl = 0.0f;
        bool has = false;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const bool in = i * kWave + (uint32_t)lane < a.nblocks;
            z += in ? (double)rc[i].sum * (double)__builtin_amdgcn_exp2f((rc[i].max - M) * kL2E) : 0.0;
            if (in && (rc[i].idx & kLmDraftBit)) { dl = rc[i].draft; has = true; }
        }
        z = wave_sum(z);
        const uint64_t own = ballot(has);
        dl = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(dl), own ? __builtin_ctzll(own) : 0));
        const double log_z = log_f64(z) + (double)M;
        if (lane == 0) {
            a.argmax_ids[row] = (int32_t)rank_idx(best);
            if (a.log_z) a.log_z[row] = (float)log_z;
            if (a.draft_lp) a.draft_lp[row] = own ? (float)((double)dl - log_z) : 0.0f;
            if (a.stats) a.stats[row] = lcs_row_stats{log_z, M, (int32_t)rank_idx(best)};
            am[j] = (int32_t)rank_idx(best);
        }
    }
    if (!a.accept_len || !a.draft) return;
    __syncthreads();
    if (tid == 0) {
        uint32_t acc = 0;
        while (acc < R && am[acc] == a.draft[seq * R + acc]) ++acc;
        a.accept_len[seq] = acc;
    }
}

// The records' merge, after a launch of the tiles.
hipError_t launch_lmhead_fin(const LmArgs& a, hipStream_t st) {
    const uint32_t nseq = a.rows_per_seq ? a.rows / a.rows_per_seq : a.rows;
    constexpr uint32_t kMost = kLmMaxBlocks / kWave, kHalf = kMost / 2;
    const bool half = a.nblocks <= kHalf * kWave;
    if (a.rows_per_seq > 1u) {
        if (half) hipLaunchKernelGGL((lmhead_fin<8, kHalf>), dim3(nseq), dim3(8 * kWave), 0, st, a);
        else hipLaunchKernelGGL((lmhead_fin<8, kMost>), dim3(nseq), dim3(8 * kWave), 0, st, a);
    } else {
        if (half) hipLaunchKernelGGL((lmhead_fin<1, kHalf>), dim3(nseq), dim3(kWave), 0, st, a);
        else hipLaunchKernelGGL((lmhead_fin<1, kMost>), dim3(nseq), dim3(kWave), 0, st, a);
    }
    return hipGetLastError();
}

// Column blocks of 64 vt columns that a context's record buffer has to hold for
// a vocabulary (see lmhead_shape's limits).
uint32_t lmhead_max_blocks(uint32_t vocab, uint32_t cus) {
    auto n = [&](uint32_t c) { return (vocab + c - 1u) / c; };
    auto least = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
    const uint32_t n1 = least(n(64u), cus * 2u), n2 = least(n(128u), cus * 4u);
    const uint32_t m = least(n1 > n2 ? n1 : n2, kLmMaxBlocks);
    return m > n(256u) ? m : n(256u);
}

// The tile of a launch. Rows: 64-row tiles up to 64 rows; above, a 128-row tile
// where that leaves out a 256-row tile more than half empty (128 rows: 225
// against 288 us, 384 rows: 479 against 505; 256 rows: 357 against 308).
// Columns: a CU runs its workgroups' columns one after the other, whether two
// are resident or one, so the time goes by ceil(workgroups / CUs) x columns;
// narrow tiles read x more often for the same columns (64 x 128256 x 4096,
// 2 x 256, 4 x 128 and 8 x 64 columns a CU: 209, 227, 276 us), hence the
// weights. 64 rows x 4096, us by 320 / 256 / 128 / 64 columns (the rule's
// first): 20000: 51 (128), 62, 72; 40000: 89 (256), 99, 102; 80000: 131
// (320), 156, 162, 169; 128256: 209 (256), 226, 271; 151936 x 3584: 224 (320),
// 249, 251, 325.
struct LmShape { uint32_t vt, br; };
static LmShape lmhead_shape(uint32_t rows, uint32_t vocab, uint32_t hidden, uint32_t cus) {
    if (hidden > kBigHidden) return {4u, 64u};
    const uint32_t br = rows <= 64u ? 64u : rows <= 128u || (rows > 256u && rows <= 384u) ? 128u : 256u;
    const uint32_t chunks = (rows + br - 1u) / br;
    struct { uint32_t vt, br, weight; } const shapes[] = {   // (widest first; weight in 1/64)
        {5, 64, 64}, {4, 64, 64}, {2, 64, 69}, {1, 64, 85}, {4, 128, 64}, {2, 128, 77}, {4, 256, 64}, {2, 256, 77}};
    LmShape best{4u, br};
    uint64_t least = ~0ull;
    for (const auto& s : shapes) {
        if (s.br != br) continue;
        const uint64_t n = ((uint64_t)vocab + 64u * s.vt - 1u) / (64u * s.vt);
        if ((s.vt == 1u && n > 2u * cus) || (s.vt == 2u && n > 4u * cus) || n > kLmMaxBlocks) continue;   // (lmhead_max_blocks)
        const uint64_t cost = (n * chunks + cus - 1u) / cus * s.vt * s.weight;
        if (cost < least) {
            least = cost;
            best.vt = s.vt;
        }
    }
    return best;
}

hipError_t launch_lmhead(const LmArgs& a0, uint32_t cus, hipStream_t st) {
    LmArgs a = a0;
    const LmShape sh = lmhead_shape(a.rows, a.vocab, a.hidden, cus);
    const uint32_t cols = 64u * sh.vt;
    a.nblocks = (a.vocab + cols - 1u) / cols;
    a.nchunks = (a.rows + sh.br - 1u) / sh.br;
    const dim3 grid(8u * ((a.nblocks + 7u) / 8u) * a.nchunks), block(kLmThreads);
    // (stages: as deep as two workgroups a CU leave room for, or one where
    // there is no second; two of 64 k where two 256-column tiles a CU are all
    // there is: 199 us against 209 with two of 32 k and 212 with three)
    if (a.hidden > kBigHidden) hipLaunchKernelGGL((lmhead_tile<4, 64, 3, 4, 2, true>), grid, block, 0, st, a);
    else if (sh.br == 256u && sh.vt == 4u) hipLaunchKernelGGL((lmhead_tile<4, 256, 2, 8, 4>), grid, dim3(8 * kWave), 0, st, a);
    else if (sh.br == 256u) hipLaunchKernelGGL((lmhead_tile<2, 256, 3>), grid, block, 0, st, a);
    else if (sh.br == 128u && sh.vt == 4u) hipLaunchKernelGGL((lmhead_tile<4, 128, 3>), grid, block, 0, st, a);
    else if (sh.br == 128u) hipLaunchKernelGGL((lmhead_tile<2, 128, 4>), grid, block, 0, st, a);
    else if (sh.vt == 5u) hipLaunchKernelGGL((lmhead_tile<5, 64, 3>), grid, block, 0, st, a);
    else if (sh.vt == 4u && a.nblocks > cus && a.nblocks <= 2u * cus)
        hipLaunchKernelGGL((lmhead_tile<4, 64, 2, 4, 4>), grid, block, 0, st, a);
    else if (sh.vt == 4u) hipLaunchKernelGGL((lmhead_tile<4, 64, 4>), grid, block, 0, st, a);
    else if (sh.vt == 2u) hipLaunchKernelGGL((lmhead_tile<2, 64, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((lmhead_tile<1, 64, 6>), grid, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_lmhead_fin(a, st);
}

void lmhead_shape_of(uint32_t rows, uint32_t vocab, uint32_t hidden, uint32_t cus, uint32_t* vt, uint32_t* br) {
    const LmShape s = lmhead_shape(rows, vocab, hidden, cus);
    *vt = s.vt;
    *br = s.br;
}

}  // namespace lcs
