// Attention of a step's new tokens over a paged cache and over each other, for MI355X
// (gfx950): o = sum_j p_j v_j with p = softmax_j(scale q.k_j), j over the sequence's
// cached tokens and over the new tokens that the row's mask names.
//
// The cache's rows are read once and bound it: rows_per_seq x (heads / kv_heads) rows
// share each key, and up to a few hundred of them are done before the next keys
// arrive. So the kernel is a stream of keys and values through LDS:
//
// - A wave takes 32 keys at a time, their keys and values brought to its own part of
//   LDS by 16-byte DMA loads, so that no register holds data in flight and waves need
//   no barrier; four waves take 128 consecutive tokens, a step.
//   Where rows and pairs are many, two or four waves share a tile, of which each brings its
//   part, with barriers.
// - Scores are computed transposed, S^T = K Q^T, with Q in registers as the B
//   operand: a lane then holds eight keys of one row, so that its softmax is the
//   lane's own, and the weights are already laid out as the B operand of O^T = V^T P^T.
//   V^T comes from LDS by transposing reads. One row's statistics and sums stay in
//   one lane column all the way.
// - The running maximum moves only when a score exceeds it by 2^8 (wave-uniform), so
//   that most tiles rescale nothing; weights are then up to 2^8, which f32 sums and
//   bf16 weights hold as well as 1.
// - The steps of all (sequence, kv head) pairs form one line that is cut into as many
//   equal pieces as there are workgroups on the card, whatever the lengths (and so that
//   pieces end with a pair, where that costs little): each workgroup finds its piece from
//   the lengths on the device. A pair that several workgroups share is joined by a
//   second launch from their partial sums.
//
// A weight is rounded to bf16 for the product with the values (2^-8 of itself at most,
// as the values themselves are); scores, maxima, sums and the normaliser are f32.
// e4m3 rows are widened to bf16, which is exact; a key's scale multiplies its scores, a
// value's scale its weight ahead of the rounding.
//
// What is not seen must not matter: cached rows past the length and in missing pages
// are replaced by zeros on their way to LDS and have weight 0. Among the new tokens a
// row that some see and others do not may hold infinities or NaNs: those elements
// are taken out of the product, counted for the rows that see them by another, and
// added there.
//
// (This file is compiled with NaNs honoured: a NaN in a row has to stay one.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"

namespace lcs {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
#define LCS_LDS __attribute__((address_space(3)))

constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;
constexpr float kUnset = -3.0e38f;   // the running maximum of a row that has seen nothing
constexpr float kSlack = 8.0f;       // log2 of the weights' bound
constexpr uint32_t kTileKeys = 32, kStepKeys = 128;

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A workgroup barrier for LDS: waits for no global store.
__device__ __forceinline__ void lds_sync() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// 16 bytes per lane from offset vo of a buffer to LDS at dst + 16 lane (dst is wave-uniform);
// what lies past the buffer's size arrives as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const unsigned char* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned char* dst, uint32_t vo) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LCS_LDS void*)dst, 16, (int)vo, 0, 0, 0);
}
__device__ __forceinline__ void dma4(const void* src, unsigned char* dst) {   // from a per-lane address to dst + 4 lane
    __builtin_amdgcn_global_load_lds((const LCS_GLOBAL void*)src, (LCS_LDS void*)dst, 4, 0, 0);
}
constexpr uint32_t kNoByte = 0x80000000u;   // an offset past every buffer
// Transposing reads of eight keys' elements by four (16-bit) or eight (8-bit) dim tiles, waited for here:
// the compiler would have the builtins wait for every DMA load that is under way.
template <int ROWS16>   // bytes of 16 rows
__device__ __forceinline__ void read_tr16(const uint32_t (&at)[4], u32x4 (&o)[4]) {
    u32x2 r[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(ROWS16)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = u32x4{r[2 * k][0], r[2 * k][1], r[2 * k + 1][0], r[2 * k + 1][1]};
}
__device__ __forceinline__ void read_tr8(const uint32_t (&at)[4], u32x2 (&o)[4]) {
    asm volatile("ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\tds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
                 : "memory");
}
// Plain reads, likewise: 16 bytes at each address and NEXT bytes behind it.
template <int NEXT>
__device__ __forceinline__ void read_one(const uint32_t (&at)[1], u32x4 (&lo)[1], u32x4 (&hi)[1]) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0])
                 : "v"(at[0]), "n"(NEXT)
                 : "memory");
}
template <int NEXT>
__device__ __forceinline__ void read_two(const uint32_t (&at)[2], u32x4 (&lo)[2], u32x4 (&hi)[2]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%6\n\tds_read_b128 %2, %5\n\tds_read_b128 %3, %5 offset:%6\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
                 : "v"(at[0]), "v"(at[1]), "n"(NEXT)
                 : "memory");
}
template <int NEXT>
__device__ __forceinline__ void read_four(const uint32_t (&at)[4], u32x4 (&lo)[4], u32x4 (&hi)[4]) {
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:%12\n\tds_read_b128 %2, %9\n\tds_read_b128 %3, %9 offset:%12\n\t"
                 "ds_read_b128 %4, %10\n\tds_read_b128 %5, %10 offset:%12\n\tds_read_b128 %6, %11\n\tds_read_b128 %7, %11 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(NEXT)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds_at(const unsigned char* p) { return (uint32_t)(uintptr_t)(LCS_LDS const unsigned char*)p; }
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
// Over the four lanes that hold a row (lane, lane ^ 16, lane ^ 32, lane ^ 48).
template <class F>
__device__ __forceinline__ float across(float x, F f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {   // to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// A tile's row is a power of two of 16-byte chunks in LDS; chunk c of row r lies at place c
// ^ x(r), so that the reads of a half wave cover the 64 banks once. x picks bits of r.
template <int ROWB>   // bytes of a row
__device__ __forceinline__ constexpr uint32_t swz_k(uint32_t r) {   // 16 rows, one chunk
    return ROWB == 64 ? r >> 2 & 3u : ROWB == 128 ? r >> 1 & 7u : r & 15u;
}
template <int ROWB, bool B8>
__device__ __forceinline__ constexpr uint32_t swz_v(uint32_t r) {
    if (!B8) return ROWB == 128 ? 2u * (r >> 1 & 3u) : 2u * (r & 7u);   // 8 rows, two chunks
    return ROWB == 64 ? (r >> 2 & 1u) | (r >> 3 & 2u) : ROWB == 128 ? (r >> 1 & 3u) | (r >> 2 & 4u) : (r & 7u) | (r >> 1 & 8u);   // rows 0-7 and 16-23, one chunk
}

// Where each sequence's steps lie on the line of all: lane l holds sequences per * l ..
// per * (l + 1) - 1 (at most 16).
struct Seq {
    uint32_t len, steps;   // cached tokens; steps, those of the new tokens included
    int32_t slot;
};
struct Line {
    uint32_t per, before, total;   // units ahead of the lane's sequences, of all sequences (of one kv head)
    uint32_t unit, share;          // steps of a unit; units of a piece
    Seq one;                       // the lane's last sequence
    bool bad;
    __device__ __forceinline__ uint32_t units(const Seq& q) const { return unit == 1u ? q.steps : (q.steps + unit - 1u) / unit; }
};
__device__ __forceinline__ Seq seq_of(const TreeArgs& a, uint32_t i, bool& bad) {
    const int32_t slot = a.c.seq ? a.c.seq[i] : (int32_t)i;
    const uint64_t most = (uint64_t)a.c.max_pages << a.c.page_shift;
    const int32_t n = a.length[i];
    uint32_t len = slot == -1 || n < 0 ? 0u : (uint32_t)n;
    if (slot < -1 || slot >= (int64_t)a.c.seqs) {
        bad = true;
        len = 0u;
    } else if (len > most) {
        bad = true;
        len = (uint32_t)most;
    }
    return Seq{len, (len + kStepKeys - 1u) / kStepKeys + a.new_steps, slot};
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
// The line is cut into a.pieces equal pieces, of `share` steps each. A piece that begins with one
// pair's end and goes on with another's start pays twice for what a pair costs by itself
// (about three steps), so pairs of up to 64 sequences, one a lane, are cut by themselves instead,
// into units of up to kMoreShare steps more than `share`, a piece each, if there are pieces enough (16 trees of 16 nodes over
// 300 to 6000 tokens, 8 kv heads: 64.7 -> 59.5 us; 16 of 48 over 600: 40.3 -> 31.1; 32 single
// tokens over 4096: 106 -> 99; 7 trees of 13 over up to 1777, 5 heads: 24.3 -> 19.5).
constexpr uint32_t kMoreShare = 3;
__device__ __forceinline__ Line line_of(const TreeArgs& a) {
    Line l{(a.c.n + kWave - 1u) / kWave, 0u, 0u, 1u, 0u, Seq{0u, 0u, 0}, false};
    uint32_t sum = 0;
    for (uint32_t k = 0; k < l.per; ++k) {
        const uint32_t i = (uint32_t)lane_id() * l.per + k;
        if (i < a.c.n) {
            l.one = seq_of(a, i, l.bad);
            sum += l.one.steps;
        }
    }
    uint32_t incl = wave_scan_incl_u(sum);
    l.before = incl - sum;
    l.total = (uint32_t)__builtin_amdgcn_readlane((int)incl, kWave - 1);
    const uint32_t H = a.c.kv_heads;
    l.share = max((l.total * H + a.pieces - 1u) / a.pieces, 1u);
    if (l.per == 1u && l.share > 1u) {   // (uniform; lanes without a sequence have 0 steps)
        for (uint32_t unit = l.share; unit <= l.share + kMoreShare; ++unit) {
            const uint32_t mine = (l.one.steps + unit - 1u) / unit;
            incl = wave_scan_incl_u(mine);
            const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, kWave - 1);
            if (total * H <= a.pieces) {
                l.before = incl - mine;
                l.total = total;
                l.unit = unit;
                l.share = 1u;
                break;
            }
        }
    }
    return l;
}

template <int DP>
constexpr int kTreePerCu = DP == 256 ? 1 : 2;   // workgroups a CU

// A partial result: the rows' unnormalised sums, then their maxima (log2) and sums of weights.
template <int DP, int MT>
struct Part {
    static constexpr uint32_t kRows = 16u * MT;
    static constexpr uint32_t kFloats = kRows * DP + 2u * kRows;
};

}  // namespace

// A workgroup has NW tiles before it at once, each shared by WR waves of 16 MT rows.
template <int DP, int MT, bool F8, int ST, int WR, int NW>
__global__ __launch_bounds__(NW * WR * kWave, NW * WR == 4 ? kTreePerCu<DP> : 1) void tree_attn(TreeArgs a) {
    static_assert(WR == 1 || ((WR == 2 || WR == 4) && ST == 2 && !F8), "the schedule of shared tiles");
    constexpr uint32_t kStride = NW * kTileKeys, kPer = kStepKeys / kStride;   // keys from tile to tile of a wave, its tiles a step
    constexpr uint32_t kMine = 16u * MT, kRows = kMine * WR, kDT = DP / 16, kKS = DP / 32;   // rows of a wave, of the workgroup
    constexpr uint32_t kRowB = DP * (F8 ? 1 : 2), kNewB = DP * 2;                 // bytes of a cached row and of a new one in LDS
    constexpr uint32_t kScaleB = F8 ? 256u : 0u;
    constexpr uint32_t kStage = 2u * kTileKeys * kRowB + kScaleB;
    constexpr uint32_t kMergeB = kRows * DP * 4u;
    constexpr uint32_t kMax1 = 2u * kTileKeys * kNewB > ST * kStage ? 2u * kTileKeys * kNewB : ST * kStage;
    constexpr uint32_t kRegion = kMax1 > kMergeB ? kMax1 : kMergeB;
    constexpr int kNI = (int)(kTileKeys * kRowB / 1024u);      // DMA loads of a tile's keys, and of its values
    constexpr int kNK = kNI + (F8 ? 1 : 0);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[NW * kRegion];
    __shared__ float stat[NW][2][kRows];
    const uint32_t lane = (uint32_t)lane_id(), wave = uniform(tid_x() / kWave), w = wave % NW, wr = wave / NW, n = lane & 15u, g = lane >> 4;
    unsigned char* const mine = lds + w * kRegion;
    const uint32_t b = wg_x(), piece = b / 8u / a.row_tiles * 8u + b % 8u, rt = b / 8u % a.row_tiles + a.row_tile0;
    const Line line = line_of(a);
    if (line.bad && b == 0u && wave == 0u) atomicOr(a.c.status, kStatusPages);
    const uint32_t H = a.c.kv_heads, all = line.total * H, share = line.share;
    const uint32_t end = min(all, (piece + 1u) * share);   // (all < 2^31 / ...: checked on the host)
    const uint32_t D = a.c.head_dim, N = a.rows_per_seq, R = N * a.group;
    const uint64_t ts = a.c.token_stride * (F8 ? 1u : 2u);
    const float sc = (a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale)) * kLog2e;
    // a score's dims: k-slot (ks, g, j) of the products is dim 8 chunk8(ks) + j of both operands
    auto chunk8 = [&](uint32_t ks) -> uint32_t { return F8 ? 2u * (g + 4u * (ks / 2u)) + (ks & 1u) : 4u * ks + g; };

    uint32_t x = piece * share;
    while (x < end) {
        // ---- the segment: the steps of one (sequence, kv head) pair in this piece ----
        // the lane that holds the sequence is the last whose steps begin at or ahead of x
        const uint64_t le = ballot(line.before * H <= x && lane * line.per < a.c.n);
        const uint32_t who = 63u - (uint32_t)__builtin_clzll(le);
        uint32_t i = who * line.per, at = uniform((uint32_t)__builtin_amdgcn_readlane((int)line.before, (int)who)) * H;
        Seq sq;
        if (line.per == 1u) {   // (uniform)
            sq.len = (uint32_t)__builtin_amdgcn_readlane((int)line.one.len, (int)who);
            sq.steps = (uint32_t)__builtin_amdgcn_readlane((int)line.one.steps, (int)who);
            sq.slot = __builtin_amdgcn_readlane(line.one.slot, (int)who);
        } else {
            bool dummy = false;
            sq = seq_of(a, i, dummy);
            while (x - at >= sq.steps * H) {   // (units of one step)
                at += sq.steps * H;
                sq = seq_of(a, ++i, dummy);
            }
        }
        i = uniform(i);
        const uint32_t len = uniform(sq.len), steps = uniform(sq.steps);
        const int32_t slot = (int32_t)uniform((uint32_t)sq.slot);
        const uint32_t units = line.units(Seq{len, steps, slot}), y = x - uniform(at), kvh = y / units, u0 = y % units, u1 = min(units, u0 + (end - x));
        const uint32_t s0 = u0 * line.unit, s1 = min(steps, u1 * line.unit);
        const uint32_t ctx_steps = steps - a.new_steps;
        const int32_t* row = a.c.table + (uint64_t)(len > 0u ? (uint32_t)slot : 0u) * a.c.max_pages;
        const unsigned char* kb = static_cast<const unsigned char*>(a.c.k) + (a.c.layer * a.c.layer_stride + kvh * a.c.head_stride) * (F8 ? 1u : 2u);
        const unsigned char* vb = static_cast<const unsigned char*>(a.c.v) + (a.c.layer * a.c.layer_stride + kvh * a.c.head_stride) * (F8 ? 1u : 2u);

        // ---- the wave's cached tiles: tile j starts at token first + kStride j ----
        const uint32_t c1 = min(s1, ctx_steps), first = s0 * kStepKeys + w * kTileKeys;
        const uint32_t nct = s0 < c1 ? (c1 - s0) * kPer : 0u;   // (the last ones may lie past the length: all zeros, unseen)
        struct Tile {
            uint32_t p0, p1;   // the pages of its first and last 16 tokens
            uint32_t there;    // its keys that are there (settle)
        };
        auto pages_of = [&](uint32_t j) -> Tile {
            const uint32_t t0 = first + (j < nct ? j : 0u) * kStride;
            const uint32_t q0 = min(t0 >> a.c.page_shift, a.c.max_pages - 1u), q1 = min((t0 + 16u) >> a.c.page_shift, a.c.max_pages - 1u);
            if (nct == 0u) return Tile{0u, 0u, 0u};
            return Tile{(uint32_t)scalar_load(row + q0), (uint32_t)scalar_load(row + q1), 0u};
        };
        auto expected = [&](uint32_t j) -> uint32_t {   // the keys of tile j ahead of the length
            const uint32_t t0 = first + j * kStride, left = t0 < len ? len - t0 : 0u;
            return left >= 32u ? ~0u : (1u << left) - 1u;
        };
        auto settle = [&](Tile& t, uint32_t j) {   // (a page that is missing: none of its keys, page 0 in its place)
            t.there = expected(j) & (t.p0 < a.c.pages ? ~0u : 0xffff0000u) & (t.p1 < a.c.pages ? ~0u : 0x0000ffffu);
            t.p0 = t.p0 < a.c.pages ? t.p0 : 0u;
            t.p1 = t.p1 < a.c.pages ? t.p1 : 0u;
        };
        // A tile's 16-row halves lie in one page each; DMA load ii of a half covers rows RPI ii + lane /
        // CPR, a chunk per lane. A half's buffer ends with its last row that is there.
        constexpr uint32_t CPR = kRowB / 16u, RPI = 64u / CPR;
        constexpr int kHalf = kNI / 2, kShare = WR == 4 ? kHalf / 2 : kHalf;   // DMA loads of a half, and those of it that the wave issues
        static_assert(kShare > 0, "a load for each wave");
        const uint32_t part0 = WR == 4 ? (wr & 1u) * (uint32_t)kShare : 0u;
        const uint32_t tsb = (uint32_t)ts;
        auto offset_of = [&](bool values, uint32_t r) -> uint32_t {   // the lane's chunk of row r
            const uint32_t ch = (lane % CPR) ^ (values ? swz_v<kRowB, F8>(r) : swz_k<kRowB>(r));
            return 16u * ch < D * (F8 ? 1u : 2u) ? (r & 15u) * tsb + 16u * ch : kNoByte;
        };
        constexpr int kVo = F8 ? kNI : kShare;   // (8-bit values: the second half is permuted by other bits)
        uint32_t vo_k[kShare], vo_v[kVo];
#pragma unroll
        for (int ii = 0; ii < kShare; ++ii) vo_k[ii] = offset_of(false, RPI * (part0 + (uint32_t)ii) + lane / CPR);
#pragma unroll
        for (int ii = 0; ii < kVo; ++ii) vo_v[ii] = offset_of(true, RPI * (part0 + (uint32_t)ii) + lane / CPR);
        const uint32_t psb = (uint32_t)a.c.page_stride * (F8 ? 1u : 2u);   // (below 2^32, and so is a row's place in its page)
        auto issue_rows = [&](bool values, const Tile& t, uint32_t j, unsigned char* dst) {
            const unsigned char* base = values ? vb : kb;
#pragma unroll
            for (uint32_t q = 0; q < (WR == 1 ? 2u : 1u); ++q) {   // (waves that share a tile bring a half or a quarter each)
                const uint32_t h = WR == 1 ? q : wr / (WR / 2u), first_page = t.p0, second_page = t.p1, in_page = ((first + j * kStride + 16u * h) & (a.c.page_tokens - 1u)) * tsb;
                const __amdgpu_buffer_rsrc_t rs = buffer_of(base + (uint64_t)(h ? second_page : first_page) * psb + in_page,
                                                            (uint32_t)__builtin_popcount(t.there >> (16u * h) & 0xffffu) * tsb);
#pragma unroll
                for (int ii = 0; ii < kShare; ++ii)
                    dma16(rs, dst + 1024 * (kHalf * h + part0 + ii), values ? vo_v[F8 ? kHalf * q + ii : ii] : vo_k[ii]);
            }
        };
        auto issue_k = [&](const Tile& t, uint32_t j, uint32_t stage) {
            unsigned char* dst = mine + stage;
            if constexpr (F8) {   // the keys' scales by the lower half, the values' by the upper
                const uint32_t r = lane & 31u, tok = (first + j * kStride + r) & (a.c.page_tokens - 1u), first_page = t.p0, second_page = t.p1;
                const float* s = lane < 32u ? a.c.k_scale : a.c.v_scale;
                const uint64_t e = ((((uint64_t)a.c.layer * a.c.pages + (r < 16u ? first_page : second_page)) * H + kvh) << a.c.page_shift) + tok;
                dma4(t.there >> r & 1u ? static_cast<const void*>(s + e) : a.zeros, dst + 2u * kTileKeys * kRowB);
            }
            issue_rows(false, t, j, dst);
        };
        auto issue_v = [&](const Tile& t, uint32_t j, uint32_t stage) { issue_rows(true, t, j, mine + stage + kTileKeys * kRowB); };

        Tile tile[ST + 1];   // of tiles j, j + 1, .. j + ST
#pragma unroll
        for (int k = 0; k <= ST; ++k) tile[k] = pages_of((uint32_t)k);
#pragma unroll
        for (int k = 0; k < ST; ++k) settle(tile[k], (uint32_t)k);
        // ---- the new tokens' tiles (bf16 always), the first one's loads issued where LDS is free ahead of it ----
        constexpr int kNew = (int)(kTileKeys * kNewB / 1024u);   // DMA loads of a tile's keys, and of its values
        const uint32_t st0 = max(s0, ctx_steps);
        auto new_first = [&](uint32_t st) -> uint32_t { return (st - ctx_steps) * kStepKeys + w * kTileKeys; };   // (and every kStride on)
        const bool ahead = st0 < s1 && new_first(st0) < N;
        auto issue_new = [&](bool values, uint32_t n0, unsigned char* dst) {
            constexpr uint32_t CPN = kNewB / 16u, RPN = 64u / CPN;
            const uint32_t rows = min(N - n0, kTileKeys), stride = (uint32_t)(values ? a.v_stride : a.k_stride) * 2u;
            const uint16_t* src = (values ? a.v : a.k) + ((uint64_t)i * N + n0) * (values ? a.v_stride : a.k_stride) + kvh * D;
            const __amdgpu_buffer_rsrc_t rs = buffer_of(reinterpret_cast<const unsigned char*>(src), (rows - 1u) * stride + 2u * D);
            uint32_t ln = lane;   // (opaque: what follows from it is not kept over the cached tiles)
            asm volatile("" : "+v"(ln));
#pragma unroll
            for (int q = 0; q < kNew / WR; ++q) {
                const int ii = q + (int)wr * (kNew / WR);
                const uint32_t r = RPN * (uint32_t)ii + ln / CPN, c = ln % CPN ^ (values ? swz_v<kNewB, false>(r) : swz_k<kNewB>(r));
                dma16(rs, dst + 1024 * ii, r < rows && 8u * c < D ? r * stride + 16u * c : kNoByte);
            }
        };
        // their places: with one stage its keys' and values' places; with two the other stage, and
        // for 8-bit rows (a new row takes two cached ones' room) the last tile's own for the values
        unsigned char* new_k = mine;
        unsigned char* new_v = mine + kTileKeys * kNewB;

        // ---- the rows: packed as (new token, query head of the group) ----
        u32x4 qr[MT][kKS];
        uint32_t node[MT];
        bool live[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint32_t pr = rt * kRows + wr * kMine + 16u * m + n;
            live[m] = pr < R;
            node[m] = live[m] ? pr / a.group : 0u;
            const uint16_t* q = a.q + ((uint64_t)i * N + node[m]) * a.q_stride + (kvh * a.group + (live[m] ? pr - node[m] * a.group : 0u)) * D;
#pragma unroll
            for (uint32_t ks = 0; ks < kKS; ++ks) qr[m][ks] = *reinterpret_cast<const u32x4*>(q + (8u * chunk8(ks) < D ? 8u * chunk8(ks) : 0u));
        }

        // (rows past the last and dims past the head's count as zeros; so do all at a scale of 0,
        // whose scores are 0; a scale below 0 changes the sign here)
        bf16x8 qf[MT][kKS];
        auto take_q = [&] {
            const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (uint32_t ks = 0; ks < kKS; ++ks) {
                    const bool in = live[m] && 8u * chunk8(ks) < D && a.scale != 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) qr[m][ks][k] = in ? qr[m][ks][k] ^ flip : 0u;
                    qf[m][ks] = __builtin_bit_cast(bf16x8, qr[m][ks]);
                }
        };
        // (the queries are waited for where the loads behind them are the same on every path: the
        // compiler counts those that surely follow)
        if (nct != 0u) {
            issue_k(tile[0], 0u, 0u);
            issue_v(tile[0], 0u, 0u);
            take_q();
            if (ST == 2 && nct > 1u) {
                issue_k(tile[1], 1u, kStage);
                if (WR == 1) issue_v(tile[1], 1u, kStage);
            }
        } else {
            if (ahead) {
                issue_new(false, new_first(st0), new_k);
                issue_new(true, new_first(st0), new_v);
            }
            take_q();
        }
        f32x4 acc[MT][kDT];
        float top[MT], sum[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            top[m] = kUnset;
            sum[m] = 0.0f;
#pragma unroll
            for (uint32_t t = 0; t < kDT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // Scores of a tile to weights, packed as the second product's operand.
        f32x4 s[MT][2];
        bf16x8 pf[MT];
        auto hide = [&](int m, uint32_t see) {   // bit k of see: the lane's row m sees key k
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[m][h][r] = see >> (16u * h + 4u * g + r) & 1u ? s[m][h][r] : -__builtin_huge_valf();
        };
        auto weigh = [&](const f32x4 (&vs)[2], bool scaled) {
            float big[MT];
            bool up = false;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                big[m] = -__builtin_huge_valf();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) big[m] = f_max(big[m], s[m][h][r]);
                up = up || big[m] * sc > top[m] + kSlack;
            }
            if (ballot(up) != 0ull) {   // (uniform)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const float now = f_max(top[m], across(big[m], f_max) * sc), f = exp2_f(top[m] - now);
                    top[m] = now;
                    sum[m] *= f;
#pragma unroll
                    for (uint32_t t = 0; t < kDT; ++t) acc[m][t] *= f;
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                u32x4 p;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[m][h][r] = exp2_f(__builtin_fmaf(s[m][h][r], sc, -top[m]));
                        sum[m] += s[m][h][r];
                        if (scaled) s[m][h][r] *= vs[h][r];
                    }
                    p[2 * h] = pack_bf16(s[m][h][0], s[m][h][1]);
                    p[2 * h + 1] = pack_bf16(s[m][h][2], s[m][h][3]);
                }
                pf[m] = __builtin_bit_cast(bf16x8, p);
            }
        };
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        // where the lane's transposing reads of dim tile t begin (the permutation repeats after kTr tiles)
        constexpr uint32_t kTr = F8 ? (kDT < 8u || DP == 256 ? kDT : 8u) : (kDT < 8u ? kDT : 8u);
        uint32_t tr_at[kTr];
#pragma unroll
        for (uint32_t t = 0; t < kTr; ++t) {
            const uint32_t q = n >> 1, r = !F8 ? 4u * g + (n >> 2) : q < 4u ? 4u * g + q : 12u + 4u * g + q;
            const uint32_t c = F8 ? t : 2u * t + (lane >> 1 & 1u);
            tr_at[t] = r * kRowB + (c ^ swz_v<kRowB, F8>(r)) * 16u + 8u * (lane & 1u);
        }

        uint32_t stage = 0;
#pragma clang loop unroll(disable)
        for (uint32_t j = 0; j < nct; ++j) {
            uint32_t fresh_stage = stage;   // (opaque: the loads' LDS places follow from it by additions, and take no registers)
            asm volatile("" : "+s"(fresh_stage));
            unsigned char* const at_k = mine + stage;
            unsigned char* const at_v = at_k + kTileKeys * kRowB;
            const bool full = j + ST <= nct;   // (ST tiles are under way)
            constexpr int kIK = kShare, kIV = kShare;   // (shared tiles) loads of a wave
            if constexpr (WR > 1) {
                // A step of shared tiles: the next values go out once all have taken the last ones', the keys
                // after the next once all have read these, so that three half steps are under way.
                if (full) wait_vm<kIV + kIK>();
                else wait_vm<kIV>();
                lds_sync();
                if (j + 1u < nct) issue_v(tile[1], j + 1u, fresh_stage ? 0u : kStage);
            } else if (full) {
                wait_vm<kNI + (ST - 1) * (kNK + kNI)>();
            } else {
                wait_vm<kNI>();
            }
            u32x4 kc[2][F8 ? kKS / 2 : kKS];
            f32x4 ks[2] = {zero, zero}, vs[2] = {zero, zero};
            constexpr uint32_t kKC = F8 ? kKS / 2 : kKS;   // 16-byte chunks of a key that a lane takes
            const uint32_t lk = lds_at(at_k) + n * kRowB;
#pragma unroll
            for (uint32_t c0 = 0; c0 < kKC; c0 += 4u) {
                constexpr uint32_t kAt = kKC < 4u ? kKC : 4u;
                uint32_t ad[kAt];
                u32x4 lo[kAt], hi[kAt];
#pragma unroll
                for (uint32_t c = 0; c < kAt; ++c) ad[c] = lk + ((4u * (c0 + c) + g) ^ swz_k<kRowB>(n)) * 16u;
                if constexpr (kAt == 4u) {
                    read_four<16 * kRowB>(ad, lo, hi);
                } else if constexpr (kAt == 2u) {
                    read_two<16 * kRowB>(ad, lo, hi);
                } else {
                    read_one<16 * kRowB>(ad, lo, hi);
                }
#pragma unroll
                for (uint32_t c = 0; c < kAt; ++c) {
                    kc[0][c0 + c] = lo[c];
                    kc[1][c0 + c] = hi[c];
                }
            }
            if constexpr (F8) {   // the scales of keys 4 g .. and 16 + 4 g ..; the values' 128 bytes behind
                const uint32_t sa = lds_at(at_k) + 2u * kTileKeys * kRowB + 16u * g, ad[2] = {sa, sa + 64u};
                u32x4 lo[2], hi[2];
                read_two<128>(ad, lo, hi);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ks[h] = __builtin_bit_cast(f32x4, lo[h]);
                    vs[h] = __builtin_bit_cast(f32x4, hi[h]);
                }
            }
            const bool more = j + ST < nct;
            settle(tile[ST], j + ST);
            const bool then = ahead && j + 1u == nct;   // (the new tokens come next)
            if (then) {
                if constexpr (WR > 1) {
                    new_k = mine + (stage ? 0u : kStage);
                    new_v = new_k + kTileKeys * kNewB;
                    issue_new(false, new_first(st0), new_k);
                    issue_new(true, new_first(st0), new_v);
                } else if constexpr (ST == 1) {
                    issue_new(false, new_first(st0), new_k);
                } else {
                    new_k = mine + (stage ? 0u : kStage);
                    issue_new(false, new_first(st0), new_k);
                    new_v = F8 ? mine + stage : new_k + kTileKeys * kNewB;
                    if constexpr (!F8) issue_new(true, new_first(st0), new_v);
                }
            }
            if (WR == 1 && more) issue_k(tile[ST], j + ST, fresh_stage);
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][0] = s[m][1] = zero;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t k = 0; k < kKS; ++k) {
                    bf16x8 kf;
                    if constexpr (F8) {
                        union { bf16x2 p[4]; bf16x8 v; } u;
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            u.p[2 * d] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kc[h][k / 2][2 * (k & 1) + d], 1.0f, false);
                            u.p[2 * d + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kc[h][k / 2][2 * (k & 1) + d], 1.0f, true);
                        }
                        kf = u.v;
                    } else {
                        kf = __builtin_bit_cast(bf16x8, kc[h][k]);
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) s[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[m][k], s[m][h], 0, 0, 0);
                }
            if constexpr (F8) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[m][h] *= ks[h];
            }
            if (tile[0].there != ~0u) {   // (uniform)
#pragma unroll
                for (int m = 0; m < MT; ++m) hide(m, tile[0].there);
                if (tile[0].there != expected(j) && lane == 0u) atomicOr(a.c.status, kStatusPages);   // (a page is missing)
            }
            weigh(vs, F8);
            if constexpr (WR > 1) {
                if (then) wait_vm<2 * kNew / WR>();   // (its shares of both)
                else if (full) wait_vm<kIK + kIV>();
                else wait_vm<0>();
                lds_sync();
                if (more) issue_k(tile[ST], j + ST, fresh_stage);
            } else if (then) wait_vm<ST == 2 && !F8 ? 2 * kNew : kNew>();
            else if (!full) wait_vm<0>();
            else if (more) wait_vm<(ST - 1) * (kNK + kNI) + kNK>();
            else wait_vm<(ST - 1) * (kNK + kNI)>();
            const uint32_t lv = lds_at(at_v);
            using Raw = std::conditional_t<F8, u32x2, u32x4>;
            Raw vc[kDT];
#pragma unroll
            for (uint32_t t = 0; t < kDT; t += 4u) {
                uint32_t ad[4];
                Raw o[4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) ad[k] = lv + tr_at[(t + k) % kTr] + (t + k) / kTr * (kTr * (F8 ? 16u : 32u));
                if constexpr (F8) read_tr8(ad, o);
                else read_tr16<16 * kRowB>(ad, o);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) vc[t + k] = o[k];
            }
            if constexpr (WR == 1 && (ST == 1 || F8)) {
                if (then) issue_new(true, new_first(st0), new_v);
            }
            if (WR == 1 && more) issue_v(tile[ST], j + ST, fresh_stage);
            stage = stage + kStage == ST * kStage ? 0u : stage + kStage;
#pragma unroll
            for (int k = 0; k < ST; ++k) tile[k] = tile[k + 1];
            tile[ST] = pages_of(j + 1u + ST);
#pragma unroll
            for (uint32_t t = 0; t < kDT; ++t) {
                bf16x8 vf;
                if constexpr (F8) {
                    union { bf16x2 p[4]; bf16x8 v; } u;
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        u.p[2 * d] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc[t][d], 1.0f, false);
                        u.p[2 * d + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc[t][d], 1.0f, true);
                    }
                    vf = u.v;
                } else {
                    vf = __builtin_bit_cast(bf16x8, vc[t]);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[m], acc[m][t], 0, 0, 0);
            }
        }

        // ---- the new tokens' products ----
        const uint32_t nnt = st0 < s1 ? (s1 - st0) * kPer : 0u;
        for (uint32_t jn = 0; jn < nnt; ++jn) {
            const uint32_t n0 = new_first(st0) + jn * kStride;
            if (n0 - w * kTileKeys >= N) break;   // (uniform over the workgroup)
            const bool in = n0 < N;   // (uniform over the waves that share a tile; all take part in the barriers)
            if (WR == 1 && !in) continue;
            uint32_t ln = lane;   // (opaque, as above)
            asm volatile("" : "+v"(ln));
            const uint32_t lane_n = ln & 15u, lg = ln >> 4;
            if (jn != 0u) {   // (the last tile has been read)
                if constexpr (WR > 1) lds_sync();
                else wait_lds();
                if (in) {
                    issue_new(false, n0, new_k);
                    issue_new(true, n0, new_v);
                }
            }
            unsigned char* const at_v = new_v;
            uint32_t see[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                see[m] = 0u;
                if (!in) continue;
                if (a.mask) see[m] = live[m] ? a.mask[((uint64_t)i * N + node[m]) * a.mask_words + n0 / 32u] : 0u;
                else see[m] = !live[m] || node[m] < n0 ? 0u : node[m] - n0 >= 31u ? ~0u : (2u << (node[m] - n0)) - 1u;
                if (N - n0 < 32u) see[m] &= (1u << (N - n0)) - 1u;
            }
            wait_vm<0>();
            if constexpr (WR > 1) lds_sync();
            bool wild = false;
            if (in) {
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][0] = s[m][1] = zero;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t k = 0; k < kKS; ++k) {
                    const uint32_t r = 16u * h + lane_n, c = F8 ? 2u * (lg + 4u * (k / 2u)) + (k & 1u) : 4u * k + lg;
                    const bf16x8 kf = *reinterpret_cast<const bf16x8*>(new_k + r * kNewB + (c ^ swz_k<kNewB>(r)) * 16u);
#pragma unroll
                    for (int m = 0; m < MT; ++m) s[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[m][k], s[m][h], 0, 0, 0);
                }
#pragma unroll
            for (int m = 0; m < MT; ++m) hide(m, see[m]);
            const f32x4 none[2] = {zero, zero};
            weigh(none, false);
            // Infinities and NaNs are kept out of the product, where a weight of 0 would not keep them
            // from the rows that do not see them: they are replaced by 0 in LDS, and what they were noted
            // in the keys' place (+inf 1, -inf 2, a NaN both).
#pragma unroll 1
            for (int ii = 0; ii < kNew; ++ii) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(at_v + 1024 * ii + 16u * ln);
#pragma unroll
                for (int k = 0; k < 4; ++k) wild = wild || (v[k] & 0x7f80u) == 0x7f80u || (v[k] & 0x7f800000u) == 0x7f800000u;
            }
            }
            const bool any_wild = ballot(wild) != 0ull;
            if constexpr (WR > 1) lds_sync();   // (keys and values have been read by both)
            if (any_wild && wr == 0u) {
                wait_lds();
#pragma unroll 1
                for (int ii = 0; ii < kNew; ++ii) {
                    u32x4* const pv = reinterpret_cast<u32x4*>(at_v + 1024 * ii + 16u * ln);
                    u32x4 v = *pv, kind;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        auto kind_of = [](uint32_t e) -> uint32_t { return (e & 0x7f80u) != 0x7f80u ? 0u : e == 0x7f80u ? 1u : e == 0xff80u ? 2u : 3u; };
                        const uint32_t lo = kind_of(v[k] & 0xffffu), hi = kind_of(v[k] >> 16);
                        kind[k] = lo | hi << 16;
                        v[k] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                    }
                    *pv = v;
                    *reinterpret_cast<u32x4*>(new_k + 1024 * ii + 16u * ln) = kind;
                }
                wait_lds();
            }
            if constexpr (WR > 1) {
                lds_sync();
                if (!in) continue;
            }
            const uint32_t rv = 4u * lg + (lane_n >> 2), lv = lds_at(at_v) + rv * kNewB + 8u * (ln & 1u);
            auto tr_of = [&](uint32_t t) -> uint32_t { return ((2u * t + (ln >> 1 & 1u)) ^ swz_v<kNewB, false>(rv)) * 16u; };
#pragma unroll
            for (uint32_t t0 = 0; t0 < kDT; t0 += 4u) {
                uint32_t ad[4];
                u32x4 v[4];
#pragma unroll
                for (uint32_t t = 0; t < 4u; ++t) ad[t] = lv + tr_of(t0 + t);
                read_tr16<16 * kNewB>(ad, v);
#pragma unroll
                for (uint32_t t = 0; t < 4u; ++t)
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        acc[m][t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v[t]), pf[m], acc[m][t0 + t], 0, 0, 0);
            }
            if (any_wild) {   // 2^127 times 2 for each that is seen: infinite sums, of both signs for a NaN
                const uint32_t lk = lds_at(new_k) + (lv - lds_at(at_v));
                bf16x8 two[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    u32x4 w2;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t b2 = see[m] >> (16u * (k / 2) + 4u * lg + 2u * (k % 2));
                        w2[k] = (b2 & 1u ? 0x4000u : 0u) | (b2 & 2u ? 0x40000000u : 0u);
                    }
                    two[m] = __builtin_bit_cast(bf16x8, w2);
                }
#pragma unroll
                for (uint32_t t0 = 0; t0 < kDT; t0 += 4u) {
                    uint32_t ad[4];
                    u32x4 v[4];
#pragma unroll
                    for (uint32_t t = 0; t < 4u; ++t) ad[t] = lk + tr_of(t0 + t);
                    read_tr16<16 * kNewB>(ad, v);
#pragma unroll
                    for (uint32_t t = 0; t < 4u; ++t) {
                        u32x4 up, down;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            up[k] = (v[t][k] & 0x10001u) * 0x7f00u;
                            down[k] = (v[t][k] >> 1 & 0x10001u) * 0xff00u;
                        }
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            acc[m][t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, up), two[m], acc[m][t0 + t], 0, 0, 0);
                            acc[m][t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, down), two[m], acc[m][t0 + t], 0, 0, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }

        // ---- the waves' sums joined ----
        if constexpr (WR > 1) lds_sync();   // (the tiles' place)
        else wait_lds();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const float z = across(sum[m], [](float p, float q) { return p + q; });
            if (g == 0u) {
                stat[w][0][wr * kMine + 16u * m + n] = top[m];
                stat[w][1][wr * kMine + 16u * m + n] = z;
            }
#pragma unroll
            for (uint32_t t = 0; t < kDT; ++t)
                *reinterpret_cast<f32x4*>(mine + (wr * kMine + 16u * m + n) * DP * 4u + ((4u * t + g) ^ n) * 16u) = acc[m][t];
        }
        lds_sync();
        const bool complete = s0 == 0u && s1 == steps;
        // (who shares the pair: its first and last pieces, and whether it begins inside the first)
        if (s0 == 0u && rt == a.row_tile0 && tid_x() == 0u) a.spans[i * H + kvh] = piece | (x + units - 1u) / share << 15 | (x != piece * share ? 1u << 31 : 0u);
        // (a workgroup has at most two incomplete segments: one that begins with the piece, one that ends with it)
        float* part = a.part + ((uint64_t)b * 2u + (x == piece * share ? 0u : 1u)) * Part<DP, MT * WR>::kFloats;
        for (uint32_t it = tid_x(); it < kRows * (DP / 4u); it += NW * WR * kWave) {
            const uint32_t rr = it / (DP / 4u), c = it % (DP / 4u), pr = rt * kRows + rr;
            float M = stat[0][0][rr];
#pragma unroll
            for (int k = 1; k < NW; ++k) M = f_max(M, stat[k][0][rr]);
            f32x4 o = zero;
            float z = 0.0f;
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const float f = exp2_f(stat[k][0][rr] - M);
                z += stat[k][1][rr] * f;
                o += *reinterpret_cast<const f32x4*>(lds + (uint32_t)k * kRegion + rr * DP * 4u + (c ^ (rr & 15u)) * 16u) * f;
            }
            if (!complete) {
                *reinterpret_cast<f32x4*>(part + rr * DP + 4u * c) = o;
                if (c == 0u) {
                    part[kRows * DP + rr] = M;
                    part[kRows * DP + kRows + rr] = z;
                }
            } else if (pr < R && 4u * c < D) {
                const bool empty = z == 0.0f;
                const float f = 1.0f / z;
                const uint64_t rw = (uint64_t)i * N + pr / a.group;
                const uint32_t h = kvh * a.group + pr % a.group;
                *reinterpret_cast<u32x2*>(a.o + rw * a.o_stride + h * D + 4u * c) =
                    empty ? u32x2{0u, 0u} : u32x2{pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f)};
                if (c == 0u && a.lse) a.lse[rw * a.heads + h] = empty ? -__builtin_huge_valf() : (M + __builtin_amdgcn_logf(z)) * kLn2;
            }
        }
        lds_sync();
        x += u1 - u0;
    }
}

// Joins the partial sums of the pairs that several workgroups share: DP / 4 threads a row, four
// elements each, and SPLIT such groups that take the partial results in turn, eight under way
// in each (131000 tokens of 8 heads over 512 workgroups: 25 us with one at a time, of one group).
template <int DP, int MT, int SPLIT>
__global__ __launch_bounds__(256) void tree_join(TreeArgs a) {
    using P = Part<DP, MT>;
    constexpr uint32_t kPer = 1024u / DP / SPLIT, kBlocks = P::kRows / kPer, U = 8;
    __shared__ f32x4 os[SPLIT > 1 ? 256 : 1];
    __shared__ float ms[SPLIT > 1 ? 256 : 1], zs[SPLIT > 1 ? 256 : 1];
    const uint32_t span = a.spans[wg_x()];
    const uint32_t p0 = span & 0x7fffu, p1 = span >> 15 & 0xffffu;
    if (p0 == p1) return;
    const uint32_t i = wg_x() / a.c.kv_heads, kvh = wg_x() % a.c.kv_heads;
    const uint32_t rt = __builtin_amdgcn_workgroup_id_y() / kBlocks, row = tid_x() / (DP / 4u);
    const uint32_t rr = __builtin_amdgcn_workgroup_id_y() % kBlocks * kPer + row % kPer, split = row / kPer;
    const uint32_t c = tid_x() % (DP / 4u), pr = (rt + a.row_tile0) * P::kRows + rr;
    float M = kUnset, z = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t q = p0 + split; q <= p1; q += U * SPLIT) {
        float m[U], s[U], now = M;
        f32x4 v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t p = q + u * SPLIT, pu = p <= p1 ? p : q;
            const uint32_t b = (pu / 8u * a.row_tiles + rt) * 8u + pu % 8u;
            const float* part = a.part + ((uint64_t)b * 2u + (pu == p0 ? span >> 31 : 0u)) * P::kFloats;
            m[u] = p <= p1 ? part[P::kRows * DP + rr] : kUnset;
            s[u] = p <= p1 ? part[P::kRows * DP + P::kRows + rr] : 0.0f;
            v[u] = *reinterpret_cast<const f32x4*>(part + rr * DP + 4u * c);
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) now = f_max(now, m[u]);
        const float f = exp2_f(M - now);
        z *= f;
        o *= f;
        M = now;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (q + u * SPLIT <= p1) {   // (what is not there weighs nothing, whatever it repeats)
                const float g = exp2_f(m[u] - now);
                z += s[u] * g;
                o += v[u] * g;
            }
        }
    }
    if constexpr (SPLIT > 1) {
        os[tid_x()] = o;
        ms[tid_x()] = M;
        zs[tid_x()] = z;
        __syncthreads();
        if (split != 0u) return;
        float now = M;
#pragma unroll
        for (uint32_t k = 1; k < SPLIT; ++k) now = f_max(now, ms[tid_x() + k * (256u / SPLIT)]);
        float f = exp2_f(M - now);
        z *= f;
        o *= f;
#pragma unroll
        for (uint32_t k = 1; k < SPLIT; ++k) {
            const uint32_t at = tid_x() + k * (256u / SPLIT);
            f = exp2_f(ms[at] - now);
            z += zs[at] * f;
            o += os[at] * f;
        }
        M = now;
    }
    const uint32_t D = a.c.head_dim, h = kvh * a.group + pr % a.group;
    if (pr >= a.rows_per_seq * a.group || 4u * c >= D) return;
    const bool empty = z == 0.0f;
    const float f = 1.0f / z;
    const uint64_t rw = (uint64_t)i * a.rows_per_seq + pr / a.group;
    *reinterpret_cast<u32x2*>(a.o + rw * a.o_stride + h * D + 4u * c) =
        empty ? u32x2{0u, 0u} : u32x2{pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f)};
    if (c == 0u && a.lse) a.lse[rw * a.heads + h] = empty ? -__builtin_huge_valf() : (M + __builtin_amdgcn_logf(z)) * kLn2;
}

namespace {

constexpr uint32_t kTreeTiles = 32;   // row tiles of a launch

template <int DP, int MT, bool F8, int ST, int WR, int NW>
hipError_t launch(TreeArgs a, uint32_t cus, hipStream_t st) {
    constexpr uint32_t per_cu = NW * WR == 4 ? kTreePerCu<DP> : 1, per = 16u * MT * WR;
    const uint32_t rows = a.rows_per_seq * a.group, tiles = (rows + per - 1u) / per;
    for (uint32_t t0 = 0; t0 < tiles; t0 += kTreeTiles) {
        a.row_tile0 = t0;
        a.row_tiles = tiles - t0 < kTreeTiles ? tiles - t0 : kTreeTiles;
        const uint32_t most = per_cu * kTreeSlots / 2u, slots = cus * per_cu < most ? cus * per_cu : most;
        a.pieces = slots / a.row_tiles / 8u * 8u;
        if (a.pieces == 0u) a.pieces = 8u;
        hipLaunchKernelGGL((tree_attn<DP, MT, F8, ST, WR, NW>), dim3(a.pieces * a.row_tiles), dim3(NW * WR * kWave), 0, st, a);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const uint32_t pairs = a.c.n * a.c.kv_heads, blocks = a.row_tiles * (per * DP / 1024u);
        // (many partial results a pair: more threads for them)
        if (pairs * 8u <= a.pieces) hipLaunchKernelGGL((tree_join<DP, MT * WR, 4>), dim3(pairs, 4u * blocks), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((tree_join<DP, MT * WR, 1>), dim3(pairs, blocks), dim3(256), 0, st, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return hipSuccess;
}

// Rows of a wave: 16, or 32 where there are more (64 leave one wave a SIMD, whose products
// wait for its softmax: 256 rows a head, 32 sequences x 4096 tokens x 8 heads 294 us, of 32
// 276). Over bf16, waves share tiles where there are enough rows: what the L2 and LDS's
// write side bring is by a workgroup then and not by a wave.
// - Four a tile, 128 rows a workgroup, where the last 128 are more than half full (the same
//   sequences, us of one wave / four a tile: 72 rows 154 / 120, 128 rows 164 / 117, 256 rows
//   250 (of two) / 226; 512 rows, 8 x 8192 tokens 234 (of two) / 217). One short context is slower
//   (72 rows over 1000 tokens 14.3 / 16), and heads of 64 up to 128 rows (16 x 6000 tokens
//   58 / 63).
// - Else two, 64 rows: above 128 rows (136 rows 214 of four / 192, 320 rows over 16 x 4096 tokens
//   182 of four / 160), and up to there where the pairs are a quarter of the workgroups or more,
//   whose lengths then matter little (us of one / two a tile, 40 or 64 rows, 8 kv heads: 64
//   sequences over up to 1300 tokens 73 / 56, 32 over up to 4096 81 / 69, all of 4096 105 / 112;
//   16 over up to 6000 67 / 60; fewer: 8 over up to 8000 40 / 43, 1 over 100000 87 / 90).
// - Heads of 256: four a tile of 16 rows each, 64 rows a workgroup, above 32 rows, so that two waves
//   fit a SIMD (us of one, of 32 rows / four, 8 kv heads: 44 rows, 12 sequences over 800 to 3187
//   tokens 72 / 47, 256 rows, 2 over up to 4000 49 / 37, 128 rows, 8 over up to 2000 50 / 48; 24 rows 57 / 59).
// - Not for 8 bits, whose tiles are half as large (256 rows 261 / 276 of two).
template <int DP, bool F8>
hipError_t launch_rows(const TreeArgs& a, uint32_t cus, hipStream_t st) {
    constexpr int ST = F8 || DP == 64 ? 2 : 1;
    const uint32_t rows = a.rows_per_seq * a.group, pairs = a.c.n * a.c.kv_heads;
    if (rows <= 16u) return launch<DP, 1, F8, ST, 1, 4>(a, cus, st);
    if constexpr (DP != 256 && !F8) {
        if (rows > (DP == 64 ? 128u : 64u) && (rows - 1u) % 128u >= 64u) return launch<DP, 2, F8, 2, 4, 2>(a, cus, st);
        if (rows > 128u || (rows > 32u && pairs * 2u >= cus)) return launch<DP, 2, F8, 2, 2, 2>(a, cus, st);
    }
    if constexpr (DP == 256 && !F8) {
        if (rows > 32u) return launch<DP, 1, F8, 2, 4, 2>(a, cus, st);
    }
    return launch<DP, 2, F8, ST, 1, 4>(a, cus, st);
}

}  // namespace

// Floats of a context's partial results: two of 64 rows for each of two workgroups a CU (of 128 rows
// or heads of 256: one workgroup a CU).
uint64_t tree_part_floats() { return 4ull * kTreeSlots * Part<128, 2>::kFloats; }
static_assert(Part<256, 4>::kFloats <= 4u * Part<128, 2>::kFloats && Part<256, 2>::kFloats <= 2u * Part<128, 2>::kFloats && Part<128, 8>::kFloats <= 4u * Part<128, 2>::kFloats, "the partial results' room");

hipError_t launch_tree_attn(const TreeArgs& args, uint32_t cus, hipStream_t st) {
    TreeArgs a = args;
    a.new_steps = (a.rows_per_seq + kStepKeys - 1u) / kStepKeys;
    const uint32_t d = a.c.head_dim;
    if (a.c.f8) return d <= 64 ? launch_rows<64, true>(a, cus, st) : d <= 128 ? launch_rows<128, true>(a, cus, st) : launch_rows<256, true>(a, cus, st);
    return d <= 64 ? launch_rows<64, false>(a, cus, st) : d <= 128 ? launch_rows<128, false>(a, cus, st) : launch_rows<256, false>(a, cus, st);
}

}  // namespace lcs
