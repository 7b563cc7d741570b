// The bookkeeping of a paged cache of keys and values, for MI355X (gfx950): pages
// given out, shared, copied on write and given back, rows appended and moved.
//
// Reference: the ref-counted copy-on-write cache (src/locus/kv/block_allocator.hpp:25-55,
// paged_cache.hpp:24-120) and the rollback after a speculative step
// (engine.cpp:399-401), both on the host.
//
// A pool's only state is the slots' table of pages and the pages' reference counts, so
// that a call's outcome does not depend on the order of earlier frees: the free pages
// are those of count 0, and the lowest are given out first. Requests are decided
// against the state ahead of the call; counts move by integer atomics, whose order
// does not change the sum.
//
// Memory bounds the calls that move rows (lcs_kv_append, lcs_kv_compact, the copies of
// lcs_kv_grow): a row is read once and written once, 16 bytes a lane. Launches and
// dependent loads (slot, table, count) bound the small ones.
//
// (This file is compiled with NaNs honoured: a NaN in a row has to stay one.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"

namespace lcs {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kKvThreads = 256;
constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126: a scale below the normal numbers would lose its bits

__device__ __forceinline__ void refuse(const KvArgs& a, int32_t* result) {
    *result = -1;
    atomicOr(a.status, kStatusPages);
}
__device__ __forceinline__ bool page_ok(const KvArgs& a, int32_t page) { return (uint32_t)page < a.pages; }

// Whether one of ids[0 .. n) is `id` (a whole workgroup asks).
__device__ __forceinline__ bool named(const int32_t* ids, uint32_t n, int32_t id) {
    bool hit = false;
    for (uint32_t j = tid_x(); j < n; j += blockDim.x) hit = hit || ids[j] == id;
    return __syncthreads_or(hit) != 0;
}

// An element's place: bytes from the base of k or v.
__device__ __forceinline__ uint64_t place(const KvArgs& a, uint32_t layer, uint32_t page, uint32_t head, uint32_t row) {
    return (layer * a.layer_stride + page * a.page_stride + head * a.head_stride + row * a.token_stride) * (a.f8 ? 1u : 2u);
}
__device__ __forceinline__ uint64_t scale_place(const KvArgs& a, uint32_t layer, uint32_t page, uint32_t head, uint32_t row) {
    return ((((uint64_t)layer * a.pages + page) * a.kv_heads + head) << a.page_shift) + row;
}

}  // namespace

// ---- lcs_kv_free: a workgroup per request ----
__global__ __launch_bounds__(kKvThreads) void kv_free(KvArgs a) {
    const uint32_t i = wg_x();
    const int32_t slot = a.seq[i];
    if (slot == -1) {
        if (tid_x() == 0) a.result[i] = 0;
        return;
    }
    const bool again = named(a.seq, i, slot);
    if ((uint32_t)slot >= a.seqs || again) {
        if (tid_x() == 0) refuse(a, &a.result[i]);
        return;
    }
    const int32_t keep = a.end ? a.end[i] : 0;
    const uint32_t first = keep > 0 ? (uint32_t)(((int64_t)keep + a.page_tokens - 1) >> a.page_shift) : 0u;
    int32_t* row = a.table + (uint64_t)slot * a.max_pages;
    for (uint32_t p = first + tid_x(); p < a.max_pages; p += kKvThreads) {
        const int32_t page = row[p];
        if (page_ok(a, page) && atomicSub(&a.refs[page], 1) <= 0) {   // (a table that holds what its counts do not)
            atomicAdd(&a.refs[page], 1);
            atomicOr(a.status, kStatusPages);
        }
        if (page != -1) row[p] = -1;
    }
    if (tid_x() == 0) a.result[i] = 0;
}

// ---- lcs_kv_fork: a workgroup per request. No slot that is read here is written by
// another request (src is nobody's dst), so the requests need no order. ----
__global__ __launch_bounds__(kKvThreads) void kv_fork(KvArgs a) {
    const uint32_t i = wg_x();
    const int32_t src = a.seq[i], dst = a.dst[i];
    if (src == -1 || dst == -1) {
        if (tid_x() == 0) a.result[i] = 0;
        return;
    }
    const int32_t tokens = a.end[i];
    const bool again = named(a.dst, i, dst), other = named(a.dst, a.n, src);
    bool ok = !again && !other && (uint32_t)src < a.seqs && (uint32_t)dst < a.seqs && tokens >= 0 &&
              (uint64_t)(uint32_t)tokens <= (uint64_t)a.max_pages << a.page_shift;
    const int32_t* from = a.table + (uint64_t)(ok ? src : 0) * a.max_pages;
    int32_t* to = a.table + (uint64_t)(ok ? dst : 0) * a.max_pages;
    const uint32_t np = ok ? (uint32_t)(((uint64_t)(uint32_t)tokens + a.page_tokens - 1u) >> a.page_shift) : 0u;
    bool bad = !ok;
    if (ok) {   // (uniform)
        for (uint32_t p = tid_x(); p < a.max_pages; p += kKvThreads)
            bad = bad || page_ok(a, to[p]) || (p < np && !page_ok(a, from[p]));
    }
    if (__syncthreads_or(bad)) {
        if (tid_x() == 0) refuse(a, &a.result[i]);
        return;
    }
    for (uint32_t p = tid_x(); p < np; p += kKvThreads) {
        const int32_t page = from[p];
        to[p] = page;
        atomicAdd(&a.refs[page], 1);
    }
    if (tid_x() == 0) a.result[i] = 0;
}

// ---- lcs_kv_grow: one workgroup decides and gives out pages ----
// 1024 / n lanes (up to a wave) look at a request's pages. The counts do not move until
// every request has read them. Its time is its chain of dependent loads (table, count,
// table), so up to kGrowLocal pages are passed on by way of LDS.
constexpr int kGrowThreads = 1024;
constexpr uint32_t kGrowPer = 16;   // pages a thread looks at for free ones in a round
constexpr uint32_t kGrowLocal = 2048;
__global__ __launch_bounds__(kGrowThreads) void kv_grow(KvArgs a) {
    constexpr uint32_t NW = kGrowThreads / kWave;
    __shared__ __attribute__((aligned(16))) int32_t slots[kKvMaxReq];
    __shared__ uint32_t need[kKvMaxReq], off[kKvMaxReq], first[kKvMaxReq], past[kKvMaxReq];
    __shared__ int32_t fresh_s[kGrowLocal], from_s[kGrowLocal];
    __shared__ uint32_t red[NW], used, copies;
    const uint32_t tid = tid_x(), n = a.n;
    int32_t slot = -1, s = 0, e = 0;
    if (tid < n) {
        slot = a.seq[tid];
        s = a.start[tid];
        e = a.end[tid];
    }
    slots[tid] = tid < n ? slot : -1;
    if (tid == 0) used = copies = 0u;
    __syncthreads();
    bool ok = false;
    if (tid < n) {
        ok = slot == -1 || ((uint32_t)slot < a.seqs && s >= 0 && e >= s && (uint64_t)(uint32_t)e <= (uint64_t)a.max_pages << a.page_shift);
        if (slot != -1) {
            bool again = false;
            for (uint32_t j = 0; j < tid; j += 4u) {
                const int4 q = *reinterpret_cast<const int4*>(slots + j);
                again = again || q.x == slot || (j + 1u < tid && q.y == slot) || (j + 2u < tid && q.z == slot) || (j + 3u < tid && q.w == slot);
            }
            ok = ok && !again;
        }
        const bool none = !ok || slot == -1 || s == e;
        first[tid] = none ? 0u : (uint32_t)s >> a.page_shift;
        past[tid] = none ? 0u : (uint32_t)(((uint64_t)(uint32_t)e + a.page_tokens - 1u) >> a.page_shift);
    }
    __syncthreads();
    uint32_t L = kWave;   // lanes a request
    while (L > 1u && L * n > (uint32_t)kGrowThreads) L >>= 1;
    const uint32_t req = tid / L, sub = tid % L;
    const uint64_t mine = (L == 64u ? ~0ull : (1ull << L) - 1ull) << ((uint32_t)lane_id() / L * L);
    const uint64_t below = (1ull << lane_id()) - 1ull;
    const bool act = req < n;
    const uint32_t p0 = act ? first[req] : 0u, p1 = act ? past[req] : 0u;
    int32_t* row = a.table + (uint64_t)(act && p1 > p0 ? slots[req] : 0) * a.max_pages;
    // what a page of the request needs: 0 nothing, 1 a page, 2 a copy
    auto wants = [&](uint32_t p, int32_t& page) -> uint32_t {
        page = p < p1 ? row[p] : 0;
        return p >= p1 ? 0u : !page_ok(a, page) ? 1u : a.refs[page] > 1 ? 2u : 0u;
    };
    uint32_t cnt = 0, w0 = 0;
    int32_t page0 = 0;   // (the lane's first page, looked up once)
    for (uint32_t b = p0; __any(b < p1); b += L) {
        int32_t page;
        const uint32_t w = wants(b + sub, page);
        if (b == p0) {
            w0 = w;
            page0 = page;
        }
        cnt += (uint32_t)__builtin_popcountll(ballot(w != 0u) & mine);
    }
    if (act && sub == 0u) need[req] = cnt;
    __syncthreads();
    uint32_t excl;
    const uint32_t total = block_exclusive_scan<kGrowThreads>(tid < n ? need[tid] : 0u, excl, red);
    if (tid < n) off[tid] = excl;
    // the lowest free pages, as many as are asked for
    const uint32_t want = min(total, a.cap);
    uint32_t found = 0;
    for (uint32_t base = 0; base < a.pages && found < want; base += kGrowThreads * kGrowPer) {
        const uint32_t g0 = base + tid * kGrowPer;
        uint32_t bits = 0;
#pragma unroll
        for (uint32_t g = 0; g < kGrowPer; g += 4) {
            if (g0 + g + 4u <= a.pages) {
                const int4 r = *reinterpret_cast<const int4*>(a.refs + g0 + g);
                bits |= (uint32_t)(r.x == 0) << g | (uint32_t)(r.y == 0) << (g + 1) | (uint32_t)(r.z == 0) << (g + 2) |
                        (uint32_t)(r.w == 0) << (g + 3);
            } else {
                for (uint32_t k = 0; k < 4u; ++k)
                    if (g0 + g + k < a.pages) bits |= (uint32_t)(a.refs[g0 + g + k] == 0) << (g + k);
            }
        }
        uint32_t at;
        const uint32_t here = block_exclusive_scan<kGrowThreads>((uint32_t)__builtin_popcount(bits), at, red);
        at += found;
        while (bits != 0u && at < want) {
            const int32_t page = (int32_t)(g0 + (uint32_t)__builtin_ctz(bits));
            if (at < kGrowLocal) fresh_s[at] = page;
            else a.fresh[at] = page;
            ++at;
            bits &= bits - 1u;
        }
        found += here;
    }
    found = min(found, want);
    __syncthreads();   // (the list is complete)
    auto fresh_of = [&](uint32_t k) -> int32_t { return k < kGrowLocal ? fresh_s[k] : a.fresh[k]; };
    if (tid < n) {
        const bool served = ok && off[tid] + need[tid] <= found;
        if (served) a.result[tid] = 0;
        else refuse(a, &a.result[tid]);
        if (served && need[tid] != 0u) atomicMax(&used, off[tid] + need[tid]);
        if (!served) past[tid] = first[tid];
    }
    __syncthreads();
    if (act && past[req] > first[req]) {   // (a request's lanes together; the loop below waits for none of another's)
        uint32_t at = off[req];
        for (uint32_t b = p0; b < p1; b += L) {
            int32_t page = page0;
            const uint32_t w = b == p0 ? w0 : wants(b + sub, page);
            const uint64_t m = ballot(w != 0u) & mine;
            const uint32_t k = at + (uint32_t)__builtin_popcountll(m & below);
            if (w != 0u && k < found) {
                const int32_t src = w == 2u ? page : -1;
                row[b + sub] = fresh_of(k);
                if (k < kGrowLocal) from_s[k] = src;
                else a.from[k] = src;
            }
            at += (uint32_t)__builtin_popcountll(m);
        }
    }
    __syncthreads();
    // the counts; and what is to be copied, in any order, moved to the front of the lists
    const uint32_t n_used = used;
    for (uint32_t b = 0; b < n_used; b += kGrowThreads) {
        const uint32_t k = b + tid;
        const int32_t src = k >= n_used ? -1 : k < kGrowLocal ? from_s[k] : a.from[k];
        const int32_t page = k < n_used ? fresh_of(k) : 0;
        if (k < n_used) a.refs[page] = 1;
        if (src >= 0) atomicSub(&a.refs[src], 1);
        __syncthreads();   // (the round's entries have been read: no more than b of them precede)
        if (src >= 0) {
            const uint32_t c = atomicAdd(&copies, 1u);
            a.fresh[c] = page;
            a.from[c] = src;
        }
    }
    __syncthreads();
    if (tid == 0) *a.n_fresh = copies;
}

// The copies that kv_grow has planned, by units of 256 chunks of 16 bytes: a part of the rows of
// one head of k or v of one layer, cp lanes a row. Many short workgroups with stores past
// the caches (nobody reads the copies soon) come nearest to the memory's rate: 64 pages of
// 32 tokens x 32 layers x 8 heads, us for the three calls of a fork, one unit a turn in
// 16384 workgroups 69 and 8192 74, with plain stores 88 and 85; two units a turn in 8192
// 74 and 88, eight in 1024 - / 112.
__global__ __launch_bounds__(kKvThreads) void kv_copy(KvArgs a) {
    const uint32_t copies = *a.n_fresh;
    const uint32_t per = a.layers * 2u * a.kv_heads, passes = 1u << a.pass_shift;
    const uint64_t units = (uint64_t)copies * per << a.pass_shift;
    const uint32_t chunk = tid_x() & (a.cp - 1u), row0 = tid_x() / a.cp, step = kKvThreads / a.cp, es = a.f8 ? 1u : 2u;
    if (chunk >= a.chunks || row0 >= a.page_tokens) return;
    for (uint64_t unit = wg_x(); unit < units; unit += gridDim.x) {
        const uint64_t it = unit >> a.pass_shift;
        const uint32_t k = (uint32_t)(it / per), r = (uint32_t)(it % per), row = ((uint32_t)unit & (passes - 1u)) * step + row0;
        const uint32_t src = (uint32_t)a.from[k], dst = (uint32_t)a.fresh[k];
        const uint32_t head = r % a.kv_heads, kv = r / a.kv_heads & 1u, layer = r / (2u * a.kv_heads);
        unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k) + place(a, layer, 0, head, row) + 16u * chunk;
        const u32x4 x = *reinterpret_cast<const u32x4*>(base + src * a.page_stride * es);
        if (a.f8 && chunk == 0u) {
            float* sc = (kv ? a.v_scale : a.k_scale) + scale_place(a, layer, 0, head, row);
            sc[(uint64_t)dst * a.kv_heads << a.page_shift] = sc[(uint64_t)src * a.kv_heads << a.page_shift];
        }
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(base + dst * a.page_stride * es));
    }
}

// ---- lcs_kv_compact ----
// Whether a request can be served, a workgroup each. Its time is the chain of place, table and
// count that a thread walks every kCheckThreads rows (16 contexts cut to 4096 rows:
// 10 us more for the call by 256 threads than by 1024; 610 rows alike).
constexpr int kCheckThreads = 1024;
__global__ __launch_bounds__(kCheckThreads) void kv_compact_check(KvArgs a) {
    const uint32_t i = wg_x();
    const int32_t slot = a.seq[i];
    if (slot == -1) {
        if (tid_x() == 0) a.result[i] = 0;
        return;
    }
    const bool again = named(a.seq, i, slot);
    bool bad = again || (uint32_t)slot >= a.seqs;
    if (!bad) {   // (uniform)
        const uint32_t n = min((uint32_t)max(a.count[i], 0), a.max_keep);
        const int32_t* keep = a.index + (uint64_t)i * a.max_keep;
        const int32_t* row = a.table + (uint64_t)slot * a.max_pages;
        for (uint32_t j = tid_x(); j < n; j += kCheckThreads) {
            const int32_t pos = keep[j], last = j ? keep[j - 1u] : -1;
            const uint32_t pp = (uint32_t)pos >> a.page_shift, pj = j >> a.page_shift;
            if (pos <= last || pos < (int32_t)j || pp >= a.max_pages) {
                bad = true;
            } else if ((uint32_t)pos != j) {
                const int32_t to = row[pj];
                bad = bad || !page_ok(a, row[pp]) || !page_ok(a, to) || a.refs[page_ok(a, to) ? to : 0] > 1;
            } else {
                bad = bad || !page_ok(a, row[pj]);
            }
        }
    }
    const bool no = __syncthreads_or(bad) != 0;
    if (tid_x() == 0) {
        if (no) refuse(a, &a.result[i]);
        else a.result[i] = 0;
    }
}

// A workgroup moves one head's rows of k or v of one layer of one request (or 16-byte chunks
// from part * cp of them), in order, by rounds of U rows a lane group. Rows never move up:
// a round writes below the next round's places, which lie at or below its sources, so
// that only a round's own rows have to be read by all lanes before the first is
// written. The next round's rows are under way meanwhile, the places of the one after it too
// (16 contexts of 4000 to 8192 tokens, half kept, 4 layers: 547 us without, 367 so, 356 with
// stores past the caches). The rounds of a workgroup follow each other, so a long list is
// walked by 1024 threads; a short one by 256, which start sooner (us a call in a graph of
// 256 / 1024 threads, half of the tokens kept, bf16, 8 heads of 128: the same 352 / 334; 10
// contexts of 13000, one layer, 190 / 133; one of 3000, 6 layers, 32 / 21; 32 of 1200, 16
// layers, 523 / 517, of 700 307 / 306, of 520 217 / 236, of 260 102 / 132; 4 of 900, 8 layers,
// 27 / 26, of 512 16.3 / 16.8, of 260 11 / 13; 5 of 200, a third kept, 13 layers, 12 / 20). The
// rule goes by the list's room, since the counts are on the device; lists of 257 to
// 400 rows would be up to a tenth faster by 256.
// 8 rows of a lane are no faster by 256 threads (346 of the first) and spill by 1024 (550).
template <int NT>
__global__ __launch_bounds__(NT) void kv_compact(KvArgs a) {
    constexpr uint32_t U = 4;
    uint32_t b = wg_x();
    const uint32_t part = b % a.parts;
    b /= a.parts;
    const uint32_t head = b % a.kv_heads, kv = b / a.kv_heads;
    const uint32_t layer = __builtin_amdgcn_workgroup_id_y(), i = __builtin_amdgcn_workgroup_id_z();
    const int32_t slot = a.seq[i];
    if (slot == -1 || a.result[i] != 0) return;
    const uint32_t n = min((uint32_t)max(a.count[i], 0), a.max_keep);
    const int32_t* keep = a.index + (uint64_t)i * a.max_keep;
    const int32_t* row = a.table + (uint64_t)slot * a.max_pages;
    const uint32_t chunk = part * a.cp + (tid_x() & (a.cp - 1u)), r0 = tid_x() / a.cp, step = NT / a.cp;
    const uint32_t es = a.f8 ? 1u : 2u, in = a.page_tokens - 1u;
    unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k) + (layer * a.layer_stride + head * a.head_stride) * es + 16u * chunk;
    float* sc = kv ? a.v_scale : a.k_scale;
    const bool data = chunk < a.chunks, scale = a.f8 && chunk == 0u;
    struct Places {
        uint32_t pos[U];
        int32_t pf[U], pt[U];   // the pages that it comes from and goes to; pt -1: it stays
    };
    struct Rows {
        u32x4 x[U];
        float s[U];
    };
    // (a row that is not moved is read where it is: no load depends on a branch)
    auto places = [&](uint32_t j0) -> Places {
        Places p;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t j = j0 + u * step + r0;
            p.pos[u] = j < n ? (uint32_t)keep[j] : 0u;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t j = j0 + u * step + r0;
            p.pf[u] = row[p.pos[u] >> a.page_shift];
            p.pt[u] = j < n && p.pos[u] != j ? row[j >> a.page_shift] : -1;
        }
        return p;
    };
    auto read = [&](const Places& p) -> Rows {
        Rows r;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            r.x[u] = u32x4{0, 0, 0, 0};
            r.s[u] = 0.0f;
            if (p.pt[u] >= 0) {
                if (data) r.x[u] = *reinterpret_cast<const u32x4*>(base + ((uint32_t)p.pf[u] * a.page_stride + (p.pos[u] & in) * a.token_stride) * es);
                if (scale) r.s[u] = sc[scale_place(a, layer, (uint32_t)p.pf[u], head, p.pos[u] & in)];
            }
        }
        return r;
    };
    const uint32_t round = U * step;
    if (n == 0u) return;
    Places now = places(0u), next = places(round);
    Rows x = read(now);
    for (uint32_t j0 = 0; j0 < n; j0 += round) {
        const Rows y = read(next);
        const Places then = places(j0 + 2u * round);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) asm volatile("" : "+v"(x.x[u]), "+v"(x.s[u]));   // (the round's rows have arrived)
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (now.pt[u] >= 0) {
                const uint32_t j = j0 + u * step + r0;
                if (data) __builtin_nontemporal_store(x.x[u], reinterpret_cast<u32x4*>(base + ((uint32_t)now.pt[u] * a.page_stride + (j & in) * a.token_stride) * es));
                if (scale) sc[scale_place(a, layer, (uint32_t)now.pt[u], head, j & in)] = x.s[u];
            }
        }
        now = next;
        next = then;
        x = y;
    }
}

// ---- lcs_kv_append ----
// A workgroup writes kAppendTokens tokens of one layer and sequence: cp lanes a row of 8
// elements each, both k's and v's heads. Where each token comes from and goes to is looked
// up once, ahead of the rows. A lane keeps its head from token to token, and quotients
// take three operations each, since arithmetic bounds the 8-bit form (64 x 4.5 tokens of
// 32 layers x 8 heads: 59 us with divisions for both).
// (Few tokens a workgroup, the layers of one sequence side by side: CUs then take like shares
// where the sequences' counts differ. 64 sequences of 0 to 16 kept tokens, 32 layers, with
// the verdict and the pages: 88.9 us; 16 tokens a workgroup, one layer's sequences side
// by side 90.7. All 16 kept: 39 us by either, 5.2 TB/s.)
constexpr uint32_t kAppendTokens = 4;
constexpr uint32_t kAppendBlocks = 2048;   // workgroups of a sequence and layer along x: 2^31 threads with 4096 layers

// x / scale to nearest: RN(1 / scale), a product, and its remainder's share (exact by an fma),
// which makes the quotient the correctly rounded one. An infinite scale gives 0, and NaN
// for an infinite x.
struct Quotient {
    float scale, inv;
    __device__ __forceinline__ explicit Quotient(float s) : scale(s > 3.4e38f ? 0.0f : s), inv(fdiv(1.0f, s)) {}
    __device__ __forceinline__ float of(float x) const {
        const float q = fmul(x, inv);
        return fmaf(fmaf(-q, scale, x), inv, q);
    }
};

// The low half, a bf16: a number or an infinity cut to +-448 (0x43e0), a NaN as it is.
__device__ __forceinline__ uint32_t cut448(uint32_t w) {
    const uint32_t m = w & 0x7fffu;
    return (w & 0x8000u) | (m > 0x7f80u ? m : min(m, 0x43e0u));
}

// The largest of cp neighbouring lanes' values (cp a power of two up to 32): pairs, quads, and
// their mirror images, in which the quads and eights are already alike.
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t cp) {
    auto with = [](uint32_t x, int y) { return max(x, (uint32_t)y); };
    if (cp > 1u) v = with(v, __builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));    // lane ^ 1
    if (cp > 2u) v = with(v, __builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));    // lane ^ 2
    if (cp > 4u) v = with(v, __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));   // 7 - lane of eight
    if (cp > 8u) v = with(v, __builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));   // 15 - lane of sixteen
    if (cp > 16u) v = with(v, __shfl_xor((int)v, 16));
    return v;
}

template <bool F8>
__global__ __launch_bounds__(kKvThreads) void kv_append(KvAppendArgs p) {
    constexpr uint32_t U = 4;
    __shared__ int32_t page_s[kAppendTokens], src_s[kAppendTokens];
    const KvArgs& a = p.a;
    const uint32_t l = wg_x() % p.n_layers, i = __builtin_amdgcn_workgroup_id_z();
    const uint32_t j0 = (wg_x() / p.n_layers + __builtin_amdgcn_workgroup_id_y() * kAppendBlocks) * kAppendTokens;
    const int32_t slot = a.seq ? a.seq[i] : (int32_t)i;
    const uint32_t n = a.count ? min((uint32_t)max(a.count[i], 0), p.rows_per_seq) : p.rows_per_seq;
    const int32_t pos0 = a.start[i];
    if (slot == -1 || j0 >= n) return;
    const uint32_t tokens = min(n - j0, kAppendTokens);
    if (tid_x() < tokens) {
        const uint32_t j = j0 + tid_x();
        const int64_t pos = (int64_t)pos0 + j;
        const int32_t src = a.index ? a.index[(uint64_t)i * p.rows_per_seq + j] : (int32_t)j;
        const bool in = (uint32_t)slot < a.seqs && pos >= 0 && (uint64_t)pos < (uint64_t)a.max_pages << a.page_shift && (uint32_t)src < p.rows_per_seq;
        int32_t page = in ? a.table[(uint64_t)slot * a.max_pages + ((uint64_t)pos >> a.page_shift)] : -1;
        if (!page_ok(a, page) || a.refs[page_ok(a, page) ? page : 0] > 1) {
            page = -1;
            atomicOr(a.status, kStatusPages);
        }
        page_s[tid_x()] = page;
        src_s[tid_x()] = src;
    }
    __syncthreads();
    // a pass covers `per` whole tokens, or a part of one's rows
    const uint32_t chunk = tid_x() & (a.cp - 1u), g = tid_x() / a.cp, step = kKvThreads / a.cp, rows = 2u * a.kv_heads;
    const uint32_t per = step > rows ? step / rows : 1u, t0 = step > rows ? g / rows : 0u;
    const bool data = chunk < a.head_dim / 8u;
    if (t0 >= per) return;
    const uint32_t layer = a.layer + l;
    // A row that holds a NaN has scale 1, and what of it is not one is cut to +-448, which the conversion
    // would not do. A lane that has met such a row writes its rows again, cut: a branch at each row costs
    // more than it looks (64 x 16 tokens of 32 layers x 8 heads 48.5 us with it, 46.0 so).
    uint32_t worst = 0;   // the largest of the rows' |x|, by its bits
    auto write = [&](auto cut) {
        constexpr bool CUT = decltype(cut)::value;
        for (uint32_t r = g - t0 * rows; r < rows; r += step) {
            const bool kv = r >= a.kv_heads;
            const uint32_t head = kv ? r - a.kv_heads : r;
            const uint16_t* from = static_cast<const uint16_t*>(kv ? p.v : p.k) + (uint64_t)l * p.new_layer_stride +
                                   (uint64_t)i * p.rows_per_seq * (kv ? p.v_stride : p.k_stride) + head * a.head_dim + 8u * chunk;
            const uint64_t stride = kv ? p.v_stride : p.k_stride;
            unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k) + place(a, layer, 0, head, 0) + (F8 ? 8u : 16u) * chunk;
            float* sc = F8 ? (kv ? a.v_scale : a.k_scale) + scale_place(a, layer, 0, head, 0) : nullptr;
            for (uint32_t t = t0; t < tokens; t += U * per) {
                u32x4 x[U];
                int32_t page[U];
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    const uint32_t tu = t + u * per;
                    page[u] = tu < tokens ? page_s[tu] : -1;
                    x[u] = u32x4{0, 0, 0, 0};
                    if (page[u] >= 0 && data) x[u] = *reinterpret_cast<const u32x4*>(from + (uint32_t)src_s[tu] * stride);
                }
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    if (t + u * per >= tokens) break;   // (the lanes of a row together)
                    const bool ok = page[u] >= 0;
                    const uint32_t tok = ((uint32_t)pos0 + j0 + t + u * per) & (a.page_tokens - 1u);
                    const uint64_t at = ((uint32_t)page[u] * a.page_stride + tok * a.token_stride) * (F8 ? 1u : 2u);
                    if constexpr (F8) {
                        uint32_t top = 0;   // the largest |x|, by its bits (a NaN's lie above infinity's)
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = max(top, max(x[u][k] & 0x7fffu, x[u][k] >> 16 & 0x7fffu));
                        top = row_max(top, a.cp);
                        if constexpr (CUT) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) x[u][k] = top > 0x7f80u ? cut448(x[u][k]) | cut448(x[u][k] >> 16) << 16 : x[u][k];
                        } else {
                            worst = max(worst, top);
                        }
                        const float f = __uint_as_float(top << 16);
                        const float scale = f > 0.0f ? fmaxf(fdiv(f, kE4m3Max), kLeastScale) : 1.0f;   // (a NaN is not above 0)
                        const Quotient by(scale);   // (448 at most, and a rounding)
                        uint32_t q[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float e[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t w = x[u][2 * h + k / 2];
                                e[k] = by.of(__uint_as_float(k % 2 ? w & 0xffff0000u : w << 16));
                            }
                            const int w = __builtin_amdgcn_cvt_pk_fp8_f32(e[0], e[1], 0, false);
                            q[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e[2], e[3], w, true);
                        }
                        if (ok && data) __builtin_nontemporal_store(u32x2{q[0], q[1]}, reinterpret_cast<u32x2*>(base + at));
                        if (ok && chunk == 0u) sc[((uint64_t)(uint32_t)page[u] * a.kv_heads << a.page_shift) + tok] = scale;
                    } else {
                        if (ok && data) __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4*>(base + at));
                    }
                }
            }
        }
    };
    write(std::false_type{});
    if constexpr (F8) {
        if (ballot(worst > 0x7f80u) != 0ull) write(std::true_type{});
    }
}

static uint32_t pow2_from(uint32_t n) {
    uint32_t p = 1;
    while (p < n) p <<= 1;
    return p;
}

hipError_t launch_kv_free(const KvArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(kv_free, dim3(a.n), dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_fork(const KvArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(kv_fork, dim3(a.n), dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_grow(const KvArgs& args, hipStream_t st) {
    KvArgs a = args;
    a.chunks = a.head_dim * (a.f8 ? 1u : 2u) / 16u;
    a.cp = pow2_from(a.chunks);
    hipLaunchKernelGGL(kv_grow, dim3(1), dim3(kGrowThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.pass_shift = 0;
    while (((uint32_t)kKvThreads << a.pass_shift) < a.page_tokens * a.cp) ++a.pass_shift;
    // (as many workgroups as a page of every request takes)
    const uint64_t units = (uint64_t)a.n * a.layers * 2u * a.kv_heads << a.pass_shift;
    hipLaunchKernelGGL(kv_copy, dim3(units < 16384u ? (uint32_t)units : 16384u), dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const KvArgs& args, hipStream_t st) {
    KvArgs a = args;
    a.chunks = a.head_dim * (a.f8 ? 1u : 2u) / 16u;
    a.cp = pow2_from(a.chunks);
    hipLaunchKernelGGL(kv_compact_check, dim3(a.n), dim3(kCheckThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // (few rows' heads: their chunks apart, in pieces of 128 bytes at least, so that the CUs have more in flight)
    const bool wide = a.max_keep > kKvThreads;
    const uint32_t heads = a.n * a.layers * 2u * a.kv_heads, enough = wide ? 512u : 2048u;
    a.parts = 1;
    while (heads * a.parts < enough && a.cp > 8u) {
        a.parts *= 2u;
        a.cp /= 2u;
    }
    // (a dimension's threads are counted in 32 bits, and past them go missing without an error:
    // layers and requests have dimensions of their own, and x has 2^21 at most)
    const dim3 grid(2u * a.kv_heads * a.parts, a.layers, a.n);
    if (wide) hipLaunchKernelGGL(kv_compact<1024>, grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(kv_compact<kKvThreads>, grid, dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppendArgs& args, hipStream_t st) {
    KvAppendArgs p = args;
    p.a.cp = pow2_from(p.a.head_dim / 8u);
    // (sequences and what is left of a long one's tokens in dimensions of their own, as kv_compact's)
    const uint32_t blocks = (p.rows_per_seq + kAppendTokens - 1u) / kAppendTokens;
    const dim3 grid(p.n_layers * (blocks < kAppendBlocks ? blocks : kAppendBlocks), (blocks + kAppendBlocks - 1u) / kAppendBlocks, p.a.n);
    if (p.a.f8) hipLaunchKernelGGL(kv_append<true>, grid, dim3(kKvThreads), 0, st, p);
    else hipLaunchKernelGGL(kv_append<false>, grid, dim3(kKvThreads), 0, st, p);
    return hipGetLastError();
}

}  // namespace lcs
