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
// every request has read them.
constexpr int kGrowThreads = 1024;
constexpr uint32_t kGrowPer = 16;   // pages a thread looks at for free ones in a round
__global__ __launch_bounds__(kGrowThreads) void kv_grow(KvArgs a) {
    constexpr uint32_t NW = kGrowThreads / kWave;
    __shared__ int32_t slots[kKvMaxReq];
    __shared__ uint32_t need[kKvMaxReq], off[kKvMaxReq], first[kKvMaxReq], past[kKvMaxReq];
    __shared__ uint32_t red[NW], used;
    const uint32_t tid = tid_x(), n = a.n;
    const int32_t slot = tid < n ? a.seq[tid] : -1;
    if (tid < n) slots[tid] = slot;
    if (tid == 0) used = 0u;
    __syncthreads();
    bool ok = false;
    if (tid < n) {
        const int32_t s = a.start[tid], e = a.end[tid];
        ok = slot == -1 || ((uint32_t)slot < a.seqs && s >= 0 && e >= s && (uint64_t)(uint32_t)e <= (uint64_t)a.max_pages << a.page_shift);
        if (slot != -1)
            for (uint32_t j = 0; j < tid; ++j) ok = ok && slots[j] != slot;
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
    uint32_t cnt = 0;
    for (uint32_t b = p0; __any(b < p1); b += L) {
        int32_t page;
        cnt += (uint32_t)__builtin_popcountll(ballot(wants(b + sub, page) != 0u) & mine);
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
            a.fresh[at++] = (int32_t)(g0 + (uint32_t)__builtin_ctz(bits));
            bits &= bits - 1u;
        }
        found += here;
    }
    found = min(found, want);
    __syncthreads();   // (the list is complete)
    if (tid < n) {
        const bool served = ok && off[tid] + need[tid] <= found;
        if (served) a.result[tid] = 0;
        else refuse(a, &a.result[tid]);
        if (served && need[tid] != 0u) atomicMax(&used, off[tid] + need[tid]);
        if (!served) past[tid] = first[tid];
    }
    __syncthreads();
    if (act && past[req] > first[req]) {   // (a request's lanes together; the loops below wait for none of another's)
        uint32_t at = off[req];
        for (uint32_t b = p0; b < p1; b += L) {
            int32_t page;
            const uint32_t w = wants(b + sub, page);
            const uint64_t m = ballot(w != 0u) & mine;
            const uint32_t k = at + (uint32_t)__builtin_popcountll(m & below);
            if (w != 0u && k < found) {
                const int32_t f = a.fresh[k];
                row[b + sub] = f;
                a.from[k] = w == 2u ? page : -1;
            }
            at += (uint32_t)__builtin_popcountll(m);
        }
    }
    __syncthreads();
    for (uint32_t k = tid; k < used; k += kGrowThreads) {
        a.refs[a.fresh[k]] = 1;
        const int32_t f = a.from[k];
        if (f >= 0) atomicSub(&a.refs[f], 1);
    }
    if (tid == 0) *a.n_fresh = used;
}

// The copies that kv_grow has planned: (copy, layer, k or v, head) by workgroup, in turn.
// CP lanes a row of 16-byte chunks.
__global__ __launch_bounds__(kKvThreads) void kv_copy(KvArgs a) {
    const uint32_t used = *a.n_fresh;
    const uint32_t per = a.layers * 2u * a.kv_heads;
    const uint64_t items = (uint64_t)used * per;
    const uint32_t chunk = tid_x() & (a.cp - 1u), row0 = tid_x() / a.cp, step = kKvThreads / a.cp;
    for (uint64_t it = wg_x(); it < items; it += gridDim.x) {
        const uint32_t k = (uint32_t)(it / per), r = (uint32_t)(it % per);
        const int32_t src = a.from[k];
        if (src < 0) continue;
        const uint32_t dst = (uint32_t)a.fresh[k];
        const uint32_t head = r % a.kv_heads, kv = r / a.kv_heads & 1u, layer = r / (2u * a.kv_heads);
        unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k);
        const uint64_t f = place(a, layer, (uint32_t)src, head, 0), t = place(a, layer, dst, head, 0);
        const uint64_t ts = a.token_stride * (a.f8 ? 1u : 2u);
        if (chunk < a.chunks) {
            for (uint32_t row = row0; row < a.page_tokens; row += 4u * step) {
                u32x4 x[4];
#pragma unroll
                for (uint32_t u = 0; u < 4u; ++u)
                    if (row + u * step < a.page_tokens)
                        x[u] = *reinterpret_cast<const u32x4*>(base + f + (row + u * step) * ts + 16u * chunk);
#pragma unroll
                for (uint32_t u = 0; u < 4u; ++u)
                    if (row + u * step < a.page_tokens)
                        *reinterpret_cast<u32x4*>(base + t + (row + u * step) * ts + 16u * chunk) = x[u];
            }
        }
        if (a.f8) {
            float* sc = kv ? a.v_scale : a.k_scale;
            const uint64_t sf = scale_place(a, layer, (uint32_t)src, head, 0), st = scale_place(a, layer, dst, head, 0);
            for (uint32_t row = tid_x(); row < a.page_tokens; row += kKvThreads) sc[st + row] = sc[sf + row];
        }
    }
}

// ---- lcs_kv_compact ----
// Whether a request can be served, a workgroup each.
__global__ __launch_bounds__(kKvThreads) void kv_compact_check(KvArgs a) {
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
        for (uint32_t j = tid_x(); j < n; j += kKvThreads) {
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

// A workgroup moves one head's rows of k or v of one layer of one request, in order, by rounds
// of U rows a lane group: a round's rows are read by all its lanes before the first
// of them is written. Rows never move up, so a round overwrites no row of a later one:
// its places lie below the next round's first, and sources at or above their places.
__global__ __launch_bounds__(kKvThreads) void kv_compact(KvArgs a) {
    constexpr uint32_t U = 8;
    uint32_t b = wg_x();
    const uint32_t head = b % a.kv_heads;
    b /= a.kv_heads;
    const uint32_t kv = b & 1u;
    b >>= 1;
    const uint32_t layer = b % a.layers, i = b / a.layers;
    const int32_t slot = a.seq[i];
    if (slot == -1 || a.result[i] != 0) return;
    const uint32_t n = min((uint32_t)max(a.count[i], 0), a.max_keep);
    const int32_t* keep = a.index + (uint64_t)i * a.max_keep;
    const int32_t* row = a.table + (uint64_t)slot * a.max_pages;
    const uint32_t chunk = tid_x() & (a.cp - 1u), r0 = tid_x() / a.cp, step = kKvThreads / a.cp;
    unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k) + 16u * chunk;
    float* sc = kv ? a.v_scale : a.k_scale;
    const uint32_t in = a.page_tokens - 1u;
    const bool data = chunk < a.chunks;
    for (uint32_t j0 = 0; j0 < n; j0 += U * step) {
        u32x4 x[U];
        float s[U];
        uint64_t to[U], st[U];
        bool move[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t j = j0 + u * step + r0;
            const uint32_t pos = j < n ? (uint32_t)keep[j] : j;
            move[u] = j < n && pos != j;
            s[u] = 0.0f;
            to[u] = st[u] = 0;
            x[u] = u32x4{0, 0, 0, 0};
            if (move[u]) {
                const uint32_t pf = (uint32_t)row[pos >> a.page_shift], pt = (uint32_t)row[j >> a.page_shift];
                to[u] = place(a, layer, pt, head, j & in);
                if (data) x[u] = *reinterpret_cast<const u32x4*>(base + place(a, layer, pf, head, pos & in));
                if (a.f8 && chunk == 0u) {
                    st[u] = scale_place(a, layer, pt, head, j & in);
                    s[u] = sc[scale_place(a, layer, pf, head, pos & in)];
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (a barrier by itself waits for no load)
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (move[u]) {
                if (data) *reinterpret_cast<u32x4*>(base + to[u]) = x[u];
                if (a.f8 && chunk == 0u) sc[st[u]] = s[u];
            }
        }
    }
}

// ---- lcs_kv_append ----
// A workgroup writes kAppendTokens tokens of one layer and sequence: cp lanes a row of 8
// elements each, both k's and v's heads.
constexpr uint32_t kAppendTokens = 16;
template <bool F8>
__global__ __launch_bounds__(kKvThreads) void kv_append(KvAppendArgs p) {
    const KvArgs& a = p.a;
    const uint32_t i = wg_x() / p.blocks, j0 = wg_x() % p.blocks * kAppendTokens, l = __builtin_amdgcn_workgroup_id_y();
    const int32_t slot = a.seq ? a.seq[i] : (int32_t)i;
    if (slot == -1) return;
    const uint32_t n = a.count ? min((uint32_t)max(a.count[i], 0), p.rows_per_seq) : p.rows_per_seq;
    if (j0 >= n) return;
    if ((uint32_t)slot >= a.seqs) {
        if (tid_x() == 0) atomicOr(a.status, kStatusPages);
        return;
    }
    const int32_t pos0 = a.start[i];
    const int32_t* row = a.table + (uint64_t)slot * a.max_pages;
    const uint32_t chunk = tid_x() & (a.cp - 1u), step = kKvThreads / a.cp;
    const uint32_t items = min(n - j0, kAppendTokens) * 2u * a.kv_heads, elems = a.head_dim / 8u;
    for (uint32_t it = tid_x() / a.cp; it < items; it += step) {
        const uint32_t head = it % a.kv_heads, kv = it / a.kv_heads & 1u, j = j0 + it / (2u * a.kv_heads);
        const int64_t pos = (int64_t)pos0 + j;
        const int32_t src = a.index ? a.index[(uint64_t)i * p.rows_per_seq + j] : (int32_t)j;
        const bool in = pos >= 0 && (uint64_t)pos < (uint64_t)a.max_pages << a.page_shift && (uint32_t)src < p.rows_per_seq;
        const int32_t page = in ? row[(uint64_t)pos >> a.page_shift] : -1;
        const bool ok = page_ok(a, page) && a.refs[page_ok(a, page) ? page : 0] <= 1;
        u32x4 x = {0, 0, 0, 0};
        if (ok && chunk < elems) {
            const uint64_t r = (uint64_t)i * p.rows_per_seq + (uint32_t)src;
            const uint64_t at = (uint64_t)l * p.new_layer_stride + r * (kv ? p.v_stride : p.k_stride) + head * a.head_dim + 8u * chunk;
            x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(kv ? p.v : p.k) + at);
        }
        const uint32_t layer = a.layer + l, tok = (uint32_t)pos & (a.page_tokens - 1u);
        unsigned char* base = static_cast<unsigned char*>(kv ? a.v : a.k);
        if constexpr (F8) {
            uint32_t top = 0;   // the largest |x|, by its bits (a NaN's lie above infinity's)
#pragma unroll
            for (int k = 0; k < 4; ++k) top = max(top, max(x[k] & 0x7fffu, x[k] >> 16 & 0x7fffu));
            for (uint32_t m = 1; m < a.cp; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, (int)m));
            const float t = __uint_as_float(top << 16);
            const float scale = t > 0.0f ? fmaxf(fdiv(t, kE4m3Max), kLeastScale) : 1.0f;   // (a NaN is not above 0)
            uint32_t q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t w = x[2 * h + k / 2];
                    const float v = fdiv(__uint_as_float(k % 2 ? w & 0xffff0000u : w << 16), scale);
                    f[k] = v > kE4m3Max ? kE4m3Max : v < -kE4m3Max ? -kE4m3Max : v;
                }
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                q[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
            }
            if (ok && chunk < elems) *reinterpret_cast<u32x2*>(base + place(a, layer, (uint32_t)page, head, tok) + 8u * chunk) = u32x2{q[0], q[1]};
            if (ok && chunk == 0u) (kv ? a.v_scale : a.k_scale)[scale_place(a, layer, (uint32_t)page, head, tok)] = scale;
        } else {
            if (ok && chunk < elems) *reinterpret_cast<u32x4*>(base + place(a, layer, (uint32_t)page, head, tok) + 16u * chunk) = x;
        }
        if (!ok && chunk == 0u) atomicOr(a.status, kStatusPages);
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
    hipLaunchKernelGGL(kv_copy, dim3(2048), dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const KvArgs& args, hipStream_t st) {
    KvArgs a = args;
    a.chunks = a.head_dim * (a.f8 ? 1u : 2u) / 16u;
    a.cp = pow2_from(a.chunks);
    hipLaunchKernelGGL(kv_compact_check, dim3(a.n), dim3(kKvThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kv_compact, dim3(a.n * a.layers * 2u * a.kv_heads), dim3(kKvThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppendArgs& args, hipStream_t st) {
    KvAppendArgs p = args;
    p.a.cp = pow2_from(p.a.head_dim / 8u);
    p.blocks = (p.rows_per_seq + kAppendTokens - 1u) / kAppendTokens;
    const dim3 grid(p.a.n * p.blocks, p.n_layers);
    if (p.a.f8) hipLaunchKernelGGL(kv_append<true>, grid, dim3(kKvThreads), 0, st, p);
    else hipLaunchKernelGGL(kv_append<false>, grid, dim3(kKvThreads), 0, st, p);
    return hipGetLastError();
}

}  // namespace lcs
