// Attention of a step's new tokens over a paged cache and over each other, for MI355X
// (gfx950): o = sum_j p_j v_j with p = softmax_j(scale q.k_j), j over the sequence's
// cached tokens and over the new tokens that the row's mask names.
//
// A wave per row and query head takes 64 keys at a time: a key's score per lane, the
// running maximum and sum over the wave, then the values with a few elements of the
// head per lane.
//
// (This file is compiled with NaNs honoured: a NaN in a row has to stay one.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lcs_device.hpp"
#include "lcs_internal.hpp"

namespace lcs {

namespace {

constexpr uint32_t kHeadMax = 256;

__device__ __forceinline__ float bf16_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float e4m3_f(uint32_t b) { return __builtin_amdgcn_cvt_f32_fp8((int)b, 0); }
__device__ __forceinline__ uint32_t f_bf16(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v); }

}  // namespace

template <bool F8>
__global__ __launch_bounds__(kWave) void tree_attn(TreeArgs a) {
    __shared__ float qs[kHeadMax], ps[kWave];
    __shared__ uint64_t at[kWave];   // a key's element 0 in k or v
    const uint32_t lane = tid_x(), h = wg_x() % a.heads, r = wg_x() / a.heads, i = r / a.rows_per_seq, j = r % a.rows_per_seq;
    const uint32_t D = a.c.head_dim, kvh = h / a.group, R = a.rows_per_seq;
    const int32_t slot = a.c.seq ? a.c.seq[i] : (int32_t)i;
    int64_t len = slot == -1 ? 0 : max(a.length[i], 0);
    bool bad = slot < -1 || slot >= (int64_t)a.c.seqs;
    if (bad) len = 0;
    const int64_t most = (int64_t)a.c.max_pages << a.c.page_shift;
    bad = bad || len > most;
    len = len > most ? most : len;
    const int32_t* row = a.c.table + (uint64_t)(len > 0 ? slot : 0) * a.c.max_pages;
    for (uint32_t d = lane; d < D; d += kWave) qs[d] = bf16_f(a.q[r * a.q_stride + h * D + d]);
    __syncthreads();
    float m = -__builtin_huge_valf(), z = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // cached tokens in blocks of 64, then the new ones
    const int64_t blocks = (len + kWave - 1) / kWave;
    for (int64_t b = 0; b < blocks + (R + kWave - 1) / kWave; ++b) {
        const bool fresh = b >= blocks;
        const int64_t t = (fresh ? b - blocks : b) * kWave + lane;
        bool see = false;
        float s = 0.0f, vs = 1.0f;
        uint64_t e = 0;
        if (!fresh) {
            if (t < len) {
                const int32_t page = row[t >> a.c.page_shift];
                see = (uint32_t)page < a.c.pages;
                bad = bad || !see;
                if (see) {
                    const uint32_t in = (uint32_t)t & (a.c.page_tokens - 1u);
                    e = a.c.layer * a.c.layer_stride + (uint32_t)page * a.c.page_stride + kvh * a.c.head_stride + in * a.c.token_stride;
                    float ks = 1.0f;
                    if (F8) {
                        const uint64_t w = ((((uint64_t)a.c.layer * a.c.pages + (uint32_t)page) * a.c.kv_heads + kvh) << a.c.page_shift) + in;
                        ks = a.c.k_scale[w];
                        vs = a.c.v_scale[w];
                    }
                    for (uint32_t d = 0; d < D; ++d)
                        s += qs[d] * (F8 ? e4m3_f(static_cast<const uint8_t*>(a.c.k)[e + d]) : bf16_f(static_cast<const uint16_t*>(a.c.k)[e + d]));
                    s *= ks;
                }
            }
        } else if (t < R) {
            see = a.mask ? a.mask[(uint64_t)r * a.mask_words + (uint32_t)t / 32u] >> (t % 32) & 1u : t <= j;
            if (see) {
                const uint64_t n = (uint64_t)i * R + (uint32_t)t;
                e = n * a.v_stride + kvh * D;
                for (uint32_t d = 0; d < D; ++d) s += qs[d] * bf16_f(a.k[n * a.k_stride + kvh * D + d]);
            }
        }
        s = see ? s * a.scale : -__builtin_huge_valf();
        const float top = fmaxf(m, wave_max(s));
        const float base = top == -__builtin_huge_valf() ? 0.0f : top;
        const float p = see ? expf(s - base) : 0.0f;
        const float keep = expf(m - base);
        m = top;
        z = z * keep + wave_sum_f(p);
        ps[lane] = p * vs;
        at[lane] = e;
        const uint64_t seen = ballot(see);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= keep;
        for (uint64_t w = seen; w; w &= w - 1u) {
            const uint32_t x = (uint32_t)__builtin_ctzll(w);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t d = lane + c * kWave;
                if (d < D) {
                    const float v = fresh ? bf16_f(a.v[at[x] + d])
                                    : F8  ? e4m3_f(static_cast<const uint8_t*>(a.c.v)[at[x] + d])
                                          : bf16_f(static_cast<const uint16_t*>(a.c.v)[at[x] + d]);
                    o[c] += ps[x] * v;
                }
            }
        }
        __syncthreads();
    }
    const bool none = m == -__builtin_huge_valf() && z == 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t d = lane + c * kWave;
        if (d < D) a.o[r * a.o_stride + h * D + d] = (uint16_t)f_bf16(none ? 0.0f : o[c] / z);
    }
    if (lane == 0 && a.lse) a.lse[(uint64_t)r * a.heads + h] = none ? -__builtin_huge_valf() : m + logf(z);
    if (bad) atomicOr(a.c.status, kStatusPages);
}

hipError_t launch_tree_attn(const TreeArgs& a, hipStream_t st) {
    const dim3 grid(a.c.n * a.rows_per_seq * a.heads);
    if (a.c.f8) hipLaunchKernelGGL(tree_attn<true>, grid, dim3(kWave), 0, st, a);
    else hipLaunchKernelGGL(tree_attn<false>, grid, dim3(kWave), 0, st, a);
    return hipGetLastError();
}

}  // namespace lcs
