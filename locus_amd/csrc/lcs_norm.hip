// The residual's addition and the root-mean-square norm ahead of the lm-head, for
// MI355X (gfx950): h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, per
// row, with y in bf16, f32 or in 8 bits (e4m3) with a scale per row, the operand
// that lcs_lmhead_ex takes.
//
// Reference: the output norm ahead of matvec(out_w, norm(x))
// (src/locus/model/llama.cpp:512-513, 754-761).
//
// Memory bounds it: a row is read once, held in registers, and written once.
// The sum of squares and the largest |h w| come from the same pass, so one
// exchange between the row's waves gives both. In 8 bits the norm's factor r
// cancels (y / scale = h w r / (max|h w| r / 448)), so an element costs two
// products after it. Squares, sums and h are f32 (h unrounded: the norm reads it
// from the registers and not from the rounded sum); y is rounded once.
//
// Rows, strides and widths are any: the vector loads and stores ask for the
// element's alignment only, which the hardware's unaligned access mode serves,
// and the lane that holds a row's end takes its elements one by one.
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
// (vectors at the alignment of their elements)
typedef u32x4 u32x4_2 __attribute__((aligned(2), may_alias));
typedef u32x4 u32x4_4 __attribute__((aligned(4), may_alias));
typedef u32x2 u32x2_1 __attribute__((aligned(1), may_alias));

constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126: a scale below the normal numbers would lose its bits

__device__ __forceinline__ float bf16_to_f(uint32_t u) { return __uint_as_float(u << 16); }
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t f_to_bf16x2(float a, float b) {   // to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// 8 elements from p; in a row's last lane only the first n exist.
template <typename T> struct Io;
template <> struct Io<uint16_t> {   // bf16
    static __device__ __forceinline__ void load(const uint16_t* p, uint32_t n, float (&v)[8]) {
        if (n >= 8u) {
            const u32x4 q = *reinterpret_cast<const u32x4_2*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = bf16_to_f(q[i] & 0xffffu);
                v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) v[i] = i < n ? bf16_to_f(p[i]) : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(uint16_t* p, uint32_t n, const float (&v)[8]) {
        u32x4 q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = f_to_bf16x2(v[2 * i], v[2 * i + 1]);
        if (n >= 8u) {
            __builtin_nontemporal_store(q, reinterpret_cast<u32x4_2*>(p));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
                if (i < n) p[i] = (uint16_t)(q[i / 2u] >> (16u * (i % 2u)));
        }
    }
};
template <> struct Io<float> {
    static __device__ __forceinline__ void load(const float* p, uint32_t n, float (&v)[8]) {
        if (n >= 8u) {
            const u32x4 q = *reinterpret_cast<const u32x4_4*>(p), r = *reinterpret_cast<const u32x4_4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __uint_as_float(q[i]);
                v[4 + i] = __uint_as_float(r[i]);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) v[i] = i < n ? p[i] : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(float* p, uint32_t n, const float (&v)[8]) {
        if (n >= 8u) {
            u32x4 q, r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[i] = __float_as_uint(v[i]);
                r[i] = __float_as_uint(v[4 + i]);
            }
            __builtin_nontemporal_store(q, reinterpret_cast<u32x4_4*>(p));
            __builtin_nontemporal_store(r, reinterpret_cast<u32x4_4*>(p + 4));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
                if (i < n) p[i] = v[i];
        }
    }
};
template <> struct Io<uint8_t> {   // e4m3; finite values are inside +-448 already
    static __device__ __forceinline__ void store(uint8_t* p, uint32_t n, const float (&v)[8]) {
        uint32_t q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int w = 0;
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], w, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
            q[i] = (uint32_t)w;
        }
        if (n >= 8u) {
            __builtin_nontemporal_store(u32x2{q[0], q[1]}, reinterpret_cast<u32x2_1*>(p));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
                if (i < n) p[i] = (uint8_t)(q[i / 4u] >> (8u * (i % 4u)));
        }
    }
};

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    auto u_max = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    LCS_WAVE_REDUCE_32(uint32_t, v, 0u, u_max);
    return v;
}
__device__ __forceinline__ float clamp448(float v) {   // (a NaN stays one)
    return v > kE4m3Max ? kE4m3Max : v < -kE4m3Max ? -kE4m3Max : v;
}

}  // namespace

// a.waves waves per row, each lane NV groups of 8 elements, a.per rows per workgroup.
// One group a lane up to 8192 columns, as many waves as that takes: the row's
// chain of loads, exchange and stores is then shortest, and most rows are in
// flight (bf16 into e4m3 with a residual, us by 4 / 2 / 1 groups: 8192 x 8192
// 117 / 96 / 93, 1 x 4096 6.7 / 4.3 / 3.2, 512 x 4096 10.0 / 7.1 / 6.1). Above,
// four (4096 x 16384: 115, with two 120). What is written is not read here
// again: stores past the caches' usual order (8192 x 8192 93 -> 90, 4096 x 16384
// 115 -> 106; loads like that cost 3 to 15 %).
template <typename XT, typename YT, bool RES, int NV>
__global__ __launch_bounds__(1024) void add_rmsnorm(NormArgs a) {
    constexpr bool Q8 = sizeof(YT) == 1;
    struct Part { float ss; uint32_t top; };
    __shared__ Part part[16];
    __shared__ uint32_t part2[16];
    const uint32_t WPR = a.waves;
    const uint32_t tid = tid_x(), wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid / kWave));
    const uint32_t rw = wv / WPR, first = rw * WPR;            // the row in the workgroup, its first wave
    const uint64_t row0 = (uint64_t)wg_x() * a.per + rw;
    const bool live = row0 < a.rows;                           // (no early end: the waves meet at a barrier)
    const uint64_t row = live ? row0 : a.rows - 1u;
    const uint32_t H = a.hidden, t = (wv - first) * kWave + (uint32_t)lane_id();
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
    const XT* res = static_cast<const XT*>(a.residual) + row * a.residual_stride;
    const XT* w = static_cast<const XT*>(a.weight);
    float v[NV][8], g[NV][8];
    uint32_t c[NV], n[NV];
    float ss = 0.0f;
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        c[i] = ((uint32_t)i * WPR * kWave + t) * 8u;
        n[i] = c[i] < H ? H - c[i] : 0u;
        if (n[i] == 0u) c[i] = 0u;
        Io<XT>::load(x + c[i], n[i], v[i]);
    }
    if (RES) {
        float r[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) Io<XT>::load(res + c[i], n[i], r[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] + r[i][e];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) Io<XT>::load(w + c[i], n[i], g[i]);
    if (RES && live && a.sum) {
        XT* sum = static_cast<XT*>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) Io<XT>::store(sum + c[i], n[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ss = __builtin_fmaf(v[i][e], v[i][e], ss);
            if (Q8) {
                // (as integers the bits of non-negative floats order as the floats do, NaNs above all)
                const uint32_t b = __float_as_uint(v[i][e] * g[i][e]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
        }
    ss = wave_sum_f(ss);
    if (Q8) top = wave_max_u(top);
    if (WPR > 1u) {
        if (lane_id() == 0) part[wv] = Part{ss, top};
        __syncthreads();
        const bool in = (uint32_t)lane_id() < WPR;
        const Part p = part[in ? first + (uint32_t)lane_id() : first];
        ss = wave_sum_f(in ? p.ss : 0.0f);
        if (Q8) top = wave_max_u(p.top);
    }
    const float r = 1.0f / __builtin_sqrtf(ss / (float)H + a.eps);
    YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
    if constexpr (!Q8) {
        if (!live) return;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * r * g[i][e];
            Io<YT>::store(y + c[i], n[i], v[i]);
        }
    } else {
        // The largest |h w| out of (1e-30, 1e30), which products may have left f32 to reach, a
        // row with an inf or a NaN, a sum of squares past f32, or a scale below the normal numbers:
        // the formula itself, element by element. A row whose largest |y| is 0 or a NaN has scale 1.
        const float m = __uint_as_float(top);
        const bool plain = m > 1e-30f && m < 1e30f && ss < 3e38f && m * r >= kE4m3Max * kLeastScale;
        float scale, inv;
        if (plain) {
            scale = m * r / kE4m3Max;
            inv = kE4m3Max / m;
        } else {
            uint32_t t2 = 0u;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[i][e] = v[i][e] * r * g[i][e];
                    const uint32_t b = (uint32_t)e < n[i] ? __float_as_uint(v[i][e]) & 0x7fffffffu : 0u;
                    t2 = b > t2 ? b : t2;
                }
            top = wave_max_u(t2);
            scale = inv = 1.0f;
        }
        if (WPR > 1u) {
            // (every wave of a row goes the same way; rows of one workgroup may not: the barrier is outside the branch)
            if (!plain && lane_id() == 0) part2[wv] = top;
            __syncthreads();
        }
        if (!plain) {
            if (WPR > 1u) {
                top = wave_max_u(part2[(uint32_t)lane_id() < WPR ? first + (uint32_t)lane_id() : first]);
            }
            const bool nan = top > 0x7f800000u;
            if (!nan && top != 0u) {
                scale = __uint_as_float(top) / kE4m3Max;
                scale = scale < kLeastScale ? kLeastScale : scale;
            }
        }
        if (!live) return;
        if (t == 0u) a.y_scale[row] = scale;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = clamp448(plain ? v[i][e] * g[i][e] * inv : v[i][e] / scale);
            Io<YT>::store(y + c[i], n[i], v[i]);
        }
    }
}

namespace {

template <typename XT, typename YT, bool RES, int NV>
void go(const NormArgs& a0, hipStream_t st) {
    NormArgs a = a0;
    a.waves = (a.hidden + 512u * NV - 1u) / (512u * NV);
    a.per = a.waves < 4u ? 4u / a.waves : 1u;
    // (a launch's threads are counted in 32 bits, and past them go missing without an
    // error: 2^31 at a time, 2 M rows of 8192 columns)
    const uint32_t threads = a.waves * a.per * kWave;
    const uint64_t most = (uint64_t)((1u << 31) / threads) * a.per;
    for (uint64_t r0 = 0; r0 < a0.rows; r0 += most) {
        a.rows = a0.rows - r0 < most ? a0.rows - r0 : most;
        a.x = static_cast<const XT*>(a0.x) + r0 * a.x_stride;
        if (RES) a.residual = static_cast<const XT*>(a0.residual) + r0 * a.residual_stride;
        if (a0.sum) a.sum = static_cast<XT*>(a0.sum) + r0 * a.sum_stride;
        a.y = static_cast<YT*>(a0.y) + r0 * a.y_stride;
        if (a0.y_scale) a.y_scale = a0.y_scale + r0;
        hipLaunchKernelGGL((add_rmsnorm<XT, YT, RES, NV>), dim3((uint32_t)((a.rows + a.per - 1u) / a.per)), dim3(threads), 0, st, a);
    }
}
template <typename XT, typename YT, bool RES>
void pick(const NormArgs& a, hipStream_t st) {
    if (a.hidden <= 8192u) go<XT, YT, RES, 1>(a, st);
    else go<XT, YT, RES, 4>(a, st);
}
template <typename XT, typename YT>
void pick_res(const NormArgs& a, hipStream_t st) {
    if (a.residual) pick<XT, YT, true>(a, st);
    else pick<XT, YT, false>(a, st);
}
template <typename XT>
void pick_out(const NormArgs& a, uint32_t y_dtype, hipStream_t st) {
    if (y_dtype == LCS_E4M3) pick_res<XT, uint8_t>(a, st);
    else if (y_dtype == LCS_BF16) pick_res<XT, uint16_t>(a, st);
    else pick_res<XT, float>(a, st);
}

}  // namespace

hipError_t launch_add_rmsnorm(const NormArgs& a, uint32_t x_dtype, uint32_t y_dtype, hipStream_t st) {
    if (x_dtype == LCS_BF16) pick_out<uint16_t>(a, y_dtype, st);
    else pick_out<float>(a, y_dtype, st);
    return hipGetLastError();
}

}  // namespace lcs
