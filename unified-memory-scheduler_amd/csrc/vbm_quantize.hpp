// What the activations' quantizers share: rows of fp32, fp16 or bf16 read eight values at a time, an expert's GLU to about an ulp, and
// e4m3 codes of blocks of 128 values.
#pragma once

#include "vbm_device.hpp"

namespace vbm {
namespace {

typedef unsigned u32x4q __attribute__((ext_vector_type(4)));
typedef unsigned u32x2q __attribute__((ext_vector_type(2)));

// Eight values of a row from element e0 on, as fp32. VEC: the address is 16-byte aligned.
template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const void * p, int64_t e0, float v[8]) {
    if constexpr (TYPE == VBM_TYPE_F32) {
        const float * x = static_cast<const float *>(p) + e0;
        if constexpr (VEC) {
            const float4 a = reinterpret_cast<const float4 *>(x)[0], b = reinterpret_cast<const float4 *>(x)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = x[i];
        }
        return;
    }
    const uint16_t * x = static_cast<const uint16_t *>(p) + e0;
    uint16_t h[8];
    if constexpr (VEC) {
        const u32x4q w = *reinterpret_cast<const u32x4q *>(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = x[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (TYPE == VBM_TYPE_F16) v[i] = static_cast<float>(__builtin_bit_cast(_Float16, h[i]));
        else v[i] = __builtin_bit_cast(float, static_cast<uint32_t>(h[i]) << 16);
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_with_moved(uint32_t v) {
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, true));
    return v > o ? v : o;
}

// The block of 16 lanes whose values these are (zeros past the end of the row) as codes and scale.
__device__ __forceinline__ void store_block(const float v[8], bool live, uint8_t * codes, float * scale) {
    // the magnitudes' bits order as the magnitudes do, infinities and NaNs above every number
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
    m = max_with_moved<0xB1>(m);
    m = max_with_moved<0x4E>(m);
    m = max_with_moved<0x141>(m);
    m = max_with_moved<0x140>(m);
    const float a = fmaxf(__builtin_bit_cast(float, m), 0x1p-116f);
    const bool finite = m < 0x7F800000u;
    const float a512 = a * 0x1p-9f, r = 1.0f / a512;
    uint32_t c[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = v[4 * h + i] * 0.875f, p = x * r;
            q[i] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-p, a512, x), r, p), x);   // (the step loses a zero's sign)
        }
        uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
        c[h] = finite ? w : 0u;
    }
    if (live) *reinterpret_cast<u32x2q *>(codes) = u32x2q{c[0], c[1]};
    if ((threadIdx.x & 15) == 0) *scale = finite ? a / 448.0f : __builtin_nanf("");
}

// exp(x) for x in [-104, kLastExp] to about an ulp: 2^(x log2 e) by the hardware's 2^y, corrected by what the product's rounding and log2 e's
// own lost. (expf_rn of the exact order, which rounds from double, would bound these kernels by its arithmetic.)
// kLastExp: the largest fp32 x whose e^x is one too, 88.7228317 (below ln(2^128 - 2^103) = 88.7228391, and the next one above); x log2 e
// is then at most 127.99999, and 2^y in range.
constexpr float kLastExp = 0x1.62e42ep+6f;
__device__ __forceinline__ float exp_ulp(float x) {
    const float log2e = 1.44269502e+00f, log2e_rest = 1.92596299e-08f, ln2 = 6.93147181e-01f;
    const float hi = x * log2e;
    const float lo = __builtin_fmaf(x, log2e_rest, __builtin_fmaf(x, log2e, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(e, lo * ln2, e);
}
// a / (1 + e^x): reciprocal and one Newton step on the quotient, of a quarter of both, so that the reciprocal of the largest
// e^x is a normal number. Past the fp32 range of e^x it is a zero, as a division by infinity (NaN for an infinite a).
__device__ __forceinline__ float over_one_plus_exp(float a, float x) {
    const float d = __builtin_fmaf(exp_ulp(x < -104.0f ? -104.0f : x), 0.25f, 0.25f), n = 0.25f * a;
    const float r = __builtin_amdgcn_rcpf(d), q = n * r;
    return x > kLastExp ? 0.0f * a : __builtin_fmaf(__builtin_fmaf(-q, d, n), r, q);
}
// The formulas of glu().
__device__ __forceinline__ float glu_value(int activation, float g0, float u0, float alpha, float limit) {
    if (activation == VBM_ACT_SWIGLU_OAI) {
        const float g = limit < g0 ? limit : g0;
        const float u = u0 < -limit ? -limit : (limit < u0 ? limit : u0);
        return over_one_plus_exp(g, alpha * -g) * (u + 1.0f);
    }
    return over_one_plus_exp(g0, -g0) * u0;
}

}  // namespace
}  // namespace vbm
