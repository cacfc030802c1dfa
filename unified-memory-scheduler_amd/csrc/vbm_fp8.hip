// Block-scaled FP8 activations: rows of e4m3 codes with one fp32 scale per 128 values, from rows of fp32, fp16
// or bf16, or from the gate and up halves of an expert through its GLU.
//
// A run of 128 values (the last of a row may be shorter) with a = max(max |x|, 2^-116):
//   scale = a / 448,  code = e4m3(448 x / a), rounded to nearest even.
// 448 is the largest e4m3 value, so nothing saturates. 16-bit inputs meet exact ties of the e4m3 grid often, so the
// quotient of 448 x (rounded to fp32, which is exact for them) is the correctly rounded one: with r = 1 / a correctly rounded, q = x r and one Newton step
// q + (x - q a) r with fused multiply-adds is the rounded x / a (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990), two instructions per value instead of a division. a / 512 and 0.875 x stand for a
// and 448 x, so that neither overflows. The floor under a keeps 1 / a finite; blocks of zeros get its scale. A block with a NaN
// or an infinity has no scale: it comes out as a NaN scale and zero codes, so that every product with it is NaN.
//
// Bound by bandwidth (one read of the inputs, one write of a quarter to half of them). Sixteen lanes share a block, eight values
// each: 16- or 2 x 16-byte loads, an 8-byte store of codes, and the maximum over 16 lanes by four DPP moves. 8192 x 4096 bf16 19 to
// 21 us (5.0 TB/s), GLU of 8192 x 2880 fp32 pairs 41 us (5.2 TB/s, where a large copy reaches 5.1); one row 2 us, a launch.
#include <type_traits>

#include "vbm_device.hpp"
#include "vbm_internal.hpp"

namespace vbm {
namespace {

constexpr int kFp8Threads = 256;
constexpr int kBlocksPerGroup = kFp8Threads / 16;

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

struct Fp8Args {
    const void * x, * up;          // up: null for the plain quantizer
    int64_t x_stride, up_stride;   // elements
    int64_t blocks;                // n_rows * blocks per row
    int k, kb;
    int activation;
    float alpha, limit;
    uint8_t * codes;
    float * scales;
};

template <int TYPE, bool VEC, bool GLU>
__global__ __launch_bounds__(kFp8Threads) void quantize_fp8_kernel(Fp8Args A) {
    const int lane = threadIdx.x & 15;
    for (int64_t b0 = blockIdx.x * static_cast<int64_t>(kBlocksPerGroup); b0 < A.blocks;
         b0 += gridDim.x * static_cast<int64_t>(kBlocksPerGroup)) {
        const int64_t at = b0 + (threadIdx.x >> 4);
        const uint32_t b = static_cast<uint32_t>(at < A.blocks ? at : A.blocks - 1);
        const uint32_t row = b / static_cast<uint32_t>(A.kb), kb = b - row * static_cast<uint32_t>(A.kb);
        const int e0 = static_cast<int>(kb) * 128 + lane * 8;
        const bool live = e0 < A.k;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (live) {
            load8<TYPE, VEC>(A.x, row * A.x_stride + e0, v);
            if constexpr (GLU) {
                float u[8];
                load8<TYPE, VEC>(A.up, row * A.up_stride + e0, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = glu_value(A.activation, v[i], u[i], A.alpha, A.limit);
            }
        }
        // (the last workgroup's spare lanes write the last block's values again)
        store_block(v, live, A.codes + static_cast<int64_t>(row) * A.k + e0, A.scales + b);
    }
}

template <bool GLU>
void launch_quantize_fp8(int type, const Fp8Args & a, hipStream_t stream) {
    if (a.blocks == 0) return;
    const size_t esize = type == VBM_TYPE_F32 ? 4 : 2;
    auto aligned = [&](const void * p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && static_cast<size_t>(stride) * esize % 16 == 0;
    };
    const bool vec = aligned(a.x, a.x_stride) && (!GLU || aligned(a.up, a.up_stride));
    const int64_t groups = (a.blocks + kBlocksPerGroup - 1) / kBlocksPerGroup;
    const dim3 grid(static_cast<unsigned>(groups < (1 << 20) ? groups : 1 << 20)), block(kFp8Threads);
    auto go = [&](auto type_c) {
        constexpr int TYPE = decltype(type_c)::value;
        if (vec) hipLaunchKernelGGL((quantize_fp8_kernel<TYPE, true, GLU>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((quantize_fp8_kernel<TYPE, false, GLU>), grid, block, 0, stream, a);
    };
    if (type == VBM_TYPE_F32) go(std::integral_constant<int, VBM_TYPE_F32>{});
    else if (type == VBM_TYPE_F16) go(std::integral_constant<int, VBM_TYPE_F16>{});
    else go(std::integral_constant<int, VBM_TYPE_BF16>{});
    check_hip(hipGetLastError(), "FP8 quantizer launch");
}

Fp8Args fp8_args(int x_type, int64_t n_rows, int64_t k, const void * codes, const void * scales) {
    require(x_type == VBM_TYPE_F32 || x_type == VBM_TYPE_F16 || x_type == VBM_TYPE_BF16, "x must be F32, F16 or BF16");
    require(n_rows >= 0 && k > 0 && k % 16 == 0 && k < (int64_t{1} << 31), "k must be a positive multiple of 16");
    const int64_t kb = (k + 127) / 128;
    require(n_rows < (int64_t{1} << 31) / kb, "too many blocks for one call");
    require(n_rows == 0 || (codes && scales), "null buffer");
    require(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
            "codes must be 16-byte and scales 4-byte aligned");
    Fp8Args a{};
    a.blocks = n_rows * kb;
    a.k = static_cast<int>(k);
    a.kb = static_cast<int>(kb);
    return a;
}

void require_rows(int x_type, const void * x, int64_t stride, int64_t n_rows, int64_t k) {
    require(n_rows == 0 || x, "null buffer");
    require(stride >= k, "rows must be at least k elements apart");
    require(reinterpret_cast<uintptr_t>(x) % (x_type == VBM_TYPE_F32 ? 4 : 2) == 0, "x must be aligned to its type");
}

}  // namespace
}  // namespace vbm

using namespace vbm;

extern "C" {

vbm_status vbm_quantize_fp8(int x_type, const void * x, int64_t n_rows, int64_t k, int64_t x_stride, void * codes,
                            float * scales, void * stream) {
    return guarded([&] {
        Fp8Args a = fp8_args(x_type, n_rows, k, codes, scales);
        require_rows(x_type, x, x_stride, n_rows, k);
        a.x = x;
        a.x_stride = x_stride;
        a.codes = static_cast<uint8_t *>(codes);
        a.scales = scales;
        launch_quantize_fp8<false>(x_type, a, as_stream(stream));
    });
}

vbm_status vbm_glu_quantize_fp8(int activation, int x_type, const void * gate, const void * up, int64_t n_rows,
                                int64_t width, int64_t gate_stride, int64_t up_stride, float alpha, float limit,
                                void * codes, float * scales, void * stream) {
    return guarded([&] {
        require(activation == VBM_ACT_SILU || activation == VBM_ACT_SWIGLU_OAI, "unknown activation");
        Fp8Args a = fp8_args(x_type, n_rows, width, codes, scales);
        require_rows(x_type, gate, gate_stride, n_rows, width);
        require_rows(x_type, up, up_stride, n_rows, width);
        a.x = gate;
        a.up = up;
        a.x_stride = gate_stride;
        a.up_stride = up_stride;
        a.activation = activation;
        a.alpha = alpha;
        a.limit = limit;
        a.codes = static_cast<uint8_t *>(codes);
        a.scales = scales;
        launch_quantize_fp8<true>(x_type, a, as_stream(stream));
    });
}

}  // extern "C"
