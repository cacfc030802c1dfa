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
#include "vbm_quantize.hpp"

namespace vbm {
namespace {

constexpr int kFp8Threads = 256;
constexpr int kBlocksPerGroup = kFp8Threads / 16;

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
