// Rows of activations that need the whole row before their first code: the residual addition with the root-mean-square norm, and
// 8-bit integer codes with one scale per row, from rows as they are or from an expert's gate and up halves through its GLU.
//
//   norm:      s = T(x + residual),  v = (s * (1 / sqrt(mean s^2 + eps))) * weight
//   integers:  a = max(max |v|, 2^-116) over the row,  scale = a / 127,  code = 127 v / a to the nearest integer, ties to even
//   e4m3:      per 128 values, as the FP8 quantizer does
//
// The sum is rounded to its own type first and the norm is that of the stored values, so that it does not matter whether the sum
// is kept or added again by the next reader. Squares, their sum and everything after it are fp32: a row whose sum of squares is
// no fp32 number has no norm and comes out as NaN. The integers' quotient is the correctly rounded one, by the step that the e4m3 codes
// use (127/128 v and a / 128 stand for 127 v and a, so that neither overflows), and then rounded to an integer.
//
// Bound by bandwidth: each value is read once and held in registers, eight a lane and up to eight such chunks, while the row's sum and
// maximum are found (DPP inside a wave, one exchange through LDS between the waves of a row). 8192 rows of 4096 bf16: norm with sum, y and
// e4m3 codes 59 us (5.15 TB/s, where a large copy reaches 5.1), integers 21 us (4.8); GLU of 8192 x 2880 fp32 pairs to integers 41 us (5.2), of
// bf16 pairs 29 (4.0); 1517 of 2880 fp16, norm and integers, 11.8 us (3.3); one row 3.2 us, of which a launch is 2, the rest three loads (x, the
// residual, the weight) and two exchanges one after the other: a chunk's loads stand in branches on the alignment and are waited for there, the sum's
// stores with them. Rows of more than 16384 values have up to eight chunks, whose loads so follow each other too, and spill up to 72 bytes a lane: 1024 of 32768 bf16, norm with
// sum, y and integers, 72 us (4.2 TB/s), one 9.4.
#include <type_traits>

#include "vbm_device.hpp"
#include "vbm_internal.hpp"
#include "vbm_quantize.hpp"

namespace vbm {
namespace {

enum RowSource { kPlainRows, kGluRows, kNormRows };

struct RowArgs {
    const void * x, * up;              // up: the GLU's other half
    int64_t x_stride, up_stride;       // elements
    const void * residual;             // or null
    void * sum;                        // or null
    int64_t residual_stride;           // of both
    const float * weight;              // [k] or null
    float eps;
    int activation;
    float alpha, limit;
    void * y;                          // or null
    int y_type, code_type;
    uint8_t * codes;                   // or null
    float * scales;
    int64_t n_rows;
    int k, kb;
    bool vec_x, vec_up, vec_residual, vec_weight, vec_y;   // rows aligned to 16 bytes
};

template <int TYPE>
__device__ __forceinline__ void load_values(bool vec, const void * p, int64_t e0, float v[8]) {
    if (vec) load8<TYPE, true>(p, e0, v);
    else load8<TYPE, false>(p, e0, v);
}

__device__ __forceinline__ uint32_t bits_of(int type, float v) {
    return type == VBM_TYPE_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)) : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
// Eight values to a row of `type` from element e0 on.
__device__ __forceinline__ void store_values(int type, bool vec, void * p, int64_t e0, const float v[8]) {
    if (type == VBM_TYPE_F32) {
        float * y = static_cast<float *>(p) + e0;
        if (vec) {
            reinterpret_cast<float4 *>(y)[0] = float4{v[0], v[1], v[2], v[3]};
            reinterpret_cast<float4 *>(y)[1] = float4{v[4], v[5], v[6], v[7]};
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[i];
        return;
    }
    uint16_t * y = static_cast<uint16_t *>(p) + e0;
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = bits_of(type, v[i]);
    if (vec) {
        *reinterpret_cast<u32x4q *>(y) = u32x4q{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = static_cast<uint16_t>(h[i]);
}

// Sum or maximum over the W waves of a row, the same in all of them. `place`: W words of LDS.
struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct MaxBits {                       // of non-negative numbers' bits, which order as the numbers do, NaNs above all
    __device__ __forceinline__ float operator()(float a, float b) const {
        return __builtin_bit_cast(uint32_t, a) > __builtin_bit_cast(uint32_t, b) ? a : b;
    }
};
template <int W, class F>
__device__ __forceinline__ float over_row(float v, float * place, const F & f) {
    v = f(v, dpp_move<0xB1>(v));
    v = f(v, dpp_move<0x4E>(v));
    v = f(v, dpp_move<0x141>(v));
    v = f(v, dpp_move<0x140>(v));
    auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
    v = f(f(row(0), row(16)), f(row(32), row(48)));
    if constexpr (W > 1) {
        place[threadIdx.x >> 6] = v;   // (all lanes the same word)
        __syncthreads();
        v = place[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = f(v, place[w]);
    }
    return v;
}

// W waves take a row, CHUNKS times eight values a lane; workgroups of at least four waves.
template <int TYPE, int SOURCE, int W, int CHUNKS>
__global__ __launch_bounds__(W < 4 ? 256 : W * 64) void rows_kernel(RowArgs A) {
    constexpr int ROWS = W < 4 ? 4 / W : 1, LANES = W * 64;
    __shared__ float exchange[2][ROWS][W];
    const int sub = ROWS == 1 ? 0 : static_cast<int>(threadIdx.x) / LANES, lane = static_cast<int>(threadIdx.x) % LANES;
    for (int64_t row0 = blockIdx.x * static_cast<int64_t>(ROWS); row0 < A.n_rows; row0 += gridDim.x * static_cast<int64_t>(ROWS)) {
        const int64_t row = row0 + sub;
        if (W == 1 && row >= A.n_rows) return;          // (rows of one wave meet at no barrier)
        float v[CHUNKS][8];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int e0 = (c * LANES + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
            if (e0 < A.k) load_values<TYPE>(A.vec_x, A.x, row * A.x_stride + e0, v[c]);
        }
        if constexpr (SOURCE == kGluRows) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int e0 = (c * LANES + lane) * 8;
                if (e0 >= A.k) continue;
                float u[8];
                load_values<TYPE>(A.vec_up, A.up, row * A.up_stride + e0, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = glu_value(A.activation, v[c][i], u[i], A.alpha, A.limit);
            }
        }
        if constexpr (SOURCE == kNormRows) {
            float squares = 0.0f;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int e0 = (c * LANES + lane) * 8;
                if (e0 < A.k && A.residual) {
                    float r[8];
                    load_values<TYPE>(A.vec_residual, A.residual, row * A.residual_stride + e0, r);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[c][i] += r[i];
                        if constexpr (TYPE == VBM_TYPE_F16) v[c][i] = static_cast<float>(static_cast<_Float16>(v[c][i]));
                        if constexpr (TYPE == VBM_TYPE_BF16) v[c][i] = static_cast<float>(static_cast<__bf16>(v[c][i]));
                    }
                    if (A.sum) store_values(TYPE, A.vec_residual, A.sum, row * A.residual_stride + e0, v[c]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) squares = __builtin_fmaf(v[c][i], v[c][i], squares);
            }
            squares = over_row<W>(squares, exchange[0][sub], Add{});
            float inverse = 1.0f / sqrtf(squares / static_cast<float>(A.k) + A.eps);
            if (!(squares < INFINITY)) inverse = __builtin_nanf("");
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int e0 = (c * LANES + lane) * 8;
                if (e0 >= A.k) continue;
                float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
                if (A.weight) load_values<VBM_TYPE_F32>(A.vec_weight, A.weight, e0, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * inverse * w[i];
                if (A.y) store_values(A.y_type, A.vec_y, A.y, row * A.k + e0, v[c]);
            }
        }
        if (SOURCE == kNormRows && A.code_type == VBM_TYPE_F8_E4M3) {
            if (A.codes) {
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    const int e0 = (c * LANES + lane) * 8;
                    // (sixteen lanes share a run; those of a run that has begun before the row's end all take part)
                    if ((e0 & ~127) < A.k) store_block(v[c], e0 < A.k, A.codes + row * A.k + e0, A.scales + row * A.kb + (e0 >> 7));
                }
            }
        } else if (SOURCE != kNormRows || A.codes) {
            uint32_t m = 0;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t b = __builtin_bit_cast(uint32_t, v[c][i]) & 0x7FFFFFFFu;
                    m = b > m ? b : m;
                }
            const float most = over_row<W>(__builtin_bit_cast(float, m), exchange[1][sub], MaxBits{});
            const bool finite = __builtin_bit_cast(uint32_t, most) < 0x7F800000u;
            const float a = fmaxf(most, 0x1p-116f), a128 = a * 0x1p-7f, r = 1.0f / a128;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int e0 = (c * LANES + lane) * 8;
                if (e0 >= A.k) continue;
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[c][i] * 0.9921875f, p = x * r;
                    const float q = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-p, a128, x), r, p));
                    w[i >> 2] |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu) << (8 * (i & 3));
                }
                *reinterpret_cast<u32x2q *>(A.codes + row * A.k + e0) = finite ? u32x2q{w[0], w[1]} : u32x2q{0, 0};
            }
            if (lane == 0) A.scales[row] = finite ? a / 127.0f : __builtin_nanf("");
        }
        if constexpr (W > 1) __syncthreads();           // the next row's exchange takes the same words
    }
}

constexpr int64_t kMostRowValues = 65536;

template <int SOURCE>
void launch_rows(int type, const RowArgs & a, hipStream_t stream) {
    if (a.n_rows == 0) return;
    auto go = [&](auto type_c, auto waves_c, auto chunks_c) {
        constexpr int TYPE = decltype(type_c)::value, W = decltype(waves_c)::value, CHUNKS = decltype(chunks_c)::value;
        constexpr int ROWS = W < 4 ? 4 / W : 1;
        const int64_t groups = (a.n_rows + ROWS - 1) / ROWS;
        hipLaunchKernelGGL((rows_kernel<TYPE, SOURCE, W, CHUNKS>), dim3(static_cast<unsigned>(groups < (1 << 20) ? groups : 1 << 20)),
                           dim3(W < 4 ? 256 : W * 64), 0, stream, a);
        check_hip(hipGetLastError(), "row kernel launch");
    };
    // A few rows are latency, and more waves a row shorten it: one of 2880 with its norm 3.2 us by eight waves, 3.7 by four; many are bandwidth: 8192
    // of 4096 64 and 59.
    const bool few = a.n_rows <= 512;
    auto shape = [&](auto type_c) {
        using std::integral_constant;
        if (a.k <= 512) go(type_c, integral_constant<int, 1>{}, integral_constant<int, 1>{});
        else if (a.k <= 2048) go(type_c, integral_constant<int, 4>{}, integral_constant<int, 1>{});
        else if (a.k <= 4096 && few) go(type_c, integral_constant<int, 8>{}, integral_constant<int, 1>{});
        else if (a.k <= 4096) go(type_c, integral_constant<int, 4>{}, integral_constant<int, 2>{});
        else if (a.k <= 8192 && few) go(type_c, integral_constant<int, 16>{}, integral_constant<int, 1>{});
        else if (a.k <= 8192) go(type_c, integral_constant<int, 8>{}, integral_constant<int, 2>{});
        else if (a.k <= 16384) go(type_c, integral_constant<int, 16>{}, integral_constant<int, 2>{});
        else go(type_c, integral_constant<int, 16>{}, integral_constant<int, 8>{});
    };
    if (type == VBM_TYPE_F32) shape(std::integral_constant<int, VBM_TYPE_F32>{});
    else if (type == VBM_TYPE_F16) shape(std::integral_constant<int, VBM_TYPE_F16>{});
    else shape(std::integral_constant<int, VBM_TYPE_BF16>{});
}

bool at(const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t type_size(int type) { return type == VBM_TYPE_F32 ? 4 : 2; }
bool rows_aligned(int type, const void * p, int64_t stride) { return at(p, 16) && static_cast<size_t>(stride) * type_size(type) % 16 == 0; }
void require_type(int type, const char * what) {
    require(type == VBM_TYPE_F32 || type == VBM_TYPE_F16 || type == VBM_TYPE_BF16, std::string(what) + " must be F32, F16 or BF16");
}
void require_rows(int type, const void * p, int64_t stride, int64_t n_rows, int64_t k, const char * what) {
    require(n_rows == 0 || p, "null buffer");
    require(stride >= k && stride < (int64_t{1} << 40), "rows must be at least k elements apart");
    require(at(p, type_size(type)), std::string(what) + " must be aligned to its type");
}

RowArgs row_args(int64_t n_rows, int64_t k, int code_type, void * codes, float * scales) {
    require(k > 0 && k % 16 == 0 && k <= kMostRowValues, "k must be a positive multiple of 16, at most 65536");
    require(n_rows >= 0 && n_rows < (int64_t{1} << 31), "n_rows out of range");
    require(at(codes, 16) && at(scales, 4), "codes must be 16-byte and scales 4-byte aligned");
    RowArgs a{};
    a.code_type = code_type;
    a.codes = static_cast<uint8_t *>(codes);
    a.scales = scales;
    a.n_rows = n_rows;
    a.k = static_cast<int>(k);
    a.kb = static_cast<int>((k + 127) / 128);
    return a;
}

}  // namespace
}  // namespace vbm

using namespace vbm;

extern "C" {

vbm_status vbm_quantize_i8(int x_type, const void * x, int64_t n_rows, int64_t k, int64_t x_stride, void * codes, float * scales,
                           void * stream) {
    return guarded([&] {
        require_type(x_type, "x");
        RowArgs a = row_args(n_rows, k, VBM_TYPE_I8, codes, scales);
        require(n_rows == 0 || (codes && scales), "null buffer");
        require_rows(x_type, x, x_stride, n_rows, k, "x");
        a.x = x;
        a.x_stride = x_stride;
        a.vec_x = rows_aligned(x_type, x, x_stride);
        launch_rows<kPlainRows>(x_type, a, as_stream(stream));
    });
}

vbm_status vbm_glu_quantize_i8(int activation, int x_type, const void * gate, const void * up, int64_t n_rows, int64_t width,
                               int64_t gate_stride, int64_t up_stride, float alpha, float limit, void * codes, float * scales,
                               void * stream) {
    return guarded([&] {
        require(activation == VBM_ACT_SILU || activation == VBM_ACT_SWIGLU_OAI, "unknown activation");
        require_type(x_type, "gate and up");
        RowArgs a = row_args(n_rows, width, VBM_TYPE_I8, codes, scales);
        require(n_rows == 0 || (codes && scales), "null buffer");
        require_rows(x_type, gate, gate_stride, n_rows, width, "gate");
        require_rows(x_type, up, up_stride, n_rows, width, "up");
        a.x = gate;
        a.up = up;
        a.x_stride = gate_stride;
        a.up_stride = up_stride;
        a.activation = activation;
        a.alpha = alpha;
        a.limit = limit;
        a.vec_x = rows_aligned(x_type, gate, gate_stride);
        a.vec_up = rows_aligned(x_type, up, up_stride);
        launch_rows<kGluRows>(x_type, a, as_stream(stream));
    });
}

vbm_status vbm_add_rms_norm_quantize(int x_type, const void * x, int64_t x_stride, const void * residual, void * sum,
                                     int64_t residual_stride, const float * weight, int64_t n_rows, int64_t k, float eps, int y_type,
                                     void * y, int code_type, void * codes, float * scales, void * stream) {
    return guarded([&] {
        require_type(x_type, "x");
        require(eps > 0.0f && eps < INFINITY, "eps must be positive");
        RowArgs a = row_args(n_rows, k, code_type, codes, scales);
        require_rows(x_type, x, x_stride, n_rows, k, "x");
        if (residual) {
            require_rows(x_type, residual, residual_stride, n_rows, k, "residual");
            require(at(sum, type_size(x_type)), "sum must be aligned to its type");
            // (each row is read before its sum is stored, but not before another row's is)
            require(sum != x || x_stride == residual_stride || n_rows <= 1, "sum may be x's buffer only with the same stride");
        } else {
            require(!sum, "there is no sum without a residual");
        }
        require(at(weight, 4), "weight must be aligned to its type");
        require(y || codes || n_rows == 0, "neither y nor codes are asked for");
        if (y) {
            require_type(y_type, "y");
            require(at(y, type_size(y_type)), "y must be aligned to its type");
        }
        if (codes) {
            require(code_type == VBM_TYPE_F8_E4M3 || code_type == VBM_TYPE_I8, "codes must be F8_E4M3 or I8");
            require(scales, "null buffer");
        }
        a.x = x;
        a.x_stride = x_stride;
        a.residual = residual;
        a.sum = sum;
        a.residual_stride = residual_stride;
        a.weight = weight;
        a.eps = eps;
        a.y = y;
        a.y_type = y_type;
        a.vec_x = rows_aligned(x_type, x, x_stride);
        a.vec_residual = rows_aligned(x_type, residual, residual_stride) && at(sum, 16);
        a.vec_weight = at(weight, 16);
        a.vec_y = at(y, 16);
        launch_rows<kNormRows>(x_type, a, as_stream(stream));
    });
}

}  // extern "C"
