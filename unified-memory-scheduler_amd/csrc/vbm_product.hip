// Products of weight matrices with token rows, dense or grouped by expert: FP8 (e4m3) weights with one fp32 scale per
// 128 x 128 block and activations with one per 128 values of a row, or fp16 / bf16 weights and activations.
//
//   FP8:    dst[t][n] = sum over blocks kb of ws[n / 128][kb] * bs[t][kb] * (sum over the block's k of w[n][k] b[t][k])
//   16-bit: dst[t][n] = sum over k of w[n][k] b[t][k]
//
// plus a bias. Everything is laid out along k, so the kernels see rows of bytes and take 128 of them a step: one FP8 scale
// block, or 64 16-bit values. As a matrix operand lane (q, r) = (lane / 16, lane % 16) holds 32 of row r's 128 bytes; which ones
// does not matter as long as both operands agree. The weights are the A operand and the tokens B, so that a lane's four results
// are four neighbouring outputs of one token.
#include <algorithm>
#include <type_traits>

#include "vbm_device.hpp"
#include "vbm_internal.hpp"
#include "vbm_product_rule.hpp"

namespace vbm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4p __attribute__((ext_vector_type(4)));
typedef unsigned u32x2p __attribute__((ext_vector_type(2)));
typedef _Float16 half8_p __attribute__((ext_vector_type(8)));
typedef _Float16 half2_p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_p __attribute__((ext_vector_type(8)));

struct ProductArgs {
    const uint8_t * w;             // [n_groups][rows][k_bytes]
    const float * ws;              // [n_groups][ceil(rows / 128)][kb], FP8 only
    const float * bias;            // [n_groups][rows] or null
    const uint8_t * b;             // [n_b][k_bytes]
    const float * bs;              // [n_b][kb], FP8 only
    int64_t n_b;
    const int32_t * b_rows;        // grouped row -> b row times b_div, or null (b row = grouped row)
    int64_t b_div;
    const int32_t * offsets;       // [n_groups + 1] or null (one group of n_rows)
    int64_t n_rows;
    const int32_t * dst_rows;      // grouped row -> dst row, or null
    int64_t n_dst;
    void * dst;
    int dst_type;
    int dst_vec, dst_vec16;        // four neighbouring outputs, or 16 bytes of them, can be stored at once
    int n_groups, rows, k_bytes, kb;
};

__device__ __forceinline__ int wave_inclusive_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row 0's last to row 1, row 2's to row 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // lane 31's to the upper half
    return v;
}

// The groups' bounds, 64 groups a pass, lane by lane; those of the first passes stay in registers, so that their loads are on
// their way together. Offsets are bounded to [0, n_rows]: bad ones cannot lead out of the buffers. (n_rows < 2^29, so that the tiles
// of a pass of 64 groups that all span it, 32 rows a tile, are counted in 31 bits; tiles of fewer rows are for far fewer rows. A place
// is looked for pass by pass, and found before the sum of the passes could leave them.)
struct Groups {
    static constexpr int KEPT = 4;
    const ProductArgs & A;
    int lo[KEPT], hi[KEPT];
    __device__ __forceinline__ explicit Groups(const ProductArgs & args) : A(args) {
#pragma unroll
        for (int c = 0; c < KEPT; ++c) load(64 * c, lo[c], hi[c]);
    }
    __device__ __forceinline__ void load(int g0, int & l, int & h) const {
        const int g = g0 + static_cast<int>(threadIdx.x & 63), n = static_cast<int>(A.n_rows);
        auto bounded = [&](int v) { return v < 0 ? 0 : (v > n ? n : v); };
        l = g < A.n_groups ? bounded(A.offsets[g]) : 0;
        h = g < A.n_groups ? bounded(A.offsets[g + 1]) : 0;
    }
    // Calls f(g0, lo, hi) pass by pass, until it returns true.
    template <class F>
    __device__ __forceinline__ void each(F && f) const {
        bool done = false;
#pragma unroll
        for (int c = 0; c < KEPT; ++c)
            if (!done && 64 * c < A.n_groups) done = f(64 * c, lo[c], hi[c]);
        for (int g0 = 64 * KEPT; !done && g0 < A.n_groups; g0 += 64) {
            int l, h;
            load(g0, l, h);
            done = f(g0, l, h);
        }
    }
};
// Of tiles in group order, `t` of them in this lane's group of a pass: whether number `index` is in this pass, and its group's
// lane, number of tiles and the tiles before it. `sum`: the tiles of earlier passes, brought up to date.
struct Place {
    int lane, tiles, before;
};
__device__ __forceinline__ bool find_place(int t, int index, int & sum, Place & p) {
    const int incl = sum + wave_inclusive_sum(t);
    const uint64_t past = __ballot(incl > index);
    sum = __builtin_amdgcn_readlane(incl, 63);
    if (!past) return false;
    p.lane = __builtin_ctzll(past);
    p.tiles = __builtin_amdgcn_readlane(t, p.lane);
    p.before = __builtin_amdgcn_readlane(incl, p.lane) - p.tiles;
    return true;
}

struct TokenTile {
    int group;
    int64_t first, last;           // grouped rows [first, last)
};

// The group and rows of token tile `index`, tiles of `tile_rows` in group order; false past the last one. Every wave finds it
// from the offsets by itself (the host does not know the groups' sizes, and a launch that wrote the list would cost more).
__device__ __forceinline__ bool find_token_tile(const ProductArgs & A, int index, int tile_rows, TokenTile & t) {
    if (!A.offsets) {
        t.group = 0;
        t.first = static_cast<int64_t>(index) * tile_rows;
        t.last = t.first + tile_rows < A.n_rows ? t.first + tile_rows : A.n_rows;
        return t.first < A.n_rows;
    }
    const Groups groups(A);
    int sum = 0;
    bool found = false;
    groups.each([&](int g0, int lo, int hi) {
        Place p;
        if (!find_place(hi > lo ? (hi - lo + tile_rows - 1) / tile_rows : 0, index, sum, p)) return false;
        const int start = __builtin_amdgcn_readlane(lo, p.lane) + (index - p.before) * tile_rows, end = __builtin_amdgcn_readlane(hi, p.lane);
        t.group = g0 + p.lane;
        t.first = start;
        t.last = start + tile_rows < end ? start + tile_rows : end;
        return found = true;
    });
    return found;
}

// Grouped row i's row of b; -1: none (its outputs are NaN).
__device__ __forceinline__ int64_t source_row(const ProductArgs & A, int64_t i) {
    if (!A.b_rows) return i < A.n_b ? i : -1;
    const int64_t v = A.b_rows[i];
    if (v < 0) return -1;
    const int64_t row = static_cast<uint32_t>(v) / static_cast<uint32_t>(A.b_div);
    return row < A.n_b ? row : -1;
}
// Its place in dst; -1: not written.
__device__ __forceinline__ int64_t target_row(const ProductArgs & A, int64_t i) {
    const int64_t row = A.dst_rows ? A.dst_rows[i] : i;
    return row >= 0 && row < A.n_dst ? row : -1;
}

// A lane's 32 bytes of a step.
struct Piece {
    u32x4p lo, hi;
};

__device__ __forceinline__ uint16_t to_16(int type, float v) {
    return type == VBM_TYPE_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)) : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Outputs n .. n + 3 of one dst row.
__device__ __forceinline__ void store4(const ProductArgs & A, int64_t row, int n, f32x4 v) {
    const int64_t at = row * A.rows + n;
    if (A.dst_type == VBM_TYPE_F32) {
        float * p = static_cast<float *>(A.dst) + at;
        if (A.dst_vec && n + 4 <= A.rows) {
            *reinterpret_cast<f32x4 *>(p) = v;
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < A.rows) p[i] = v[i];
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = to_16(A.dst_type, v[i]);
    uint16_t * p = static_cast<uint16_t *>(A.dst) + at;
    if (A.dst_vec && n + 4 <= A.rows) {
        *reinterpret_cast<u32x2p *>(p) = u32x2p{h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < A.rows) p[i] = h[i];
}

__device__ __forceinline__ half8_p widened(unsigned a, unsigned b) {
    const half2_p p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const half2_p p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return half8_p{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// A piece as matrix operands, and the product of two of them added to c.
template <int KIND>
struct Operand {
    static constexpr int N = KIND == kF8 ? 1 : (KIND == kF8Wide ? 4 : 2);
    using T = std::conditional_t<KIND == kF8, i32x8, std::conditional_t<KIND == kBF16, bf16x8_p, half8_p>>;
    T v[N];
    __device__ __forceinline__ void take(const Piece & p) {
        if constexpr (KIND == kF8) {
            v[0] = __builtin_bit_cast(i32x8, p);
        } else if constexpr (KIND == kF8Wide) {
            v[0] = widened(p.lo.x, p.lo.y), v[1] = widened(p.lo.z, p.lo.w);
            v[2] = widened(p.hi.x, p.hi.y), v[3] = widened(p.hi.z, p.hi.w);
        } else {
            v[0] = __builtin_bit_cast(T, p.lo), v[1] = __builtin_bit_cast(T, p.hi);
        }
    }
};
template <int KIND>
__device__ __forceinline__ f32x4 product(const Operand<KIND> & a, const Operand<KIND> & b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < Operand<KIND>::N; ++i) {
        if constexpr (KIND == kF8) c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v[i], b.v[i], c, 0, 0, 0, 0, 0, 0);
        else if constexpr (KIND == kBF16) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
        else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], c, 0, 0, 0);
    }
    return c;
}

// Loads from memory to LDS (lane l's bytes land at m0 + l * size), in inline assembly so that the compiler does not wait for
// all of them before every LDS read; the kernel waits itself before each barrier. The compiler knows of no other use of
// M0 here, and the wait state between a scalar write of M0 and the load that reads it is written out.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds_16(const void * src, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds_16(const void * base, uint32_t offset, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(base), "v"(offset), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds_4(const void * src, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(m0) : "memory", "m0");
}
// By all lanes (`all` -1) or by lane 0 alone (0), which the waits count alike; all lanes are active where it is called.
__device__ __forceinline__ void load_to_lds_4(const void * src, uint32_t m0, int all) {
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dword %0, off\n\ts_mov_b64 exec, -1" ::"v"(src), "s"(m0), "s"(all | 1), "s"(all) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until all but the wave's newest N loads have landed and its LDS reads are done, then for the workgroup's other waves.
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// All but the wave's newest N loads have landed, and its LDS reads are done.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// The last steps of a ring, at most LEFT + 1 of them, with P loads each on their way.
template <int LEFT, int P, class F>
__device__ __forceinline__ void drain(int i, int n, const F & compute) {
    if (n - i > LEFT) {
        landed<LEFT * P>();
        compute(i);
        ++i;
    }
    if constexpr (LEFT > 0) drain<LEFT - 1, P>(i, n, compute);
}

// ------------------------------------------------------------------------------- few tokens a group
// A workgroup takes 16 weight rows x up to 8 * MAX8 tokens (MAX8: 1 or 2) of one group; its W waves share the depth in runs and add their
// sums up through LDS, in wave order. The weights' bytes are the work, and they are read once; what counts is that enough of them
// are on their way. Each wave streams its own through a ring of D steps in LDS, without barriers: a load brings 128
// bytes of each of eight rows, in neighbouring lanes (loaded straight into a matrix operand's registers, 16 rows in neighbouring lanes,
// a kilobyte occupies the address unit for 64 cycles instead of 18, which alone limits a CU to 16 bytes a cycle).
// One token through eight FP8 experts of 1536 x 2048: 9.2 us (7.1 from the caches), of which the 25 MB take 5 at the rate of a large
// copy; one token through one matrix of 5760 x 2880: 6.3 us, latency: bounds and rows, the weights, the waves' sums. Deep rows of many
// experts (64 tokens top-4 over 32 experts, FP8 2880 x 7168 118 us, bf16 2880 x 4096 127) are read at 5.6 to 5.9 TB/s.
template <int KIND, int MAX8, int D>
__global__ __launch_bounds__(256) void few_rows_kernel(ProductArgs A, int row_tiles) {
    static_assert(MAX8 <= 2, "one column of sixteen tokens");
    constexpr int W = 4, RUN = 16;                           // RUN: steps whose scales a wave holds
    constexpr int STEP = (2 + MAX8) * 1024, SCALES = is_f8(KIND) ? RUN * 64 : 0, WAVE = D * STEP + SCALES;
    static_assert(1024 <= WAVE, "the ring's memory holds the waves' sums");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * WAVE];
    TokenTile t;
    const int token_tile = static_cast<int>(blockIdx.x) / row_tiles, n0 = (static_cast<int>(blockIdx.x) - token_tile * row_tiles) * 16;
    if (!find_token_tile(A, token_tile, 8 * MAX8, t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int q = lane >> 4, r = lane & 15, live = static_cast<int>(t.last - t.first);
    uint8_t * mine = lds + wave * WAVE;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(mine));
    auto token_row = [&](int i) __attribute__((always_inline)) {   // spare tokens repeat the first one, unknown ones read row 0
        const int64_t src = source_row(A, t.first + (i < live ? i : 0));
        return src < 0 ? 0 : src;
    };

    const uint8_t * wbase = A.w + (static_cast<int64_t>(t.group) * A.rows + n0) * A.k_bytes;
    uint32_t wsrc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int n = n0 + 8 * i + (lane >> 3);
        wsrc[i] = static_cast<uint32_t>((n < A.rows ? n : A.rows - 1) - n0) * static_cast<uint32_t>(A.k_bytes);
    }
    const float * wscale = is_f8(KIND) ? A.ws + (static_cast<int64_t>(t.group) * ((A.rows + 127) >> 7) + (n0 >> 7)) * A.kb : nullptr;
    const int k_begin = A.kb * wave / W, k_end = A.kb * (wave + 1) / W;

    auto run = [&](auto t8_c) __attribute__((always_inline)) {
        constexpr int T8 = decltype(t8_c)::value, P = 2 + T8;   // P: loads a step
        const uint8_t * tsrc[T8];
#pragma unroll
        for (int i = 0; i < T8; ++i) tsrc[i] = A.b + token_row(8 * i + (lane >> 3)) * A.k_bytes;
        const float * ssrc = is_f8(KIND) ? A.bs + token_row(lane >> 2) * A.kb : nullptr;
        // piece lane % 8 of a row sits at its place xor (row / 2 % 8), as in the kernels below
        const int piece_even = (lane & 7) ^ (lane >> 4), piece_odd = piece_even ^ 4;
        f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};

        for (int k0 = k_begin; k0 < k_end; k0 += RUN) {
            const int n_steps = k_end - k0 < RUN ? k_end - k0 : RUN;
            float scales = 0.0f;                             // lane l: the weights' scale of step k0 + l
            if constexpr (is_f8(KIND)) {
                scales = lane < n_steps ? wscale[k0 + lane] : 0.0f;
                asm volatile("" : "+v"(scales));
                // the tokens' scales, four steps of sixteen tokens a load: [four steps][token][4]
                for (int c = 0; c < (n_steps + 3) / 4; ++c) {
                    const int k = k0 + 4 * c + (lane & 3);
                    load_to_lds_4(ssrc + (k < A.kb ? k : A.kb - 1), lds0 + D * STEP + c * 256);
                }
            }
            auto issue = [&](int i) __attribute__((always_inline)) {
                const int k = k0 + i;
                const int64_t off = static_cast<int64_t>(k) * 128;
                const uint32_t at = lds0 + (i % D) * STEP;
                // (a piece past the row's end reads the step's first one: zeros take its place in the registers)
                const int even = k * 128 + piece_even * 16 < A.k_bytes ? piece_even * 16 : 0, odd = k * 128 + piece_odd * 16 < A.k_bytes ? piece_odd * 16 : 0;
#pragma unroll
                for (int l = 0; l < 2; ++l) load_to_lds_16(wbase + off, wsrc[l] + (l & 1 ? odd : even), at + l * 1024);
#pragma unroll
                for (int l = 0; l < T8; ++l) load_to_lds_16(tsrc[l] + off + (l & 1 ? odd : even), at + (2 + l) * 1024);
            };
            auto compute = [&](int i) __attribute__((always_inline)) {
                const uint8_t * stage = mine + (i % D) * STEP;
                const int left = A.k_bytes - (k0 + i) * 128 - 32 * q;   // bytes of the row from this lane's pieces on
                auto operand = [&](const uint8_t * rows, int rr) __attribute__((always_inline)) {
                    const uint8_t * p = rows + rr * 128;
                    Piece v{*reinterpret_cast<const u32x4p *>(p + ((2 * q) ^ (rr >> 1)) * 16), *reinterpret_cast<const u32x4p *>(p + ((2 * q + 1) ^ (rr >> 1)) * 16)};
                    if (left < 32) {
                        if (left <= 16) v.hi = u32x4p{0, 0, 0, 0};
                        if (left <= 0) v.lo = u32x4p{0, 0, 0, 0};
                    }
                    Operand<KIND> o;
                    o.take(v);
                    return o;
                };
                // (of eight tokens rows 8 .. 15 read rows 0 .. 7: their columns are not used)
                const Operand<KIND> a = operand(stage, r), b = operand(stage + 2048, T8 == 1 ? r & 7 : r);
                if constexpr (is_f8(KIND)) {
                    const float sw = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scales), i));
                    const float f = sw * *reinterpret_cast<const float *>(mine + D * STEP + (i >> 2) * 256 + r * 16 + (i & 3) * 4);
                    const f32x4 p = product<KIND>(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(p[e], f, acc[e]);
                } else {
                    acc = product<KIND>(a, b, acc);
                }
            };
            for (int i = 0; i < D && i < n_steps; ++i) issue(i);
            int i = 0;
            for (; i + D < n_steps; ++i) {
                landed<(D - 1) * P>();
                compute(i);
                landed<(D - 1) * P>();                       // (its reads are done: the wait covers them too)
                issue(i + D);
            }
            drain<D - 1, P>(i, n_steps, compute);
            landed<0>();                                     // (the next run's loads take the places of this one's last reads)
        }
        __syncthreads();                                     // the rings are free: the waves' sums go there
        f32x4 * parts = reinterpret_cast<f32x4 *>(lds);      // [wave][lane]
        parts[wave * 64 + lane] = acc;
        __syncthreads();
        if (wave) return;
        f32x4 v = parts[lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += parts[w * 64 + lane];
        const int n = n0 + 4 * q;
        const int64_t i = t.first + r;
        if (i >= t.last || n >= A.rows) return;
        const int64_t row = target_row(A, i);
        if (row < 0) return;
        if (A.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < A.rows) v[e] += A.bias[static_cast<int64_t>(t.group) * A.rows + n + e];
        }
        const float nan = __builtin_nanf("");
        store4(A, row, n, source_row(A, i) < 0 ? f32x4{nan, nan, nan, nan} : v);
    };
    if constexpr (MAX8 == 2) {
        if (live > 8) return run(std::integral_constant<int, 2>{});
    }
    run(std::integral_constant<int, 1>{});
}

// The same where there are rows enough to keep the card busy with one wave a row tile: the tokens, of all of the depth, are staged in LDS
// once and shared by the workgroup's W waves; then each wave streams `tiles` row tiles of 16 rows, one after the other through
// a ring of D steps, with no barrier and no sums to join. 64 tokens top-4 over 32 FP8 experts of 5760 x 2880, fp32 outputs: 106 us,
// 5.05 TB/s (a large copy reaches 5.1); with the depth shared among the waves (the kernel above) 135. 16 tokens top-4 over 32 bf16 experts of 2880 x
// 2880: 82 us, 5.7 TB/s. Bound by memory.
template <int KIND, int MAX8, int W, int D>
__global__ __launch_bounds__(W * 64) void stream_rows_kernel(ProductArgs A, int row_units, int tiles) {
    using L = StreamLayout<KIND, MAX8, W, D>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[L::TOTAL];
    TokenTile t;
    const int token_tile = static_cast<int>(blockIdx.x) / row_units, unit = static_cast<int>(blockIdx.x) - token_tile * row_units;
    if (!find_token_tile(A, token_tile, 8 * MAX8, t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int q = lane >> 4, r = lane & 15, live = static_cast<int>(t.last - t.first), eights = (live + 7) >> 3;
    const int n0 = unit * (W * 16) * tiles, row_tiles = (A.rows + 15) >> 4;
    const int first_tile = (n0 >> 4) + wave;                 // this wave's: first_tile + W i
    const int my_tiles = first_tile >= row_tiles ? 0 : ((row_tiles - first_tile + W - 1) / W < tiles ? (row_tiles - first_tile + W - 1) / W : tiles);
    const uint8_t * weights = A.w + static_cast<int64_t>(t.group) * A.rows * A.k_bytes;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)), ring0 = lds0 + wave * (D * 2048);
    const int piece_even = (lane & 7) ^ (lane >> 4), piece_odd = piece_even ^ 4;

    // the weights' steps, in order over the wave's tiles: the next one to load is step kb_next of tile tile_next (the last one again past the end)
    int tile_next = 0, kb_next = 0, slot_next = 0;
    const uint8_t * base = nullptr;
    uint32_t wsrc[2];
    auto enter_tile = [&](int i) __attribute__((always_inline)) {
        const int n = (first_tile + W * i) * 16;
        base = weights + static_cast<int64_t>(n) * A.k_bytes;
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            const int row = 8 * l + (lane >> 3);
            wsrc[l] = static_cast<uint32_t>(n + row < A.rows ? row : A.rows - 1 - n) * static_cast<uint32_t>(A.k_bytes);
        }
    };
    auto issue = [&]() __attribute__((always_inline)) {
        const int64_t off = static_cast<int64_t>(kb_next) * 128;
        // (a piece past the row's end reads the step's first one: zeros take its place in the registers)
        const int even = kb_next * 128 + piece_even * 16 < A.k_bytes ? piece_even * 16 : 0, odd = kb_next * 128 + piece_odd * 16 < A.k_bytes ? piece_odd * 16 : 0;
        load_to_lds_16(base + off, wsrc[0] + even, ring0 + slot_next * 2048);
        load_to_lds_16(base + off, wsrc[1] + odd, ring0 + slot_next * 2048 + 1024);
        slot_next = slot_next + 1 == D ? 0 : slot_next + 1;
        if (kb_next + 1 < A.kb) {
            ++kb_next;
        } else if (tile_next + 1 < my_tiles) {
            kb_next = 0;
            enter_tile(++tile_next);
        }
    };
    if (my_tiles) {
        enter_tile(0);
#pragma unroll
        for (int i = 0; i < D; ++i) issue();
    }

    // the tokens: [eight tokens][step] x 1 KB, place as for the weights; scales [four steps][token][4]
    auto token_row = [&](int i) __attribute__((always_inline)) {   // spare tokens repeat the first one, unknown ones read row 0
        const int64_t src = source_row(A, t.first + (i < live ? i : 0));
        return src < 0 ? 0 : src;
    };
    for (int e = 0; e < eights; ++e) {
        const uint8_t * src = A.b + token_row(8 * e + (lane >> 3)) * A.k_bytes;
        const int piece = e & 1 ? piece_odd : piece_even;
        for (int kb = wave; kb < A.kb; kb += W) {
            const uint32_t at = L::TOKENS + (e * A.kb + kb) * 1024;
            if (kb * 128 + piece * 16 < A.k_bytes) load_to_lds_16(src + static_cast<int64_t>(kb) * 128 + piece * 16, lds0 + at);
            else *reinterpret_cast<u32x4p *>(lds + at + lane * 16) = u32x4p{0, 0, 0, 0};
        }
    }
    const int scales_at = L::TOKENS + eights * A.kb * 1024;
    const int blocks = (A.rows + 127) >> 7;
    if constexpr (is_f8(KIND)) {
        const float * src = A.bs + token_row(lane >> 2) * A.kb;
        for (int c = wave; 4 * c < A.kb; c += W) {
            const int kb = 4 * c + (lane & 3);
            load_to_lds_4(src + (kb < A.kb ? kb : A.kb - 1), lds0 + scales_at + c * 256);
        }
        for (int i = wave; i < L::BLOCKS; i += W) {
            const int block = (n0 >> 7) + i < blocks ? (n0 >> 7) + i : blocks - 1;
            load_to_lds_4(A.ws + (static_cast<int64_t>(t.group) * blocks + block) * A.kb + (lane < A.kb ? lane : A.kb - 1), lds0 + L::BLOCK_SCALES + i * 256);
        }
    }
    float * bias = reinterpret_cast<float *>(lds + L::BIAS);
    for (int i = threadIdx.x; i < W * 16 * tiles; i += W * 64)
        bias[i] = A.bias && n0 + i < A.rows ? A.bias[static_cast<int64_t>(t.group) * A.rows + n0 + i] : 0.0f;
    const int64_t mine = t.first + r, to = mine < t.last ? target_row(A, mine) : -1;   // the dst row of token r; -1: none
    const bool bad = to >= 0 && source_row(A, mine) < 0;
    landed<0>();
    __syncthreads();

    auto run = [&](auto t8_c) __attribute__((always_inline)) {
        constexpr int T8 = decltype(t8_c)::value;
        const uint8_t * ring = lds + wave * (D * 2048);
        int slot = 0;
        for (int i = 0; i < my_tiles; ++i) {
            const int n = (first_tile + W * i) * 16;
            const float * wscale = reinterpret_cast<const float *>(lds + L::BLOCK_SCALES + ((n >> 7) - (n0 >> 7)) * 256);
            f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
            for (int kb = 0; kb < A.kb; ++kb) {
                landed<(D - 1) * 2>();
                const int left = A.k_bytes - kb * 128 - 32 * q;   // bytes of the row from this lane's pieces on
                auto operand = [&](const uint8_t * rows, int rr, bool weights) __attribute__((always_inline)) {
                    const uint8_t * p = rows + rr % 8 * 128;
                    Piece v{*reinterpret_cast<const u32x4p *>(p + ((2 * q) ^ (rr >> 1)) * 16), *reinterpret_cast<const u32x4p *>(p + ((2 * q + 1) ^ (rr >> 1)) * 16)};
                    if (weights && left < 32) {
                        if (left <= 16) v.hi = u32x4p{0, 0, 0, 0};
                        if (left <= 0) v.lo = u32x4p{0, 0, 0, 0};
                    }
                    Operand<KIND> o;
                    o.take(v);
                    return o;
                };
                const Operand<KIND> a = operand(ring + slot * 2048 + (r >> 3) * 1024, r, true);
                // (of eight tokens rows 8 .. 15 read rows 0 .. 7: their columns are not used)
                const int rr = T8 == 1 ? r & 7 : r;
                const Operand<KIND> b = operand(lds + L::TOKENS + ((rr >> 3) * A.kb + kb) * 1024, rr, false);
                if constexpr (is_f8(KIND)) {
                    const f32x4 p = product<KIND>(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                    const float f = wscale[kb] * *reinterpret_cast<const float *>(lds + scales_at + (kb >> 2) * 256 + r * 16 + (kb & 3) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(p[e], f, acc[e]);
                } else {
                    acc = product<KIND>(a, b, acc);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot has been read
                issue();
                slot = slot + 1 == D ? 0 : slot + 1;
            }
            const f32x4 extra = *reinterpret_cast<const f32x4 *>(bias + (n - n0) + 4 * q);
            const float nan = __builtin_nanf("");
            if (to >= 0 && n + 4 * q < A.rows) store4(A, to, n + 4 * q, bad ? f32x4{nan, nan, nan, nan} : acc + extra);
        }
        landed<0>();                                         // no load may land after the workgroup has ended
    };
    if constexpr (MAX8 == 2) {
        if (eights > 1) return run(std::integral_constant<int, 2>{});
    }
    run(std::integral_constant<int, 1>{});
}

// ----------------------------------------------------------------------------------- many tokens
// Sixteen tokens' outputs from n on, fp32 in LDS (`row_bytes` a token), to their dst rows: PIECES of N values a token.
template <int PIECES, int N>
__device__ __forceinline__ void store_column(const ProductArgs & A, const uint8_t * from, int row_bytes, const int * rows, int n) {
    constexpr int AT_ONCE = 64 / PIECES;                     // tokens
    const int lane = threadIdx.x & 63, at = n + lane % PIECES * N;
#pragma unroll
    for (int t = lane / PIECES; t < 16; t += AT_ONCE) {
        const f32x4 * v4 = reinterpret_cast<const f32x4 *>(from + t * row_bytes + lane % PIECES * N * 4);
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v4[i / 4][i % 4];
        int64_t row = rows[t];
        if (row == -1 || at >= A.rows) continue;
        if (row < 0) {
            row = -2 - row;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __builtin_nanf("");
        }
        if constexpr (N == 4) {
            float * p = static_cast<float *>(A.dst) + row * A.rows + at;
            if (A.dst_vec16) {
                *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
                continue;
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < A.rows) p[i] = v[i];
        } else {
            uint16_t * p = static_cast<uint16_t *>(A.dst) + row * A.rows + at;
            uint16_t h[N];
            if (A.dst_type == VBM_TYPE_BF16) {
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v[i]));
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[i]));
            }
            if (A.dst_vec16) {
                u32x4p w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | static_cast<uint32_t>(h[2 * i + 1]) << 16;
                *reinterpret_cast<u32x4p *>(p) = w;
                continue;
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < A.rows) p[i] = h[i];
        }
    }
}

struct Work {
    int group, row_tile;
    int first, live;               // grouped rows
};
// The calling workgroup's share: a row tile x a token tile of at most `most` 16-token columns of one group. Workgroup i runs on XCD
// i % 8, so each XCD takes a contiguous run of the list (group by group, row tile by row tile): the token tiles that share a row
// tile's weights, and the row tiles that share the tokens, then meet in one L2. A group's tiles share its columns evenly. `launched`: the
// most token tiles that rows grouped in order can have; offsets out of order may count more, and have the first ones done.
__device__ __forceinline__ bool find_work(const ProductArgs & A, int most, int row_tiles, int launched, Work & w) {
    const int n_rows = static_cast<int>(A.n_rows), slot = static_cast<int>(blockIdx.x >> 3);
    auto columns = [&](int lo, int hi) { return hi > lo ? (hi - lo + 15) >> 4 : 0; };
    auto tiles_of = [&](int lo, int hi) { return (columns(lo, hi) + most - 1) / most; };
    int item = 0, lo = 0, hi = n_rows, tiles = 0, before = 0;
    auto mine = [&](int total) {                             // this workgroup's item of so many token tiles
        const int items = total * row_tiles, per_xcd = (items + 7) >> 3;
        item = static_cast<int>(blockIdx.x & 7) * per_xcd + slot;
        return slot < per_xcd && item < items;
    };
    w.group = 0;
    if (!A.offsets) {
        tiles = tiles_of(0, n_rows);
        if (!mine(tiles)) return false;
    } else {
        const Groups groups(A);
        int part = 0, sum = 0;
        groups.each([&](int, int l, int h) {
            part = std::min(part + tiles_of(l, h), launched);    // (below 2^24: the sum of 64 lanes is counted in 31 bits)
            return false;
        });
        if (!mine(std::min(__builtin_amdgcn_readlane(wave_inclusive_sum(part), 63), launched))) return false;
        const int index = item / row_tiles;
        groups.each([&](int g0, int l, int h) {
            Place p;
            if (!find_place(tiles_of(l, h), index, sum, p)) return false;
            w.group = g0 + p.lane;
            lo = __builtin_amdgcn_readlane(l, p.lane);
            hi = __builtin_amdgcn_readlane(h, p.lane);
            tiles = p.tiles;
            before = p.before;
            return true;
        });
        if (!tiles) return false;
    }
    const int local = item - before * row_tiles;
    w.row_tile = local / tiles;
    const int tile = local - w.row_tile * tiles, share = (columns(lo, hi) + tiles - 1) / tiles;
    w.first = lo + tile * share * 16;
    w.live = hi - w.first < share * 16 ? hi - w.first : share * 16;
    return w.live > 0;
}

// A workgroup of WN x WT waves takes BN = 16 SN WN weight rows x up to BT = 16 ST WT tokens of one group; a wave 16 SN rows x every WT-th
// 16-token column. A step's 128 bytes of every row are staged in LDS, as many stages as the live columns leave room for, with one
// wait and one barrier a step. Piece p (16 bytes) of row r lies at place p ^ (r / 2 % 8) of the row's 128 bytes: sixteen rows'
// reads of one piece then cover all banks (unswizzled they took twice as long).
//
// FP8 4096 x 4096 x 4096 with bf16 outputs: 65 to 67 us, 2.1 PFLOP/s, where a library's product without block scales reaches 2.7.
// Per step of 256 x 256 (1.75 us): the matrix instructions alone 1.0, with the fp32 sums of the scaled blocks 1.25 (an FMA per output and
// block, half of a matrix instruction's time), the LDS reads under them; the rest is the loads' issue: a wave stands still until
// the address unit has taken its kilobyte (18 cycles each, 64 of them a step), and the waves of a workgroup ask for it together.
// What was tried: all of a step's loads at once 1.78; four-wave workgroups of 256 x 128 84 us; items dealt to the XCDs in turn, not in
// runs: the same here, 5 % slower for ragged groups. Grouped prefill is bound by the weights' stream and what a workgroup
// does not overlap with it: one of them fits a CU, and its start (bounds, rows, first stages) and end cost about 8 us of some 40.
template <int KIND, int SN, int ST, int WN, int WT, int LDS>
__global__ __launch_bounds__(WN * WT * 64) void many_rows_kernel(ProductArgs A, int row_tiles, int launched) {
    constexpr int W = WN * WT, BN = 16 * SN * WN, BT = 16 * ST * WT;
    constexpr int DW = BN / 8 / W;                           // a wave's loads of weights a step: 8 rows each
    static_assert(DW * 8 * W == BN && BT % 32 == 0, "the waves share the loads");
    constexpr int STAGE_BYTES = LDS - BT * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
    Work work;
    if (!find_work(A, ST * WT, row_tiles, launched, work)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int q = lane >> 4, r = lane & 15, wn = wave / WT, wt = wave % WT;
    const int n0 = work.row_tile * BN;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));

    const uint8_t * wbase = A.w + (static_cast<int64_t>(work.group) * A.rows + n0) * A.k_bytes;
    uint32_t wsrc[DW];                                       // (rows of a tile are at most 2^32 bytes apart)
    // the piece that this lane brings of row lane / 8 of eight: place lane % 8, of rows 0 .. 7 or 8 .. 15 of sixteen (loads k = wave + W i
    // with even or odd k; W is even, so all of a wave's are alike)
    static_assert(W % 2 == 0, "a wave's loads are all of even or all of odd eights");
    const int piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
#pragma unroll
    for (int i = 0; i < DW; ++i) {
        const int n = n0 + 8 * (wave + W * i) + (lane >> 3);
        wsrc[i] = static_cast<uint32_t>((n < A.rows ? n : A.rows - 1) - n0) * static_cast<uint32_t>(A.k_bytes) + piece * 16;
    }
    auto token_row = [&](int i) __attribute__((always_inline)) {   // spare tokens repeat the first one, unknown ones read row 0
        const int64_t src = source_row(A, work.first + (i < work.live ? i : 0));
        return src < 0 ? 0 : src;
    };
    const float * wscale = nullptr;
    if constexpr (is_f8(KIND)) {
        const int block = (n0 + 16 * SN * wn) >> 7, last = (A.rows - 1) >> 7;
        wscale = A.ws + (static_cast<int64_t>(work.group) * (last + 1) + (block < last ? block : last)) * A.kb;
    }

    int * rows = reinterpret_cast<int *>(lds + STAGE_BYTES);   // the tokens' dst rows, -1: none, -2 - row: all NaN
    for (int c = threadIdx.x; c < BT; c += W * 64) {
        const int64_t i = static_cast<int64_t>(work.first) + c;
        const int row = c < work.live ? static_cast<int>(target_row(A, i)) : -1;
        rows[c] = row >= 0 && source_row(A, i) < 0 ? -2 - row : row;
    }

    const int live_cols = (work.live + 15) >> 4;
    auto run = [&](auto live_c) __attribute__((always_inline)) {
        constexpr int NT = decltype(live_c)::value;
        constexpr int EIGHTS = NT * WT * 2, LOADS = DW + (EIGHTS + W - 1) / W;   // only the live columns' tokens
        constexpr int PARTS = LOADS + (is_f8(KIND) ? 1 : 0), SCALE_WAVES = (EIGHTS + 7) / 8;
        constexpr int SCALES = (BN + 8 * EIGHTS) * 128, STAGE = SCALES + (is_f8(KIND) ? SCALE_WAVES * 256 : 0);
        constexpr int STAGES = STAGE_BYTES / STAGE < 4 ? STAGE_BYTES / STAGE : 4;
        static_assert(STAGES >= 2 && SCALE_WAVES <= W, "two stages at least");
        // Every wave issues the same number of loads, which the waits count: past the live columns it loads eight tokens that another one
        // loads too (of the same parity, so that the pieces' places agree); and the first waves bring the tokens' scales, the others
        // one of the same.
        const float * ssrc = is_f8(KIND) ? A.bs + token_row(64 * (wave % SCALE_WAVES) + lane) * A.kb : nullptr;
        const int scale_lanes = (wave - SCALE_WAVES) >> 31;
        const uint8_t * tsrc[LOADS - DW];
        int place[LOADS - DW];
#pragma unroll
        for (int i = 0; i < LOADS - DW; ++i) {
            const int eight = (wave + W * i) % EIGHTS;
            tsrc[i] = A.b + token_row(8 * eight + (lane >> 3)) * A.k_bytes + piece * 16;
            place[i] = BN * 128 + eight * 1024;
        }
        f32x4 acc[SN][NT];
#pragma unroll
        for (int s = 0; s < SN; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[s][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float scales = 0.0f;                                 // lane l: the weights' scale of step l (mod 64)
        auto fetch_scales = [&](int kb) __attribute__((always_inline)) {
            if constexpr (is_f8(KIND)) scales = kb + lane < A.kb ? wscale[kb + lane] : 0.0f;
            asm volatile("" : "+v"(scales));                 // (the wait for it here, not in every step, where it would wait for the stages too)
        };
        // Loads [begin, end) of a step's PARTS (weights, tokens, the tokens' scales) into stage `to`. A stage's loads go out a few (EACH) a
        // column, from the last column of the step that frees it on: together they would hold up the reads and products behind them, and
        // later ones would not have landed in time. (A wave of at most two columns has little to hold up and takes them together: 100 tokens,
        // 2880 rows, k 2880 9.7 us against 10.2; 500, 1536, 4096 14.2 against 15.2; 2048, 2880, 2880, a wide tile, 32.5 together against 29.5
        // apart.) Past the last step it is loaded again, for nobody, so that the waits' counts
        // hold; a piece past a row's end reads the step's first one (zeros take its place before it is used).
        constexpr int EACH = ST <= 2 ? PARTS : (PARTS + NT / 2) / (NT / 2 + 1);
        auto load_parts = [&](int to, int begin, int end) __attribute__((always_inline)) {
            const int kb = to < A.kb ? to : A.kb - 1;
            const int64_t off = static_cast<int64_t>(kb) * 128;
            const int back = kb * 128 + piece * 16 < A.k_bytes ? 0 : -16 * piece;
            const uint32_t at = lds0 + (to % STAGES) * STAGE;
#pragma unroll
            for (int i = begin; i < end; ++i) {
                if (i < DW) load_to_lds_16(wbase + off, wsrc[i < DW ? i : 0] + back, at + (wave + W * i) * 1024);
                else if (i < LOADS) load_to_lds_16(tsrc[i - DW < LOADS - DW ? i - DW : 0] + off + back, at + place[i - DW < LOADS - DW ? i - DW : 0]);
                else load_to_lds_4(ssrc + kb, at + SCALES + wave % SCALE_WAVES * 256, scale_lanes);
            }
        };
#pragma unroll
        for (int kb = 0; kb < STAGES; ++kb) load_parts(kb, 0, kb == STAGES - 1 ? EACH : PARTS);
        // this lane's places in a stage: pieces 2q and 2q + 1 of row r of sixteen, and the token columns' scales
        const uint32_t lo = r * 128 + ((2 * q) ^ (r >> 1)) * 16, hi = r * 128 + ((2 * q + 1) ^ (r >> 1)) * 16;
        constexpr int COL = 16 * WT;                         // rows from one of a wave's token columns to the next
        uint32_t a_lo, a_hi, b_lo, b_hi, b_scale;
        auto enter = [&](int kb) __attribute__((always_inline)) {
            const uint32_t stage = (kb % STAGES) * STAGE;
            a_lo = stage + 2048 * SN * wn + lo, a_hi = stage + 2048 * SN * wn + hi;
            b_lo = stage + BN * 128 + 2048 * wt + lo, b_hi = stage + BN * 128 + 2048 * wt + hi;
            b_scale = stage + SCALES + 64 * wt + 4 * r;
            asm volatile("" : "+v"(a_lo), "+v"(a_hi), "+v"(b_lo), "+v"(b_hi), "+v"(b_scale));   // (offsets then fit the reads' own)
        };
        auto operand = [&](uint32_t at_lo, uint32_t at_hi, int rows) __attribute__((always_inline)) {
            Operand<KIND> o;
            o.take(Piece{*reinterpret_cast<const u32x4p *>(lds + at_lo + rows * 128), *reinterpret_cast<const u32x4p *>(lds + at_hi + rows * 128)});
            return o;
        };
        auto token_scale = [&](int j) __attribute__((always_inline)) {
            return *reinterpret_cast<const float *>(lds + b_scale + j * COL * 4);
        };
        // Software pipeline over the columns: the products p[s] of a column are summed under the matrix instructions of the next one, whose
        // operand is read a column ahead. Before a step's last column the waves meet: the next step's stage has landed, and this
        // step's has been read (its last operands are in registers) and takes the bytes of a later one; the next step's
        // first operands are read under the last column, the weights' into the registers that it has just used.
        Operand<KIND> a[SN], b[2];
        float sb[2] = {0.0f, 0.0f}, factor = 0.0f;
        f32x4 p[SN];
#pragma unroll
        for (int s = 0; s < SN; ++s) p[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        auto first_operands = [&](int kb) __attribute__((always_inline)) {
            enter(kb);
            b[0] = operand(b_lo, b_hi, 0);
            if constexpr (is_f8(KIND)) sb[0] = token_scale(0);
#pragma unroll
            for (int s = 0; s < SN; ++s) a[s] = operand(a_lo, a_hi, 16 * s);
        };
        meet<(STAGES - 2) * PARTS + EACH>();
        first_operands(0);
        auto step = [&](int kb, auto more_c) __attribute__((always_inline)) {
            constexpr bool MORE = decltype(more_c)::value;   // another step follows
            float sw = 0.0f;
            if constexpr (is_f8(KIND)) {
                sw = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scales), kb & 63));
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const bool last = j + 1 == NT, read = !last || MORE;
                if (last && MORE) {
                    meet<(STAGES - 2) * PARTS>();
                    enter(kb + 1);
                }
                const Operand<KIND> now = b[j & 1];
                const float scale_now = sb[j & 1];
                const int next = last ? 0 : (j + 1) & 1;
                if (read) b[next] = operand(b_lo, b_hi, last ? 0 : (j + 1) * COL);
                if (is_f8(KIND) && read) sb[next] = token_scale(last ? 0 : j + 1);
                const int before = j ? j - 1 : NT - 1;
#pragma unroll
                for (int s = 0; s < SN; ++s) {
                    if constexpr (is_f8(KIND)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[s][before][i] = __builtin_fmaf(p[s][i], factor, acc[s][before][i]);
                        p[s] = product<KIND>(a[s], now, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                    } else {
                        acc[s][j] = product<KIND>(a[s], now, acc[s][j]);
                    }
                    if (last && MORE) a[s] = operand(a_lo, a_hi, 16 * s);
                }
                if constexpr (is_f8(KIND)) factor = sw * scale_now;
                // (left to itself the compiler sums a product right behind its matrix instruction and waits for it)
                if constexpr (KIND == kF8) {
                    if (read) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);          // the next column's reads
#pragma unroll
                    for (int s = 0; s < SN; ++s) {
                        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);                  // a product's sums,
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                  // the next product
                        if (last && MORE) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (last && MORE) load_parts(kb + STAGES, 0, EACH);
                if (!last && MORE) load_parts(kb + STAGES - 1, std::min((j + 1) * EACH, PARTS), std::min((j + 2) * EACH, PARTS));
            }
        };
        const int whole = A.k_bytes >> 7;
        for (int kb = 0; kb < whole;) {
            fetch_scales(kb);
            const int end = kb + 64 < whole ? kb + 64 : whole;
            for (; kb < end; ++kb) step(kb, std::true_type{});   // (no branch inside a step: the compiler would move sums behind it)
        }
        if (whole < A.kb) {                                  // a row's last bytes, less than a step
            if (!(whole & 63)) fetch_scales(whole);
            if (whole * 128 + piece * 16 >= A.k_bytes) {
                uint8_t * mine = lds + (whole % STAGES) * STAGE + wave * 1024 + lane * 16;
#pragma unroll
                for (int i = 0; i < DW; ++i) *reinterpret_cast<u32x4p *>(mine + W * i * 1024) = u32x4p{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < LOADS - DW; ++i)
                    if (wave + W * i < EIGHTS) *reinterpret_cast<u32x4p *>(mine + BN * 128 + W * i * 1024) = u32x4p{0, 0, 0, 0};
            }
            meet<0>();
            first_operands(whole);
            step(whole, std::false_type{});
        }
        if constexpr (is_f8(KIND)) {
#pragma unroll
            for (int s = 0; s < SN; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[s][NT - 1][i] = __builtin_fmaf(p[s][i], factor, acc[s][NT - 1][i]);
        }
        meet<0>();                                           // no load may land after the workgroup has ended
        // A wave's 16-token column at a time goes through LDS, so that neighbouring lanes store neighbouring bytes of a dst row:
        // straight from the registers (16 rows x 32 bytes a store) the stores of a 4096 x 4096 output took 6 us longer.
        constexpr int ROW = 16 * SN * 4 + 16;                // bytes of a token's outputs there
        static_assert(W * 16 * ROW <= STAGE_BYTES, "the stages' memory holds them");
        const int nw = n0 + 16 * SN * wn;                    // the wave's first output
        f32x4 bias[SN];
#pragma unroll
        for (int s = 0; s < SN; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = nw + 16 * s + 4 * q + e;
                bias[s][e] = A.bias && n < A.rows ? A.bias[static_cast<int64_t>(work.group) * A.rows + n] : 0.0f;
            }
        uint8_t * mine = lds + wave * 16 * ROW;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int s = 0; s < SN; ++s) *reinterpret_cast<f32x4 *>(mine + r * ROW + 64 * s + 16 * q) = acc[s][j] + bias[s];
            const int * to = rows + 16 * (j * WT + wt);
            if (A.dst_type == VBM_TYPE_F32) store_column<4 * SN, 4>(A, mine, ROW, to, nw);
            else store_column<2 * SN, 8>(A, mine, ROW, to, nw);
        }
    };
    // the wave columns' most live 16-token columns, the same for all waves (they meet at the barriers)
    const int nt = (live_cols + WT - 1) / WT;
    if constexpr (ST >= 8) {
        if (nt > 6) return run(std::integral_constant<int, 8>{});
    }
    if constexpr (ST >= 6) {
        if (nt > 5) return run(std::integral_constant<int, 6>{});
    }
    if constexpr (ST >= 5) {
        if (nt > 4) return run(std::integral_constant<int, 5>{});
    }
    if constexpr (ST >= 4) {
        if (nt > 3) return run(std::integral_constant<int, 4>{});
        if (nt > 2) return run(std::integral_constant<int, 3>{});
    }
    if (nt > 1) return run(std::integral_constant<int, 2>{});
    run(std::integral_constant<int, 1>{});
}

template <int KIND, int MAX8, int D>
void launch_few_rows(const ProductArgs & a, const ProductSize & s, hipStream_t stream) {
    const int64_t row_tiles = (a.rows + 15) / 16, blocks = row_tiles * s.most_token_tiles(8 * MAX8);
    require(blocks < (int64_t{1} << 24), "too many outputs for one launch");
    hipLaunchKernelGGL((few_rows_kernel<KIND, MAX8, D>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a,
                       static_cast<int>(row_tiles));
    check_hip(hipGetLastError(), "product launch");
}

template <int KIND, int MAX8, int W, int D>
void launch_stream_rows(const ProductArgs & a, const ProductSize & s, hipStream_t stream) {
    using L = StreamLayout<KIND, MAX8, W, D>;
    require(a.kb <= L::MAX_KB, "the tokens do not fit in LDS");
    const int64_t row_tiles = (a.rows + 15) / 16;
    const int tiles = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(L::MAX_TILES, s.groups() * row_tiles / 4096)));
    const int64_t units = (row_tiles + W * tiles - 1) / (W * tiles), blocks = units * s.most_token_tiles(8 * MAX8);
    require(blocks < (int64_t{1} << 32) / (W * 64), "too many outputs for one launch");
    hipLaunchKernelGGL((stream_rows_kernel<KIND, MAX8, W, D>), dim3(static_cast<unsigned>(blocks)), dim3(W * 64), 0, stream, a,
                       static_cast<int>(units), tiles);
    check_hip(hipGetLastError(), "product launch");
}

template <int KIND, int SN, int ST, int WN, int WT, int LDS>
void launch_many_rows(const ProductArgs & a, const ProductSize & s, hipStream_t stream) {
    constexpr int BN = 16 * SN * WN, BT = 16 * ST * WT;
    const int64_t row_tiles = (a.rows + BN - 1) / BN, tiles = s.most_token_tiles(BT), items = row_tiles * tiles;
    require(items < (int64_t{1} << 32) / (WN * WT * 64) - 8, "too many outputs for one launch");
    hipLaunchKernelGGL((many_rows_kernel<KIND, SN, ST, WN, WT, LDS>), dim3(static_cast<unsigned>((items + 7) / 8 * 8)),
                       dim3(WN * WT * 64), 0, stream, a, static_cast<int>(row_tiles), static_cast<int>(tiles));
    check_hip(hipGetLastError(), "product launch");
}

template <int KIND>
void launch_product(const ProductArgs & a, hipStream_t stream) {
    constexpr int FEW = KIND == kF8 ? kF8Wide : KIND;
    const ProductSize s{a.offsets != nullptr, a.n_rows, a.n_groups, a.rows, a.kb};
    switch (product_kernel<KIND>(s)) {
        case ProductKernel::few8: return launch_few_rows<FEW, 1, 4>(a, s, stream);
        case ProductKernel::few16: return launch_few_rows<FEW, 2, 3>(a, s, stream);
        case ProductKernel::stream8_4: return launch_stream_rows<FEW, 1, 4, 4>(a, s, stream);
        case ProductKernel::stream8_8: return launch_stream_rows<FEW, 1, 8, 4>(a, s, stream);
        case ProductKernel::stream16_4: return launch_stream_rows<FEW, 2, 4, 3>(a, s, stream);
        case ProductKernel::stream16_8: return launch_stream_rows<FEW, 2, 8, 4>(a, s, stream);
        case ProductKernel::tile256x256:
            if constexpr (KIND != kF8Wide) launch_many_rows<KIND, 4, 8, 4, 2, 160 * 1024>(a, s, stream);
            return;
        case ProductKernel::tile256x160:
            if constexpr (KIND != kF8Wide) launch_many_rows<KIND, 4, 5, 4, 2, 160 * 1024>(a, s, stream);
            return;
        case ProductKernel::tile256x128: return launch_many_rows<KIND, 2, 8, 8, 1, 160 * 1024>(a, s, stream);
        case ProductKernel::tile128x64: return launch_many_rows<KIND, 2, 4, 4, 1, 80 * 1024>(a, s, stream);
        case ProductKernel::tile64x32: return launch_many_rows<KIND, 1, 2, 4, 1, 40 * 1024>(a, s, stream);
    }
}

void product(const vbm_weights & w, const void * b, const float * b_scales, ProductArgs a, int dst_type, void * dst, hipStream_t stream) {
    const bool f8 = w.type == VBM_TYPE_F8_E4M3;
    require(f8 || w.type == VBM_TYPE_F16 || w.type == VBM_TYPE_BF16, "weights must be F8_E4M3, F16 or BF16");
    require(dst_type == VBM_TYPE_F32 || dst_type == VBM_TYPE_F16 || dst_type == VBM_TYPE_BF16, "dst must be F32, F16 or BF16");
    require(w.n_groups > 0 && w.n_groups <= 1024, "n_groups must be in 1..1024");
    require(w.rows > 0 && w.rows < (int64_t{1} << 30) && w.k > 0 && w.k < (int64_t{1} << 23), "rows and k out of range");
    const int64_t k_bytes = w.k * (f8 ? 1 : 2);
    require(k_bytes % 16 == 0, f8 ? "k must be a multiple of 16" : "k must be a multiple of 8");
    require(a.n_rows >= 0 && a.n_rows < (int64_t{1} << 29) && a.n_b >= 0 && a.n_dst >= 0 && a.n_dst < (int64_t{1} << 31) - 2, "row counts out of range");
    require(a.b_div > 0 && a.b_div < (int64_t{1} << 31), "b_div must be positive");
    if (a.n_rows == 0) return;
    require(w.data && b && dst && a.n_b > 0 && (!f8 || (w.scales && b_scales)), "null buffer");
    auto at = [](const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    require(at(w.data, 16) && at(b, 16), "weights and b must be 16-byte aligned");
    const size_t dsize = dst_type == VBM_TYPE_F32 ? 4 : 2;
    require(at(dst, dsize) && at(w.scales, 4) && at(w.bias, 4) && at(b_scales, 4) && at(a.offsets, 4) && at(a.b_rows, 4) && at(a.dst_rows, 4),
            "buffers must be aligned to their types");
    a.w = static_cast<const uint8_t *>(w.data);
    a.ws = w.scales;
    a.bias = w.bias;
    a.b = static_cast<const uint8_t *>(b);
    a.bs = b_scales;
    a.dst = dst;
    a.dst_type = dst_type;
    a.dst_vec = at(dst, 4 * dsize) && w.rows % 4 == 0;
    a.dst_vec16 = at(dst, 16) && static_cast<size_t>(w.rows) * dsize % 16 == 0;
    a.n_groups = static_cast<int>(w.n_groups);
    a.rows = static_cast<int>(w.rows);
    a.k_bytes = static_cast<int>(k_bytes);
    a.kb = static_cast<int>((k_bytes + 127) / 128);
    if (f8 && dst_type == VBM_TYPE_BF16) launch_product<kF8>(a, stream);
    else if (f8) launch_product<kF8Wide>(a, stream);
    else if (w.type == VBM_TYPE_F16) launch_product<kF16>(a, stream);
    else launch_product<kBF16>(a, stream);
}

}  // namespace
}  // namespace vbm

using namespace vbm;

extern "C" {

vbm_status vbm_mul_mat_fp8(const vbm_weights * w, const void * b, const float * b_scales, int64_t n_tokens, int dst_type,
                           void * dst, void * stream) {
    return guarded([&] {
        require(w != nullptr, "null weights");
        require(w->type == VBM_TYPE_F8_E4M3 && w->n_groups == 1, "weights must be one F8_E4M3 matrix");
        ProductArgs a{};
        a.n_b = a.n_rows = a.n_dst = n_tokens;
        a.b_div = 1;
        product(*w, b, b_scales, a, dst_type, dst, as_stream(stream));
    });
}

vbm_status vbm_grouped_mul_mat(const vbm_weights * w, const void * b, const float * b_scales, int64_t n_b,
                               const int32_t * b_rows, int64_t b_div, const int32_t * offsets, int64_t n_rows,
                               const int32_t * dst_rows, int64_t n_dst, int dst_type, void * dst, void * stream) {
    return guarded([&] {
        require(w != nullptr, "null weights");
        require(offsets != nullptr || n_rows == 0, "null offsets");
        ProductArgs a{};
        a.n_b = n_b;
        a.b_rows = b_rows;
        a.b_div = b_div;
        a.offsets = offsets;
        a.n_rows = n_rows;
        a.dst_rows = dst_rows;
        a.n_dst = n_dst;
        product(*w, b, b_scales, a, dst_type, dst, as_stream(stream));
    });
}

}  // extern "C"
