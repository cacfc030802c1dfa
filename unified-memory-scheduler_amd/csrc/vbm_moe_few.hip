// A routed-expert layer for a few tokens, weights as they are stored, in two launches:
//
//   h[t, r] = act(Wg[e] x[t] + bg[e], Wu[e] x[t] + bu[e])            e = ids[t, r]
//   out[t]  = sum over ranks r of weights[t, r] * (Wd[e] h[t, r] + bd[e])
//
// The first launch routes (top-k of the logits and the softmax over it, every workgroup for itself) and makes h, the second multiplies
// by the down weights and adds the ranks up, in their order. What such a step has to do is read the touched experts' weights once; the kernels
// differ from the grouped products in what they save around that: five launches, and the rows between them.
//
// The activations are not quantized. The weights are widened to bf16, exactly (e4m3 has 4 significant bits, 8-bit integers have 8; fp16's 11
// are two bf16 values), and so are the activations, as sums of bf16 values: fp32 ones of three (8 + 8 + 8 bits, each the leading
// bits of what is left, so the last one is exact, but for bits below bf16's smallest value, 2^-133), fp16 of two, bf16 of one. Each term is a column of the matrix instruction's B operand, whose
// 16 columns a few tokens would leave unused anyway: 5 rows of three terms or 8 of one or two. All products are exact in fp32, as in an fp32
// program, and summed in fp32, FP8 blocks and integer rows before their scales; h is kept as its three terms. (An infinity's second term is a NaN.)
//
// Rows are grouped by expert into slots of up to as many (token, rank) entries as there are columns, in the order in which they first
// appear; every wave finds its slot by itself from the ids: with two ballots for each of an id's ten bits a lane knows the entries of its entry's
// expert. An expert with more entries than a slot holds has its weights read once for each slot: sixteen tokens all through four bf16 experts of 2880 x 2880
// take 84 + 47 us, two slots an expert and four in the second launch; four such tokens, one slot, 31 + 21.
// The weights stream as in the grouped products: 16 rows by 128 bytes a step, loaded straight to a ring in LDS of each wave, with the
// activations of the step behind them (they come from the L2, and the waits count all loads alike).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vbm_device.hpp"
#include "vbm_internal.hpp"
#include "vbm_lds_stream.hpp"
#include "vbm_quantize.hpp"

namespace vbm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMostTokens = 16, kMostEntries = 128, kMostTiles = 4;   // (tiles of a wave)
constexpr int kTerms = -1;                     // the type of h: three bf16 terms of each value, a step's first, second, third

constexpr bool one_byte(int kind) { return kind == VBM_TYPE_F8_E4M3 || kind == VBM_TYPE_I8; }

// A step's activations of one entry.
template <int KIND, int X>
struct Rows {
    static constexpr int VALUES = one_byte(KIND) ? 128 : 64;                      // of k, a step
    static constexpr int TERMS = X == VBM_TYPE_BF16 ? 1 : (X == VBM_TYPE_F16 ? 2 : 3);
    static constexpr int MOST = TERMS < 3 ? 8 : (X == kTerms && one_byte(KIND) ? 4 : 5);   // entries a slot: (the fifth's pieces take a fourth load)
    static constexpr int BYTES = VALUES * (X == kTerms ? 6 : (X == VBM_TYPE_F32 ? 4 : 2)), PIECES = BYTES / 16;
    static constexpr int loads(int entries) { return (entries * PIECES + 63) / 64; }   // of a wave, 64 pieces each
};

struct FewArgs {
    const uint8_t * w;             // [n_expert][rows][k_bytes]
    const float * ws, * bias;      // as vbm_weights has them
    const void * x;                // x [n_tokens][k], or h [entries][kb][three terms of a step]
    const int32_t * ids;           // [entries]
    const float * logits;          // or null: then ids are read
    int32_t * ids_out;             // with logits
    float * weights_out;
    const float * weights;         // [entries], the second launch's
    uint8_t * h;                   // the first launch's outputs
    void * out;
    int out_type;
    int n_tokens, top_k, n_expert, entries, capacity;   // capacity: most entries a slot
    int rows, k_bytes, kb;         // of this launch's matrix
    int inter, h_kb, h_step;       // I; steps of a row of h, and their bytes
    int row_units, tiles;          // workgroups a slot; row tiles a wave
    int activation;
    float alpha, limit;
};

// The entries' grouping by expert, as every wave finds it: lane l holds entries l and 64 + l.
struct Slots {
    int id[2], position[2];        // of the entry among those of its expert
    uint64_t same[2][2];           // the entries of its expert
    uint64_t leads[2];             // entries that begin a slot
    __device__ __forceinline__ Slots(const int32_t * ids, int entries, int n_expert, int capacity) {
        const int lane = threadIdx.x & 63;
        const uint64_t below = (uint64_t{1} << lane) - 1;
        uint64_t valid[2], plane[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            id[s] = lane + 64 * s < entries ? ids[lane + 64 * s] : -1;
            if (static_cast<unsigned>(id[s]) >= static_cast<unsigned>(n_expert)) id[s] = -1;
            valid[s] = __ballot(id[s] >= 0);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int o = 0; o < 2; ++o) same[s][o] = valid[o];
#pragma unroll
        for (int b = 0; b < 10; ++b) {
#pragma unroll
            for (int o = 0; o < 2; ++o) plane[o] = __ballot(id[o] >> b & 1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int o = 0; o < 2; ++o) same[s][o] &= id[s] >> b & 1 ? plane[o] : ~plane[o];
        }
        position[0] = __popcll(same[0][0] & below);
        position[1] = __popcll(same[1][0]) + __popcll(same[1][1] & below);
#pragma unroll
        for (int s = 0; s < 2; ++s) leads[s] = __ballot(id[s] >= 0 && position[s] % capacity == 0);
    }
    __device__ __forceinline__ int count() const { return __popcll(leads[0]) + __popcll(leads[1]); }
    // The number of the slot that entry (s, this lane) begins.
    __device__ __forceinline__ int number(int s) const {
        const uint64_t below = (uint64_t{1} << (threadIdx.x & 63)) - 1;
        return s ? __popcll(leads[0]) + __popcll(leads[1] & below) : __popcll(leads[0] & below);
    }
    // Slot `index`: its expert, and its entries into list[]; their number.
    __device__ __forceinline__ int find(int index, int capacity, int & expert, int * list) const {
        const int lane = threadIdx.x & 63;
        int first = 0, n = 0;
        expert = -1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint64_t at = __ballot((leads[s] >> lane & 1) && number(s) == index);
            if (!at) continue;
            const int l = __builtin_ctzll(at);
            expert = __builtin_amdgcn_readlane(id[s], l);
            first = __builtin_amdgcn_readlane(position[s], l);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool mine = expert >= 0 && id[s] == expert && position[s] >= first && position[s] < first + capacity;
            if (mine) list[position[s] - first] = lane + 64 * s;
            n += __popcll(__ballot(mine));
        }
        return n;
    }
    // All slots: experts, numbers of entries, entries [slot][capacity]. By one wave.
    __device__ __forceinline__ void table(int capacity, int * experts, int * counts, int * list) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (id[s] < 0) continue;
            uint64_t m0 = same[s][0], m1 = same[s][1];
            const int total = __popcll(m0) + __popcll(m1), first = position[s] / capacity * capacity;
            for (int j = 0; j < first; ++j) {                // (the first entry of its slot: a slot holds almost always all of them)
                if (m0) m0 &= m0 - 1;
                else m1 &= m1 - 1;
            }
            const uint64_t below = (uint64_t{1} << __builtin_ctzll(m0 ? m0 : m1)) - 1;
            const int slot = m0 ? __popcll(leads[0] & below) : __popcll(leads[0]) + __popcll(leads[1] & below);
            list[slot * capacity + position[s] - first] = lane + 64 * s;
            if (position[s] == first) {
                experts[slot] = id[s];
                counts[slot] = total - first < capacity ? total - first : capacity;
            }
        }
    }
};

// Maximum over the wave, the same in all lanes.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
        v = o > v ? o : v;
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});   // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});   // row 0's last to row 1, row 2's to row 3
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});   // lane 31's to the upper half
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
// One wave's top-k of n <= 64 NPL logits, lg[c]: that of expert lane + 64 c, in the router's order (value desc, then lower index, NaN as -inf):
// lane j < k gets pick j. The keys are the values' bits, which order as they do once the sign is taken care of; 0 is none left. A round is
// a maximum over lanes in registers (with an exchange through LDS in it, as the router's has, a token took about 1 us more).
template <int NPL>
__device__ __forceinline__ void top_k(const float (&lg)[NPL], int n, int k, float & value, int & id) {
    const int lane = threadIdx.x & 63;
    uint32_t key[NPL];
#pragma unroll
    for (int c = 0; c < NPL; ++c) {
        const uint32_t b = __builtin_bit_cast(uint32_t, route_key(lg[c]) + 0.0f);   // (-0 as 0)
        key[c] = lane + 64 * c < n ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
    }
    uint32_t mine = 0;
    id = -1;
    for (int j = 0; j < k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int c = 1; c < NPL; ++c) best = key[c] > best ? key[c] : best;
        const uint32_t top = wave_max(best);
        int pick = -1;
#pragma unroll
        for (int c = NPL - 1; c >= 0; --c) {
            const uint64_t m = __ballot(key[c] == top);
            if (m) pick = 64 * c + __builtin_ctzll(m);
        }
#pragma unroll
        for (int c = 0; c < NPL; ++c) key[c] = pick == lane + 64 * c ? 0u : key[c];
        if (lane == j) mine = top, id = pick;
    }
    value = __builtin_bit_cast(float, mine & 0x80000000u ? mine & 0x7FFFFFFFu : ~mine);
}

// ids (and weights) of the tokens into LDS, by top-k of the logits or from the caller; W waves.
template <int W>
__device__ __forceinline__ void route(const FewArgs & A, int32_t * ids, bool writes) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (!A.logits) {
        for (int i = threadIdx.x; i < A.entries; i += W * 64) ids[i] = A.ids[i];
        return;
    }
    auto pick = [&](auto npl_c) {
        constexpr int NPL = decltype(npl_c)::value;
        for (int t = wave; t < A.n_tokens; t += W) {
            float lg[NPL], value;
            int id;
#pragma unroll
            for (int c = 0; c < NPL; ++c) lg[c] = lane + 64 * c < A.n_expert ? A.logits[static_cast<int64_t>(t) * A.n_expert + lane + 64 * c] : 0.0f;
            top_k<NPL>(lg, A.n_expert, A.top_k, value, id);
            if (lane < A.top_k) ids[t * A.top_k + lane] = id;
            if (writes) {
                const float w = wave_pick_softmax(value, A.top_k);
                if (lane < A.top_k) {
                    A.ids_out[t * A.top_k + lane] = id;
                    A.weights_out[t * A.top_k + lane] = w;
                }
            }
        }
    };
    if (A.n_expert <= 128) pick(std::integral_constant<int, 2>{});
    else if (A.n_expert <= 256) pick(std::integral_constant<int, 4>{});
    else pick(std::integral_constant<int, 16>{});
}

__device__ __forceinline__ unsigned upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060302u);
}
__device__ __forceinline__ float without(float v, unsigned mask) {   // v minus the bits of it that `mask` keeps
    return v - __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & mask);
}

// Eight weights as bf16 values; fp16's upper parts, and what is left of them in `rest`.
template <int KIND>
__device__ __forceinline__ bf16x8 widened(const unsigned * w, bf16x8 & rest) {
    if constexpr (KIND == VBM_TYPE_BF16) {
        return __builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[2], w[3]});
    } else if constexpr (KIND == VBM_TYPE_F8_E4M3) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, true);
        const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, true);
        return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    } else if constexpr (KIND == VBM_TYPE_I8) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned two = w[i >> 1] >> (16 * (i & 1));
            v[i] = upper_halves(static_cast<float>(static_cast<int8_t>(two)), static_cast<float>(static_cast<int8_t>(two >> 8)));
        }
        return __builtin_bit_cast(bf16x8, v);
    } else {
        u32x4 v, u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
            const float b = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
            v[i] = upper_halves(a, b);
            u[i] = upper_halves(without(a, 0xFFFF0000u), without(b, 0xFFFF0000u));
        }
        rest = __builtin_bit_cast(bf16x8, u);
        return __builtin_bit_cast(bf16x8, v);
    }
}

// The same in all lanes, which the compiler does not see everywhere. (A load needs five wait states behind a vector instruction that writes
// its scalar base; the compiler does not count into the inline assembly of the loads.)
__device__ __forceinline__ const uint8_t * uniform(const uint8_t * p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
    uint64_t u = static_cast<uint64_t>(hi) << 32 | lo;
    asm volatile("s_nop 4" : "+s"(u));
    return reinterpret_cast<const uint8_t *>(u);
}

// What a wave streams: G times 16 weight rows x 128 bytes a step, the step's activations of up to 64 NB pieces, FP8 scales.
template <int KIND, int X, int NB, int G>
struct Ring {
    using R = Rows<KIND, X>;
    static constexpr bool F8 = KIND == VBM_TYPE_F8_E4M3;
    // (FEWEST, MOST: a step's loads; how many depends on its slot's entries. As many for all steps, those for nobody by one lane, took the down
    // launch of four tokens 37.5 us instead of 35.4. gate_up's waits count them as they are: on the fewest, and so for later steps too, sixteen tokens
    // over integers took 119 us instead of 110; down's, where it makes 1 % the other way, on the fewest.)
    static constexpr int FEWEST = 2 * G + 1 + (F8 ? 1 : 0), MOST = FEWEST + NB - 1, ACTIVATIONS = G * 2048, SCALES = ACTIVATIONS + NB * 1024, STEP = SCALES + (F8 ? 256 : 0);
    static constexpr int NJ = R::VALUES / 32;

    // What the lane loads: its rows of weights (offset from the groups' bases), the entry's row and the piece of each load of activations; `live` loads
    // are for the slot's entries.
    struct Source {
        const uint8_t * base[G];
        uint32_t offset[2 * G];
        const uint8_t * rows[NB];
        int piece[NB], live;
        const float * scale;
    };
    // list: the n entries of the slot; row_of(entry): its activations.
    template <class F>
    static __device__ __forceinline__ void enter(Source & s, const int * list, int n, const F & row_of) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int flat = 64 * i + lane, c = flat / R::PIECES;
            s.rows[i] = row_of(list[c < n ? c : 0]);
            s.piece[i] = (flat % R::PIECES) ^ (c & 7);
        }
        s.live = __builtin_amdgcn_readfirstlane(R::loads(n));
    }

    // Places of the weights' 16-byte pieces as in the grouped products' rings: piece p of row r at place p ^ (r / 2 % 8) of
    // its 128 bytes. Activations: entry c's pieces behind each other, p at place p ^ (c % 8), so that the lanes' reads
    // of one piece of several entries spread over the banks.
    // Returns the number of loads.
    static __device__ __forceinline__ int load(uint32_t at, const Source & s, int kb, int k_bytes, int row_bytes) {
        const int lane = threadIdx.x & 63, even = (lane & 7) ^ (lane >> 4), odd = even ^ 4;
        const int64_t off = static_cast<int64_t>(kb) * 128;
        // (a piece past the row's end reads the step's first one: zeros take its place in the registers)
        const int e = kb * 128 + even * 16 < k_bytes ? even * 16 : 0, o = kb * 128 + odd * 16 < k_bytes ? odd * 16 : 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint8_t * base = uniform(s.base[g] + off);
            load_to_lds_16(base, s.offset[2 * g] + e, at + g * 2048);
            load_to_lds_16(base, s.offset[2 * g + 1] + o, at + g * 2048 + 1024);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (i && i >= s.live) break;
            const int b = kb * R::BYTES + s.piece[i] * 16;
            load_to_lds_16(s.rows[i] + (b < row_bytes ? b : kb * R::BYTES), at + ACTIVATIONS + i * 1024);
        }
        if constexpr (F8) load_to_lds_4(s.scale + kb, at + SCALES);
        return FEWEST - 1 + s.live;
    }

    // The step in `stage` added to acc: lane (q, r) has rows 4q .. 4q + 3 of column r of each group. entry, term: this lane's column.
    static __device__ __forceinline__ void multiply(const uint8_t * stage, int entry, int term, int kb, int k_bytes, f32x4 (&acc)[G]) {
        if ((kb + 1) * 128 <= k_bytes) multiply_step<false>(stage, entry, term, 128, acc);
        else multiply_step<true>(stage, entry, term, k_bytes - kb * 128 - 32 * static_cast<int>(threadIdx.x >> 4 & 3), acc);
    }
    // TAIL: the row's last step is not a whole one; `left` bytes of it are from this lane's 32 on.
    template <bool TAIL>
    static __device__ __forceinline__ void multiply_step(const uint8_t * stage, int entry, int term, int left, f32x4 (&acc)[G]) {
        const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
        unsigned w[G][8];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            *reinterpret_cast<u32x4 *>(w[g]) = *reinterpret_cast<const u32x4 *>(stage + g * 2048 + r * 128 + ((2 * q) ^ (r >> 1)) * 16);
            *reinterpret_cast<u32x4 *>(w[g] + 4) = *reinterpret_cast<const u32x4 *>(stage + g * 2048 + r * 128 + ((2 * q + 1) ^ (r >> 1)) * 16);
        }
        const uint8_t * row = stage + ACTIVATIONS + entry * R::BYTES;
        auto piece = [&](int p) { return *reinterpret_cast<const u32x4 *>(row + (p ^ (entry & 7)) * 16); };
        f32x4 sum[G];
#pragma unroll
        for (int g = 0; g < G; ++g) sum[g] = F8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[g];
        // term t of a value is what its first 8 (t + 1) significant bits have over its first 8 t
        const unsigned kept = term == 1 ? 0xFFFFFF00u : 0xFFFFFFFFu, gone = term == 0 ? 0u : (term == 1 ? 0xFFFF0000u : 0xFFFFFF00u);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            u32x4 b;
            if constexpr (X == VBM_TYPE_BF16) {
                b = piece(q * NJ + j);
            } else if constexpr (X == kTerms) {
                b = piece(term * (R::VALUES / 8) + q * NJ + j);
            } else {
                float v[8];
                if constexpr (X == VBM_TYPE_F32) {
                    const f32x4 lo = __builtin_bit_cast(f32x4, piece((q * NJ + j) * 2)), hi = __builtin_bit_cast(f32x4, piece((q * NJ + j) * 2 + 1));
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
                } else {
                    const u32x4 h = piece(q * NJ + j);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h[i >> 1] >> (16 * (i & 1)))));
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned bits = __builtin_bit_cast(unsigned, static_cast<float>(v[i]));
                    // (fp16 has two terms, and the second one is all the rest)
                    v[i] = __builtin_bit_cast(float, X == VBM_TYPE_F32 ? bits & kept : bits) - __builtin_bit_cast(float, bits & gone);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = upper_halves(v[2 * i], v[2 * i + 1]);
            }
            const bool past = TAIL && left <= (j * 2 / NJ) * 16;   // (k ends at a multiple of 16 bytes)
            if (past) b = u32x4{0, 0, 0, 0};
            const bf16x8 x = __builtin_bit_cast(bf16x8, b);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                constexpr int N = one_byte(KIND) ? 2 : 4;        // words of eight weights
                unsigned a[N];
#pragma unroll
                for (int i = 0; i < N; ++i) a[i] = past ? 0u : w[g][N * j + i];
                bf16x8 rest;
                const bf16x8 v = widened<KIND>(a, rest);
                sum[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, x, sum[g], 0, 0, 0);
                if constexpr (KIND == VBM_TYPE_F16) sum[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(rest, x, sum[g], 0, 0, 0);
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if constexpr (F8) {
                const float f = *reinterpret_cast<const float *>(stage + SCALES + g * (256 / G));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][i] = __builtin_fmaf(sum[g][i], f, acc[g][i]);
            } else {
                acc[g] = sum[g];
            }
        }
    }
};

// The loads of the N newest steps.
template <int N>
struct Newest {
    int loads[N] = {};
    __device__ __forceinline__ void add(int n) {
#pragma unroll
        for (int i = N - 1; i > 0; --i) loads[i] = loads[i - 1];
        loads[0] = n;
    }
    // All others have landed, and the wave's LDS reads are done. FEWEST, MOST: of a step.
    template <int FEWEST, int MOST>
    __device__ __forceinline__ void landed_before() const {
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += loads[i];
        wait<N * FEWEST, N * MOST>(n);
    }
    template <int LEAST, int MOST>
    static __device__ __forceinline__ void wait(int n) {
        if constexpr (LEAST < MOST) {
            if (n > LEAST) return wait<LEAST + 1, MOST>(n);
        }
        landed<LEAST>();
    }
};

// Lane (q, r) with an entry's first column: its terms' columns, which are the neighbouring lanes, added up.
template <int TERMS>
__device__ __forceinline__ f32x4 over_terms(f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float sum = acc[e];                            // (a bit cast of the vector's element itself would take the first one's)
        const int v = __builtin_bit_cast(int, sum);
        float rest = 0.0f;
        if constexpr (TERMS > 2) rest = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, v, 0x102, 0xF, 0xF, true));
        if constexpr (TERMS > 1) rest += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, v, 0x101, 0xF, 0xF, true));
        acc[e] = sum + rest;
    }
    return acc;
}

// ------------------------------------------------------------------------------------ gate and up
// A row tile is 16 gate rows and the 16 up rows of the same values of h. SHARE waves share a tile's depth and join their sums through LDS; or
// (SHARE 1) each wave takes `tiles` of its own, one after the other through its ring, without barriers.
//
// One token through eight of 128 FP8 experts of 2048 x 768 (25 MB): 11 us, 2 of them the routing, some 5 a launch and the first loads (16 tokens, 84
// experts: 56 us from logits, 49 with the routing given; every workgroup routes before its first load, also those past the last slot); 16 tokens, 30 bf16
// experts of 2880 x 2880 touched: 166 us, 6.0 TB/s (reads alone reach 5.6 to 6); four tokens in fp32, 16 integer experts: 61 us, 4.4 TB/s, of which splitting
// x into its terms takes 8 (bf16 tokens 53). 8 + 8 rows a tile took 86 there, and 168 for bf16; an even share of all tiles for 512
// workgroups, split inside tiles, 61 and 179; rings of two steps with three workgroups a CU the same as of three with two.
template <int KIND, int X, int NB, int SHARE>
__global__ __launch_bounds__(256) void few_gate_up_kernel(FewArgs A) {
    using S = Ring<KIND, X, NB, 2>;
    using R = Rows<KIND, X>;
    constexpr int W = 4, D = NB <= 2 ? 3 : 2, MOST_TILES = SHARE == 1 ? kMostTiles : 1, TILES = W / SHARE * MOST_TILES;   // (two workgroups a CU)
    constexpr bool kScaled = KIND == VBM_TYPE_I8;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[W * D * S::STEP];
    __shared__ __attribute__((aligned(16))) float row_bias[TILES * 32], row_scale[kScaled ? TILES * 32 : 4];   // [tile][gate, up][16]
    __shared__ int32_t ids[kMostEntries];
    __shared__ int list[W][8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int q = lane >> 4, r = lane & 15;
    route<W>(A, ids, blockIdx.x == 0);
    __syncthreads();
    const int index = static_cast<int>(blockIdx.x) / A.row_units, unit = static_cast<int>(blockIdx.x) - index * A.row_units;
    int expert;
    const int n = Slots(ids, A.entries, A.n_expert, A.capacity).find(index, A.capacity, expert, list[wave]);
    if (!n) return;                                          // (the whole workgroup)
    expert = __builtin_amdgcn_readfirstlane(expert);

    const int row_tiles = (A.inter + 15) >> 4;
    constexpr int AT_ONCE = W / SHARE;                       // tiles
    const int local0 = wave / SHARE, tile0 = unit * A.tiles * AT_ONCE, first_tile = tile0 + local0;   // this wave's: first_tile + AT_ONCE i
    const int my_tiles = first_tile >= row_tiles ? 0 : std::min((row_tiles - first_tile + AT_ONCE - 1) / AT_ONCE, A.tiles);
    const int k_begin = A.kb * (wave % SHARE) / SHARE, k_end = A.kb * (wave % SHARE + 1) / SHARE;
    const uint8_t * weights = A.w + static_cast<int64_t>(expert) * A.rows * A.k_bytes;
    uint8_t * mine = ring + wave * (D * S::STEP);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(mine));

    const int row_bytes = A.k_bytes / (one_byte(KIND) ? 1 : 2) * (X == VBM_TYPE_F32 ? 4 : 2);
    typename S::Source source;
    S::enter(source, list[wave], n, [&](int entry) { return static_cast<const uint8_t *>(A.x) + static_cast<int64_t>(entry / A.top_k) * row_bytes; });
    const int column = r / R::TERMS < n ? r / R::TERMS : 0, term = r % R::TERMS;

    int tile_next = 0, kb_next = k_begin, place_next = 0;
    Newest<D - 1> newest;
    auto enter = [&](int i) __attribute__((always_inline)) {
        const int i0 = (first_tile + AT_ONCE * i) * 16;
#pragma unroll
        for (int g = 0; g < 2; ++g) source.base[g] = weights + static_cast<int64_t>(i0 + g * A.inter) * A.k_bytes;
#pragma unroll
        for (int l = 0; l < 2; ++l) {                        // (the last tile's rows past I read its last one)
            const int row = 8 * l + (lane >> 3);
            source.offset[l] = source.offset[2 + l] = static_cast<uint32_t>(i0 + row < A.inter ? row : A.inter - 1 - i0) * static_cast<uint32_t>(A.k_bytes);
        }
        if constexpr (S::F8) source.scale = A.ws + (static_cast<int64_t>(expert) * ((A.rows + 127) >> 7) + ((i0 + (lane >= 32 ? A.inter : 0)) >> 7)) * A.kb;
    };
    auto issue = [&]() __attribute__((always_inline)) {
        newest.add(S::load(lds0 + place_next * S::STEP, source, kb_next, A.k_bytes, row_bytes));
        place_next = place_next + 1 == D ? 0 : place_next + 1;
        if (kb_next + 1 < k_end) {                           // (past the end the last step again, so that the waits' counts hold)
            ++kb_next;
        } else if (tile_next + 1 < my_tiles) {
            kb_next = k_begin;
            enter(++tile_next);
        }
    };
    const bool streams = my_tiles > 0 && k_begin < k_end;
    if (streams) {
        enter(0);
#pragma unroll
        for (int i = 0; i < D; ++i) issue();
    }
    for (int i = threadIdx.x; i < AT_ONCE * A.tiles * 32; i += W * 64) {
        const int value = (tile0 + (i >> 5)) * 16 + (i & 15), at = value + (i & 16 ? A.inter : 0);
        row_bias[i] = A.bias && value < A.inter ? A.bias[static_cast<int64_t>(expert) * A.rows + at] : 0.0f;
        if constexpr (kScaled) row_scale[i] = value < A.inter ? A.ws[static_cast<int64_t>(expert) * A.rows + at] : 0.0f;
    }
    __syncthreads();

    // Tile i's sums to h, as their three terms: lane (q, first column of an entry) has four values.
    auto finish = [&](int i, f32x4 gate, f32x4 up) __attribute__((always_inline)) {
        gate = over_terms<R::TERMS>(gate);
        up = over_terms<R::TERMS>(up);
        const int local = (local0 + AT_ONCE * i) * 32 + 4 * q, first = (first_tile + AT_ONCE * i) * 16 + 4 * q;
        if (term || r / R::TERMS >= n || first >= A.inter) return;
        if constexpr (kScaled) gate *= *reinterpret_cast<const f32x4 *>(row_scale + local), up *= *reinterpret_cast<const f32x4 *>(row_scale + local + 16);
        gate += *reinterpret_cast<const f32x4 *>(row_bias + local);
        up += *reinterpret_cast<const f32x4 *>(row_bias + local + 16);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = glu_value(A.activation, gate[e], up[e], A.alpha, A.limit);
        uint8_t * to = A.h + (static_cast<int64_t>(list[wave][column]) * A.h_kb + first / R::VALUES) * A.h_step + first % R::VALUES * 2;
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            *reinterpret_cast<u32x2q *>(to + t * R::VALUES * 2) = u32x2q{upper_halves(v[0], v[1]), upper_halves(v[2], v[3])};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = without(v[e], 0xFFFF0000u);
        }
    };

    int place = 0;
    for (int i = 0; i < (SHARE == 1 ? my_tiles : 1); ++i) {
        f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        if (streams) {
            for (int kb = k_begin; kb < k_end; ++kb) {
                newest.template landed_before<S::FEWEST, S::MOST>();
                S::multiply(mine + place * S::STEP, column, term, kb, A.k_bytes, acc);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the place has been read
                issue();
                place = place + 1 == D ? 0 : place + 1;
            }
        }
        if constexpr (SHARE == 1) {
            finish(i, acc[0], acc[1]);
        } else {
            landed<0>();                                     // (the waves' sums take the ring's memory)
            f32x4 * parts = reinterpret_cast<f32x4 *>(mine);
            parts[lane] = acc[0];
            parts[64 + lane] = acc[1];
            __syncthreads();
            if (wave % SHARE || !my_tiles) return;
#pragma unroll
            for (int w = 1; w < SHARE; ++w) {
                const f32x4 * other = reinterpret_cast<const f32x4 *>(mine + w * (D * S::STEP));
                acc[0] += other[lane];
                acc[1] += other[64 + lane];
            }
            finish(0, acc[0], acc[1]);
        }
    }
    landed<0>();                                             // no load may land after the workgroup has ended
}

// ------------------------------------------------------------------------------- down and combine
// One token as above: 8.5 us for 12.6 MB, of which all but the 2.5 of the stream are a launch, the ids, the first loads and the combine; 30 bf16 experts 98 us
// (5.1 TB/s), 16 integer ones 35. H / 16 workgroups, one a CU, leave CUs idle (180 of 256 work for 2880, 128 for 2048), and each reads at up to 12 bytes a cycle: 8, 12 or
// 16 waves, with rings as deep as fit, take the same time. From H = 4096 to 5120 the launch needs a second round: eight FP8 experts of 1536 values
// 15.4 and 25.5 us, 56 of them 72 and 126.
//
// A workgroup takes 16 rows of the output for all slots; its waves share all their steps in contiguous runs, slot by slot. A wave's sums of a slot
// go to the entries' places in LDS, except for a slot that an earlier wave began: those are added up behind it, in the waves' order.
template <int KIND, int NB>
__global__ __launch_bounds__(512) void few_down_kernel(FewArgs A) {
    using S = Ring<KIND, kTerms, NB, 1>;
    using R = Rows<KIND, kTerms>;
    constexpr int W = 8, D = NB <= 2 ? 4 : 3;              // (what fits in LDS)
    constexpr bool kScaled = KIND == VBM_TYPE_I8;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[W * D * S::STEP];
    __shared__ __attribute__((aligned(16))) float y[kMostEntries * 16], heads[W][R::MOST * 16];
    __shared__ int32_t ids[kMostEntries];
    __shared__ float shares[kMostEntries];
    __shared__ int experts[kMostEntries], counts[kMostEntries], list[kMostEntries * R::MOST], head_slot[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int q = lane >> 4, r = lane & 15, n0 = static_cast<int>(blockIdx.x) * 16;
    if (static_cast<int>(threadIdx.x) < A.entries) ids[threadIdx.x] = A.ids[threadIdx.x], shares[threadIdx.x] = A.weights[threadIdx.x];
    __syncthreads();
    const Slots slots(ids, A.entries, A.n_expert, A.capacity);
    const int n_slots = slots.count();
    if (wave == 0) slots.table(A.capacity, experts, counts, list);
    __syncthreads();

    const int total = n_slots * A.kb, begin = static_cast<int>(static_cast<int64_t>(total) * wave / W), end = static_cast<int>(static_cast<int64_t>(total) * (wave + 1) / W);
    uint8_t * mine = ring + wave * (D * S::STEP);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(mine));
    const int row_bytes = A.kb * R::BYTES;

    int next = begin, slot_next = A.kb ? begin / A.kb : 0, kb_next = begin - slot_next * A.kb, place_next = 0;
    typename S::Source source;
#pragma unroll
    for (int l = 0; l < 2; ++l) {
        const int n = n0 + 8 * l + (lane >> 3);
        source.offset[l] = static_cast<uint32_t>((n < A.rows ? n : A.rows - 1) - n0) * static_cast<uint32_t>(A.k_bytes);
    }
    auto enter = [&](int s) __attribute__((always_inline)) {
        const int expert = __builtin_amdgcn_readfirstlane(experts[s]);
        source.base[0] = A.w + (static_cast<int64_t>(expert) * A.rows + n0) * A.k_bytes;
        if constexpr (S::F8) source.scale = A.ws + (static_cast<int64_t>(expert) * ((A.rows + 127) >> 7) + (n0 >> 7)) * A.kb;
        S::enter(source, list + s * A.capacity, counts[s], [&](int entry) { return static_cast<const uint8_t *>(A.x) + static_cast<int64_t>(entry) * row_bytes; });
    };
    auto issue = [&]() __attribute__((always_inline)) {
        S::load(lds0 + place_next * S::STEP, source, kb_next, A.k_bytes, row_bytes);
        place_next = place_next + 1 == D ? 0 : place_next + 1;
        if (next + 1 < end) {                                // (past the end the last step again, so that the waits' counts hold)
            ++next;
            if (++kb_next == A.kb) {
                kb_next = 0;
                enter(++slot_next);
            }
        }
    };
    if (lane == 0) head_slot[wave] = -1;
    const int first_slot = slot_next, first_kb = kb_next;
    if (begin < end) {
        enter(first_slot);
#pragma unroll
        for (int i = 0; i < D; ++i) issue();
    }
    // This thread's output is that of token mine_t and row mine_n: the first ranks' scales and biases are asked for here, so that
    // nobody waits for them at the end.
    constexpr int AHEAD = 8;
    const int mine_t = static_cast<int>(threadIdx.x) >> 4, mine_n = n0 + (lane & 15);
    const bool puts = mine_t < A.n_tokens && mine_n < A.rows;
    auto row_at = [&](int k) {                               // of rank k's expert; -1: none
        const int e = ids[mine_t * A.top_k + k];
        return static_cast<unsigned>(e) < static_cast<unsigned>(A.n_expert) ? static_cast<int64_t>(e) * A.rows + mine_n : -1;
    };
    float scales[AHEAD], biases[AHEAD];
    if (puts) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t at = k < A.top_k ? row_at(k) : -1;
            scales[k] = kScaled && at >= 0 ? A.ws[at] : 1.0f;
            biases[k] = A.bias && at >= 0 ? A.bias[at] : 0.0f;
        }
    }
    if (begin < end) {
        int s = first_slot, kb = first_kb, place = 0;
        const int column = r / 3, term = r % 3;
        bool head = kb > 0;
        int n = counts[s];
        f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int i = begin; i < end; ++i) {
            landed<(D - 1) * S::FEWEST>();
            S::multiply(mine + place * S::STEP, column < n ? column : 0, term, kb, A.k_bytes, acc);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the place has been read
            issue();
            place = place + 1 == D ? 0 : place + 1;
            if (++kb == A.kb || i + 1 == end) {
                acc[0] = over_terms<3>(acc[0]);
                if (term == 0 && column < n) {
                    float * to = head ? &heads[wave][column * 16] : y + list[s * A.capacity + column] * 16;
                    *reinterpret_cast<f32x4 *>(to + 4 * q) = acc[0];
                }
                if (head && lane == 0) head_slot[wave] = s;
                acc[0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                head = false;
                kb = 0;
                if (i + 1 < end) n = counts[++s];
            }
        }
        landed<0>();                                         // no load may land after the workgroup has ended
    }
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < W; ++w) {
            const int s = head_slot[w];
            if (s < 0) continue;
            for (int i = lane; i < counts[s] * 16; i += 64) y[list[s * A.capacity + (i >> 4)] * 16 + (i & 15)] += heads[w][i];
        }
    }
    __syncthreads();
    if (!puts) return;
    float v = 0.0f;
    auto add = [&](int k, float scale, float bias) __attribute__((always_inline)) {   // the ranks in their order
        const int entry = mine_t * A.top_k + k, expert = ids[entry];
        if (expert == -1) return;
        float e = static_cast<unsigned>(expert) < static_cast<unsigned>(A.n_expert) ? y[entry * 16 + (lane & 15)] : __builtin_nanf("");
        if constexpr (kScaled) e *= scale;
        if (A.bias) e += bias;
        v += shares[entry] * e;
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (k < A.top_k) add(k, scales[k], biases[k]);
    for (int k = AHEAD; k < A.top_k; ++k) {
        const int64_t at = row_at(k);
        add(k, kScaled && at >= 0 ? A.ws[at] : 1.0f, A.bias && at >= 0 ? A.bias[at] : 0.0f);
    }
    const int64_t at = static_cast<int64_t>(mine_t) * A.rows + mine_n;
    if (A.out_type == VBM_TYPE_F32) static_cast<float *>(A.out)[at] = v;
    else if (A.out_type == VBM_TYPE_BF16) static_cast<__bf16 *>(A.out)[at] = static_cast<__bf16>(v);
    else static_cast<_Float16 *>(A.out)[at] = static_cast<_Float16>(v);
}

struct FewCall {
    int kind, x_type;
    FewArgs up, down;              // of the two launches
    int64_t slots;                 // at most
    double expected;               // experts that are hit
    size_t h_at, bytes;            // of the workspace
};

int64_t align_256(int64_t n) { return (n + 255) / 256 * 256; }

// Checks everything but the buffers of one call.
FewCall few_call(const vbm_moe_few_desc * d, int64_t n_tokens) {
    require(d != nullptr, "null description");
    const vbm_weights & g = d->gate_up, & w = d->down;
    const bool bytes = one_byte(g.type);
    require(bytes || g.type == VBM_TYPE_F16 || g.type == VBM_TYPE_BF16, "weights must be I8, F8_E4M3, F16 or BF16");
    require(w.type == g.type, "gate_up and down must be of one type");
    require(g.n_groups > 0 && g.n_groups <= kMaxRouteExperts && w.n_groups == g.n_groups, "gate_up and down need the same number of experts, 1..1024");
    require(g.k > 0 && g.k < (int64_t{1} << 23) && w.k > 0 && w.k < (int64_t{1} << 23), "rows and k out of range");
    require(w.rows == g.k && g.rows == 2 * w.k, "gate_up must be [2 * I][H] and down [H][I]");
    require(g.k % (bytes ? 16 : 8) == 0 && w.k % (bytes ? 16 : 8) == 0, bytes ? "H and I must be multiples of 16" : "H and I must be multiples of 8");
    require(g.data && w.data && (!bytes || (g.scales && w.scales)), "null weights");
    auto at = [](const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    require(at(g.data, 16) && at(w.data, 16), "weights must be 16-byte aligned");
    require(at(g.scales, 4) && at(w.scales, 4) && at(g.bias, 4) && at(w.bias, 4), "buffers must be aligned to their types");
    require(d->activation == VBM_ACT_SILU || d->activation == VBM_ACT_SWIGLU_OAI, "unknown activation");
    require(d->top_k > 0 && d->top_k <= g.n_groups && d->top_k <= 64, "top_k must be 1..n_experts, at most 64");
    require(n_tokens >= 0 && n_tokens <= kMostTokens && n_tokens * d->top_k <= kMostEntries, "at most 16 tokens and 128 (token, rank) pairs");

    FewCall c{};
    c.kind = g.type;
    FewArgs & a = c.up;
    a.w = static_cast<const uint8_t *>(g.data);
    a.ws = g.scales;
    a.bias = g.bias;
    a.n_tokens = static_cast<int>(n_tokens);
    a.top_k = static_cast<int>(d->top_k);
    a.n_expert = static_cast<int>(g.n_groups);
    a.entries = a.n_tokens * a.top_k;
    a.inter = static_cast<int>(w.k);
    a.activation = d->activation;
    a.alpha = d->alpha;
    a.limit = d->limit;
    const int size = bytes ? 1 : 2;
    a.rows = static_cast<int>(g.rows);
    a.k_bytes = static_cast<int>(g.k) * size;
    a.kb = (a.k_bytes + 127) / 128;
    a.h_kb = (a.inter * size + 127) / 128;
    a.h_step = bytes ? Rows<VBM_TYPE_I8, kTerms>::BYTES : Rows<VBM_TYPE_BF16, kTerms>::BYTES;
    FewArgs & b = c.down;
    b = a;
    b.w = static_cast<const uint8_t *>(w.data);
    b.ws = w.scales;
    b.bias = w.bias;
    b.rows = static_cast<int>(w.rows);
    b.k_bytes = a.inter * size;
    b.kb = a.h_kb;
    // experts that are hit if every token takes top_k of them at random
    double missed = 1.0;
    for (int64_t t = 0; t < n_tokens; ++t) missed *= 1.0 - static_cast<double>(a.top_k) / a.n_expert;
    c.expected = std::max(1.0, a.n_expert * (1.0 - missed));
    c.slots = a.entries;
    c.h_at = static_cast<size_t>(2 * align_256(4 * kMostEntries));
    c.bytes = c.h_at + static_cast<size_t>(a.entries) * a.h_kb * a.h_step;
    return c;
}

// All workgroups at once, two a CU (2048 waves): four or two waves a tile where there are few (384 tiles, one token: 13 us either way, 16 unshared), several
// tiles a wave where there are many, so that fewer workgroups route and start. 131 layers of 141 to 21674 tiles, all weights, H of 1024 to 4096, by
// every choice: this one takes 3 % longer than the best on average, 16 % at most. us a layer by 1, 2, 3, 4 tiles a wave: 21674 tiles, FP8, H 1024: 471, 396, 377, 366 (4 are
// taken); 10550, FP8, H 2048: 267, 245, 235, 237 (4); 5076, bf16, H 2880: 273, 282, 269, 296 (3); 9172, FP8, H 2880: 326, 311, 330, 352 (4); 4033,
// integers, H 4096: 186, 197, 174, 193 (2). Waves a tile: 305 tiles of integers 24 by four, 27 by two, 34 by one; 1609 101, 81, 73; 508 42, 37, 40 (four).
template <int KIND, int X>
void launch_gate_up(const FewCall & c, hipStream_t stream) {
    using R = Rows<KIND, X>;
    FewArgs a = c.up;
    a.capacity = std::min(R::MOST, a.n_tokens);
    const int64_t row_tiles = (a.inter + 15) / 16;
    const double tiles = c.expected * static_cast<double>(row_tiles);
    auto go = [&](auto nb_c, auto share_c) {
        constexpr int NB = decltype(nb_c)::value, SHARE = decltype(share_c)::value, AT_ONCE = 4 / SHARE;
        a.tiles = SHARE == 1 ? static_cast<int>(std::max(1.0, std::min<double>(kMostTiles, std::ceil(tiles / 2048 - 0.25)))) : 1;
        a.row_units = static_cast<int>((row_tiles + AT_ONCE * a.tiles - 1) / (AT_ONCE * a.tiles));
        const int64_t blocks = c.slots * a.row_units;
        require(blocks < (int64_t{1} << 24), "too many outputs for one launch");
        hipLaunchKernelGGL((few_gate_up_kernel<KIND, X, NB, SHARE>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
        check_hip(hipGetLastError(), "few tokens gate_up launch");
    };
    auto shape = [&](auto nb_c) {
        if (tiles > 1024) go(nb_c, std::integral_constant<int, 1>{});
        else if (tiles > 512) go(nb_c, std::integral_constant<int, 2>{});
        else go(nb_c, std::integral_constant<int, 4>{});
    };
    const int nb = R::loads(a.capacity);
    if (nb == 1) return shape(std::integral_constant<int, 1>{});
    if constexpr (R::loads(R::MOST) >= 2) {
        if (nb == 2) return shape(std::integral_constant<int, 2>{});
    }
    if constexpr (R::loads(R::MOST) >= 3) shape(std::integral_constant<int, 3>{});
}

template <int KIND>
void launch_down(const FewCall & c, hipStream_t stream) {
    using R = Rows<KIND, kTerms>;
    FewArgs b = c.down;
    b.capacity = std::min(R::MOST, b.n_tokens);
    auto go = [&](auto nb_c) {
        hipLaunchKernelGGL((few_down_kernel<KIND, decltype(nb_c)::value>), dim3(static_cast<unsigned>((b.rows + 15) / 16)), dim3(512), 0, stream, b);
        check_hip(hipGetLastError(), "few tokens down launch");
    };
    const int nb = R::loads(b.capacity);
    if (nb == 1) return go(std::integral_constant<int, 1>{});
    if (nb == 2) return go(std::integral_constant<int, 2>{});
    if constexpr (R::loads(R::MOST) >= 3) go(std::integral_constant<int, 3>{});
}

template <int KIND>
void launch_few(const FewCall & c, hipStream_t stream) {
    if (c.x_type == VBM_TYPE_F32) launch_gate_up<KIND, VBM_TYPE_F32>(c, stream);
    else if (c.x_type == VBM_TYPE_F16) launch_gate_up<KIND, VBM_TYPE_F16>(c, stream);
    else launch_gate_up<KIND, VBM_TYPE_BF16>(c, stream);
    launch_down<KIND>(c, stream);
}

}  // namespace
}  // namespace vbm

using namespace vbm;

extern "C" {

vbm_status vbm_moe_few_workspace(const vbm_moe_few_desc * desc, int64_t n_tokens, size_t * bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null bytes");
        *bytes = few_call(desc, n_tokens).bytes;
    });
}

vbm_status vbm_moe_few_forward(const vbm_moe_few_desc * desc, int x_type, const void * x, const float * logits, int32_t * ids, float * weights,
                               int64_t n_tokens, int out_type, void * out, void * workspace, size_t workspace_bytes, void * stream) {
    return guarded([&] {
        FewCall c = few_call(desc, n_tokens);
        auto type = [](int t) { return t == VBM_TYPE_F32 || t == VBM_TYPE_F16 || t == VBM_TYPE_BF16; };
        require(type(x_type), "x must be F32, F16 or BF16");
        require(type(out_type), "out must be F32, F16 or BF16");
        if (n_tokens == 0) return;
        auto at = [](const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
        require(x && out && workspace, "null buffer");
        require(logits || (ids && weights), "neither logits nor ids and weights");
        require(at(x, 16) && at(workspace, 16), "x and workspace must be 16-byte aligned");
        require(at(out, out_type == VBM_TYPE_F32 ? 4 : 2) && at(logits, 4) && at(ids, 4) && at(weights, 4), "buffers must be aligned to their types");
        require(workspace_bytes >= c.bytes, "workspace too small");
        uint8_t * space = static_cast<uint8_t *>(workspace);
        int32_t * chosen = ids ? ids : reinterpret_cast<int32_t *>(space);
        float * shares = weights ? weights : reinterpret_cast<float *>(space + align_256(4 * kMostEntries));
        c.x_type = x_type;
        c.up.x = x;
        c.up.logits = logits;
        c.up.ids = c.down.ids = chosen;
        c.up.ids_out = chosen;
        c.up.weights_out = shares;
        c.up.h = space + c.h_at;
        c.down.x = space + c.h_at;
        c.down.weights = shares;
        c.down.out = out;
        c.down.out_type = out_type;
        if (c.kind == VBM_TYPE_F8_E4M3) launch_few<VBM_TYPE_F8_E4M3>(c, as_stream(stream));
        else if (c.kind == VBM_TYPE_I8) launch_few<VBM_TYPE_I8>(c, as_stream(stream));
        else if (c.kind == VBM_TYPE_F16) launch_few<VBM_TYPE_F16>(c, as_stream(stream));
        else launch_few<VBM_TYPE_BF16>(c, as_stream(stream));
    });
}

}  // extern "C"
