// What the dense attention kernels share: the score rule, which keys a row sees, the matrix-core
// operand types and the partial results of a split key range with their join.
#pragma once

#include <math.h>

#include <type_traits>

#include "common.h"

namespace pqhsa {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// never quite zero: an infinite partial sum stays one under any other base
__device__ inline float exp2_something(float x) { return fmaxf(exp2_fast(x), 0x1p-149f); }

// Weights are 2^(z2 - m) for a running base m, a former maximum, which is only moved (and what was summed
// under it rescaled) when a score passes it by more than a slack, in log2 units: most tiles need no exchange
// between lanes at all.  fp32 and bf16 hold such weights at any size.
constexpr float kMaxSlack = 8.0f;
// fp16 does not: below 2^-14 it has steps of 2^-24, whatever the size.  So its weights are 2^(z2 - m + 13), at most
// 2^15, and the base also moves DOWN where all of a tile's scores for a row lie more than a drop (of the
// kernel's) below it: keys far below the largest one, which only count together (those behind an attention
// sink, say), then have the same bits.  It stays within 2^40 of the row's maximum: what is rounded away below that is
// under 2^31 keys * 2^-78 * 2^16, less than fp16 outputs resolve.  Sums hold 2^15 * 2^40 * 2^16 * 2^31 keys.
// A new maximum becomes the base itself, up to 2^-15 (the weight of a key that stands out is then a power of two,
// and not rounded); all other moves are by whole numbers, and exact, as multiples of 2^-14 below 2^10 are.
constexpr float kHalfSlack = 2.0f, kHalfShift = 13.0f, kHalfFall = 40.0f;
template <int DT>
struct WeightBase {
    static constexpr bool kHalf = DT == PQHSA_F16;
    static constexpr float kSlack = kHalf ? kHalfSlack : kMaxSlack;
    float m = -INFINITY;                                 // the base; -inf: no visible key so far
    float most = -INFINITY;                              // fp16: the row's maximum so far
    __device__ inline bool raises(float top) const { return top > m + kSlack; }
    __device__ inline bool falls(float top, float drop) const { return kHalf && top < m - drop; }
    // moves to a tile's maximum `top` of the row; returns what sums so far are multiplied by
    __device__ inline float move(float top, float drop) {
        if constexpr (kHalf) {
            if (top > most) {
                const float to = (top + 768.0f) - 768.0f, f = exp2_fast(m - to);   // (the sum drops what is below 2^-14)
                m = to;
                most = top;
                return f;
            }
            float by = 0.0f;                             // upwards
            if (top > m) by = ceilf(top - m);
            else if (falls(top, drop) && top > -INFINITY && m < INFINITY) by = -fminf(floorf(m - top), floorf(m - most + kHalfFall));
            m += by;
            return __builtin_ldexpf(1.0f, -(int)by);
        } else {
            const float to = fmaxf(m, top), f = m == to ? 1.0f : exp2_fast(m - to);
            m = to;
            return f;
        }
    }
    // what exponents are taken relative to
    __device__ inline float origin() const { return m == -INFINITY ? 0.0f : kHalf ? m - kHalfShift : m; }
    // At the end: the base m to which a sum of weights belongs once it is multiplied by what this returns (fp16: brought
    // to [1/2, 1), so that m + log2 of it, the log-sum-exp, is rounded once).
    __device__ inline float settle(float sum) {
        if constexpr (!kHalf) return 1.0f;
        const int e = __builtin_amdgcn_frexp_expf(sum);  // (0 for zero, infinities and NaN)
        m += (float)e - kHalfShift;
        return __builtin_ldexpf(1.0f, -e);
    }
};

// ---- score rule ---------------------------------------------------------------------
// Scores are kept in units of log2: z2 = log2(e) * z, so that a weight is one exp2.
struct ScoreArgs {
    float scale2;             // scale * log2(e)
    float in_cap, cap2;       // softcap: z2 = cap2 * tanh(dot * in_cap); in_cap = scale / softcap, cap2 = softcap * log2(e)
    int capped;
    int window;               // 0: none
    int prefix;               // of every sequence when prefixes is NULL
    const int32_t *prefixes;  // [B]
    const float *slopes;      // [H * G]
    const int32_t *docs;      // [B, docs_stride]
    int64_t docs_stride;
};

inline ScoreArgs make_score(const pqhsa_score *s) {
    ScoreArgs a = {};
    a.scale2 = s->scale * kLog2e;
    a.capped = s->softcap > 0.0f;
    if (a.capped) {
        a.in_cap = s->scale / s->softcap;
        a.cap2 = s->softcap * kLog2e;
    }
    a.window = s->window;
    a.prefix = s->prefix;
    a.prefixes = s->prefixes;
    a.slopes = s->slopes;
    a.docs = s->docs;
    a.docs_stride = s->docs_stride;
    return a;
}

int validate_score(const pqhsa_score *s, int n_max, const char *what);
int validate_mass(const pqhsa_mass *m, int n_max, const char *what);
// host-side bound of the keys a row at the end of a sequence can see
int64_t visible_bound(const pqhsa_score *s, int64_t n_max);

// tanh to fp32 accuracy relative to the result.  Up to 1: x + x y p(y) with y = x^2, p the polynomial that meets
// (tanh(x) / x - 1) / y at the seven Chebyshev points of y in [0, 1] (evaluated in fp32, 9e-8 of the result at most:
// 1.5 half steps).  Above: (1 - e) / (1 + e) with e = exp(-2 |x|) <= 0.14.  inf gives 1, NaN stays NaN.
constexpr float kTanhSmall = 1.0f;
__device__ inline float tanh_small(float x) {
    const float y = x * x;
    float p = -0.000420695494f;
    p = fmaf(p, y, 0.00251045933f);
    p = fmaf(p, y, -0.0082189219f);
    p = fmaf(p, y, 0.0216601154f);
    p = fmaf(p, y, -0.0539347889f);
    p = fmaf(p, y, 0.133331285f);
    p = fmaf(p, y, -0.333333313f);
    return fmaf(p * y, x, x);
}
__device__ inline float tanh_score(float x) {
    const float e = exp2_fast(-2.0f * kLog2e * fabsf(x));
    const float big = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    return fabsf(x) < kTanhSmall ? tanh_small(x) : copysignf(big, x);
}

__device__ inline int sequence_length(const int32_t *seq_lens, int b, int n_max) {
    return min(max(seq_lens[b], 0), n_max);
}
__device__ inline int sequence_prefix(const ScoreArgs &s, int b) {
    return max(s.prefixes ? s.prefixes[b] : s.prefix, 0);
}

// Byte offset of K/V row (b, h, pos), or -1 where the block table names a block outside the cache (such
// a key is treated as masked).
__device__ inline int64_t checked_row_bytes(const KvView &v, int blocks, int b, int h, int pos) {
    int64_t off;
    if (v.paged) {
        const int blk = pos / v.block_size;
        const int row = pos - blk * v.block_size;
        const int phys = v.block_table[(int64_t)b * v.max_blocks + blk];
        if (phys < 0 || phys >= blocks) return -1;
        off = (int64_t)phys * v.stride_block + (int64_t)row * v.stride_tok + (int64_t)h * v.stride_head;
    } else {
        off = (int64_t)b * v.stride_seq + (int64_t)pos * v.stride_tok + (int64_t)h * v.stride_head;
    }
    return off * v.esize;
}

// ---- matrix-core operands of the 2-byte types -----------------------------------------
template <int DT>
struct Half16;
template <>
struct Half16<PQHSA_BF16> {
    typedef bf16x8 vec8;
    static __device__ inline f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
    static __device__ inline f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
    // two floats rounded to the type (to nearest even), the first in the low half
    static __device__ inline uint32_t pack(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
    }
    static __device__ inline float low(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ inline float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <>
struct Half16<PQHSA_F16> {
    typedef f16x8 vec8;
    static __device__ inline f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
    static __device__ inline f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
    }
    static __device__ inline uint32_t pack(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, f16x2));
    }
    static __device__ inline float low(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
    static __device__ inline float high(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
};

// w's two halves (one fp32 number) with infinite and NaN ones set to zero
template <int DT>
__device__ inline uint32_t finite_part(uint32_t w) {
    if constexpr (DT == PQHSA_F32) {
        return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    } else {
        constexpr uint32_t e = DT == PQHSA_BF16 ? 0x7f80u : 0x7c00u;
        return ((w & e) == e ? 0u : w & 0xffffu) | ((w & (e << 16)) == (e << 16) ? 0u : w & 0xffff0000u);
    }
}

// ---- partial results of a split key range, and their join ---------------------------------
// Row r (query row * heads + head) of split s: part_o[(r * splits + s) * 128 ..] the weighted value sum
// relative to the maximum m, part_ml[r * splits + s] = (m, l); a split without a visible key has m = -inf,
// l = 0 and no sums.
struct JoinArgs {
    const float *part_o;
    const float2 *part_ml;
    int splits;
    int heads;                 // query heads H * G
    char *out;
    int64_t out_row, out_head; // strides in elements
    float *lse;                // [rows, heads] or NULL
    float2 *row_ml;            // [rows, heads] maximum and sum, or NULL
    const int32_t *row_count;  // rows in use (device), NULL: all
};
int launch_join(const JoinArgs &a, int dtype, int64_t rows, hipStream_t stream);

}  // namespace pqhsa
