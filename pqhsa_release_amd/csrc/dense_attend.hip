// Dense attention of one new token per sequence over its whole (paged) cache.
//
//   z_j = score(q, k_j),  o = sum_j exp(z_j) v_j / sum_j exp(z_j),  lse = log sum_j exp(z_j)
//
// Every K and V row has to be read once and nothing else is large: 512 bytes per key and KV head in the
// 2-byte types against 4 * 128 * G operations, far below what the matrix cores do in that time.  So
// the kernel is built around the loads.  A workgroup takes one chunk of keys of one (sequence, KV head)
// for all G query rows of the group; its four waves walk the chunk independently of each other, 32 keys
// (16 in fp32) a step, K and V straight from memory into the registers the matrix cores read, the next
// step's 16 KB requested before this step is computed.  No LDS is in that loop but the list of row
// addresses, which the workgroup resolves through the block table beforehand.
//
//   S^T = K Q^T  (16 keys x 16 query rows): rows of the tile are assigned to keys so that a lane ends up
//     with the scores of 8 consecutive keys of one query row, which is exactly what the second product's
//     weight operand holds: no exchange between lanes.
//   O^T = V^T P  (16 dims x 16 query rows): a lane loads 16 bytes of each of its 8 keys' V rows (16 lanes
//     read a whole row) and transposes the 8 x 8 block with byte permutes.
//
// The weights enter the second product as the sum of two 2-byte numbers (the rounded weight and its
// rounded remainder), because a second product costs nothing here: 2^-17 of a weight is rounded away at most in
// bf16, 2^-22 in fp16 (there by a base near the step's own scores, and a remainder of its own scale).
//
// Measured (bf16, 16-token pages): 4 x 131 072 tokens of 8 KV heads 392 us, 5.5 TB/s; 1 x 32 768 34 us, 4 of them
// the join (30 us called again and again on one cache of 134 MB, part of which then stays in the last-level
// cache); 16 x 700 12 to 15 us, which are two launches and the chain length -> block -> row -> partial -> output, not
// bytes.  The launch is sized by the bound of the lengths: 1 x 8 192 takes 15 us under its own, 33 under 131 072.
#include "dense_common.h"

namespace pqhsa {

constexpr int kDenseThreads = 256;
constexpr int kDenseWaves = kDenseThreads / kWave;
constexpr int kDenseRows = 16;         // query rows of a matrix tile
constexpr int kDenseChunkMin = 128, kDenseChunkMax = 4096;
// fp16: the remainder enters times 2^11 (at most 2^14) and is summed by itself, so that a weight, at most 2^15, is off
// by 2^-22 of itself or by 2^-36.  A step whose 32 keys all lie more than the drop (log2) below the base moves it:
// otherwise its largest weight is 2^(13 - 22) at least, and 32 roundings of 2^-36 are 2^-22 of that.
constexpr float kLowScale = 2048.0f, kDenseDrop = 22.0f;
constexpr int kMassKeys = 1024;        // keys per workgroup of the weight accumulation

struct DenseArgs {
    const char *q;
    int64_t q_row, q_head;             // strides in elements
    char *out;
    int64_t out_row, out_head;
    float *lse;
    KvView kv;
    int blocks, B, H, G;
    const int32_t *seq_lens;
    int n_max;
    ScoreArgs score;
    int chunk, splits;
    float *part_o;                     // [B * H * G, splits, 128]
    float2 *part_ml;                   // [B * H * G, splits]
    float *scores;                     // [B * H * G, score_stride] z2 of every enumerated key, or NULL
    int64_t score_stride;
};

// The keys a row at the end of a sequence of `len` tokens sees by position: [0, prefix) and [start, len).
// They are numbered 0 .. count - 1 in ascending order.
struct KeyRange {
    int first, gap, count;             // key of number v: v < first ? v : v + gap
    __device__ inline int key(int v) const { return v < first ? v : v + gap; }
};
__device__ inline KeyRange key_range(const ScoreArgs &s, int b, int len) {
    const int start = s.window > 0 ? max(0, len - s.window) : 0;
    const int prefix = min(sequence_prefix(s, b), len);
    KeyRange r;
    if (prefix >= start) {
        r.first = len; r.gap = 0; r.count = len;
    } else {
        r.first = prefix; r.gap = start - prefix; r.count = prefix + (len - start);
    }
    return r;
}

template <int DT, bool SCORES>
__global__ __launch_bounds__(kDenseThreads, 2) void dense_attend_kernel(DenseArgs a) {
    constexpr bool kF32 = DT == PQHSA_F32;
    constexpr int kTiles = kF32 ? 1 : 2;                 // 16-key tiles per step
    constexpr int kPer = 4 * kTiles;                     // keys per lane and step
    constexpr int kStep = 16 * kTiles;
    constexpr int kSlices = kF32 ? 8 : 4;                // 16-byte loads of a lane per key row
    constexpr int kVWords = kF32 ? 2 : 1;                // 16-byte loads of a lane per value row
    extern __shared__ __align__(16) char lds[];
    int64_t *offs = reinterpret_cast<int64_t *>(lds);    // [chunk] byte offsets of the rows, -1: masked

    const int tid = threadIdx.x, lane = tid & 63, wave = tid / kWave;
    const int n = lane & 15, kg = lane >> 4;             // query row, group of keys
    const int bh = blockIdx.x, split = blockIdx.y;
    const int b = bh / a.H, h = bh - b * a.H;
    const int len = sequence_length(a.seq_lens, b, a.n_max);
    const KeyRange range = key_range(a.score, b, len);
    const int v0 = split * a.chunk;
    const int count = min(a.chunk, range.count - v0);
    const int g = n < a.G ? n : 0;                       // lanes without a query row repeat row 0

    if (count <= 0) {                                    // nothing in this chunk
        if (tid < a.G) {
            const int64_t r = (int64_t)bh * a.G + tid;
            if (a.splits > 1) a.part_ml[r * a.splits + split] = make_float2(-INFINITY, 0.0f);
            else {
                if (a.part_ml) a.part_ml[r] = make_float2(-INFINITY, 0.0f);
                if (a.lse) a.lse[r] = -INFINITY;
            }
        }
        if (a.splits == 1)
            for (int x = tid; x < a.G * kD; x += kDenseThreads)
                store1<DT>(a.out + ((int64_t)b * a.out_row + (int64_t)(h * a.G + x / kD) * a.out_head) * a.kv.esize, x % kD, 0.0f);
        return;
    }

    // query rows as the second operand of the score product: lane (n, kg) holds row n
    uint4 qf[kSlices];
    {
        const char *qrow = a.q + ((int64_t)b * a.q_row + (int64_t)(h * a.G + g) * a.q_head) * a.kv.esize;
#pragma unroll
        for (int u = 0; u < kSlices; ++u) qf[u] = *reinterpret_cast<const uint4 *>(qrow + u * 64 + kg * 16);
    }
    // addresses of the chunk's rows
    const int padded = (count + kDenseWaves * kStep - 1) / (kDenseWaves * kStep) * (kDenseWaves * kStep);
    const int32_t *docs = a.score.docs ? a.score.docs + (int64_t)b * a.score.docs_stride : nullptr;
    const int doc = docs ? docs[len - 1] : 0;
    for (int v = tid; v < padded; v += kDenseThreads) {
        int64_t off = -1;
        if (v < count) {
            const int pos = range.key(v0 + v);
            if (!docs || docs[pos] == doc) off = checked_row_bytes(a.kv, a.blocks, b, h, pos);
        }
        offs[v] = off;
    }
    const float slope2 = a.score.slopes ? a.score.slopes[h * a.G + g] * kLog2e : 0.0f;
    __syncthreads();

    uint4 kf[kTiles][kSlices], vf[kPer][kVWords];
    auto request = [&](int at) {                         // the step at local key `at`
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            // row n of tile t is the key that puts 8 (4) consecutive keys into a lane's scores
            const int64_t off = offs[at + (n >> 2) * kPer + t * 4 + (n & 3)];
            const char *p = a.kv.k_base + (off < 0 ? 0 : off) + kg * 16;
#pragma unroll
            for (int u = 0; u < kSlices; ++u) kf[t][u] = *reinterpret_cast<const uint4 *>(p + u * 64);
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int64_t off = offs[at + kg * kPer + e];
            const char *p = a.kv.v_base + (off < 0 ? 0 : off) + n * (16 * kVWords);
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vf[e][w] = *reinterpret_cast<const uint4 *>(p + 16 * w);
        }
    };

    WeightBase<DT> base;
    float l;
    f32x4 acc[8];                                        // dim (kg * 4 + r) * 8 + d of query row n in acc[d][r]
    f32x4 rem[base.kHalf ? 8 : 1];                       // fp16: sums of the scaled remainders
    // A remainder of zero or below turns an infinite value into NaN, and so does a weight too small for its type.
    // The walk is made without a thought for that; a wave whose sums are not all finite makes it again, with such
    // values set aside and summed by themselves (all rows see the same keys, and no weight of theirs is nothing).
    auto walk = [&](auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        base = WeightBase<DT>();
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (base.kHalf) {
#pragma unroll
            for (int d = 0; d < 8; ++d) rem[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (!CAREFUL && wave * kStep < padded) request(wave * kStep);
        for (int at = wave * kStep; at < padded; at += kDenseWaves * kStep) {
            uint4 kc[kTiles][kSlices], vc[kPer][kVWords];
            if (CAREFUL) request(at);                    // (nothing in flight: a walk for few)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int u = 0; u < kSlices; ++u) kc[t][u] = kf[t][u];
#pragma unroll
            for (int e = 0; e < kPer; ++e)
#pragma unroll
                for (int w = 0; w < kVWords; ++w) vc[e][w] = vf[e][w];
            if (!CAREFUL && at + kDenseWaves * kStep < padded) request(at + kDenseWaves * kStep);

            f32x4 s[kTiles];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                s[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < kSlices; ++u) {
                    if constexpr (kF32) {
                        const f32x4 x = __builtin_bit_cast(f32x4, kc[t][u]), y = __builtin_bit_cast(f32x4, qf[u]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[c], y[c], s[t], 0, 0, 0);
                    } else {
                        s[t] = Half16<DT>::mfma16(kc[t][u], qf[u], s[t]);
                    }
                }
            }
            // (one branch a rule, not one a key)
            float z[kPer];
            bool live[kPer];
            float top = -INFINITY;
            if (a.score.capped) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) z[e] = a.score.cap2 * tanh_score(s[e >> 2][e & 3] * a.score.in_cap);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) z[e] = s[e >> 2][e & 3] * a.score.scale2;
            }
            if (a.score.slopes) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) z[e] -= slope2 * (float)(len - 1 - range.key(v0 + at + kg * kPer + e));
            }
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                live[e] = offs[at + kg * kPer + e] >= 0;
                z[e] = live[e] ? z[e] : -INFINITY;
                top = fmaxf(top, z[e]);
            }
            if constexpr (SCORES) {
                // Every lane stores, the ones that repeat row 0 what row 0's lane does: with a branch around them the
                // compiler could not count the stores, and waited for them where it waits for the next step's rows
                // (330 instead of 322 us in 16 sequences of 16 384 to 65 536 keys).
                float4 *p = reinterpret_cast<float4 *>(a.scores + ((int64_t)bh * a.G + g) * a.score_stride + v0 + at + kg * kPer);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) p[t] = make_float4(z[4 * t], z[4 * t + 1], z[4 * t + 2], z[4 * t + 3]);
            }
            uint64_t low = __ballot(base.falls(top, kDenseDrop));
            low &= low << 32 | low >> 32;                    // in all four lanes of a row
            low &= low << 16 | low >> 48;
            if (__ballot(base.raises(top)) | low) {          // a row's base moves: once or a few times per chunk
                top = fmaxf(top, __shfl_xor(top, 16, kWave));
                top = fmaxf(top, __shfl_xor(top, 32, kWave));
                const float f = base.move(top, kDenseDrop);
                l *= f;
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[d] *= f;
                if constexpr (base.kHalf) {
#pragma unroll
                    for (int d = 0; d < 8; ++d) rem[d] *= f;
                }
            }
            if constexpr (CAREFUL) {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
#pragma unroll
                    for (int w = 0; w < kVWords; ++w)
                        vc[e][w] = make_uint4(finite_part<DT>(vc[e][w].x), finite_part<DT>(vc[e][w].y), finite_part<DT>(vc[e][w].z), finite_part<DT>(vc[e][w].w));
            }
            const float origin = base.origin();
            float p[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                p[e] = exp2_fast(z[e] - origin);
                l += p[e];
#pragma unroll
                for (int w = 0; w < kVWords; ++w)
                    if (!live[e]) vc[e][w] = make_uint4(0u, 0u, 0u, 0u);  // whatever lies there must not reach the product
            }
            if constexpr (kF32) {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        const f32x4 x = __builtin_bit_cast(f32x4, vc[e][d >> 2]);
                        acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[d & 3], p[e], acc[d], 0, 0, 0);
                    }
            } else {
                uint4 hi, lo;
                uint32_t *hw = reinterpret_cast<uint32_t *>(&hi), *lw = reinterpret_cast<uint32_t *>(&lo);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    hw[w] = Half16<DT>::pack(p[2 * w], p[2 * w + 1]);
                    const float x = p[2 * w] - Half16<DT>::low(hw[w]), y = p[2 * w + 1] - Half16<DT>::high(hw[w]);
                    lw[w] = base.kHalf ? Half16<DT>::pack(kLowScale * x, kLowScale * y) : Half16<DT>::pack(x, y);
                }
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    uint32_t t[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t x = reinterpret_cast<const uint32_t *>(&vc[2 * w][0])[d >> 1];
                        const uint32_t y = reinterpret_cast<const uint32_t *>(&vc[2 * w + 1][0])[d >> 1];
                        t[w] = __builtin_amdgcn_perm(y, x, d & 1 ? 0x07060302u : 0x05040100u);
                    }
                    const uint4 vt = make_uint4(t[0], t[1], t[2], t[3]);
                    acc[d] = Half16<DT>::mfma16(vt, hi, acc[d]);
                    if constexpr (base.kHalf) rem[d] = Half16<DT>::mfma16(vt, lo, rem[d]);
                    else acc[d] = Half16<DT>::mfma16(vt, lo, acc[d]);
                }
            }
        }
    };
    walk(std::false_type{});
    float zero[4] = {};                                  // NaN where a sum is not finite
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            zero[r] = __builtin_fmaf(acc[d][r], 0.0f, zero[r]);
            if constexpr (base.kHalf) zero[r] = __builtin_fmaf(rem[d][r], 0.0f, zero[r]);
        }
    if (__builtin_expect(__ballot(zero[0] + zero[1] + (zero[2] + zero[3]) != 0.0f) != 0, 0)) {
        walk(std::true_type{});
        float odd[8] = {};                               // dims n * 8 + d of this lane's keys
#pragma unroll 1
        for (int at = wave * kStep; at < padded; at += kDenseWaves * kStep)
#pragma unroll 1
            for (int e = 0; e < kPer; ++e) {
                const int64_t off = offs[at + kg * kPer + e];
                if (off < 0) continue;
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const float x = load1<DT>(a.kv.v_base + off, n * 8 + d);
                    if (!(fabsf(x) < INFINITY)) odd[d] += x;
                }
            }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            odd[d] += __shfl_xor(odd[d], 16, kWave);
            odd[d] += __shfl_xor(odd[d], 32, kWave);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[d][r] += __shfl(odd[d], kg * 4 + r, kWave);
        }
    }
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    const float settled = base.settle(l);
    l *= settled;
    if constexpr (base.kHalf) {
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = (acc[d] + rem[d] * (1.0f / kLowScale)) * settled;
    }

    // the four waves' results under the chunk's maximum
    __syncthreads();                                     // the address list is no longer read
    float *red_m = reinterpret_cast<float *>(lds);       // [waves][16]
    float *red_l = red_m + kDenseWaves * kDenseRows;
    float *red_o = red_l + kDenseWaves * kDenseRows;     // [waves][G][128]
    if (kg == 0) {
        red_m[wave * kDenseRows + n] = base.m;
        red_l[wave * kDenseRows + n] = l;
    }
    if (n < a.G) {
        float *o = red_o + ((size_t)wave * a.G + n) * kD + kg * 32;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            *reinterpret_cast<float4 *>(o + r * 8) = make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]);
            *reinterpret_cast<float4 *>(o + r * 8 + 4) = make_float4(acc[4][r], acc[5][r], acc[6][r], acc[7][r]);
        }
    }
    __syncthreads();
    for (int x = tid; x < a.G * kD; x += kDenseThreads) {
        const int g = x / kD, d = x % kD;                // (of the output element)
        float top = red_m[g];
#pragma unroll
        for (int w = 1; w < kDenseWaves; ++w) top = fmaxf(top, red_m[w * kDenseRows + g]);
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kDenseWaves; ++w) {
            const float mw = red_m[w * kDenseRows + g];
            const float f = mw == top ? 1.0f : exp2_something(mw - top);   // (a wave without a visible key holds zeros)
            sum += f * red_l[w * kDenseRows + g];
            o += f * red_o[((size_t)w * a.G + g) * kD + d];
        }
        const int64_t r = (int64_t)bh * a.G + g;
        if (a.splits > 1) {
            a.part_o[(r * a.splits + split) * kD + d] = o;
        } else {
            store1<DT>(a.out + ((int64_t)b * a.out_row + (int64_t)(h * a.G + g) * a.out_head) * a.kv.esize, d,
                       sum == 0.0f ? 0.0f : o / sum);
            if (d == 0 && a.lse) a.lse[r] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
        }
        if (d == 0 && a.part_ml) a.part_ml[r * a.splits + split] = make_float2(top, sum);
    }
}

// ---- join of the split partials: one workgroup per row -------------------------------------
// Eight groups of 32 lanes (four dims a lane) take every eighth split, `kBatch` of them at a time with all
// loads in flight at once: the time is one or two round trips to memory.  Each group keeps a running
// maximum and sum; the groups meet in LDS.
template <int DT, int kBatch>
__global__ __launch_bounds__(256) void dense_join_kernel(JoinArgs a) {
    constexpr int kGroups = 8;
    __shared__ float red[kGroups][kD];
    __shared__ float2 red_ml[kGroups];
    const int64_t r = blockIdx.x;
    const int64_t token = r / a.heads;
    if (a.row_count && token >= *a.row_count) return;
    const int tid = threadIdx.x, group = tid / 32, d4 = tid % 32;
    const float2 *ml = a.part_ml + r * a.splits;
    const float *part = a.part_o + r * a.splits * kD + d4 * 4;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = group; s0 < a.splits; s0 += kGroups * kBatch) {
        float2 y[kBatch];
        float4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int s = min(s0 + i * kGroups, a.splits - 1);
            y[i] = ml[s];
            x[i] = *reinterpret_cast<const float4 *>(part + (int64_t)s * kD);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (s0 + i * kGroups >= a.splits) y[i] = make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, y[i].x);
        }
        const float back = m == top ? 1.0f : exp2_something(m - top);
        m = top;
        l *= back;
        o.x *= back; o.y *= back; o.z *= back; o.w *= back;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            // a split without a visible key wrote no sums: whatever lies there is not used
            const bool some = y[i].y != 0.0f;            // (NaN counts)
            const float f = y[i].x == m ? 1.0f : exp2_something(y[i].x - m);
            l += some ? f * y[i].y : 0.0f;
            o.x += some ? f * x[i].x : 0.0f;
            o.y += some ? f * x[i].y : 0.0f;
            o.z += some ? f * x[i].z : 0.0f;
            o.w += some ? f * x[i].w : 0.0f;
        }
    }
    *reinterpret_cast<float4 *>(&red[group][d4 * 4]) = o;
    if (d4 == 0) red_ml[group] = make_float2(m, l);
    __syncthreads();
    if (tid < kD) {
        float2 y[kGroups];
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kGroups; ++w) { y[w] = red_ml[w]; m = fmaxf(m, y[w].x); }
        float x = 0.0f;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < kGroups; ++w) {
            const float f = y[w].x == m ? 1.0f : exp2_something(y[w].x - m);   // (a group without a visible key holds zeros)
            l += f * y[w].y;
            x += f * red[w][tid];
        }
        constexpr int esize = DT == PQHSA_F32 ? 4 : 2;
        store1<DT>(a.out + (token * a.out_row + (r - token * a.heads) * a.out_head) * esize, tid, l == 0.0f ? 0.0f : x / l);
        if (tid == 0 && a.lse) a.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        if (tid == 0 && a.row_ml) a.row_ml[r] = make_float2(m, l);
    }
}

int launch_join(const JoinArgs &a, int dtype, int64_t rows, hipStream_t stream) {
    PQHSA_DISPATCH_DTYPE(dtype,
                         if (a.splits <= 16) hipLaunchKernelGGL((dense_join_kernel<DT, 2>), dim3((unsigned)rows), dim3(256), 0, stream, a);
                         else hipLaunchKernelGGL((dense_join_kernel<DT, 8>), dim3((unsigned)rows), dim3(256), 0, stream, a));
    return check_launch("dense_join");
}

// ---- accumulated weight of every key -----------------------------------------------------
// The group's rows have their (m, l) per split and the scores of all enumerated keys in memory (4 bytes each
// against the 512 of a key's K and V; a second product would read K again): a workgroup folds the
// statistics once and turns 1024 keys' scores into weights.  No atomics: a key has one owner, which adds the
// G rows in order.  16 sequences of 16 384 to 65 536 keys, 4 x 7 heads: 26 us, and 52 us more in the attention for
// writing the scores.
struct MassArgs {
    const float *scores;
    int64_t score_stride;
    const float2 *part_ml;
    int splits, B, H, G;
    const int32_t *seq_lens;
    int n_max;
    ScoreArgs score;
    const float *in;
    float *out;
    int64_t stride;
    float decay;
};

__global__ __launch_bounds__(256) void dense_mass_kernel(MassArgs a) {
    __shared__ float2 row[kDenseRows];                   // maximum and 1 / sum of every row
    const int bh = blockIdx.y, b = bh / a.H;
    const int len = sequence_length(a.seq_lens, b, a.n_max);
    const int j0 = blockIdx.x * kMassKeys;
    if (j0 >= len) return;
    const KeyRange range = key_range(a.score, b, len);
    const int tid = threadIdx.x, lane = tid & 63;
    for (int g = tid / 64; g < a.G; g += 4) {
        const float2 *ml = a.part_ml + ((int64_t)bh * a.G + g) * a.splits;
        float m = -INFINITY, l = 0.0f;
        for (int s = lane; s < a.splits; s += 64) {
            const float2 x = ml[s];
            const float to = fmaxf(m, x.x);
            l = (m == to ? l : l * exp2_fast(m - to)) + (x.x == to ? x.y : x.y * exp2_fast(x.x - to));
            m = to;
        }
        const float top = wave_max_all(m);
        l = wave_total(m == top ? l : l * exp2_fast(m - top));
        if (lane == 0) row[g] = l == 0.0f ? make_float2(INFINITY, 0.0f) : make_float2(top, 1.0f / l);   // +inf: the row gives no weight
    }
    __syncthreads();
    // four keys a thread: 16-byte loads of every row's scores, several rows in flight
    const float *scores = a.scores + (int64_t)bh * a.G * a.score_stride;
    const int64_t at = (int64_t)bh * a.stride;
    const int j = j0 + 4 * tid;
    if (j >= len) return;
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float &to, float z, float2 r) {       // (-inf: masked, also from a row of NaN)
        to += z == -INFINITY ? 0.0f : exp2_fast(z - r.x) * r.y;
    };
    if (a.in) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < len) w[e] = a.decay * a.in[at + j + e];
    }
    const bool front = j + 3 < range.first, behind = j - range.gap >= range.first && (range.gap & 3) == 0;
    if (j + 3 < len && (front || behind)) {
        const float *p = scores + (front ? j : j - range.gap);
#pragma unroll 4
        for (int g = 0; g < a.G; ++g) {
            const float4 z = *reinterpret_cast<const float4 *>(p + g * a.score_stride);
            const float2 r = row[g];
            add(w[0], z.x, r); add(w[1], z.y, r); add(w[2], z.z, r); add(w[3], z.w, r);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int v = j + e < range.first ? j + e : j + e - range.gap;
            if (j + e < len && (j + e < range.first || v >= range.first))
                for (int g = 0; g < a.G; ++g) add(w[e], scores[g * a.score_stride + v], row[g]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < len) a.out[at + j + e] = w[e];
}

// ---- host side ---------------------------------------------------------------------------
int64_t visible_bound(const pqhsa_score *s, int64_t n_max) {
    if (s->window <= 0) return n_max;
    const int64_t prefix = s->prefixes ? n_max : (s->prefix > 0 ? s->prefix : 0);
    return prefix + s->window < n_max ? prefix + s->window : n_max;
}

int validate_score(const pqhsa_score *s, int n_max, const char *what) {
    PQHSA_REQUIRE(s != nullptr, "%s: score rule is NULL", what);
    PQHSA_REQUIRE(n_max <= 0x7fffffff - 65536, "%s: n_max %d is too large (key numbers are 32 bits)", what, n_max);
    PQHSA_REQUIRE(isfinite(s->scale), "%s: scale is not finite", what);
    PQHSA_REQUIRE(isfinite(s->softcap) && s->softcap >= 0.0f, "%s: softcap must be finite and not negative", what);
    PQHSA_REQUIRE(isfinite(s->scale * kLog2e) && isfinite(s->softcap * kLog2e) && (s->softcap == 0.0f || isfinite(s->scale / s->softcap)),
                  "%s: scale %g with softcap %g is out of range", what, s->scale, s->softcap);
    PQHSA_REQUIRE(s->window >= 0 && s->prefix >= 0, "%s: window %d and prefix %d must not be negative", what, s->window, s->prefix);
    PQHSA_REQUIRE(!s->docs || s->docs_stride >= n_max, "%s: docs_stride %lld below n_max %d", what, (long long)s->docs_stride, n_max);
    return PQHSA_OK;
}

int validate_mass(const pqhsa_mass *m, int n_max, const char *what) {
    if (!m) return PQHSA_OK;
    PQHSA_REQUIRE(m->out != nullptr, "%s: mass without an output", what);
    PQHSA_REQUIRE(m->stride >= n_max, "%s: mass stride %lld below n_max %d", what, (long long)m->stride, n_max);
    PQHSA_REQUIRE(isfinite(m->decay), "%s: decay is not finite", what);
    PQHSA_REQUIRE(m->rows >= 0, "%s: mass rows must not be negative", what);
    return PQHSA_OK;
}

namespace {

struct DensePlan {
    int chunk, splits;
    int64_t score_stride;
    size_t scores_at, ml_at, bytes;
};

DensePlan plan_dense(int B, int H, int G, int n_max, const pqhsa_score *score, bool mass) {
    DensePlan p = {};
    const int64_t streams = (int64_t)B * H;
    const int64_t keys = visible_bound(score, n_max) > 0 ? visible_bound(score, n_max) : 1;
    // The chip holds 512 workgroups at once.  One sequence's chunks are equally long, so it is cut into one
    // such round (1 x 32768, one resident cache: 30.8 us, 33.7 in three rounds); several are as long as the longest at
    // most, and three rounds even that out (16 of 16384 to 65536 keys: 360 us, 381 in two).
    const int64_t want = B == 1 ? 512 : 1536;
    int64_t chunk = (streams * keys + want - 1) / want;
    // No join where it costs more than walking on: two steps a wave (8 heads of 256 keys 8.9 us, 10.2 joined), and
    // streams that fill the chip by themselves (512 of up to 512 keys 21.4 us, 25.4 joined; of up to 1024 33.9 and 34.8).
    if (keys <= 256 || (streams >= 512 && keys <= 1024)) chunk = keys;
    chunk = (chunk + kDenseChunkMin - 1) / kDenseChunkMin * kDenseChunkMin;
    if (chunk > kDenseChunkMax) chunk = kDenseChunkMax;
    p.chunk = (int)chunk;
    p.splits = (int)((keys + chunk - 1) / chunk);
    p.score_stride = (int64_t)p.splits * chunk;
    const size_t rows = (size_t)streams * G;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    if (p.splits > 1) take(rows * p.splits * kD * sizeof(float));
    p.ml_at = p.splits > 1 || mass ? take(rows * p.splits * sizeof(float2)) : 0;
    p.scores_at = mass ? take(rows * p.score_stride * sizeof(float)) : 0;
    p.bytes = at;
    return p;
}

}  // namespace

}  // namespace pqhsa

using namespace pqhsa;

extern "C" size_t pqhsa_dense_attend_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t n_max,
                                                     const pqhsa_score *score, int32_t with_mass) {
    if (B <= 0 || H <= 0 || G <= 0 || n_max <= 0 || !score) return 256;
    const size_t need = plan_dense(B, H, G, n_max, score, with_mass != 0).bytes;
    return need < 256 ? 256 : need;
}

extern "C" int pqhsa_dense_attend_paged(const void *q, int32_t q_dtype, int64_t q_stride_row, int64_t q_stride_head,
                                        void *out, int64_t out_stride_row, int64_t out_stride_head,
                                        const pqhsa_kv_view *kv, int32_t blocks, int32_t B, int32_t H, int32_t G,
                                        const int32_t *seq_lens, int32_t n_max, const pqhsa_score *score, float *lse,
                                        const pqhsa_mass *mass, void *workspace, size_t workspace_bytes, void *stream_v) {
    const char *what = "dense_attend_paged";
    int rc = validate_view(kv);
    if (rc) return rc;
    PQHSA_REQUIRE(B >= 0 && H > 0 && G > 0 && G <= kDenseRows, "%s: B %d, H %d, G %d (1 to 16 query heads per KV head)", what, B, H, G);
    PQHSA_REQUIRE(n_max >= 0, "%s: n_max %d is negative", what, n_max);
    rc = validate_score(score, n_max, what);
    if (rc) return rc;
    rc = validate_mass(mass, n_max, what);
    if (rc) return rc;
    if (B == 0) return PQHSA_OK;
    PQHSA_REQUIRE(q && out && seq_lens && workspace, "%s: NULL argument", what);
    PQHSA_REQUIRE(q_dtype == kv->dtype, "%s: q dtype %d differs from the cache's %d", what, q_dtype, kv->dtype);
    const int64_t vec = kv->dtype == PQHSA_F32 ? 4 : 8;
    PQHSA_REQUIRE((uintptr_t)q % 16 == 0 && q_stride_row % vec == 0 && q_stride_head % vec == 0,
                  "%s: query rows must be 16-byte aligned", what);
    PQHSA_REQUIRE((uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", what);
    if (kv->paged)
        PQHSA_REQUIRE(blocks > 0 && (int64_t)kv->max_blocks * kv->block_size >= n_max,
                      "%s: %d blocks, and a table of %d x %d tokens for n_max %d", what, blocks, kv->max_blocks, kv->block_size, n_max);
    PQHSA_REQUIRE((int64_t)B * H <= (mass ? 65535 : 0x7fffffff / kDenseRows), "%s: too many sequences and heads", what);
    const DensePlan p = plan_dense(B, H, G, n_max, score, mass != nullptr);
    PQHSA_REQUIRE(p.splits <= 65535, "%s: n_max %d too large for one launch", what, n_max);
    if (workspace_bytes < p.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, p.bytes);
        return PQHSA_ENOSPC;
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    char *w = static_cast<char *>(workspace);
    DenseArgs a = {};
    a.q = static_cast<const char *>(q); a.q_row = q_stride_row; a.q_head = q_stride_head;
    a.out = static_cast<char *>(out); a.out_row = out_stride_row; a.out_head = out_stride_head;
    a.lse = lse;
    a.kv = make_view(kv);
    a.blocks = blocks; a.B = B; a.H = H; a.G = G; a.seq_lens = seq_lens; a.n_max = n_max;
    a.score = make_score(score);
    a.chunk = p.chunk; a.splits = p.splits;
    a.part_o = reinterpret_cast<float *>(w);
    a.part_ml = p.splits > 1 || mass ? reinterpret_cast<float2 *>(w + p.ml_at) : nullptr;
    a.scores = mass ? reinterpret_cast<float *>(w + p.scores_at) : nullptr;
    a.score_stride = p.score_stride;
    const size_t list = (size_t)p.chunk * sizeof(int64_t);
    const size_t fold = (size_t)kDenseWaves * (2 * kDenseRows + G * kD) * sizeof(float);
    const size_t lds = list > fold ? list : fold;
    const dim3 grid((unsigned)(B * H), (unsigned)p.splits);
    PQHSA_DISPATCH_DTYPE(kv->dtype,
                         if (mass) hipLaunchKernelGGL((dense_attend_kernel<DT, true>), grid, dim3(kDenseThreads), lds, stream, a);
                         else hipLaunchKernelGGL((dense_attend_kernel<DT, false>), grid, dim3(kDenseThreads), lds, stream, a));
    rc = check_launch(what);
    if (rc) return rc;
    if (p.splits > 1) {
        JoinArgs j = {a.part_o, a.part_ml, p.splits, H * G, a.out, a.out_row, a.out_head, lse, nullptr, nullptr};
        rc = launch_join(j, kv->dtype, (int64_t)B * H * G, stream);
        if (rc) return rc;
    }
    if (mass && n_max > 0) {
        MassArgs s = {a.scores, a.score_stride, a.part_ml, p.splits, B, H, G, seq_lens, n_max, a.score,
                      mass->in, mass->out, mass->stride, mass->decay};
        hipLaunchKernelGGL(dense_mass_kernel, dim3((unsigned)((n_max + kMassKeys - 1) / kMassKeys), (unsigned)(B * H)),
                           dim3(256), 0, stream, s);
        rc = check_launch("dense_mass");
    }
    return rc;
}
