// Dense attention of packed prompt rows over a (paged) cache: whole prompts, or rows that continue a
// cached one, under the score rule of dense_common.h.
//
// A prompt of R rows over n keys costs 4 * 128 operations per (row, key) pair that is visible and reads
// K and V once per 128 query rows: the matrix cores bound it.  The rows of all G heads of a KV head are
// packed into one row space (row = token * G + g), so a workgroup's 128 rows share every K/V tile it
// fetches, and a short piece of a prompt still fills a tile.  Four waves own 32 rows each; K/V tiles of
// 64 keys (32 in fp32) go through LDS in two buffers, the next tile's rows requested from memory while
// this one is computed.
//
//   S^T = K Q^T (32 keys x 32 rows): a lane holds 16 keys' scores of ONE query row, so the running maximum
//     and sum need one exchange between two lanes, and only when the maximum moves (kMaxSlack).
//   O^T = V^T P: the lane's scores are, in place, the second operand's layout.  V is transposed on its way
//     into LDS (4 keys x 8 dims a thread, byte permutes) with the keys in the order in which the scores lie.
//
// Tiles no row of the workgroup sees are left out of the walk (causal order, window, prefix from the
// positions; documents from a bit per tile); a tile every row sees skips all mask arithmetic.  Where the
// launch would not fill the chip the key range is split over workgroups and joined by a second launch.
#include "dense_common.h"

namespace pqhsa {

constexpr int kPromptThreads = 256;
constexpr int kPromptRows = 128;       // packed rows per workgroup
constexpr int kPromptSlots = 4;        // tiles whose row addresses are kept
constexpr int kPromptBuffer = 32768;   // bytes of a K/V tile pair in LDS

struct PromptArgs {
    const char *q;
    int64_t q_row, q_head;
    char *out;
    int64_t out_row, out_head;
    float *lse;                        // [T, H * G]
    KvView kv;
    int blocks, B, H, G;
    const int32_t *cu_rows;            // [B + 1]
    int64_t T;
    const int32_t *seq_lens;
    int n_max;
    ScoreArgs score;
    int tiles;                         // row tiles of the launch
    int splits;
    int mask_words;                    // words of the per-tile bit mask in LDS (documents)
    float *part_o;                     // [T * H * G, splits, 128]
    float2 *part_ml;                   // [T * H * G, splits]
    // accumulated weights
    const float *mass_in;
    float *mass_out;
    int64_t mass_stride;
    float decay;
    int mass_rows;
};

struct PromptRows {
    int64_t first;                     // first row of the sequence in q
    int rows;
};
__device__ inline PromptRows sequence_rows(const int32_t *cu, int64_t T, int b) {
    const int64_t lo = min(max((int64_t)cu[b], (int64_t)0), T);
    const int64_t hi = min(max((int64_t)cu[b + 1], lo), T);
    return {lo, (int)(hi - lo)};
}

// The workgroup's row tile: sequence and tile number inside it (b < 0: none).  Every wave finds it by itself.
__device__ inline void find_row_tile(const PromptArgs &a, int want, int &b_out, int &tile_out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.B; base += 64) {
        int tiles = 0;
        if (base + lane < a.B) {
            const PromptRows r = sequence_rows(a.cu_rows, a.T, base + lane);
            tiles = (int)(((int64_t)r.rows * a.G + kPromptRows - 1) / kPromptRows);
        }
        const int upto = (int)wave_prefix_u32((uint32_t)tiles);
        const uint64_t hit = __ballot(before + upto > want);
        if (hit) {
            const int who = __ffsll((unsigned long long)hit) - 1;
            b_out = base + who;
            tile_out = want - before - (__shfl(upto, who, kWave) - __shfl(tiles, who, kWave));
            return;
        }
        before += __shfl(upto, 63, kWave);
    }
    b_out = -1;
    tile_out = 0;
}

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

template <int DT, bool GENERAL>
__global__ __launch_bounds__(kPromptThreads, 2) void prompt_attend_kernel(PromptArgs a) {
    constexpr bool kF32 = DT == PQHSA_F32;
    constexpr int KT = kF32 ? 32 : 64;                   // keys per tile
    constexpr int kTT = KT / 32;                         // matrix tiles of keys
    constexpr int kRowBytes = kD * (kF32 ? 4 : 2);
    constexpr int kSlices = kRowBytes / 32;              // 16-byte pieces of a row per lane of a pair
    constexpr int kRowLanes = kRowBytes / 16;            // lanes that fetch one row
    constexpr int kPass = 64 / kRowLanes;                // rows a wave fetches per instruction
    extern __shared__ __align__(16) char lds[];
    int64_t *offs = reinterpret_cast<int64_t *>(lds + 2 * kPromptBuffer);          // [slots][64]
    int32_t *kdoc = reinterpret_cast<int32_t *>(offs + kPromptSlots * 64);         // [slots][64]
    uint64_t *valid = reinterpret_cast<uint64_t *>(kdoc + kPromptSlots * 64);      // [slots]
    int32_t *poison = reinterpret_cast<int32_t *>(valid + kPromptSlots);           // [2]: an infinity or NaN was set aside
    int32_t *doc_range = poison + 2;                                               // [2]
    uint32_t *wanted = reinterpret_cast<uint32_t *>(doc_range + 2);                // [mask_words]

    const int tid = threadIdx.x, lane = tid & 63, wave = tid / kWave;
    const int n = lane & 31, kg = lane >> 5;
    const int h = blockIdx.x, split = blockIdx.z;
    int b, tile;
    find_row_tile(a, a.tiles - 1 - (int)blockIdx.y, b, tile);    // the longest rows of a prompt first
    if (b < 0) return;
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const PromptRows rows = sequence_rows(a.cu_rows, a.T, b);
    const int len = sequence_length(a.seq_lens, b, a.n_max);
    const int first_pos = len - rows.rows;
    const int64_t packed = (int64_t)rows.rows * a.G;
    const int64_t pr = (int64_t)tile * kPromptRows + wave * 32 + n;
    const bool mine = pr < packed;
    const int prc = (int)(mine ? pr : packed - 1);       // rows past the end repeat the last one
    const int token = prc / a.G, g = prc - token * a.G;
    const int pos = first_pos + token;
    const int prefix_all = min(sequence_prefix(a.score, b), len);
    // positions of the workgroup's rows, and of the wave's
    const int wg_lo = first_pos + (int)((int64_t)tile * kPromptRows / a.G);
    const int wg_hi = first_pos + (int)((min((int64_t)(tile + 1) * kPromptRows, packed) - 1) / a.G);
    const int w_first = (int)min((int64_t)tile * kPromptRows + wave * 32, packed - 1);
    const int w_last = (int)min((int64_t)tile * kPromptRows + wave * 32 + 31, packed - 1);
    const int w_lo = first_pos + w_first / a.G, w_hi = first_pos + w_last / a.G;
    const int window = a.score.window > 0 ? a.score.window : 0x7fffffff;
    const int32_t *docs = a.score.docs ? a.score.docs + (int64_t)b * a.score.docs_stride : nullptr;

    // the walk: tiles [0, walk_a), then walk_b onwards, `count` in all
    const int end = max(0, min(len, wg_hi + 1));
    const int begin = a.score.window > 0 ? max(0, wg_lo - window + 1) : 0;
    const int walk_a = wg_hi >= 0 ? (prefix_all + KT - 1) / KT : 0;
    const int walk_b = max(begin / KT, walk_a);
    const int count = wg_hi >= 0 ? walk_a + max(0, (end + KT - 1) / KT - walk_b) : 0;
    const int per = (count + a.splits - 1) / a.splits;
    const int t_begin = min(split * per, count), t_end = min(t_begin + per, count);
    auto key_tile = [&](int t) { return (t < walk_a ? t : walk_b + t - walk_a) * KT; };

    if (docs) {                                          // a bit per tile of the walk: some key of the rows' documents
        if (tid == 0) { doc_range[0] = 0x7fffffff; doc_range[1] = -0x7fffffff - 1; }
        for (int w = tid; w < a.mask_words; w += kPromptThreads) wanted[w] = 0u;
        __syncthreads();
        for (int p = max(wg_lo, 0) + tid; p <= wg_hi; p += kPromptThreads) {
            atomicMin(&doc_range[0], docs[p]);
            atomicMax(&doc_range[1], docs[p]);
        }
        __syncthreads();
        const int d_lo = doc_range[0], d_hi = doc_range[1];
        for (int x = tid; x < (t_end - t_begin) * KT; x += kPromptThreads) {
            const int j = key_tile(t_begin + x / KT) + x % KT;
            if (j < len) {
                const int d = docs[j];
                if (d >= d_lo && d <= d_hi) atomicOr(&wanted[x / KT / 32], 1u << (x / KT % 32));
            }
        }
        __syncthreads();
    }
    // the first tile at or after t that has to be walked (t_end: none)
    auto next = [&](int t) {
        if (!docs) return t;
        while (t < t_end) {
            const int x = t - t_begin;
            const uint32_t bits = wanted[x / 32] >> (x % 32);
            if (bits) return min(t + __ffs((int)bits) - 1, t_end);
            t = t_begin + (x / 32 + 1) * 32;
        }
        return t_end;
    };

    // query rows as the second operand: lane (n, kg) holds row n
    uint4 qf[kSlices];
    {
        const char *p = a.q + ((rows.first + token) * a.q_row + (int64_t)(h * a.G + g) * a.q_head) * a.kv.esize;
#pragma unroll
        for (int u = 0; u < kSlices; ++u) qf[u] = *reinterpret_cast<const uint4 *>(p + (u * 2 + kg) * 16);
    }
    const float slope2 = GENERAL && a.score.slopes ? a.score.slopes[h * a.G + g] * kLog2e : 0.0f;
    const int row_doc = docs && pos >= 0 ? docs[pos] : 0;
    const int row_prefix = pos >= 0 ? prefix_all : 0;
    const int row_from = pos >= 0 ? max(pos - window + 1, 0) : 0;   // keys [row_from, pos] and [0, row_prefix)

    // addresses of a tile's rows (the first KT threads), -1: past the sequence or outside the cache
    auto resolve = [&](int t, int slot) {
        if (tid < 64) {
            const int j = key_tile(t) + tid;
            const bool in = tid < KT && j < len;
            int64_t off = -1;
            if (in) off = checked_row_bytes(a.kv, a.blocks, b, h, j);
            offs[slot * 64 + tid] = off;
            if (docs) kdoc[slot * 64 + tid] = in ? docs[j] : 0;
            const uint64_t ok = __ballot(off >= 0);
            if (tid == 0) valid[slot] = ok;
        }
    };
    // K: four rows' pieces a thread; V: four consecutive rows (2-byte types; four passes in fp32)
    u32x4 ks[4], vs[4];
    auto fetch = [&](int slot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (wave * 4 + i) * kPass + lane / kRowLanes;
            const int64_t off = offs[slot * 64 + r];
            ks[i] = *reinterpret_cast<const u32x4 *>(a.kv.k_base + (off < 0 ? 0 : off) + (lane % kRowLanes) * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = kF32 ? (wave * 4 + i) * kPass + lane / kRowLanes : (wave * 4 + lane / 16) * 4 + i;
            const int64_t off = offs[slot * 64 + r];
            const u32x4 x = *reinterpret_cast<const u32x4 *>(a.kv.v_base + (off < 0 ? 0 : off) + (lane % kRowLanes) * 16);
            vs[i] = off < 0 ? (u32x4){0u, 0u, 0u, 0u} : x;
        }
    };
    // K rows by 16-byte pieces, the piece number xored with the row; V^T (2-byte types) rows of 64 keys by
    // dim, 16-byte slots of 8 keys (slot 2u + kg: keys 16u + 4kg + {0..3, 8..11}), xored with the dim
    // `watch`: a tile that some rows do not see whole.  A weight of zero would not cancel an infinite or NaN
    // value there, so these are left out of the product and come back at the end, for the rows that see them.
    auto store = [&](int buf, bool watch) {
        if (watch) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = finite_part<DT>(vs[i][w]);
                    bad |= x != vs[i][w];
                    vs[i][w] = x;
                }
            if (bad) poison[0] = 1;
        }
        char *kl = lds + buf * kPromptBuffer, *vl = kl + kPromptBuffer / 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (wave * 4 + i) * kPass + lane / kRowLanes;
            *reinterpret_cast<u32x4 *>(kl + r * kRowBytes + (((lane % kRowLanes) ^ (r & 15)) * 16)) = ks[i];
        }
        if constexpr (kF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (wave * 4 + i) * kPass + lane / kRowLanes;
                *reinterpret_cast<u32x4 *>(vl + r * kRowBytes + (lane % kRowLanes) * 16) = vs[i];
            }
        } else {
            const int q4 = wave * 4 + lane / 16, i16 = lane & 15;
            const int slot16 = (q4 >> 2) * 2 + (q4 & 1), half = (q4 >> 1) & 1;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                uint32_t w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    w[x] = __builtin_amdgcn_perm(vs[2 * x + 1][d >> 1], vs[2 * x][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
                *reinterpret_cast<uint2 *>(vl + (i16 * 8 + d) * 128 + ((slot16 ^ ((i16 ^ d) & 7)) * 16) + half * 8) = make_uint2(w[0], w[1]);
            }
        }
    };
    // whether rows at positions [lo, hi] all see keys [k0, k0 + KT)
    auto all_see = [&](int k0, int lo, int hi) {
        const int last = k0 + KT - 1;
        return !docs && lo >= 0 && ((last <= lo && hi - k0 < window) || last < prefix_all);
    };

    float m = -INFINITY, l = 0.0f;
    f32x16 acc[4];                                       // dim 32 dt + 8 (r / 4) + 4 kg + r % 4 of row n in acc[dt][r]
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] = 0.0f;

    // value product of the tile: weights in the operand registers, V^T from LDS
    auto value_operand = [&](const char *vl, int u, int dt) {
        if constexpr (kF32) {                            // (u: the accumulator register of the key's score)
            const uint32_t w = *reinterpret_cast<const uint32_t *>(vl + (8 * (u / 4) + 4 * kg + u % 4) * kRowBytes + (dt * 32 + n) * 4);
            return make_uint4(w, 0u, 0u, 0u);
        } else {
            const int dim = dt * 32 + n;
            return *reinterpret_cast<const uint4 *>(vl + dim * 128 + (((u * 2 + kg) ^ (((dim >> 3) ^ dim) & 7)) * 16));
        }
    };
    auto value_mfma = [&](uint4 v, uint4 w, f32x16 o) {
        if constexpr (kF32) return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.x), __uint_as_float(w.x), o, 0, 0, 0);
        else return Half16<DT>::mfma32(v, w, o);
    };
    constexpr int kSteps = kF32 ? 16 : KT / 16;          // matrix instructions per 32 dims

    if (tid == 0) poison[0] = 0;
    int t = next(t_begin), t1 = t < t_end ? next(t + 1) : t_end;
    if (t < t_end) {
        resolve(t, 0);
        if (t1 < t_end) resolve(t1, 1);
        __syncthreads();
        fetch(0);
        store(0, !all_see(key_tile(t), wg_lo, wg_hi));
        __syncthreads();
    }
    for (int it = 0; t < t_end; ++it) {
        const int slot = it & 3;
        const char *kl = lds + (it & 1) * kPromptBuffer, *vl = kl + kPromptBuffer / 2;
        const int t2 = t1 < t_end ? next(t1 + 1) : t_end;
        const int k0 = key_tile(t);
        if (t1 < t_end) fetch((it + 1) & 3);
        if (t2 < t_end) resolve(t2, (it + 2) & 3);

        f32x16 s[kTT];
#pragma unroll
        for (int T = 0; T < kTT; ++T) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[T][r] = 0.0f;
            const int key = T * 32 + n;
#pragma unroll
            for (int u = 0; u < kSlices; ++u) {
                const uint4 x = *reinterpret_cast<const uint4 *>(kl + key * kRowBytes + (((u * 2 + kg) ^ (key & 15)) * 16));
                if constexpr (kF32) {
                    const f32x4 y = __builtin_bit_cast(f32x4, x), z = __builtin_bit_cast(f32x4, qf[u]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[T] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[c], z[c], s[T], 0, 0, 0);
                } else {
                    s[T] = Half16<DT>::mfma32(x, qf[u], s[T]);
                }
            }
        }
        const bool whole = all_see(k0, w_lo, w_hi) && valid[slot] == (KT == 64 ? ~0ull : 0xffffffffull);
        // scores; where GENERAL is false they stay unscaled, the scale goes into the exponent
        const float unit = GENERAL ? 1.0f : a.score.scale2;
        if constexpr (GENERAL) {
#pragma unroll
            for (int T = 0; T < kTT; ++T)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = k0 + T * 32 + 8 * (r / 4) + 4 * kg + r % 4;
                    const float x = s[T][r];
                    s[T][r] = (a.score.capped ? a.score.cap2 * tanh_score(x * a.score.in_cap) : x * a.score.scale2)
                              - slope2 * (float)abs(pos - j);
                }
        }
        if (!whole) {
            const uint64_t ok = valid[slot] >> (4 * kg);
#pragma unroll
            for (int T = 0; T < kTT; ++T)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    int4 kd = make_int4(0, 0, 0, 0);
                    if (docs) kd = *reinterpret_cast<const int4 *>(&kdoc[slot * 64 + T * 32 + 8 * r4 + 4 * kg]);
                    const int d[4] = {kd.x, kd.y, kd.z, kd.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = k0 + T * 32 + 8 * r4 + 4 * kg + e;
                        bool see = ((j >= row_from && j <= pos) || j < row_prefix) && ((ok >> (T * 32 + 8 * r4 + e)) & 1);
                        if (docs) see = see && d[e] == row_doc;
                        s[T][4 * r4 + e] = see ? s[T][4 * r4 + e] : -INFINITY;
                    }
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[T][r]);
        top *= unit;
        if (__ballot(top > m + kMaxSlack)) {
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            const float to = fmaxf(m, top);
            const float f = m == to ? 1.0f : exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) acc[dt] *= f;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float p[kTT][16];
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[T][r] = exp2_fast(GENERAL ? s[T][r] - base : __builtin_fmaf(s[T][r], unit, -base));
                l += p[T][r];
            }
        // weights rounded to the value type for the product (their sum l is not): each at most half a
        // step off, independently, no more than the output's own rounding
        uint4 pw[kSteps];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            if constexpr (kF32) {
                pw[u] = make_uint4(__float_as_uint(p[0][u]), 0u, 0u, 0u);
            } else {
                const float *x = &p[u / 2][(u % 2) * 8];
                pw[u] = make_uint4(Half16<DT>::pack(x[0], x[1]), Half16<DT>::pack(x[2], x[3]), Half16<DT>::pack(x[4], x[5]), Half16<DT>::pack(x[6], x[7]));
            }
        }
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) acc[dt] = value_mfma(value_operand(vl, u, dt), pw[u], acc[dt]);
        if (t1 < t_end) store((it + 1) & 1, !all_see(key_tile(t1), wg_lo, wg_hi));
        __syncthreads();
        t = t1;
        t1 = t2;
    }
    l += __shfl_xor(l, 32, kWave);
    if (t_begin < t_end && poison[0]) {                  // the infinities and NaN that were set aside
#pragma unroll 1
        for (t = next(t_begin); t < t_end; t = next(t + 1)) {
            const int k0 = key_tile(t);
            if (all_see(k0, wg_lo, wg_hi)) continue;
#pragma unroll 1
            for (int j = k0; j < min(k0 + KT, len); ++j) {
                const int64_t off = checked_row_bytes(a.kv, a.blocks, b, h, j);
                bool see = off >= 0 && ((j >= row_from && j <= pos) || j < row_prefix);
                if (docs) see = see && docs[j] == row_doc;
                if (!see) continue;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float x = load1<DT>(a.kv.v_base + off, dt * 32 + 8 * (r / 4) + 4 * kg + r % 4);
                        if (!(fabsf(x) < INFINITY)) acc[dt][r] += x;
                    }
            }
        }
    }
    if (!mine) return;
    const int64_t r = (rows.first + token) * (int64_t)(a.H * a.G) + h * a.G + g;
    if (a.splits > 1) {
        if (kg == 0) a.part_ml[r * a.splits + split] = make_float2(m, l);
        if (l != 0.0f) {
            float *o = a.part_o + (r * a.splits + split) * kD;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4)
                    *reinterpret_cast<float4 *>(o + dt * 32 + 8 * r4 + 4 * kg) =
                        make_float4(acc[dt][4 * r4], acc[dt][4 * r4 + 1], acc[dt][4 * r4 + 2], acc[dt][4 * r4 + 3]);
        }
        return;
    }
    if (kg == 0 && a.lse) a.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    char *o = a.out + ((rows.first + token) * a.out_row + (int64_t)(h * a.G + g) * a.out_head) * a.kv.esize;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = l == 0.0f ? 0.0f : acc[dt][4 * r4 + e] * inv;
            const int d = dt * 32 + 8 * r4 + 4 * kg;
            if constexpr (kF32) *reinterpret_cast<float4 *>(o + d * 4) = make_float4(x[0], x[1], x[2], x[3]);
            else *reinterpret_cast<uint2 *>(o + d * 2) = make_uint2(Half16<DT>::pack(x[0], x[1]), Half16<DT>::pack(x[2], x[3]));
        }
}

// ---- weight of every key, summed over the last rows of the prompts -----------------------------
// With every row's log-sum-exp known the weights are one product K Q^T and an exp2 away.  A wave keeps 32
// keys as the first operand in registers and walks the counted rows; every lane sums its rows' weights
// of 16 keys, the lanes are summed at the end: no atomics, one owner per key.
template <int DT>
__global__ __launch_bounds__(kPromptThreads, 2) void prompt_mass_kernel(PromptArgs a) {
    constexpr bool kF32 = DT == PQHSA_F32;
    constexpr int kSlices = kD * (kF32 ? 4 : 2) / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid / kWave;
    const int n = lane & 31, kg = lane >> 5;
    const int b = blockIdx.y / a.H, h = blockIdx.y - b * a.H;
    const int len = sequence_length(a.seq_lens, b, a.n_max);
    const int k0 = (blockIdx.x * 4 + wave) * 32;
    if (k0 >= len) return;                               // (no barrier below: waves are independent)
    const PromptRows rows = sequence_rows(a.cu_rows, a.T, b);
    const int first_pos = len - rows.rows;
    const int prefix = min(sequence_prefix(a.score, b), len);
    const int window = a.score.window > 0 ? a.score.window : 0x7fffffff;
    const int32_t *docs = a.score.docs ? a.score.docs + (int64_t)b * a.score.docs_stride : nullptr;

    uint4 kf[kSlices];
    const int64_t off = k0 + n < len ? checked_row_bytes(a.kv, a.blocks, b, h, k0 + n) : -1;
#pragma unroll
    for (int u = 0; u < kSlices; ++u)
        kf[u] = *reinterpret_cast<const uint4 *>(a.kv.k_base + (off < 0 ? 0 : off) + (u * 2 + kg) * 16);
    const uint32_t ok = (uint32_t)__ballot(off >= 0);    // (both halves of the wave hold the same 32 keys)
    int kd[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int j = k0 + 8 * (r / 4) + 4 * kg + r % 4;
        kd[r] = docs && j < len ? docs[j] : 0;
    }
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.0f;

    const int from = a.mass_rows > 0 ? max(0, rows.rows - a.mass_rows) : 0;
    const int64_t packed = (int64_t)rows.rows * a.G;
    int64_t at = (int64_t)from * a.G;
    // rows before the first that can see a key of this tile (causal order, unless the prefix reaches it)
    if (k0 >= prefix) at = max(at, (int64_t)max(k0 - first_pos, 0) * a.G);
    for (; at < packed; at += 32) {
        const bool mine = at + n < packed;
        const int prc = (int)(mine ? at + n : packed - 1);
        const int token = prc / a.G, g = prc - token * a.G, pos = first_pos + token;
        // past the window of all the tile's keys, and these are not in the prefix: no later row sees them
        if (k0 >= prefix && first_pos + (int)(at / a.G) - (k0 + 31) >= window) break;
        const char *p = a.q + ((rows.first + token) * a.q_row + (int64_t)(h * a.G + g) * a.q_head) * a.kv.esize;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int u = 0; u < kSlices; ++u) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + (u * 2 + kg) * 16);
            if constexpr (kF32) {
                const f32x4 y = __builtin_bit_cast(f32x4, kf[u]), z = __builtin_bit_cast(f32x4, x);
#pragma unroll
                for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_32x32x2f32(y[c], z[c], s, 0, 0, 0);
            } else {
                s = Half16<DT>::mfma32(kf[u], x, s);
            }
        }
        const float lse = a.lse[(rows.first + token) * (int64_t)(a.H * a.G) + h * a.G + g];
        const float total = !mine || lse == -INFINITY ? INFINITY : lse * kLog2e;   // +inf: the row gives no weight
        const float slope2 = a.score.slopes ? a.score.slopes[h * a.G + g] * kLog2e : 0.0f;
        const int row_doc = docs && pos >= 0 ? docs[pos] : 0;
        const int row_prefix = pos >= 0 ? prefix : 0, row_from = pos >= 0 ? max(pos - window + 1, 0) : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int jj = 8 * (r / 4) + 4 * kg + r % 4, j = k0 + jj;
            float z = a.score.capped ? a.score.cap2 * tanh_score(s[r] * a.score.in_cap) : s[r] * a.score.scale2;
            z -= slope2 * (float)abs(pos - j);
            const bool see = ((j >= row_from && j <= pos) || j < row_prefix) && ((ok >> jj) & 1) && (!docs || kd[r] == row_doc);
            sum[r] += see && mine ? exp2_fast(z - total) : 0.0f;
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float x = sum[r];
        x += __shfl_xor(x, 1, kWave);
        x += __shfl_xor(x, 2, kWave);
        x += __shfl_xor(x, 4, kWave);
        x += __shfl_xor(x, 8, kWave);
        x += __shfl_xor(x, 16, kWave);
        const int j = k0 + 8 * (r / 4) + 4 * kg + r % 4;
        if (n == r && j < len) {                         // one lane of each half writes key r's sum
            const int64_t o = (int64_t)blockIdx.y * a.mass_stride + j;
            a.mass_out[o] = (a.mass_in ? a.decay * a.mass_in[o] : 0.0f) + x;
        }
    }
}

namespace {

struct PromptPlan {
    int64_t tiles;
    int splits;
    size_t ml_at, lse_at, bytes;
};

PromptPlan plan_prompt(int64_t T, int B, int H, int G, int n_max, int rows_hint, int key_tile, bool own_lse) {
    PromptPlan p = {};
    p.tiles = (T * G + kPromptRows - 1) / kPromptRows + B;          // every sequence may end inside a tile
    int64_t busy = p.tiles - B;
    if (rows_hint > 0 && rows_hint * (int64_t)B <= T) {             // about as many tiles as sequences have
        const int64_t each = ((int64_t)rows_hint * G + kPromptRows - 1) / kPromptRows;
        if (each * B > busy) busy = each * B;
    }
    if (busy < 1) busy = 1;
    // two workgroups per compute unit, at least four key tiles each
    const int64_t want = (512 + busy * H - 1) / (busy * H);
    const int64_t most = ((int64_t)n_max + 4 * key_tile - 1) / (4 * key_tile);
    p.splits = (int)(want < most ? want : most);
    if (p.splits < 1) p.splits = 1;
    const size_t rows = (size_t)T * H * G;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    if (p.splits > 1) {
        take(rows * p.splits * kD * sizeof(float));
        p.ml_at = take(rows * p.splits * sizeof(float2));
    }
    if (own_lse) p.lse_at = take(rows * sizeof(float));
    p.bytes = at;
    return p;
}

template <int DT, bool GENERAL>
int launch_prompt(const PromptArgs &a, size_t lds, hipStream_t stream) {
    auto kern = prompt_attend_kernel<DT, GENERAL>;
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) {
        set_error("prompt_attend: cannot raise the LDS limit to %zu: %s", lds, hipGetErrorString(e));
        return PQHSA_ELAUNCH;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)a.H, (unsigned)a.tiles, (unsigned)a.splits), dim3(kPromptThreads), lds, stream, a);
    return check_launch("prompt_attend");
}

}  // namespace

}  // namespace pqhsa

using namespace pqhsa;

extern "C" size_t pqhsa_prompt_attend_workspace_bytes(int64_t T, int32_t B, int32_t H, int32_t G, int32_t n_max,
                                                      int32_t rows_hint, int32_t dtype, int32_t with_lse) {
    if (T <= 0 || B <= 0 || H <= 0 || G <= 0 || n_max <= 0) return 256;
    const size_t need = plan_prompt(T, B, H, G, n_max, rows_hint, dtype == PQHSA_F32 ? 32 : 64, with_lse == 0).bytes;
    return need < 256 ? 256 : need;
}

extern "C" int pqhsa_prompt_attend_paged(const void *q, int32_t q_dtype, int64_t q_stride_row, int64_t q_stride_head,
                                         void *out, int64_t out_stride_row, int64_t out_stride_head, int64_t T,
                                         const int32_t *cu_rows, const pqhsa_kv_view *kv, int32_t blocks, int32_t B,
                                         int32_t H, int32_t G, const int32_t *seq_lens, int32_t n_max, int32_t rows_hint,
                                         const pqhsa_score *score, float *lse, const pqhsa_mass *mass, void *workspace,
                                         size_t workspace_bytes, void *stream_v) {
    const char *what = "prompt_attend_paged";
    int rc = validate_view(kv);
    if (rc) return rc;
    PQHSA_REQUIRE(B >= 0 && H > 0 && G > 0 && G <= 16, "%s: B %d, H %d, G %d (1 to 16 query heads per KV head)", what, B, H, G);
    PQHSA_REQUIRE(n_max >= 0 && T >= 0, "%s: n_max %d or T %lld is negative", what, n_max, (long long)T);
    rc = validate_score(score, n_max, what);
    if (rc) return rc;
    rc = validate_mass(mass, n_max, what);
    if (rc) return rc;
    if (B == 0 || (T == 0 && !mass)) return PQHSA_OK;
    PQHSA_REQUIRE(cu_rows && seq_lens && workspace && (T == 0 || (q && out)), "%s: NULL argument", what);
    PQHSA_REQUIRE(q_dtype == kv->dtype, "%s: q dtype %d differs from the cache's %d", what, q_dtype, kv->dtype);
    const int64_t vec = kv->dtype == PQHSA_F32 ? 4 : 8;
    PQHSA_REQUIRE((uintptr_t)q % 16 == 0 && q_stride_row % vec == 0 && q_stride_head % vec == 0,
                  "%s: query rows must be 16-byte aligned", what);
    PQHSA_REQUIRE((uintptr_t)out % 16 == 0 && out_stride_row % vec == 0 && out_stride_head % vec == 0,
                  "%s: output rows must be 16-byte aligned", what);
    PQHSA_REQUIRE((uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", what);
    if (kv->paged)
        PQHSA_REQUIRE(blocks > 0 && (int64_t)kv->max_blocks * kv->block_size >= n_max,
                      "%s: %d blocks, and a table of %d x %d tokens for n_max %d", what, blocks, kv->max_blocks, kv->block_size, n_max);
    PQHSA_REQUIRE(T * G < 0x7fffffff && T * H * G < 0x7fffffff, "%s: %lld rows of %d x %d heads are too many", what, (long long)T, H, G);
    PQHSA_REQUIRE((int64_t)B * H <= 65535, "%s: too many sequences and heads", what);
    const int key_tile = kv->dtype == PQHSA_F32 ? 32 : 64;
    const PromptPlan p = plan_prompt(T, B, H, G, n_max, rows_hint, key_tile, lse == nullptr);
    PQHSA_REQUIRE(p.tiles <= 65535 && p.splits <= 65535, "%s: %lld row tiles are too many for one launch", what, (long long)p.tiles);
    if (workspace_bytes < p.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, p.bytes);
        return PQHSA_ENOSPC;
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    char *w = static_cast<char *>(workspace);
    PromptArgs a = {};
    a.q = static_cast<const char *>(q); a.q_row = q_stride_row; a.q_head = q_stride_head;
    a.out = static_cast<char *>(out); a.out_row = out_stride_row; a.out_head = out_stride_head;
    a.lse = lse ? lse : reinterpret_cast<float *>(w + p.lse_at);
    a.kv = make_view(kv);
    a.blocks = blocks; a.B = B; a.H = H; a.G = G; a.cu_rows = cu_rows; a.T = T; a.seq_lens = seq_lens; a.n_max = n_max;
    a.score = make_score(score);
    a.tiles = (int)p.tiles;
    a.splits = p.splits;
    a.mask_words = score->docs ? (n_max / key_tile + 2 + 31) / 32 + 1 : 0;
    a.part_o = reinterpret_cast<float *>(w);
    a.part_ml = reinterpret_cast<float2 *>(w + p.ml_at);
    const size_t lds = 2 * kPromptBuffer + kPromptSlots * (64 * 8 + 64 * 4 + 8) + 16 + (size_t)a.mask_words * 4;
    PQHSA_REQUIRE(lds <= 160 * 1024, "%s: n_max %d too large for a document mask", what, n_max);
    if (T > 0) {
        const bool general = score->softcap > 0.0f || score->slopes || !(score->scale > 0.0f);
        PQHSA_DISPATCH_DTYPE(kv->dtype, rc = general ? launch_prompt<DT, true>(a, lds, stream) : launch_prompt<DT, false>(a, lds, stream));
        if (rc) return rc;
        if (p.splits > 1) {
            JoinArgs j = {a.part_o, a.part_ml, p.splits, H * G, a.out, a.out_row, a.out_head, a.lse, cu_rows + B};
            rc = launch_join(j, kv->dtype, T * H * G, stream);
            if (rc) return rc;
        }
    }
    if (mass && n_max > 0) {
        a.mass_in = mass->in; a.mass_out = mass->out; a.mass_stride = mass->stride; a.decay = mass->decay; a.mass_rows = mass->rows;
        const dim3 grid((unsigned)((n_max + 127) / 128), (unsigned)(B * H));
        PQHSA_DISPATCH_DTYPE(kv->dtype, hipLaunchKernelGGL(prompt_mass_kernel<DT>, grid, dim3(kPromptThreads), 0, stream, a));
        rc = check_launch("prompt_mass");
    }
    return rc;
}
