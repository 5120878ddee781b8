// Dense attention of packed prompt rows over a (paged) cache: whole prompts, or rows that continue a
// cached one, under the score rule of dense_common.h.
//
// A prompt of R rows over n keys costs 4 * 128 operations per visible (row, key) pair and reads K and V
// once per row tile: the matrix cores bound it.  The rows of all G heads of a KV head are packed into one
// row space (row = token * G + g), so a workgroup's rows share every K/V tile it fetches, and a short piece of
// a prompt still fills a tile.  A wave owns 32 rows; K/V tiles of 64 keys (32 in fp32) come straight from memory
// into a ring of LDS stages, several on their way while one is computed (through registers: 2.84 ms instead
// of 2.35 at 16 384 rows of 8 x 4 heads).
//
//   S^T = K Q^T (32 keys x 32 rows): a lane holds 16 keys' scores of ONE query row, so the running maximum
//     and sum need one exchange between two lanes, and only when the maximum moves (kMaxSlack).
//   O^T = V^T P: the lane's scores are, in place, the second operand's layout.  V lies in LDS as in memory; a
//     transposing read hands a lane the four keys of its dim.
//
// Tiles no row of the workgroup sees are left out of the walk (causal order, window, prefix from the
// positions; documents from a bit per tile); a tile every row of a wave sees skips all mask arithmetic.
//
// Measured: 16 384 rows of 8 x 4 heads in bf16 2.25 ms, 980 TFLOP/s of visible pairs (a large library product reaches
// 1165 here): per tile and wave 1 000 cycles of matrix instructions, 1 000 of exp2, sums and rounding, and
// 1 000 of requests and waits overlap between two waves of a SIMD only in part.  6 prompts of 300 to 1 801
// rows in 5 documents 95 us: 25 us a workgroup, 8 of them the chain of dependent reads before the first tile.  64
// rows of 4 x 7 heads behind 32 704 keys, fp16, 60 us + 8 us join.  8 192 rows of 8 x 4 heads: 600 us as they are, 750 with a bias,
// 800 capped at 50 with scores far below the cap and 910 with scores around it (a tile with one of these evaluates
// quotients for all of its scores).
#include <atomic>

#include "dense_common.h"

namespace pqhsa {

constexpr int kTileBytes = 16384;      // a K or V tile in LDS
// fp16: a tile whose 64 keys all lie more than this (log2) below a row's base moves it.  Its largest weight is 2^(13 - 16)
// at least otherwise, and 64 roundings of 2^-25 are 2^-16 of that.
constexpr float kPromptDrop = 16.0f;

// Two shapes of workgroup (32 rows a wave either way).
template <int WAVES>
struct PromptShape {
    static constexpr int kWaves = WAVES;
    static constexpr int kThreads = WAVES * kWave;
    static constexpr int kRows = WAVES * 32;             // packed rows
    static constexpr int kStages = WAVES / 2;            // K/V tiles in LDS
    static constexpr int kSlots = 2 * kStages;           // tiles whose row addresses are known or on their way
    static constexpr int kLds = 2 * kStages * kTileBytes + kSlots * (64 * 8 + 64 * 4 + 64 * 4 + 8 + 4) + 16 + kD * 4;
};

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
    uint32_t block_magic;              // (2^32 - 1) / block_size
    int mask_words;                    // words of the per-tile bit mask in LDS (documents)
    float *part_o;                     // [T * H * G, splits, 128]
    float2 *part_ml;                   // [T * H * G, splits]
    float2 *row_ml;                    // [T * H * G] maximum and sum of every row (accumulated weights only)
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

// The workgroup's row tile: its sequence (b < 0: none) with rows, length and prefix, and the tile's number in
// it.  Every wave finds it by itself; a lane reads all of a sequence's numbers at once.
struct RowTile {
    int b, tile, first, rows, len, prefix;               // (T, and so the first row, is below 2^31)
};
template <int ROWS>
__device__ inline RowTile find_row_tile(const PromptArgs &a, int want) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.B; base += 64) {
        int tiles = 0, len = 0, prefix = 0;
        PromptRows r = {0, 0};
        if (base + lane < a.B) {
            r = sequence_rows(a.cu_rows, a.T, base + lane);
            len = sequence_length(a.seq_lens, base + lane, a.n_max);
            prefix = min(sequence_prefix(a.score, base + lane), len);
            tiles = (int)(((int64_t)r.rows * a.G + ROWS - 1) / ROWS);
        }
        const int upto = (int)wave_prefix_u32((uint32_t)tiles);
        const uint64_t hit = __ballot(before + upto > want);
        if (hit) {
            const int who = __ffsll((unsigned long long)hit) - 1;
            auto its = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
            RowTile t = {base + who, want - before - (its(upto) - its(tiles)), its((int)r.first), its(r.rows), its(len), its(prefix)};
            if (t.tile < 0 || t.tile >= its(tiles)) t.b = -1;          // (cu_rows that do not ascend)
            return t;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return RowTile{-1, 0, 0, 0, 0, 0};
}

__device__ inline uint64_t uniform(uint64_t x) {         // the same in every lane
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32;
}

// The keys k0 .. k0 + 63 that a lane's query row sees, as bits: [row_from, pos] and [0, row_prefix), of these
// the ones that `exist` (the same in every lane) and, with documents, the ones of its own; kd is the
// document of key k0 + lane.
__device__ inline uint64_t seen_keys(int k0, uint64_t exist, int pos, int row_from, int row_prefix, bool docs, int kd, int row_doc) {
    auto below = [&](int j) { const int x = min(max(j - k0, 0), 64); return x == 0 ? 0ull : ~0ull >> (64 - x); };
    uint64_t see = ((below(pos + 1) & ~below(row_from)) | below(row_prefix)) & exist;
    if (docs) {                                          // one turn per document among the keys, mostly one or two
        uint64_t left = exist, own = 0;
        while (left) {
            const int d = __builtin_amdgcn_readlane(kd, __ffsll((unsigned long long)left) - 1);
            const uint64_t hit = __ballot(kd == d);
            own = d == row_doc ? hit : own;
            left &= ~hit;
        }
        see &= own;
    }
    return see;
}
// all ones where a lane's key r of 16 (bit 8 (r / 4) + r % 4 of `seen`) is seen
__device__ inline uint32_t seen_mask(uint32_t seen, int r) { return (uint32_t)((int32_t)(seen << (31 - (8 * (r / 4) + r % 4))) >> 31); }

// 16 bytes per lane from memory into LDS at the wave-uniform byte address `lds` plus 16 * lane, without
// passing through registers.  The compiler does not see the access: whoever reads the LDS waits with
// direct_loads_done() and a barrier first.  (M0, which holds the LDS address, has no other use here.)
__device__ inline void load_direct(uint32_t lds, const char *p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p) : "memory");
}
__device__ inline void load_direct4(uint32_t lds, const void *p) {   // 4 bytes per lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p) : "memory");
}
// all of this wave's direct loads but the last LEFT have arrived
template <int LEFT>
__device__ inline void direct_loads_done() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }

__device__ uint4 g_zero_row;           // what lanes of a row that does not exist load

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4v;

// RULE: 0 scores as they are (the scale goes into the exponent), 1 scaled, with a distance bias, 2 capped as well.  (One
// kernel for 1 and 2: 99 instead of 93 us for 2 048 rows with a bias.)
template <int DT, int RULE, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, WAVES == 8 ? 1 : 2) void prompt_attend_kernel(PromptArgs a) {
    using Shape = PromptShape<WAVES>;
    constexpr int kStages = Shape::kStages, kSlots = Shape::kSlots, kPromptRows = Shape::kRows, kThreads = Shape::kThreads;
    constexpr bool kF32 = DT == PQHSA_F32, GENERAL = RULE > 0;
    constexpr int KT = kF32 ? 32 : 64;                   // keys per tile
    constexpr int kTT = KT / 32;                         // matrix tiles of keys
    constexpr int kRowBytes = kD * (kF32 ? 4 : 2);
    constexpr int kSlices = kRowBytes / 32;              // 16-byte pieces of a row per lane of a pair
    constexpr int kRowLanes = kRowBytes / 16;            // lanes that fetch one row
    constexpr int kPass = 64 / kRowLanes;                // rows a wave fetches per instruction
    constexpr int kSteps = kF32 ? 16 : KT / 16;          // matrix instructions of the value product per 32 dims
    constexpr int kLoads = 16 / WAVES;                   // instructions of a wave per K or V tile
    constexpr int kVat = kStages * kTileBytes;           // K of stage i at i * kTileBytes, V behind all of K
    extern __shared__ __align__(16) char lds[];
    int64_t *offs = reinterpret_cast<int64_t *>(lds + 2 * kVat);                   // [slots][64] row addresses
    int32_t *phys = reinterpret_cast<int32_t *>(offs + kSlots * 64);               // [slots][64] blocks as looked up
    int32_t *kdoc = phys + kSlots * 64;                                            // [slots][64] documents
    uint64_t *valid = reinterpret_cast<uint64_t *>(kdoc + kSlots * 64);            // [slots] rows that exist
    int32_t *tiles = reinterpret_cast<int32_t *>(valid + kSlots);                  // [slots] tile of the walk (documents)
    int32_t *poison = tiles + kSlots;                                              // [3]: a sum is not finite; values were set aside in tiles seen in part; in whole ones
    uint32_t *odd = reinterpret_cast<uint32_t *>(poison + 4);                      // [128 dims] 1: inf, 2: -inf, 4: NaN among the latter
    uint32_t *wanted = odd + kD;                                                   // [mask_words] tiles to walk
    uint32_t *pure = wanted + a.mask_words;                                        // [mask_words] tiles of the rows' one document
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char *)lds;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane & 31, kg = lane >> 5;
    // Workgroups go to the eight XCDs in turn: where heads and splits allow it, the row tiles of one
    // (head, split) stay on one XCD, whose L2 then holds their K/V.
    const int streams = a.H * a.splits;
    int stream, order;
    if (streams % 8 == 0) {
        const int id = blockIdx.x / 8;
        order = id % a.tiles;
        stream = id / a.tiles * 8 + (int)(blockIdx.x % 8);
    } else {
        stream = blockIdx.x % streams;
        order = blockIdx.x / streams;
    }
    const int h = stream % a.H, split = stream / a.H;
    const RowTile rows = find_row_tile<kPromptRows>(a, a.tiles - 1 - order);       // the longest rows of a prompt first
    if (rows.b < 0) return;
    const int b = rows.b, tile = rows.tile, len = rows.len;
    const int first_pos = len - rows.rows;
    const int64_t packed = (int64_t)rows.rows * a.G;
    const int64_t pr = (int64_t)tile * kPromptRows + wave * 32 + n;
    const bool mine = pr < packed;
    const int prc = (int)(mine ? pr : packed - 1);       // rows past the end repeat the last one
    const int token = prc / a.G, g = prc - token * a.G;
    const int pos = first_pos + token;
    const int prefix_all = rows.prefix;
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
    const int begin = a.score.window > 0 ? max(0, max(wg_lo, 0) - window + 1) : 0;   // (rows in front of the sequence see nothing)
    const int walk_a = wg_hi >= 0 ? (prefix_all + KT - 1) / KT : 0;
    const int walk_b = max(begin / KT, walk_a);
    const int count = wg_hi >= 0 ? walk_a + max(0, (end + KT - 1) / KT - walk_b) : 0;
    const int per = (count + a.splits - 1) / a.splits;
    const int t_begin = min(split * per, count), t_end = min(t_begin + per, count);
    auto key_tile = [&](int t) { return (t < walk_a ? t : walk_b + t - walk_a) * KT; };

    // query rows as the second operand: lane (n, kg) holds row n
    u32x4 qf[kSlices];
    {
        const char *p = a.q + ((int64_t)(rows.first + token) * a.q_row + (int64_t)(h * a.G + g) * a.q_head) * a.kv.esize;
#pragma unroll
        for (int u = 0; u < kSlices; ++u) qf[u] = *reinterpret_cast<const u32x4 *>(p + (u * 2 + kg) * 16);
    }

    if (docs && t_begin < t_end) {
        // a bit per tile of the walk: some key lies in the rows' documents; every key is of their one document
        constexpr int kTokens = kPromptRows / 64, kPer = 64 / KT, kBatch = 8 / kPer;   // (8 tiles a wave and turn)
        constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
        int d_lo = 0x7fffffff, d_hi = -0x7fffffff - 1, own[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) own[i] = docs[max(min(wg_lo + i * 64 + lane, wg_hi), 0)];
#pragma unroll 1
        for (int w = wave; w * 8 < t_end - t_begin; w += WAVES) {
            int d[kBatch];
            bool in[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const int t = t_begin + w * 8 + x * kPer + lane / KT;
                const int j = key_tile(t) + lane % KT;
                in[x] = t < t_end && j < len;
                d[x] = docs[in[x] ? j : 0];
            }
            if (w == wave) {
#pragma unroll
                for (int i = 0; i < kTokens; ++i) { d_lo = min(d_lo, own[i]); d_hi = max(d_hi, own[i]); }
                constexpr uint32_t kSign = 0x80000000u;    // (the order of the bits is then that of the numbers)
                d_hi = (int)(wave_max_u32((uint32_t)d_hi ^ kSign) ^ kSign);
                d_lo = (int)(~wave_max_u32(~((uint32_t)d_lo ^ kSign)) ^ kSign);
            }
            uint32_t some = 0, whole = 0;
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const uint64_t hit = __ballot(in[x] && d[x] >= d_lo && d[x] <= d_hi);
                const uint64_t same = __ballot(in[x] && d[x] == d_lo && d_lo == d_hi);
#pragma unroll
                for (int y = 0; y < kPer; ++y) {
                    if ((hit >> (y * 32)) & kAll) some |= 1u << (x * kPer + y);
                    if (((same >> (y * 32)) & kAll) == kAll) whole |= 1u << (x * kPer + y);
                }
            }
            // (bits behind the last tile, in this byte's word or not written at all, are never looked at)
            if (lane == 0) {
                reinterpret_cast<uint8_t *>(wanted)[w] = (uint8_t)some;
                reinterpret_cast<uint8_t *>(pure)[w] = (uint8_t)whole;
            }
        }
        __syncthreads();
    }
    // the first tile at or after t that has to be walked (t_end: none)
    auto next = [&](int t) {
        if (!docs) return min(t, t_end);
        while (t < t_end) {
            const int x = t - t_begin;
            const uint32_t bits = __builtin_amdgcn_readfirstlane(wanted[x / 32]) >> (x % 32);
            if (bits) return min(t + __ffs((int)bits) - 1, t_end);
            t = t_begin + (x / 32 + 1) * 32;
        }
        return t_end;
    };
    // Tiles whose every key rows at positions [lo, hi] all see (one document aside): numbers [0, pre) and
    // [from, to) of the walk.
    struct Whole { int pre, from, to; };
    auto whole_tiles = [&](int lo, int hi) {
        Whole w = {0, 0, 0};
        if (lo < 0) return w;
        w.pre = min(prefix_all / KT, walk_a);            // tiles that end inside the prefix
        const int last = (lo + 1) / KT;                  // key tiles that end at or before lo
        const int start = a.score.window > 0 ? (max(hi - window + 1, 0) + KT - 1) / KT : 0;   // the first that begins inside hi's window
        // key tile k is number k below walk_a, walk_a + k - walk_b from walk_b on, and in neither part between them
        auto number = [&](int k) { return k < walk_a ? k : walk_a + max(k - walk_b, 0); };
        w.from = number(start);
        w.to = number(last);
        return w;
    };
    const Whole wave_whole = whole_tiles(w_lo, w_hi), wg_whole = whole_tiles(wg_lo, wg_hi);
    auto all_see = [&](int t, const Whole &w) {
        const bool one_doc = !docs || ((__builtin_amdgcn_readfirstlane(pure[(t - t_begin) / 32]) >> ((t - t_begin) % 32)) & 1);
        return one_doc && (t < w.pre || (t >= w.from && t < w.to));
    };

    const float slope2 = GENERAL && a.score.slopes ? a.score.slopes[h * a.G + g] * kLog2e : 0.0f;
    const int row_doc = docs && pos >= 0 ? docs[pos] : 0;
    const int row_prefix = pos >= 0 ? prefix_all : 0;
    const int row_from = pos >= 0 ? max(pos - window + 1, 0) : 0x7fffffff;   // keys [row_from, pos] and [0, row_prefix)

    // Tile number `x` of this workgroup's own walk, t_end behind the last.
    auto tile_at = [&](int x) { return docs ? __builtin_amdgcn_readfirstlane(tiles[x & (kSlots - 1)]) : min(t_begin + x, t_end); };
    // Addresses of a tile's rows, -1: past the sequence, outside the cache, or no tile at all.  The blocks
    // come from the table straight into LDS (a load into registers would make the compiler wait for every
    // direct load in flight); two stages later they become addresses.
    const int32_t *table = a.kv.block_table + (int64_t)b * a.kv.max_blocks;
    auto block_of = [&](int j) {                         // j / block_size: the product is one short at most
        int q = (int)__umulhi((uint32_t)j, a.block_magic);
        return j - q * a.kv.block_size >= a.kv.block_size ? q + 1 : q;
    };
    auto look_up = [&](int x, int t) {                   // (one wave)
        const int slot = x & (kSlots - 1);
        const int j = key_tile(t) + lane;
        const bool in = t < t_end && lane < KT && j < len;
        if (a.kv.paged)
            load_direct4(lds0 + 2 * kVat + kSlots * 512 + slot * 256,
                         in ? static_cast<const void *>(table + block_of(j)) : &g_zero_row);
        if (docs) {
            load_direct4(lds0 + 2 * kVat + kSlots * 768 + slot * 256, in ? static_cast<const void *>(docs + j) : &g_zero_row);
            if (lane == 0) tiles[slot] = t;
        }
    };
    auto resolve = [&](int x, int t) {                   // (one wave, once the blocks are there)
        const int slot = x & (kSlots - 1);
        const int j = key_tile(t) + lane;
        bool ok = t < t_end && lane < KT && j < len;
        int64_t off = (int64_t)h * a.kv.stride_head;
        if (a.kv.paged) {
            const int p = phys[slot * 64 + lane];
            ok = ok && p >= 0 && p < a.blocks;
            off += (int64_t)p * a.kv.stride_block + (int64_t)(j - block_of(j) * a.kv.block_size) * a.kv.stride_tok;
        } else {
            off += (int64_t)b * a.kv.stride_seq + (int64_t)j * a.kv.stride_tok;
        }
        offs[slot * 64 + lane] = ok ? off * a.kv.esize : -1;
        const uint64_t bits = __ballot(ok);
        if (lane == 0) valid[slot] = bits;
    };
    // Row r of K lies with its 16-byte piece c at place c ^ (r & 15); row r of V (2-byte types) at place
    // c ^ 2 (r & 7): the matrix operands' reads then spread over the banks.  A tile past the end is fetched
    // as zeros, so that the number of loads in flight is always the same.
    // (All addresses are read before the first load is issued: no read of LDS may move past one, and a wait for each
    // took half of the time that requesting a tile does.)
    auto fetch = [&](int x) {
        int64_t off[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) off[i] = offs[(x & (kSlots - 1)) * 64 + (wave * kLoads + i) * kPass + lane / kRowLanes];
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = (wave * kLoads + i) * kPass + lane / kRowLanes;
                const int turn = v ? (kF32 ? 0 : (r & 7) << 1) : r & 15;
                const char *p = (v ? a.kv.v_base : a.kv.k_base) + off[i] + ((lane % kRowLanes) ^ turn) * 16;
                load_direct(lds0 + (v ? kVat : 0) + (x & (kStages - 1)) * kTileBytes + (wave * kLoads + i) * 1024,
                            off[i] < 0 ? reinterpret_cast<const char *>(&g_zero_row) : p);
            }
    };
    // A weight of zero does not cancel an infinite or NaN value, and one that is too small for its type loses it.  The
    // walk is made without a thought for that; where a sum then is not finite it is made again with such values
    // set aside.  They come back at the end: those of a tile that all rows of the workgroup see whole by the dim, the
    // others for the rows that see them.
    auto set_aside = [&](char *vl, bool whole) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kTileBytes / 16 / kThreads; ++i) {
            const int at = i * kThreads + tid;
            u32x4 *p = reinterpret_cast<u32x4 *>(vl + at * 16);
            const u32x4 x = *p;
            u32x4 y;
#pragma unroll
            for (int w = 0; w < 4; ++w) y[w] = finite_part<DT>(x[w]);
            if (x[0] == y[0] && x[1] == y[1] && x[2] == y[2] && x[3] == y[3]) continue;
            *p = y;
            bad = true;
            if (!whole) continue;
            const int row = at / kRowLanes, first = ((at % kRowLanes) ^ (kF32 ? 0 : (row & 7) << 1)) * (kD / kRowLanes);
#pragma unroll
            for (int e = 0; e < kD / kRowLanes; ++e) {
                float v;
                if constexpr (kF32) v = __uint_as_float(x[e]);
                else v = e & 1 ? Half16<DT>::high(x[e / 2]) : Half16<DT>::low(x[e / 2]);
                if (!(fabsf(v) < INFINITY)) atomicOr(odd + first + e, v > 0.0f ? 1u : v < 0.0f ? 2u : 4u);
            }
        }
        if (bad) poison[whole ? 2 : 1] = 1;
        __syncthreads();
    };

    WeightBase<DT> base;
    float l;
    f32x16 acc[4];                                       // dim 32 dt + 8 (r / 4) + 4 kg + r % 4 of row n in acc[dt][r]
    // where GENERAL is false scores stay unscaled, the scale goes into the exponent
    const float unit = GENERAL ? 1.0f : a.score.scale2;

    // S^T of a tile: key 32 T + 8 (r / 4) + 4 kg + r % 4 of row n in s[T][r]
    auto score_product = [&](const char *kl, f32x16 (&s)[kTT]) {
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[T][r] = 0.0f;
#pragma unroll
        for (int u = 0; u < kSlices; ++u)
#pragma unroll
            for (int T = 0; T < kTT; ++T) {
                const int key = T * 32 + n;
                const u32x4 x = *reinterpret_cast<const u32x4 *>(kl + key * kRowBytes + (((u * 2 + kg) ^ (n & 15)) * 16));
                if constexpr (kF32) {
                    const f32x4 y = __builtin_bit_cast(f32x4, x), z = __builtin_bit_cast(f32x4, qf[u]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[T] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[c], z[c], s[T], 0, 0, 0);
                } else {
                    s[T] = Half16<DT>::mfma32(__builtin_bit_cast(uint4, x), __builtin_bit_cast(uint4, qf[u]), s[T]);
                }
            }
    };
    // the score rule on them: cap and bias (GENERAL), and the mask where the wave does not see the tile whole
    auto finish_scores = [&](f32x16 (&s)[kTT], int t, int slot) {
        const int k0 = key_tile(t);
        if constexpr (GENERAL) {
            if constexpr (RULE == 2) {
                float most = 0.0f;
#pragma unroll
                for (int T = 0; T < kTT; ++T)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        s[T][r] *= a.score.in_cap;
                        most = fmaxf(most, fabsf(s[T][r]));
                    }
                if (__ballot(most >= kTanhSmall) == 0) {         // scores far below the cap: no exponential, no quotient
#pragma unroll
                    for (int T = 0; T < kTT; ++T)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[T][r] = a.score.cap2 * tanh_small(s[T][r]);
                } else {
#pragma unroll
                    for (int T = 0; T < kTT; ++T)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[T][r] = a.score.cap2 * tanh_score(s[T][r]);
                }
            } else {
#pragma unroll
                for (int T = 0; T < kTT; ++T)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[T][r] *= a.score.scale2;
            }
            if (a.score.slopes) {
#pragma unroll
                for (int T = 0; T < kTT; ++T)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[T][r] -= slope2 * (float)abs(pos - (k0 + T * 32 + 8 * (r / 4) + 4 * kg + r % 4));
            }
        }
        const uint64_t exist = uniform(valid[slot]);
        if (all_see(t, wave_whole) && exist == (KT == 64 ? ~0ull : 0xffffffffull)) return;
        const uint64_t see = seen_keys(k0, exist, pos, row_from, row_prefix, docs != nullptr, docs ? kdoc[slot * 64 + lane] : 0, row_doc);
#pragma unroll
        for (int T = 0; T < kTT; ++T) {
            const uint32_t seen = (uint32_t)(see >> (32 * T)) >> (4 * kg);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t keep = seen_mask(seen, r);
                s[T][r] = __uint_as_float((__float_as_uint(s[T][r]) & keep) | (0xff800000u & ~keep));   // (-inf)
            }
        }
    };
    auto largest = [&](const f32x16 (&s)[kTT]) {
        float top = -INFINITY;
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[T][r]);
        return top * unit;
    };
    auto move_base = [&](float top) {
        uint64_t low = __ballot(base.falls(top, kPromptDrop));
        low &= low << 32 | low >> 32;                    // in both lanes of a row
        if (__ballot(base.raises(top)) | low) {
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            const float f = base.move(top, kPromptDrop);
            l *= f;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) acc[dt] *= f;
        }
    };
    // Weights, rounded to the value type for the product (their sum l is not): each at most half a step off,
    // independently, no more than the output's own rounding.  (fp16 ones that lie more than 2^27 below the
    // largest of their tile are subnormal: 2^-38 of that one off, at most.  A second product for the remainders, as
    // in the single token's kernel, would cost half as many matrix instructions again.)
    auto weigh = [&](const f32x16 (&s)[kTT], uint4 (&pw)[kSteps]) {
        const float origin = base.origin();
        float p[kTT][16];
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[T][r] = exp2_fast(GENERAL ? s[T][r] - origin : __builtin_fmaf(s[T][r], unit, -origin));
            }
        // (a tile's weights among themselves first, in pairs: one after the other into l they would lose 1e-6 of it
        // over a long walk, and every accumulated weight with it)
        float sum[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r] = kTT == 2 ? p[0][r] + p[kTT - 1][r] : p[0][r];
#pragma unroll
        for (int half = 8; half > 0; half /= 2)
#pragma unroll
            for (int r = 0; r < half; ++r) sum[r] += sum[r + half];
        l += sum[0];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            if constexpr (kF32) {
                pw[u] = make_uint4(__float_as_uint(p[0][u]), 0u, 0u, 0u);
            } else {
                const float *x = &p[u / 2][(u % 2) * 8];
                pw[u] = make_uint4(Half16<DT>::pack(x[0], x[1]), Half16<DT>::pack(x[2], x[3]), Half16<DT>::pack(x[4], x[5]), Half16<DT>::pack(x[6], x[7]));
            }
        }
    };
    // O^T += V^T P.  2-byte types: a transposing read gives a lane four keys of its dim; two of them are the
    // eight keys 16u + 4kg + {0..3, 8..11} whose weights the lane holds in pw[u].
    auto value_product = [&](uint32_t vl, const uint4 (&pw)[kSteps]) {
        if constexpr (kF32) {
#pragma unroll
            for (int u = 0; u < kSteps; ++u)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const float v = *reinterpret_cast<const float *>(lds + (vl - lds0) + (8 * (u / 4) + 4 * kg + u % 4) * kRowBytes + (dt * 32 + n) * 4);
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, __uint_as_float(pw[u].x), acc[dt], 0, 0, 0);
                }
        } else {
            const int i = lane & 15, key = 4 * kg + (i >> 2);
            const int piece = ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
#pragma unroll
            for (int u = 0; u < kSteps; ++u)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const uint32_t at = vl + key * kRowBytes + (((dt * 4 + piece) ^ ((key & 7) << 1)) * 16) + (i & 1) * 8 + u * 16 * kRowBytes;
                    const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v *)(size_t)at);
                    const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v *)(size_t)(at + 8 * kRowBytes));
                    const uint2 xw = __builtin_bit_cast(uint2, x), yw = __builtin_bit_cast(uint2, y);
                    acc[dt] = Half16<DT>::mfma32(make_uint4(xw.x, xw.y, yw.x, yw.y), pw[u], acc[dt]);
                }
        }
    };

    // The ring.  While tile x is computed, K and V of tile x + stages - 1 are requested, the blocks of tile
    // x + slots - 1 looked up and those of tile x + stages turned into addresses.  What iteration x requests has
    // arrived by the end of iteration x + stages - 2.  Tile x's own slot is still being read (its documents),
    // so the first that may be looked up anew is the one of tile x - 1.
    constexpr int kInFlight = (kStages - 2) * 2 * kLoads;
    if (tid < 3) poison[tid] = 0;
    if (tid < kD) odd[tid] = 0u;
    const int t_first = next(t_begin);
#pragma unroll 1
    for (bool careful = false;; careful = true) {
        base = WeightBase<DT>();
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[dt][r] = 0.0f;
        int t = t_first, reach = t;
        f32x16 s[kTT];
        if (t < t_end) {
            for (int x = 0; x < wave; ++x) reach = next(reach + 1);
            if (wave < kSlots - 1) look_up(wave, reach);     // (as many waves as slots; the last slot is iteration 0's)
            // the query rows with them: inside the loop the compiler's wait would also be one for the direct loads
#pragma unroll
            for (int u = 0; u < kSlices; ++u) asm volatile("" : "+v"(qf[u]));
            direct_loads_done<0>();
            if (wave < kSlots - 1) resolve(wave, reach);
            __syncthreads();
            if (docs && wave == 0) reach = tile_at(kSlots - 2);
#pragma unroll
            for (int x = 0; x < kStages - 1; ++x) fetch(x);
            direct_loads_done<kInFlight>();
            __syncthreads();
            if (careful) set_aside(lds + kVat, all_see(t, wg_whole));
        }
#pragma unroll 1
        for (int x = 0; t < t_end; ++x) {
            const int t1 = tile_at(x + 1);
            const char *kl = lds + (x & (kStages - 1)) * kTileBytes;
            char *vl = lds + kVat + (x & (kStages - 1)) * kTileBytes;
            uint4 pw[kSteps];
            fetch(x + kStages - 1);
            score_product(kl, s);
            finish_scores(s, t, x & (kSlots - 1));
            move_base(largest(s));
            weigh(s, pw);
            value_product(lds0 + (uint32_t)(vl - lds), pw);
            if (wave == 0) {
                if (x + kStages >= kSlots - 1) resolve(x + kStages, tile_at(x + kStages));
                if (docs) reach = next(reach + 1);
                look_up(x + kSlots - 1, docs ? reach : min(t_begin + x + kSlots - 1, t_end));
            }
            if (t1 < t_end) {
                direct_loads_done<kInFlight>();
                __syncthreads();
                if (careful) set_aside(lds + kVat + ((x + 1) & (kStages - 1)) * kTileBytes, all_see(t1, wg_whole));
            }
            t = t1;
        }
        direct_loads_done<0>();                              // (no load may reach the LDS after the workgroup has left it)
        if (careful || t_first >= t_end) break;
        bool finite = true;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) finite = finite & (fabsf(acc[dt][r]) < INFINITY);
        if (!finite) poison[0] = 1;
        __syncthreads();                                 // (the ring is no longer read, either)
        if (!poison[0]) break;
    }
    l += __shfl_xor(l, 32, kWave);
    if (t_first < t_end && poison[2]) {                  // the infinities and NaN that were set aside
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t x = odd[dt * 32 + 8 * (r / 4) + 4 * kg + r % 4];
                if (x) acc[dt][r] += x == 1u ? INFINITY : x == 2u ? -INFINITY : NAN;
            }
    }
    if (t_first < t_end && poison[1]) {
#pragma unroll 1
        for (int t = t_first; t < t_end; t = next(t + 1)) {
            const int k0 = key_tile(t);
            if (all_see(t, wg_whole)) continue;
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
    const float settled = base.settle(l), m = base.m;
    l *= settled;
    if constexpr (base.kHalf) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) acc[dt] *= settled;
    }
    if (!mine) return;
    const int64_t r = (int64_t)(rows.first + token) * (a.H * a.G) + h * a.G + g;
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
    if (kg == 0 && a.row_ml) a.row_ml[r] = make_float2(m, l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    char *o = a.out + ((int64_t)(rows.first + token) * a.out_row + (int64_t)(h * a.G + g) * a.out_head) * a.kv.esize;
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
// With every row's maximum m and sum l known the weights are one product K Q^T and an exp2 away (m and l
// rather than the log-sum-exp: rounding that to fp32 would put 1e-6 of error on every weight).  A wave keeps 64
// keys (32 in fp32) as the first operand in registers; the counted rows pass by in tiles of 32, which the
// four waves of a workgroup share in LDS (a row's pieces lie 256 bytes apart for the lanes of an operand:
// read from memory by every wave they took four times the requests).  Every lane sums its rows' weights
// of its keys, the lanes are summed at the end: no atomics, one owner per key.  32 rows of 4 x 7 heads over
// 32 768 keys: 26 us, 290 TFLOP/s; half of it is the chain of reads before the first tile (32 keys a wave and a
// ring of two tiles: 39 us).
constexpr int kMassWaves = 4;
constexpr int mass_keys(int dt) { return dt == PQHSA_F32 ? 32 : 64; }      // of a wave

template <int DT>
__global__ __launch_bounds__(kMassWaves * kWave, 2) void prompt_mass_kernel(PromptArgs a) {
    constexpr bool kF32 = DT == PQHSA_F32;
    constexpr int kRowBytes = kD * (kF32 ? 4 : 2), kSlices = kRowBytes / 32, kRowLanes = kRowBytes / 16, kPass = 64 / kRowLanes;
    constexpr int kTile = 32 * kRowBytes, kLoads = kTile / 1024 / kMassWaves;
    constexpr int kKeys = mass_keys(DT), kTT = kKeys / 32;
    // A ring of four tiles, each with the (m, l) of its rows: three are on their way while one is computed.
    constexpr int kRing = 4;
    __shared__ __align__(16) char tiles[kRing * kTile];
    __shared__ float2 sums[kRing][32];
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char *)tiles;
    const uint32_t sums0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char *)reinterpret_cast<char *>(&sums[0][0]);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n = lane & 31, kg = lane >> 5;
    const int b = blockIdx.y / a.H, h = blockIdx.y - b * a.H;
    const int len = __builtin_amdgcn_readfirstlane(sequence_length(a.seq_lens, b, a.n_max));
    const int wg_k0 = blockIdx.x * kMassWaves * kKeys, k0 = wg_k0 + wave * kKeys;
    if (wg_k0 >= len) return;
    const int wg_last = min(wg_k0 + kMassWaves * kKeys, len) - 1;
    PromptRows rows = sequence_rows(a.cu_rows, a.T, b);
    rows.first = __builtin_amdgcn_readfirstlane((int)rows.first);
    rows.rows = __builtin_amdgcn_readfirstlane(rows.rows);
    const int first_pos = len - rows.rows;
    const int prefix = __builtin_amdgcn_readfirstlane(min(sequence_prefix(a.score, b), len));
    const int window = a.score.window > 0 ? a.score.window : 0x7fffffff;
    const int32_t *docs = a.score.docs ? a.score.docs + (int64_t)b * a.score.docs_stride : nullptr;

    const int from = a.mass_rows > 0 ? max(0, rows.rows - a.mass_rows) : 0;
    const int packed = rows.rows * a.G;
    int at = from * a.G;
    // rows before the first that can see a key of the workgroup (causal order, unless the prefix reaches one)
    if (wg_k0 >= prefix) at = max(at, max(wg_k0 - first_pos, 0) * a.G);
    const uint32_t magic = 0xffffffffu / (uint32_t)a.G;
    auto token_of = [&](int pr) {                        // pr / G: the product is one short at most
        const int t = (int)__umulhi((uint32_t)pr, magic);
        return pr - t * a.G >= a.G ? t + 1 : t;
    };
    // A lane walks the rows it fetches 32 packed rows (step_tokens tokens and step_heads heads) at a time; behind
    // the last row it fetches that one again, so that the number of loads in flight is always the same.
    const int step_tokens = token_of(32), step_heads = 32 - step_tokens * a.G;
    struct Walk { int pr, g; int64_t off; };             // packed row, its head in the group, where it lies
    auto start = [&](int pr, int64_t row, int64_t head) {
        const int token = token_of(pr), g = pr - token * a.G;
        return Walk{pr, g, (rows.first + token) * row + (int64_t)(h * a.G + g) * head};
    };
    auto advance = [&](Walk &w, int64_t step, int64_t wrap) {
        w.pr += 32;
        w.g += step_heads;
        w.off += step;
        if (w.g >= a.G) { w.g -= a.G; w.off += wrap; }
    };
    const int64_t q_row = a.q_row * a.kv.esize, q_head = a.q_head * a.kv.esize;
    const int64_t q_step = step_tokens * q_row + step_heads * q_head, q_wrap = q_row - a.G * q_head;
    const int64_t ml_row = (int64_t)a.H * a.G, ml_step = step_tokens * ml_row + step_heads, ml_wrap = ml_row - a.G;
    Walk walk[kLoads], ml_walk = {0, 0, 0};
    int64_t q_last = 0, ml_last = 0;
    auto fetch = [&](int buf) {                          // the next tile (pieces placed as the prompt kernel's K)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (wave * kLoads + i) * kPass + lane / kRowLanes;
            load_direct(lds0 + buf * kTile + (wave * kLoads + i) * 1024,
                        a.q + (walk[i].pr < packed ? walk[i].off : q_last) + ((lane % kRowLanes) ^ (r & 15)) * 16);
            advance(walk[i], q_step, q_wrap);
        }
        if (wave == 0) {
            load_direct4(sums0 + buf * 256, reinterpret_cast<const float *>(a.row_ml + (ml_walk.pr < packed ? ml_walk.off : ml_last)) + (lane & 1));
            advance(ml_walk, ml_step, ml_wrap);
        }
    };
    if (at < packed) {
        q_last = start(packed - 1, q_row, q_head).off;
        ml_last = start(packed - 1, ml_row, 1).off;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) walk[i] = start(at + (wave * kLoads + i) * kPass + lane / kRowLanes, q_row, q_head);
        ml_walk = start(at + lane / 2, ml_row, 1);
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) fetch(i);
    }

    const int key_doc = docs && lane < kKeys && k0 + lane < len ? docs[k0 + lane] : 0;
    uint4 kf[kTT][kSlices];
    uint64_t ok = 0;                                     // keys that exist, the same in every lane
#pragma unroll
    for (int T = 0; T < kTT; ++T) {
        const int64_t off = k0 + T * 32 + n < len ? checked_row_bytes(a.kv, a.blocks, b, h, k0 + T * 32 + n) : -1;
#pragma unroll
        for (int u = 0; u < kSlices; ++u)
            kf[T][u] = *reinterpret_cast<const uint4 *>(a.kv.k_base + (off < 0 ? 0 : off) + (u * 2 + kg) * 16);
        ok |= (uint64_t)(uint32_t)__ballot(off >= 0) << (32 * T);   // (both halves of the wave hold the same 32 keys)
    }
    const bool general = a.score.capped || a.score.slopes || docs;
    float sum[kTT][16];
#pragma unroll
    for (int T = 0; T < kTT; ++T)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[T][r] = 0.0f;
    direct_loads_done<0>();
    __syncthreads();

#pragma unroll 1
    for (int buf = 0; at < packed; at += 32, buf = (buf + 1) % kRing) {
        // past the window of all the workgroup's keys, and these are not in the prefix: no later row sees them
        const int first_row = first_pos + token_of(at);
        if (wg_k0 >= prefix && first_row - wg_last >= window) break;
        fetch((buf + kRing - 1) % kRing);
        const float2 ml = sums[buf][n];
        const bool gives = at + n < packed && ml.y != 0.0f;            // m = +inf: the row gives no weight
        const float m = gives ? ml.x : INFINITY, inv = gives ? 1.0f / ml.y : 0.0f;
        f32x16 s[kTT];
#pragma unroll
        for (int T = 0; T < kTT; ++T)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[T][r] = 0.0f;
#pragma unroll
        for (int u = 0; u < kSlices; ++u) {
            const uint4 x = *reinterpret_cast<const uint4 *>(tiles + buf * kTile + n * kRowBytes + (((u * 2 + kg) ^ (n & 15)) * 16));
#pragma unroll
            for (int T = 0; T < kTT; ++T) {
                if constexpr (kF32) {
                    const f32x4 y = __builtin_bit_cast(f32x4, kf[T][u]), z = __builtin_bit_cast(f32x4, x);
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[T] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[c], z[c], s[T], 0, 0, 0);
                } else {
                    s[T] = Half16<DT>::mfma32(kf[T][u], x, s[T]);
                }
            }
        }
        const int last_row = first_pos + token_of(min(at + 31, packed - 1));
        if (!general && ok == (kTT == 2 ? ~0ull : 0xffffffffull) && first_row >= k0 + kKeys - 1 && last_row - k0 < window) {   // every row sees every key
#pragma unroll
            for (int T = 0; T < kTT; ++T)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sum[T][r] = __builtin_fmaf(exp2_fast(__builtin_fmaf(s[T][r], a.score.scale2, -m)), inv, sum[T][r]);
        } else {
            const int pr = min(at + n, packed - 1), token = token_of(pr), g = pr - token * a.G, pos = first_pos + token;
            const uint64_t see = seen_keys(k0, ok, pos, pos >= 0 ? max(pos - window + 1, 0) : 0x7fffffff, pos >= 0 ? prefix : 0,
                                           docs != nullptr, key_doc, docs && pos >= 0 ? docs[pos] : 0);
            // (one branch a rule, not one a key: few workgroups come here, but the others are done long before them)
            float unit = a.score.scale2;
            if (a.score.capped) {
                unit = a.score.cap2;
#pragma unroll
                for (int T = 0; T < kTT; ++T)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[T][r] = tanh_score(s[T][r] * a.score.in_cap);
            }
            const float slope2 = a.score.slopes ? a.score.slopes[h * a.G + g] * kLog2e : 0.0f;
#pragma unroll
            for (int T = 0; T < kTT; ++T) {
                const uint32_t seen = (uint32_t)(see >> (32 * T)) >> (4 * kg);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = k0 + T * 32 + 8 * (r / 4) + 4 * kg + r % 4;
                    const float bias = __builtin_fmaf(slope2, (float)abs(pos - j), m);
                    sum[T][r] += __uint_as_float(__float_as_uint(exp2_fast(__builtin_fmaf(s[T][r], unit, -bias)) * inv) & seen_mask(seen, r));
                }
            }
        }
        direct_loads_done<(kRing - 2) * kLoads>();
        __syncthreads();
    }
    direct_loads_done<0>();
    // Sums over the 32 lanes of each half, of 32 (16) keys at once: in every step a lane hands over the half of
    // its keys that its partner keeps, so lane n ends up with key n (n % 16) of the half.
    float x[kTT * 16];
#pragma unroll
    for (int i = 0; i < kTT * 16; ++i) x[i] = sum[i / 16][i % 16];
    if constexpr (kTT == 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] += __shfl_xor(x[i], 16, kWave);
    }
#pragma unroll
    for (int half = kTT * 8; half > 0; half /= 2)
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = n & half ? x[i + half] : x[i], give = n & half ? x[i] : x[i + half];
            x[i] = keep + __shfl_xor(give, half, kWave);
        }
    const int T = n / 16 % kTT, r = n % 16, j = k0 + T * 32 + 8 * (r / 4) + 4 * kg + r % 4;
    if (n < kTT * 16 && j < len) {
        const int64_t o = (int64_t)blockIdx.y * a.mass_stride + j;
        a.mass_out[o] = (a.mass_in ? a.decay * a.mass_in[o] : 0.0f) + x[0];
    }
}

namespace {

struct PromptPlan {
    int waves;
    int64_t tiles;
    int splits;
    size_t ml_at, row_at, bytes;
};

PromptPlan plan_prompt(int64_t T, int B, int H, int G, int n_max, int rows_hint, int key_tile, bool mass) {
    PromptPlan p = {};
    p.splits = 1;
    // Eight waves (256 rows, four stages, one workgroup per compute unit) halve the K/V traffic of four (128
    // rows, two stages, two workgroups), which overlap each other's starts and ends: 2.35 against 2.57 ms for 16 384
    // rows of 8 x 4 heads and 176 against 203 us for 4 096 (512 of the large workgroups), 95 against 98 us
    // for documents of 360 rows; fewer rows than that do not fill the chip with the large ones.
    p.waves = T * G / 256 * H >= 512 ? 8 : 4;
    const int tile_rows = p.waves * 32;
    p.tiles = (T * G + tile_rows - 1) / tile_rows + B;              // every sequence may end inside a tile
    int64_t busy = p.tiles - B;
    if (rows_hint > 0 && rows_hint * (int64_t)B <= T) {             // about as many tiles as sequences have
        const int64_t each = ((int64_t)rows_hint * G + tile_rows - 1) / tile_rows;
        if (each * B > busy) busy = each * B;
    }
    if (busy < 1) busy = 1;
    // Splitting the keys fills the chip where row tiles are few, but the partial sums go through memory and the
    // join is a launch: the number of splits with the least estimated time, in us.
    const double tile_us = key_tile == 32 ? 7.0 : 2.2, key_tiles = (double)((n_max + key_tile - 1) / key_tile);
    const int64_t room = p.waves == 8 ? 256 : 512;
    double best = 0.0;
    for (int s = 1; s <= 128 && s <= key_tiles; ++s) {
        const double turns = (double)((busy * H * s + room - 1) / room), longest = (double)(int64_t)((key_tiles + s - 1) / s);
        double us = turns * longest * tile_us;
        if (s > 1) us += 8.0 + (double)(T * H * G) * (0.0008 + s * 0.00034);
        if (s == 1 || us < best) {
            best = us;
            p.splits = s;
        }
    }
    const size_t rows = (size_t)T * H * G;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    if (p.splits > 1) {
        take(rows * p.splits * kD * sizeof(float));
        p.ml_at = take(rows * p.splits * sizeof(float2));
    }
    if (mass) p.row_at = take(rows * sizeof(float2));
    p.bytes = at;
    return p;
}

template <int DT, int RULE, int WAVES>
int launch_prompt(const PromptArgs &a, hipStream_t stream) {
    auto kern = prompt_attend_kernel<DT, RULE, WAVES>;
    const size_t lds = PromptShape<WAVES>::kLds + 2 * (size_t)a.mask_words * 4;
    static std::atomic<uint64_t> raised{0};              // devices on which the kernel's LDS limit is raised already
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (e == hipSuccess && (device > 63 || !(raised.load(std::memory_order_relaxed) & bit))) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e == hipSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) {
        set_error("prompt_attend: cannot raise the LDS limit: %s", hipGetErrorString(e));
        return PQHSA_ELAUNCH;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.H * a.tiles * a.splits)), dim3(WAVES * kWave), lds, stream, a);
    return check_launch("prompt_attend");
}

template <int DT, int WAVES>
int launch_rule(int rule, const PromptArgs &a, hipStream_t stream) {
    return rule == 2 ? launch_prompt<DT, 2, WAVES>(a, stream) : rule == 1 ? launch_prompt<DT, 1, WAVES>(a, stream) : launch_prompt<DT, 0, WAVES>(a, stream);
}

}  // namespace

}  // namespace pqhsa

using namespace pqhsa;

extern "C" size_t pqhsa_prompt_attend_workspace_bytes(int64_t T, int32_t B, int32_t H, int32_t G, int32_t n_max,
                                                      int32_t rows_hint, int32_t dtype, int32_t with_mass) {
    if (T <= 0 || B <= 0 || H <= 0 || G <= 0 || n_max <= 0) return 256;
    const size_t need = plan_prompt(T, B, H, G, n_max, rows_hint, dtype == PQHSA_F32 ? 32 : 64, with_mass != 0).bytes;
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
    PQHSA_REQUIRE(T * G < 0x7fffffff - 65536 && T * H * G < 0x7fffffff, "%s: %lld rows of %d x %d heads are too many", what, (long long)T, H, G);
    PQHSA_REQUIRE((int64_t)B * H <= 65535, "%s: too many sequences and heads", what);
    const int key_tile = kv->dtype == PQHSA_F32 ? 32 : 64;
    const PromptPlan p = plan_prompt(T, B, H, G, n_max, rows_hint, key_tile, mass != nullptr);
    PQHSA_REQUIRE(p.tiles * H * p.splits <= 0x7fffffff, "%s: %lld row tiles are too many for one launch", what, (long long)p.tiles);
    if (workspace_bytes < p.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, p.bytes);
        return PQHSA_ENOSPC;
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    char *w = static_cast<char *>(workspace);
    PromptArgs a = {};
    a.q = static_cast<const char *>(q); a.q_row = q_stride_row; a.q_head = q_stride_head;
    a.out = static_cast<char *>(out); a.out_row = out_stride_row; a.out_head = out_stride_head;
    a.lse = lse;
    a.kv = make_view(kv);
    a.blocks = blocks; a.B = B; a.H = H; a.G = G; a.cu_rows = cu_rows; a.T = T; a.seq_lens = seq_lens; a.n_max = n_max;
    a.score = make_score(score);
    a.tiles = (int)p.tiles;
    a.block_magic = kv->paged ? 0xffffffffu / (uint32_t)kv->block_size : 0u;
    a.splits = p.splits;
    a.mask_words = score->docs ? (n_max / key_tile + 2 + 31) / 32 + 1 : 0;
    a.part_o = reinterpret_cast<float *>(w);
    a.part_ml = reinterpret_cast<float2 *>(w + p.ml_at);
    a.row_ml = mass ? reinterpret_cast<float2 *>(w + p.row_at) : nullptr;
    PQHSA_REQUIRE(PromptShape<8>::kLds + 2 * (size_t)a.mask_words * 4 <= 160 * 1024, "%s: n_max %d too large for a document mask", what, n_max);
    if (T > 0) {
        const int rule = score->softcap > 0.0f ? 2 : score->slopes || !(score->scale > 0.0f) ? 1 : 0;
        PQHSA_DISPATCH_DTYPE(kv->dtype, rc = p.waves == 8 ? launch_rule<DT, 8>(rule, a, stream) : launch_rule<DT, 4>(rule, a, stream));
        if (rc) return rc;
        if (p.splits > 1) {
            JoinArgs j = {a.part_o, a.part_ml, p.splits, H * G, a.out, a.out_row, a.out_head, a.lse, a.row_ml, cu_rows + B};
            rc = launch_join(j, kv->dtype, T * H * G, stream);
            if (rc) return rc;
        }
    }
    if (mass && n_max > 0) {
        a.mass_in = mass->in; a.mass_out = mass->out; a.mass_stride = mass->stride; a.decay = mass->decay; a.mass_rows = mass->rows;
        const int keys = kMassWaves * mass_keys(kv->dtype);
        const dim3 grid((unsigned)((n_max + keys - 1) / keys), (unsigned)(B * H));
        PQHSA_DISPATCH_DTYPE(kv->dtype, hipLaunchKernelGGL(prompt_mass_kernel<DT>, grid, dim3(kMassWaves * kWave), 0, stream, a));
        rc = check_launch("prompt_mass");
    }
    return rc;
}
