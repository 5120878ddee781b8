// Eviction from a cache by accumulated attention weight: per (sequence, KV head) the first `sink` and the
// last `recent` keys stay, and of the others those with the largest weight, until `keep` are left; their
// K/V rows are copied, in ascending order of position, to the first slots of another cache.
//
// The selection is a radix search on the weights' bits (11 + 11 + 10) for the last one that stays, then a
// pass that writes the kept positions in order.  Counting digits is arithmetic more than traffic (about 15
// instructions a key and pass), so a stream of more than 16 384 keys is spread over workgroups: one launch
// per digit, each workgroup leaving the histogram of its 16 384 keys in the workspace, and the ordered
// pass.  The histograms of the chunks in front of its own also tell a workgroup where its first kept key
// goes, so nothing is counted twice and no launch clears anything.  A shorter stream is one workgroup
// and one launch, its keys in registers.
//
// The move reads and writes 2 * 256 bytes (2-byte types) per kept key and is nearly all the traffic there
// is: 16 bytes a lane, 16 lanes a row, all rows of a thread requested before the first is stored.
//
// Measured (bf16): 16 sequences of 16 384 to 65 536 keys, 8 heads, 8 192 kept each: the move 212 us, 5.0 TB/s read and
// written (a large copy reaches 4.9); the selection 58 us in four launches.  One sequence of 8 192 keys, 8
// heads, 4 096 kept: 12 + 6.5 us, the selection bound by the instructions of 8 workgroups on 8 compute units.
#include "common.h"
#include "dense_common.h"

namespace pqhsa {

constexpr int kEvictThreads = 1024;
constexpr int kEvictLoads = 16;                          // keys per thread, all requested at once
constexpr int kEvictChunk = kEvictThreads * kEvictLoads;
constexpr int kEvictCopies = 8;                          // histogram copies, by lane: a wave's equal digits rarely meet
constexpr int kEvictBins = 2048;
constexpr int kEvictStride = kEvictBins + 8;             // words of a copy: the copies of a bin lie in different banks
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 64;                            // kept keys per workgroup of the move

struct EvictArgs {
    const float *mass;
    int64_t mass_stride;
    const int32_t *seq_lens;
    int B, H, n_max, keep, sink, recent;
    int32_t *kept;                                       // [B, H, keep]
    int32_t *new_lens;                                   // [B]
    float *mass_out;                                     // [B, H, out_stride] or NULL
    int64_t out_stride;
    // streams of more than one chunk
    int chunks;
    uint32_t *hist;                                      // [3][B * H, chunks, 2048] digits of every chunk's candidates
    uint32_t *sure;                                      // [2][B * H, chunks] keys above the cut's first (second) digit
    uint2 *found;                                        // [2][B * H] digits of the cut so far, keys still wanted
};

// What is decided for a stream before any weight is looked at: keys [0, low) and [high, len) stay, `want` of the others.
struct EvictStream {
    int len, low, high;
    uint32_t want;
    bool all;
};
__device__ inline EvictStream evict_stream(const EvictArgs &a, int b) {
    EvictStream s;
    s.len = sequence_length(a.seq_lens, b, a.n_max);
    s.low = min(a.sink, s.len);
    s.high = max(s.low, s.len - a.recent);
    s.all = s.len <= a.keep;
    s.want = s.all ? 0u : (uint32_t)(a.keep - s.low - (s.len - s.high));
    return s;
}

struct EvictLds {
    uint2 copies[kEvictCopies][kEvictStride / 2];
    uint32_t found[2];
    uint32_t wave_sums[kEvictThreads / kWave];
};

constexpr int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
constexpr int digit_bits(int pass) { return pass == 2 ? 10 : 11; }

// This thread's 16 keys of the chunk at j0: wave-sized pieces, so that a load is one line and lanes are in order.
__device__ inline int chunk_key(int j0, int e) { return j0 + ((int)(threadIdx.x / kWave) * kEvictLoads + e) * kWave + (int)(threadIdx.x & 63); }
__device__ inline void load_chunk(const float *mass, int j0, int len, float (&w)[kEvictLoads]) {
#pragma unroll
    for (int e = 0; e < kEvictLoads; ++e) {
        const int j = chunk_key(j0, e);
        w[e] = j < len ? mass[j] : 0.0f;
    }
}

// whether any of this wave's keys lies below `len` (a chunk's last waves may have none: every instruction a key
// costs is one of 16 waves' on one compute unit, so these leave early)
__device__ inline bool wave_has_keys(int j0, int len) { return __builtin_amdgcn_readfirstlane(chunk_key(j0, 0) & ~63) < len; }

// sum of the waves' numbers: of those in front of this one, of all
__device__ inline uint32_t waves_before(const EvictLds &l) {
    const int lane = threadIdx.x & 63;
    return wave_total_u32(lane < (int)(threadIdx.x / kWave) ? l.wave_sums[lane] : 0u);
}
__device__ inline uint32_t waves_total(const EvictLds &l) {
    const int lane = threadIdx.x & 63;
    return wave_total_u32(lane < kEvictThreads / kWave ? l.wave_sums[lane] : 0u);
}

__device__ inline void clear_copies(EvictLds &l) {
#pragma unroll
    for (int c = 0; c < kEvictCopies; ++c) l.copies[c][threadIdx.x] = make_uint2(0u, 0u);
}

// adds the digits of the chunk's candidates, those that share `prefix` above the digit (copies cleared, barriers outside)
__device__ inline void count_digits(EvictLds &l, const float (&w)[kEvictLoads], int j0, const EvictStream &s, int pass, uint32_t prefix) {
    uint32_t *copy = reinterpret_cast<uint32_t *>(l.copies[threadIdx.x & (kEvictCopies - 1)]);
    const int shift = digit_shift(pass), above = shift + digit_bits(pass);
    if (!wave_has_keys(j0, s.high)) return;
#pragma unroll
    for (int e = 0; e < kEvictLoads; ++e) {
        const int j = chunk_key(j0, e);
        const uint32_t k = order_key(w[e]);
        if (j >= s.low && j < s.high && (pass == 0 || (k >> above) == prefix))
            atomicAdd(&copy[(k >> shift) & ((1u << digit_bits(pass)) - 1u)], 1u);
    }
}

// A thread owns two neighbouring bins, thread 0 the highest two: (higher, lower).  Read, they are cleared for the
// next digit.
__device__ inline int high_bin() { return kEvictBins - 1 - 2 * (int)threadIdx.x; }
__device__ inline uint2 fold_copies(EvictLds &l) {
    uint2 r = make_uint2(0u, 0u);
#pragma unroll
    for (int c = 0; c < kEvictCopies; ++c) {
        uint2 &x = l.copies[c][high_bin() / 2];
        r.x += x.y;
        r.y += x.x;
        x = make_uint2(0u, 0u);
    }
    return r;
}

// The highest bin b with count(bins > b) < want <= count(bins >= b), from every thread's own two bins:
// found = (b, count(bins > b)).  want >= 1 and at most the total.
__device__ inline void find_cut(EvictLds &l, uint2 mine, uint32_t want) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    const uint32_t both = mine.x + mine.y;
    uint32_t upto = wave_prefix_u32(both);
    if (lane == 63) l.wave_sums[wave] = upto;
    __syncthreads();
    upto += waves_before(l);
    const uint32_t before = upto - both;
    if (before < want && want <= upto) {
        const bool first = want <= before + mine.x;
        l.found[0] = (uint32_t)(high_bin() - (first ? 0 : 1));
        l.found[1] = first ? before : before + mine.x;
    }
    __syncthreads();
}

// sum of one number per thread, in every thread
__device__ inline uint32_t block_total(EvictLds &l, uint32_t v) {
    v = wave_total_u32(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) l.wave_sums[threadIdx.x / kWave] = v;
    __syncthreads();
    return waves_total(l);
}

// outputs that do not depend on the weights: the new length and what lies behind the kept keys
__device__ inline void write_rest(const EvictArgs &a, int bh, int b, int len) {
    const int left = min(len, a.keep);
    if (bh == b * a.H && threadIdx.x == 0) a.new_lens[b] = left;
    for (int64_t r = left + (int)threadIdx.x; r < a.keep; r += kEvictThreads) a.kept[(int64_t)bh * a.keep + r] = -1;
    if (a.mass_out)
        for (int64_t r = left + (int)threadIdx.x; r < a.out_stride; r += kEvictThreads) a.mass_out[(int64_t)bh * a.out_stride + r] = 0.0f;
}

// bits of `mask` below this lane's
__device__ inline uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// The kept keys of a chunk, in order, behind `sure` keys that stay whatever the ties do and `ties` keys of
// exactly the cut's weight; the first `quota` ties of the stream stay.
__device__ inline void write_kept(const EvictArgs &a, EvictLds &l, int bh, const EvictStream &s, const float (&w)[kEvictLoads], int j0,
                                  uint32_t cut, uint32_t quota, uint32_t sure_before, uint32_t ties_before) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    uint64_t sure[kEvictLoads], tie[kEvictLoads];        // a bit per lane
    uint32_t counts = 0;
    const bool some = wave_has_keys(j0, s.len);
    const uint32_t open = s.all ? 0u : (uint32_t)(s.high - s.low);     // keys [low, low + open) are judged by their weight
    if (s.want == 0) cut = ~0u;                          // (none of them stays: no weight is above, and no tie counts)
    if (some) {
#pragma unroll
        for (int e = 0; e < kEvictLoads; ++e) {
            const int j = chunk_key(j0, e);
            const uint32_t k = order_key(w[e]);
            const bool judged = (uint32_t)(j - s.low) < open;
            sure[e] = __ballot(j < s.len && (!judged || k > cut));
            tie[e] = __ballot(judged && k == cut);
            counts += (uint32_t)__popcll(sure[e]) | ((uint32_t)__popcll(tie[e]) << 16);
        }
    }
    __syncthreads();
    if (lane == 0) l.wave_sums[wave] = counts;           // (at most 16 384 of each: no carry between the halves)
    __syncthreads();
    if (!some) return;
    const uint32_t before = waves_before(l);
    uint32_t n = sure_before + (before & 0xffffu), q = ties_before + (before >> 16);
    int32_t *kept = a.kept + (int64_t)bh * a.keep;
    float *mass_out = a.mass_out ? a.mass_out + (int64_t)bh * a.out_stride : nullptr;
#pragma unroll
    for (int e = 0; e < kEvictLoads; ++e) {
        const uint32_t my_n = n + lanes_below(sure[e]), my_q = q + lanes_below(tie[e]);
        if (((sure[e] >> lane) & 1) || (((tie[e] >> lane) & 1) && my_q < quota)) {
            const uint32_t r = my_n + min(my_q, quota);
            kept[r] = chunk_key(j0, e);
            if (mass_out) mass_out[r] = w[e];
        }
        n += (uint32_t)__popcll(sure[e]);
        q += (uint32_t)__popcll(tie[e]);
    }
}

// streams of one chunk: everything in one workgroup
__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ EvictLds l;
    const int bh = blockIdx.x, b = bh / a.H;
    const EvictStream s = evict_stream(a, b);
    float w[kEvictLoads];
    load_chunk(a.mass + (int64_t)bh * a.mass_stride, 0, s.len, w);
    write_rest(a, bh, b, s.len);
    uint32_t prefix = 0, want = s.want;
    if (want > 0) {
        clear_copies(l);
        __syncthreads();
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            count_digits(l, w, 0, s, pass, prefix);
            __syncthreads();
            find_cut(l, fold_copies(l), want);
            prefix = (prefix << digit_bits(pass)) | l.found[0];
            want -= l.found[1];
        }
    }
    write_kept(a, l, bh, s, w, 0, prefix, want, 0, 0);
}

// Digit `PASS` of one chunk of a longer stream, once the digits in front of it are known from the chunks'
// histograms.
__device__ inline uint2 *hist_row(const EvictArgs &a, int pass, int bh, int chunk) {
    return reinterpret_cast<uint2 *>(a.hist + (((int64_t)pass * a.B * a.H + bh) * a.chunks + chunk) * kEvictBins);
}
__device__ inline uint2 sum_hist(const EvictArgs &a, int pass, int bh, int used) {
    uint2 sum = make_uint2(0u, 0u);
#pragma unroll 8
    for (int c = 0; c < used; ++c) {
        const uint2 h = hist_row(a, pass, bh, c)[threadIdx.x];
        sum.x += h.x;
        sum.y += h.y;
    }
    return sum;
}

template <int PASS>
__global__ __launch_bounds__(kEvictThreads) void evict_digit_kernel(EvictArgs a) {
    __shared__ EvictLds l;
    const int chunk = blockIdx.x, bh = blockIdx.y, b = bh / a.H, j0 = chunk * kEvictChunk;
    const EvictStream s = evict_stream(a, b);
    if (j0 >= s.len || s.want == 0) return;
    float w[kEvictLoads];
    load_chunk(a.mass + (int64_t)bh * a.mass_stride, j0, s.len, w);
    clear_copies(l);
    uint32_t prefix = 0, want = s.want;
    if constexpr (PASS > 0) {
        const int streams = a.B * a.H, used = (s.len + kEvictChunk - 1) / kEvictChunk;
        if constexpr (PASS == 2) { prefix = a.found[bh].x; want = a.found[bh].y; }
        const uint2 mine = hist_row(a, PASS - 1, bh, chunk)[threadIdx.x];
        find_cut(l, sum_hist(a, PASS - 1, bh, used), want);
        const int cut = (int)l.found[0];
        prefix = (prefix << digit_bits(PASS - 1)) | l.found[0];
        want -= l.found[1];
        const uint32_t above = block_total(l, (high_bin() > cut ? mine.x : 0u) + (high_bin() - 1 > cut ? mine.y : 0u));
        if (threadIdx.x == 0) {
            a.sure[((int64_t)(PASS - 1) * streams + bh) * a.chunks + chunk] = above;
            if (chunk == 0) a.found[(PASS - 1) * streams + bh] = make_uint2(prefix, want);
        }
    }
    __syncthreads();
    count_digits(l, w, j0, s, PASS, prefix);
    __syncthreads();
    hist_row(a, PASS, bh, chunk)[threadIdx.x] = fold_copies(l);
}

__global__ __launch_bounds__(kEvictThreads) void evict_order_kernel(EvictArgs a) {
    __shared__ EvictLds l;
    const int chunk = blockIdx.x, bh = blockIdx.y, b = bh / a.H, j0 = chunk * kEvictChunk;
    const EvictStream s = evict_stream(a, b);
    if (chunk == 0) write_rest(a, bh, b, s.len);
    if (j0 >= s.len) return;
    float w[kEvictLoads];
    load_chunk(a.mass + (int64_t)bh * a.mass_stride, j0, s.len, w);
    uint32_t prefix = 0, want = 0;
    // keys of the chunks in front that stay whatever their weight
    uint32_t sure = s.all ? (uint32_t)j0 : (uint32_t)(min(s.low, j0) + max(0, j0 - s.high)), ties = 0;
    if (s.want > 0) {
        const int streams = a.B * a.H, used = (s.len + kEvictChunk - 1) / kEvictChunk;
        prefix = a.found[streams + bh].x;
        want = a.found[streams + bh].y;
        const uint2 front = sum_hist(a, 2, bh, chunk);
        uint2 sum = front;
#pragma unroll 8
        for (int c = chunk; c < used; ++c) {
            const uint2 h = hist_row(a, 2, bh, c)[threadIdx.x];
            sum.x += h.x;
            sum.y += h.y;
        }
        find_cut(l, sum, want);
        const int cut = (int)l.found[0];
        prefix = (prefix << digit_bits(2)) | l.found[0];
        want -= l.found[1];
        uint32_t mine = (high_bin() > cut ? front.x : 0u) + (high_bin() - 1 > cut ? front.y : 0u);
        for (int c = threadIdx.x; c < chunk; c += kEvictThreads)
            mine += a.sure[(int64_t)bh * a.chunks + c] + a.sure[((int64_t)streams + bh) * a.chunks + c];
        sure += block_total(l, mine);
        ties = block_total(l, high_bin() == cut ? front.x : high_bin() - 1 == cut ? front.y : 0u);
    }
    write_kept(a, l, bh, s, w, j0, prefix, want, sure, ties);
}

struct MoveArgs {
    KvView src, dst;
    int src_blocks, dst_blocks, H, keep;
    const int32_t *kept;
    const int32_t *new_lens;
};

// BYTES of a row, 16 a lane.  A row of a block outside the cache is copied as zeros, one whose new place is
// outside is left out.
template <int BYTES>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(MoveArgs a) {
    constexpr int kLanes = BYTES / 16, kAtOnce = kMoveThreads / kLanes, kTimes = kMoveRows / kAtOnce;
    __shared__ int64_t from[kMoveRows], to[kMoveRows];
    const int tid = threadIdx.x;
    const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
    const int r0 = blockIdx.x * kMoveRows;
    const int rows = min(kMoveRows, min(a.new_lens[b], a.keep) - r0);
    if (rows <= 0) return;
    if (tid < kMoveRows) {
        int64_t x = -1, y = -1;
        if (tid < rows) {
            x = checked_row_bytes(a.src, a.src_blocks, b, h, a.kept[(int64_t)bh * a.keep + r0 + tid]);
            y = checked_row_bytes(a.dst, a.dst_blocks, b, h, r0 + tid);
        }
        from[tid] = x;
        to[tid] = y;
    }
    __syncthreads();
    const int lane = tid % kLanes, row = tid / kLanes;
    u32x4 k[kTimes], v[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const int64_t x = from[row + i * kAtOnce];
        const int64_t at = (x < 0 ? 0 : x) + lane * 16;
        k[i] = *reinterpret_cast<const u32x4 *>(a.src.k_base + at);
        v[i] = *reinterpret_cast<const u32x4 *>(a.src.v_base + at);
        if (x < 0) k[i] = v[i] = (u32x4){0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const int64_t y = to[row + i * kAtOnce];
        if (y < 0) continue;
        *reinterpret_cast<u32x4 *>(const_cast<char *>(a.dst.k_base) + y + lane * 16) = k[i];
        *reinterpret_cast<u32x4 *>(const_cast<char *>(a.dst.v_base) + y + lane * 16) = v[i];
    }
}

namespace {

struct EvictPlan {
    int chunks;
    size_t sure_at, found_at, bytes;
};
EvictPlan plan_evict(int B, int H, int n_max) {
    EvictPlan p = {};
    p.chunks = (n_max + kEvictChunk - 1) / kEvictChunk;
    if (p.chunks <= 1) return p;
    const size_t rows = (size_t)B * H * p.chunks;
    p.sure_at = 3 * rows * kEvictBins * sizeof(uint32_t);
    p.found_at = p.sure_at + ((2 * rows * sizeof(uint32_t) + 255) & ~(size_t)255);
    p.bytes = p.found_at + 2 * (size_t)B * H * sizeof(uint2);
    return p;
}

}  // namespace

}  // namespace pqhsa

using namespace pqhsa;

extern "C" size_t pqhsa_evict_workspace_bytes(int32_t B, int32_t H, int32_t n_max) {
    const size_t need = B > 0 && H > 0 && n_max > 0 ? plan_evict(B, H, n_max).bytes : 0;
    return need < 256 ? 256 : need;
}

extern "C" int pqhsa_evict(const pqhsa_kv_view *src, int32_t src_blocks, const pqhsa_kv_view *dst, int32_t dst_blocks,
                           int32_t B, int32_t H, const float *mass, int64_t mass_stride, const int32_t *seq_lens,
                           int32_t n_max, int32_t keep, int32_t sink, int32_t recent, int32_t *kept, int32_t *new_lens,
                           float *mass_out, int64_t mass_out_stride, void *workspace, size_t workspace_bytes,
                           void *stream_v) {
    const char *what = "evict";
    int rc = validate_view(src);
    if (rc) return rc;
    rc = validate_view(dst);
    if (rc) return rc;
    PQHSA_REQUIRE(src->dtype == dst->dtype, "%s: caches of dtype %d and %d", what, src->dtype, dst->dtype);
    PQHSA_REQUIRE(B >= 0 && H > 0 && (int64_t)B * H <= 65535, "%s: B %d, H %d", what, B, H);
    PQHSA_REQUIRE(n_max >= 0 && mass_stride >= n_max, "%s: n_max %d, weights of stride %lld", what, n_max, (long long)mass_stride);
    PQHSA_REQUIRE(n_max <= 0x7fffffff - 65536, "%s: n_max %d is too large (key numbers are 32 bits)", what, n_max);
    PQHSA_REQUIRE(sink >= 0 && recent >= 0 && keep > 0 && (int64_t)sink + recent <= keep, "%s: keep %d must be positive and hold sink %d + recent %d",
                  what, keep, sink, recent);
    const int left = keep < n_max ? keep : n_max;
    PQHSA_REQUIRE(!mass_out || mass_out_stride >= left, "%s: mass_out of stride %lld for %d keys", what, (long long)mass_out_stride, left);
    if (src->paged)
        PQHSA_REQUIRE(src_blocks > 0 && (int64_t)src->max_blocks * src->block_size >= n_max,
                      "%s: %d blocks, and a table of %d x %d tokens for n_max %d", what, src_blocks, src->max_blocks, src->block_size, n_max);
    if (dst->paged)
        PQHSA_REQUIRE(dst_blocks > 0 && (int64_t)dst->max_blocks * dst->block_size >= left,
                      "%s: %d new blocks, and a table of %d x %d tokens for %d keys", what, dst_blocks, dst->max_blocks, dst->block_size, left);
    PQHSA_REQUIRE(!(src->paged && dst->paged && src->block_table == dst->block_table) && !(!src->paged && !dst->paged && src->k_base == dst->k_base),
                  "%s: the new cache has to lie apart from the old one", what);
    if (B == 0) return PQHSA_OK;
    PQHSA_REQUIRE(mass && seq_lens && kept && new_lens && workspace, "%s: NULL argument", what);
    PQHSA_REQUIRE((uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", what);
    const EvictPlan p = plan_evict(B, H, n_max);
    if (workspace_bytes < p.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, p.bytes);
        return PQHSA_ENOSPC;
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    char *w = static_cast<char *>(workspace);
    const EvictArgs e = {mass, mass_stride, seq_lens, B, H, n_max, keep, sink, recent, kept, new_lens, mass_out, mass_out_stride,
                         p.chunks, reinterpret_cast<uint32_t *>(w), reinterpret_cast<uint32_t *>(w + p.sure_at),
                         reinterpret_cast<uint2 *>(w + p.found_at)};
    if (p.chunks <= 1) {
        hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)(B * H)), dim3(kEvictThreads), 0, stream, e);
        rc = check_launch("evict_select");
    } else {
        const dim3 grid((unsigned)p.chunks, (unsigned)(B * H));
        if (keep < n_max) {                              // (a length that is at most `keep` has nothing to search)
            hipLaunchKernelGGL(evict_digit_kernel<0>, grid, dim3(kEvictThreads), 0, stream, e);
            hipLaunchKernelGGL(evict_digit_kernel<1>, grid, dim3(kEvictThreads), 0, stream, e);
            hipLaunchKernelGGL(evict_digit_kernel<2>, grid, dim3(kEvictThreads), 0, stream, e);
        }
        hipLaunchKernelGGL(evict_order_kernel, grid, dim3(kEvictThreads), 0, stream, e);
        rc = check_launch("evict_order");
    }
    if (rc || left == 0) return rc;
    const MoveArgs m = {make_view(src), make_view(dst), src_blocks, dst_blocks, H, keep, kept, new_lens};
    const dim3 grid((unsigned)((left + kMoveRows - 1) / kMoveRows), (unsigned)(B * H));
    if (src->dtype == PQHSA_F32) hipLaunchKernelGGL(evict_move_kernel<512>, grid, dim3(kMoveThreads), 0, stream, m);
    else hipLaunchKernelGGL(evict_move_kernel<256>, grid, dim3(kMoveThreads), 0, stream, m);
    return check_launch("evict_move");
}
