// Eviction from a cache by accumulated attention weight: per (sequence, KV head) the first `sink` and the
// last `recent` keys stay, and of the others those with the largest weight, until `keep` are left; their
// K/V rows are copied, in ascending order of position, to the first slots of another cache.
//
// Two launches.  The selection reads the weights (4 bytes a key, a few times, from the L2 after the
// first): one workgroup per stream finds the weight of the last key to stay by a radix search on the bits
// (11 + 11 + 10) and then writes the kept positions in order with one block-wide prefix sum per 16 384
// keys.  The move reads and writes 2 * 256 bytes per kept key and is all the traffic there is: lanes of 16
// bytes, 16 lanes a row, eight rows' loads of a thread in flight.
#include "common.h"
#include "dense_common.h"
#include "select_common.h"

namespace pqhsa {

constexpr int kEvictThreads = 1024;
constexpr int kEvictRun = 16;                            // consecutive keys per thread in the ordered pass
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
};

__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ __align__(16) uint32_t hist[2048];
    __shared__ uint32_t found[2];
    __shared__ uint32_t wave_sums[kEvictThreads / kWave];
    const int tid = threadIdx.x, lane = tid & 63;
    const int bh = blockIdx.x, b = bh / a.H;
    const int len = sequence_length(a.seq_lens, b, a.n_max);
    const int left = min(len, a.keep);
    const float *mass = a.mass + (int64_t)bh * a.mass_stride;
    int32_t *kept = a.kept + (int64_t)bh * a.keep;
    float *mass_out = a.mass_out ? a.mass_out + (int64_t)bh * a.out_stride : nullptr;
    if (bh == b * a.H && tid == 0) a.new_lens[b] = left;
    for (int64_t r = left + tid; r < a.keep; r += kEvictThreads) kept[r] = -1;
    if (mass_out)
        for (int64_t r = left + tid; r < a.out_stride; r += kEvictThreads) mass_out[r] = 0.0f;

    const int low = min(a.sink, len), high = max(low, len - a.recent);
    uint32_t want = len > a.keep ? (uint32_t)(a.keep - low - (len - high)) : 0u;
    uint32_t cut = 0;                                    // order key of the last weight that stays
    const bool search = want > 0;
    if (search) {
        uint32_t prefix = 0;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const int bins = pass == 2 ? 1024 : 2048;
            for (int x = tid; x < 2048; x += kEvictThreads) hist[x] = 0u;
            __syncthreads();
            for (int j = low + tid; j < high; j += kEvictThreads) {
                const uint32_t k = order_key(mass[j]);
                if (pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
            }
            __syncthreads();
            if (tid < kWave) find_from_top(hist, bins, want, &found[0], &found[1]);
            __syncthreads();
            prefix = pass == 2 ? (prefix << 10) | found[0] : (prefix << 11) | found[0];
            want -= found[1];
            __syncthreads();
        }
        cut = prefix;                                    // `want` keys of exactly this weight stay, the first ones
    }

    // ordered pass: counts of sure keys (low half) and of ties (high half) per thread, summed over the block
    uint32_t base_sure = 0, base_tie = 0;
    for (int j0 = 0; j0 < len; j0 += kEvictThreads * kEvictRun) {
        const int j = j0 + tid * kEvictRun;
        float w[kEvictRun];
        uint32_t sure = 0, tie = 0;                      // a bit per key of the run
#pragma unroll
        for (int e = 0; e < kEvictRun; ++e) {
            w[e] = j + e < len ? mass[j + e] : 0.0f;
            const uint32_t k = order_key(w[e]);
            const bool in = j + e < len, fixed = len <= a.keep || j + e < low || j + e >= high;
            if (in && (fixed || (search && k > cut))) sure |= 1u << e;
            else if (in && search && k == cut) tie |= 1u << e;
        }
        const uint32_t counts = (uint32_t)__popc(sure) | ((uint32_t)__popc(tie) << 16);
        uint32_t upto = wave_prefix_u32(counts);         // (at most 16 384 of each: no carry between the halves)
        if (lane == 63) wave_sums[tid / kWave] = upto;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int v = 0; v < kEvictThreads / kWave; ++v) {
            before += v < tid / kWave ? wave_sums[v] : 0u;
            all += wave_sums[v];
        }
        upto += before - counts;
        uint32_t s = base_sure + (upto & 0xffffu), q = base_tie + (upto >> 16);
#pragma unroll
        for (int e = 0; e < kEvictRun; ++e) {
            const bool is_sure = (sure >> e) & 1, is_tie = (tie >> e) & 1;
            if (is_sure || (is_tie && q < want)) {
                const uint32_t r = s + min(q, want);
                kept[r] = j + e;
                if (mass_out) mass_out[r] = w[e];
            }
            s += is_sure;
            q += is_tie;
        }
        base_sure += all & 0xffffu;
        base_tie += all >> 16;
        __syncthreads();
    }
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

}  // namespace pqhsa

using namespace pqhsa;

extern "C" int pqhsa_evict(const pqhsa_kv_view *src, int32_t src_blocks, const pqhsa_kv_view *dst, int32_t dst_blocks,
                           int32_t B, int32_t H, const float *mass, int64_t mass_stride, const int32_t *seq_lens,
                           int32_t n_max, int32_t keep, int32_t sink, int32_t recent, int32_t *kept, int32_t *new_lens,
                           float *mass_out, int64_t mass_out_stride, void *stream_v) {
    const char *what = "evict";
    int rc = validate_view(src);
    if (rc) return rc;
    rc = validate_view(dst);
    if (rc) return rc;
    PQHSA_REQUIRE(src->dtype == dst->dtype, "%s: caches of dtype %d and %d", what, src->dtype, dst->dtype);
    PQHSA_REQUIRE(B >= 0 && H > 0 && (int64_t)B * H <= 65535, "%s: B %d, H %d", what, B, H);
    PQHSA_REQUIRE(n_max >= 0 && mass_stride >= n_max, "%s: n_max %d, weights of stride %lld", what, n_max, (long long)mass_stride);
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
    PQHSA_REQUIRE(mass && seq_lens && kept && new_lens, "%s: NULL argument", what);
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    const EvictArgs e = {mass, mass_stride, seq_lens, B, H, n_max, keep, sink, recent, kept, new_lens, mass_out, mass_out_stride};
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)(B * H)), dim3(kEvictThreads), 0, stream, e);
    rc = check_launch("evict_select");
    if (rc || left == 0) return rc;
    const MoveArgs m = {make_view(src), make_view(dst), src_blocks, dst_blocks, H, keep, kept, new_lens};
    const dim3 grid((unsigned)((left + kMoveRows - 1) / kMoveRows), (unsigned)(B * H));
    if (src->dtype == PQHSA_F32) hipLaunchKernelGGL(evict_move_kernel<512>, grid, dim3(kMoveThreads), 0, stream, m);
    else hipLaunchKernelGGL(evict_move_kernel<256>, grid, dim3(kMoveThreads), 0, stream, m);
    return check_launch("evict_move");
}
