// The work list of paged attention (dpk_attn_paged.cuh), made by one block: by a kernel of its own, or for
// short lists by every CTA of the attention kernel for itself.
#pragma once

#include "dpk_attn_paged.cuh"

namespace dpk {

// Sum over the block's threads, for two values at once; `sh` holds 32 pairs.  Every thread gets the
// totals and the sums of the threads before it.
__device__ __forceinline__ int2 plan_scan(int2 v, int2* sh, int2& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x.x, o), z = __shfl_up_sync(0xffffffffu, x.y, o);
        if (lane >= o) { x.x += y; x.y += z; }
    }
    __syncthreads();                       // the previous use of sh is over
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int2 w = lane < warps ? sh[lane] : make_int2(0, 0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w.x, o), z = __shfl_up_sync(0xffffffffu, w.y, o);
            if (lane >= o) { w.x += y; w.y += z; }
        }
        sh[lane] = w;
    }
    __syncthreads();
    total = sh[warps - 1];
    const int2 before = warp ? sh[warp - 1] : make_int2(0, 0);
    return make_int2(x.x - v.x + before.x, x.y - v.y + before.y);
}

// New tokens of sequence s, 0 where query_start does not make sense.
__device__ __forceinline__ int plan_new(const PagedParams& p, int s, int& tok0)
{
    tok0 = p.qstart[s];
    const int end = p.qstart[s + 1];
    if (tok0 < 0 || end < tok0 || end > p.N) {
        atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
        tok0 = 0;
        return 0;
    }
    if (s == 0 && tok0 != 0)               // rows before the first sequence belong to none, like those behind the last
        atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
    return end - tok0;
}

// Tile number `at` of an item of `rows` rows, and the units of its visible range.
__device__ __forceinline__ int plan_tile(const PagedParams& p, int seq, int kvh, int at, int rows, PagedTile& t)
{
    t.seq = seq;
    t.kvh = kvh;
    const int fresh = plan_new(p, seq, t.tok0);
    t.m0 = at * p.tile_rows;
    t.rows = min(p.tile_rows, rows - t.m0);
    t.kv_len = p.kv_lens[seq];
    if (t.kv_len < 0 || t.kv_len > static_cast<int64_t>(p.W) * p.page) {
        atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
        t.kv_len = 0;
    }
    t.pos0 = t.kv_len - fresh;
    t.kv_end = t.kv_len;
    int last = 0, head;
    if (p.rows || !p.mask) {
        if (p.causal) last = paged_row(p, t, t.rows - 1, head);
    } else {                                     // the last row that is not routed out
        last = -1;
        for (int r = t.rows - 1; r >= 0 && last < 0; --r) last = paged_row(p, t, r, head);
    }
    if (p.causal) t.kv_end = min(t.kv_len, t.pos0 + last + 1);
    return last >= 0 && t.kv_end > 0 ? paged_units(p, t) : 0;
}

// Where the tiles of (s, kvh) are put down by paged_rows_kernel: room for as many as its rows can need.
__device__ __forceinline__ int plan_slot(const PagedParams& p, int s, int kvh)
{
    int tok0;
    const int fresh = plan_new(p, s, tok0);
    return p.Hk * (tok0 * p.rep / p.tile_rows + s) + kvh * (fresh * p.rep / p.tile_rows + 1);
}

// The whole block cuts the work: `tile`, `start` [tiles + 1] and `first` [S * Hk] may be shared memory.
__device__ __forceinline__ void plan_work(const PagedParams& p, PagedTile* tile, int32_t* start, int* first,
                                          int2* sh, int& tiles_out, int& length_out)
{
    const int tid = threadIdx.x, threads = blockDim.x;
    const int items = p.S * p.Hk;
    // 1. tiles of every (sequence, KV head)
    int carry = 0;
    for (int x0 = 0; x0 < items; x0 += threads) {
        const int x = x0 + tid;
        int n = 0;
        if (x < items) {
            int tok0;
            const int rows = p.rows ? p.row_count[x] : plan_new(p, x / p.Hk, tok0) * p.rep;
            n = (rows + p.tile_rows - 1) / p.tile_rows;
        }
        int2 t;
        const int2 at = plan_scan(make_int2(n, 0), sh, t);
        if (x < items) first[x] = carry + at.x;
        carry += t.x;
    }
    const int tiles = min(carry, p.max_tiles);
    __syncthreads();
    // 2. the visible keys of every tile; tiles without any are dropped.  Worker after worker gets every
    //    workers-th tile, so that tiles that are worked on at the same time are neighbours and read the same
    //    K and V: in order, each worker would keep to its own sequences, and together they would go
    //    through more K and V than L2 holds (12 sequences of 509 tokens over 3000, 64 heads: 739 us
    //    instead of 837; where it all fits L2 the order makes no difference).
    //    Worker g's share of the T tiles is every place of the line in [g T / W, (g + 1) T / W), so that all
    //    workers pass their k-th tile at about the same time.
    const int rounds = tiles / p.workers;            // tiles that every worker has; some have one more
    int kept = 0, length = 0;
    for (int q0 = 0; q0 < tiles; q0 += threads) {
        const int q = q0 + tid;
        int n = 0;
        PagedTile pt = {};
        if (q < tiles) {
            // max_tiles * workers < 2^31 was checked
            const int g = ((q + 1) * p.workers - 1) / tiles, g_first = g * tiles / p.workers, k = q - g_first;
            const int t = k < rounds ? k * p.workers + g : rounds * p.workers + g_first - g * rounds;
            int lo = 0, hi = items - 1;
            while (lo < hi) {                        // last item that starts at or before t
                const int mid = (lo + hi + 1) >> 1;
                if (first[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int s = lo / p.Hk, kvh = lo - s * p.Hk;
            if (p.rows) {
                const int64_t slot = static_cast<int64_t>(plan_slot(p, s, kvh)) + t - first[lo];
                if (slot >= 0 && slot < p.max_tiles) {       // always, where query_start ascends
                    pt = p.slot[slot];
                    n = paged_units(p, pt);
                }
            } else {
                int tok0;
                n = plan_tile(p, s, kvh, t - first[lo], plan_new(p, s, tok0) * p.rep, pt);
            }
        }
        int2 total;
        const int2 at = plan_scan(make_int2(n > 0, n > 0 ? n + p.tile_gap : 0), sh, total);
        if (n > 0) {
            tile[kept + at.x] = pt;
            start[kept + at.x] = length + at.y;
        }
        kept += total.x;
        length += total.y;
    }
    if (tid == 0) start[kept] = length;
    __syncthreads();
    tiles_out = kept;
    length_out = length;
}

// Places per worker: an equal share, but where few tiles meet many workers no shorter than makes the walk
// through a worker's units about as long as joining the parts of a tile takes: the
// square root of a tile's units, times 0.8 for CTAs and 0.3 for warps (32 rows over 16000 keys 53 us without, 27 with;
// 8 rows over 120000 62 and 47; 0 to 1.0 were tried).
__device__ __forceinline__ int plan_range(const PagedParams& p, int tiles, int length)
{
    const int share = max((length + p.workers - 1) / p.workers, p.min_range);
    return tiles > 0 ? max(share, static_cast<int>((p.tile_rows > 16 ? 0.8f : 0.3f) * sqrtf(static_cast<float>(length) / tiles))) : share;
}

}  // namespace dpk
