// Attention of new tokens over a paged cache: what the work list, the two attention kernels and the
// joining kernel share.
//
// The work is cut into TILES and UNITS.  A tile is up to `tile_rows` (new token, query head) rows of
// one sequence and one KV head; a unit is `unit_keys` consecutive keys of a tile's visible range.
// The units of all tiles form one line, with `tile_gap` empty places behind each tile for what a
// tile costs beside its units, and worker w (a warp or a CTA) takes places [w * range, (w + 1) *
// range): sequences of very different lengths load the GPU evenly, a long cache with few rows is
// split over many workers, and nothing depends on lengths the host does not know.  A tile that one
// worker covers is finished there; of the others every worker leaves its un-normalised sum, its row
// maxima and row sums in one of its two slots (slot 0 for the tile that was begun by an earlier
// worker or starts with the range, slot 1 for the tile that starts later), and the joining kernel
// adds them in worker order: the same bits on every run.
#pragma once

#include "dpk_host.h"
#include "dpk_sm100.cuh"

namespace dpk {

struct PagedTile {
    int32_t seq, kvh;       // sequence, KV head
    int32_t m0, rows;       // rows [m0, m0 + rows) of the (sequence, KV head)'s row list
    int32_t kv_len;         // tokens of the sequence in the cache
    int32_t kv_end;         // keys [0, kv_end) are visible to some row of the tile
    int32_t pos0;           // cache position of the sequence's first new token
    int32_t tok0;           // its index in Q
};

struct PagedHead {          // written by the planning kernel
    int32_t tiles;          // tiles with work
    int32_t length;         // places of the line
    int32_t range;          // places per worker
    int32_t pad;
};

// Left by each worker for the joining kernel: the tile that starts in its range and ends behind it.
struct PagedBorder {
    PagedTile tile;
    int32_t last_worker;    // the worker that ends the tile; -1: there is no such tile
    int32_t slot;           // where this worker left its part; later ones use slot 0
    int32_t pad[2];
};

struct PagedParams {
    const uint8_t* Q;       // [N, Hq, D]
    const uint8_t* K;       // [P, page, Hk, D]
    const uint8_t* V;
    uint8_t* O;             // [N, Hq, D] packed
    const int32_t* table;   // [S, W]
    const int32_t* kv_lens; // [S]
    const int32_t* qstart;  // [S + 1]
    const uint8_t* mask;    // [N, NG] or NULL
    int64_t q_ts, page_stride, token_stride, table_stride;   // elements
    int N, S, W, P, page, Hq, Hk, NG, rep, hpg;
    int causal, clear_tail;
    float scale_log2;
    // workspace
    PagedHead* head;
    int32_t* start;         // [tiles + 1] place of each tile's first unit
    PagedTile* tile;        // [tiles]
    PagedTile* slot;        // [max_tiles] with `rows`: tiles as paged_rows_kernel leaves them
    int32_t* first_tile;    // [S * Hk] running number of tiles before dropping empty ones; more than kPlanItems only
    int32_t* rows;          // [Hk][N * rep] active rows of each (sequence, KV head), or NULL: all rows
    int32_t* row_count;     // [S * Hk] with `rows`
    PagedBorder* border;    // [workers]
    float* part_o;          // [workers][2][tile_rows][D]
    float* part_ml;         // [workers][2][tile_rows][2]
    int tile_rows, unit_keys, tile_gap, workers, min_range, max_tiles;
    int* status;
};

// Row r of a tile's list -> new token and query head; -1 where the row is routed out.  The bounds hold
// by themselves as long as query_start ascends; where it does not, two sequences may have written
// over each other's lists, and the checks keep every access inside Q, O and the lists.
__device__ __forceinline__ int paged_row(const PagedParams& p, const PagedTile& t, int r, int& head)
{
    int x = t.m0 + r;
    head = t.kvh * p.rep;
    if (x < 0) return -1;
    if (p.rows) {
        const int64_t at = static_cast<int64_t>(t.tok0) * p.rep + x;
        if (at >= static_cast<int64_t>(p.N) * p.rep) return -1;
        x = p.rows[static_cast<int64_t>(t.kvh) * p.N * p.rep + at];
    }
    const int i = x / p.rep;
    if (t.tok0 + i >= p.N) return -1;
    head += x - i * p.rep;
    if (!p.rows && p.mask && p.mask[static_cast<int64_t>(t.tok0 + i) * p.NG + head / p.hpg] == 0) return -1;
    return i;
}

// Last key that new token i of the tile's sequence sees, -1 or less where it sees none (or i is -1: no row).
__device__ __forceinline__ int paged_last_key(const PagedParams& p, const PagedTile& t, int i)
{
    return i < 0 ? -1 : p.causal ? min(t.kv_len - 1, t.pos0 + i) : t.kv_len - 1;
}

// What a row's sum of weighted values is multiplied by.  A row that sees no key is zero; any other is divided by the
// sum of its weights whatever that is: NaN where a score it sees is NaN or +inf, 0 (and so 0 * inf, NaN) where all
// its scores are -inf -- the softmax of such rows has no value, and the row says so, however the work was cut.
__device__ __forceinline__ float paged_inverse(int last_key, float l) { return last_key < 0 ? 0.f : 1.f / l; }

__device__ __forceinline__ int paged_units(const PagedParams& p, const PagedTile& t)
{
    return (t.kv_end + p.unit_keys - 1) / p.unit_keys;
}

// First tile with units at or behind `place`; the whole warp searches, 32 probes a step.
__device__ __forceinline__ int paged_find_tile(const PagedParams& p, const PagedTile* tile, const int32_t* start,
                                               int tiles, int place)
{
    int lo = 0, hi = tiles;                         // the last tile that starts at or before `place`
    const int lane = threadIdx.x & 31;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + lane * step;
        const bool ok = at < hi && start[at] <= place;
        const int n = __popc(__ballot_sync(0xffffffffu, ok));      // lane 0 always holds
        hi = min(hi, lo + n * step);
        lo = lo + (n - 1) * step;
    }
    return place < start[lo] + paged_units(p, tile[lo]) ? lo : lo + 1;
}

__device__ __forceinline__ void paged_write_border(const PagedParams& p, const PagedTile* tile, const int32_t* start,
                                                   int worker, int border, int u_begin, int range)
{
    PagedBorder b;
    b.last_worker = -1;
    if (border >= 0) {
        b.tile = tile[border];
        b.last_worker = (start[border] + paged_units(p, b.tile) - 1) / range;
        b.slot = start[border] > u_begin ? 1 : 0;
    }
    p.border[worker] = b;
}

// Kernels of one call follow each other without the gap between dependent launches: a kernel is
// resident before its predecessor has ended, and waits here for the predecessor's writes.
__device__ __forceinline__ void paged_wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void paged_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... KArgs, class... Args>
static cudaError_t paged_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                                Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

__device__ __forceinline__ float paged_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// `used`: workers that can get work
int attn_paged_tc(const PagedParams& p, int D, int dtype, int used, bool plan_here, cudaStream_t s);

// Tiles up to which the chunk kernel makes the work list itself (see dpk_attn_paged_tc.cu).
constexpr int kPtTiles = 256;

}  // namespace dpk
