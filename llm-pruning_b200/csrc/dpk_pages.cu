// Bookkeeping of a paged KV cache: extend, fork, trim, copy and compact (sm_100a).
//
// State (device memory of the caller, never read by the host):
//   table [S, W] int32   page ids of each sequence, -1 behind its last page
//   lens  [S]    int32   tokens of each sequence; it holds ceil(len / page_size) pages
//   refs  [P]    int32   how many sequences hold a page; 0 = free
// and the pools k, v: [L, P, page_size * Hk * D] 16-bit elements, pages contiguous, layer and page
// strides free.
//
// Everything the integers decide is deterministic: free pages are taken in ascending order by the
// sequences in row order, and holes are filled in ascending order.  That takes prefix sums over the
// P counts, so these operators run as ONE cluster of eight CTAs: every CTA scans an eighth of the
// counts, the partial sums meet in distributed shared memory, and no second launch or host round
// trip is needed between "how many are free" and "who gets which".  They are latency bound (4 bytes
// per page are read): extending 256 sequences in a pool of 131072 pages takes 14 us.  One CTA instead
// of eight is as fast up to 262144 pages there (its launch is cheaper, its scan longer) but twice as
// slow on compacting 65536 and four times on 262144.  The bytes of pages are moved by a second launch over a list the first one
// wrote, bound by HBM (each byte read once and written once).
#define DPK_KERNEL_ID 16   // thousands digit of the device status word
#include <cooperative_groups.h>

#include "dpk_host.h"
#include "dpk_sm100.cuh"

namespace cg = cooperative_groups;

namespace dpk {

constexpr int kPgCluster = 8;         // CTAs of the bookkeeping cluster (portable size)
constexpr int kPgThreads = 1024;

// one page (or its first rows) to be moved in every layer of both pools
struct PageMove {
    int32_t src, dst, rows;
};

struct PageState {
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    int64_t table_stride;
    int S, W, P, page;
    int32_t* count;          // workspace: number of entries of `moves`
    PageMove* moves;         // workspace
    int* status;
};

__device__ __forceinline__ void page_report(int* status)
{
    atomicCAS(status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
}

__device__ __forceinline__ int pages_of(int len, int page) { return (len + page - 1) / page; }

// Sum over the block's threads; `sh` holds 33 ints.  Every thread gets the total and the sum of the
// threads before it.
__device__ __forceinline__ int block_scan(int v, int* sh, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                       // the previous use of sh is over
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = lane < warps ? sh[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sh[lane] = w;
    }
    __syncthreads();
    total = sh[warps - 1];
    return x - v + (warp ? sh[warp - 1] : 0);
}

// ---- extend ------------------------------------------------------------------------------------

struct ExtendWork {        // workspace, one entry per sequence
    int32_t* tail;         // id of a shared last page that this sequence will write to, else -1
    int32_t* keeper;       // with shared tails: 0 nothing shared; 1 copies its tail; 2 + j: keeps it, j = last sharer
    int32_t* upto;         // pages needed by the sequences up to and including this one, for more than kPgRows
};

constexpr int kPgRows = 4096;       // sequences whose running sums fit shared memory

// pages that sequence s will hold with `add` more tokens; more than any table has where that is refused
__device__ __forceinline__ int64_t pages_wanted(int len, int add, int page)
{
    return add < 0 || len < 0 ? INT64_MAX : (static_cast<int64_t>(len) + add + page - 1) / page;
}

// Every CTA sums up the needs of all sequences for itself (a scan over S, against a round trip through
// the cluster and one more barrier), so that two cluster barriers are enough: one behind the count
// of the free pages, one before the lengths change.  Shared tails cost a third.
__global__ void __cluster_dims__(kPgCluster, 1, 1) __launch_bounds__(kPgThreads)
page_extend_kernel(const PageState st, const ExtendWork wk, const int32_t* __restrict__ add,
                   uint8_t* __restrict__ granted)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), tid = threadIdx.x;
    const int gt = rank * kPgThreads + tid;
    constexpr int kAll = kPgCluster * kPgThreads;
    __shared__ int sh[33];
    __shared__ int sh_upto[kPgRows];
    __shared__ int sh_free;            // free pages of this CTA's slice of the counts
    __shared__ int sh_shared;          // is any tail of this CTA's rows shared
    int32_t* upto = st.S <= kPgRows ? sh_upto : wk.upto;    // beyond: every CTA writes the same values

    // 1. who writes to a shared, partly filled last page
    if (rank == 0 && tid == 0) *st.count = 0;
    int any = 0;
    for (int s = gt; s < st.S; s += kAll) {
        const int len = st.lens[s], a = add[s];
        int tail = -1;
        if (a > 0 && len > 0 && len % st.page != 0 && pages_wanted(len, a, st.page) <= st.W) {
            const int id = st.table[s * st.table_stride + pages_of(len, st.page) - 1];
            if (id < 0 || id >= st.P) page_report(st.status);
            else if (st.refs[id] > 1) tail = id;
        }
        wk.tail[s] = tail;
        any |= tail >= 0;
    }
    // free pages of this slice; a slice is a contiguous range of the counts
    const int per = ((st.P + kPgCluster - 1) / kPgCluster + 3) & ~3;
    const int p0 = min(st.P, rank * per), p1 = min(st.P, p0 + per);
    const bool wide = (reinterpret_cast<uintptr_t>(st.refs) & 15u) == 0;
    int mine = 0;
    if (wide) {
#pragma unroll 4
        for (int p = p0 + tid * 4; p < p1; p += kPgThreads * 4) {
            if (p + 4 <= p1) {
                const int4 r = *reinterpret_cast<const int4*>(st.refs + p);
                mine += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
            } else {
                for (int q = p; q < p1; ++q) mine += st.refs[q] == 0;
            }
        }
    } else {
#pragma unroll 8
        for (int p = p0 + tid; p < p1; p += kPgThreads) mine += st.refs[p] == 0;
    }
    any = __syncthreads_or(any);
    int total;
    block_scan(mine, sh, total);
    if (tid == 0) {
        sh_free = total;
        sh_shared = any;
    }
    cluster.sync();
    int shared_tails = 0, before = 0, free_pages = 0;
    for (int r = 0; r < kPgCluster; ++r) {
        shared_tails |= *cluster.map_shared_rank(&sh_shared, r);
        const int f = *cluster.map_shared_rank(&sh_free, r);
        free_pages += f;
        if (r < rank) before += f;
    }

    // 2. of the sharers of such a page everybody takes a copy, but where all its holders write to
    //    it the first one keeps it.  A warp per sharer compares it with every row.
    if (shared_tails) {
        const int lane = tid & 31;
        for (int s = gt >> 5; s < st.S; s += kAll / 32) {
            const int tail = wk.tail[s];
            int keep = 0;
            if (tail >= 0) {
                int holders = 0, first = st.S, last = -1;
#pragma unroll 4
                for (int j = lane; j < st.S; j += 32)
                    if (wk.tail[j] == tail) {
                        ++holders;
                        first = min(first, j);
                        last = max(last, j);
                    }
                holders = __reduce_add_sync(0xffffffffu, holders);
                first = __reduce_min_sync(0xffffffffu, first);
                last = __reduce_max_sync(0xffffffffu, last);
                keep = (first == s && holders == st.refs[tail]) ? 2 + last : 1;
            }
            if (lane == 0) wk.keeper[s] = keep;
        }
        cluster.sync();
    }

    // 3. running sum of the needs
    int wanted = 0;
    for (int s0 = 0; s0 < st.S; s0 += kPgThreads) {
        const int s = s0 + tid;
        int need = 0;
        if (s < st.S) {
            const int len = st.lens[s];
            const int64_t want = pages_wanted(len, add[s], st.page);
            if (want <= st.W) need = static_cast<int>(want) - pages_of(len, st.page);
            if (shared_tails) need += wk.keeper[s] == 1;
        }
        const int x = block_scan(need, sh, total);
        if (s < st.S) upto[s] = wanted + x + need;
        wanted += total;
    }
    __syncthreads();

    // 4. who is granted: in row order while the free pages last
    auto is_granted = [&](int s, int keep) {
        if (pages_wanted(st.lens[s], add[s], st.page) > st.W) return false;
        const int need = upto[s] - (s > 0 ? upto[s - 1] : 0);
        return (need == 0 || upto[s] <= free_pages) && (keep < 2 || upto[keep - 2] <= free_pages);
    };
    for (int s = gt; s < st.S; s += kAll) {
        const int keep = shared_tails ? wk.keeper[s] : 0;
        const bool ok = is_granted(s, keep);
        granted[s] = ok ? 1 : 0;
        if (ok && keep == 1) atomicSub(&st.refs[wk.tail[s]], 1);     // its holders stay above zero: see step 2
    }

    // 5. the k-th free page goes to the row whose needs cover k
    int base = before;
    for (int c0 = p0; c0 < p1 && base < wanted; c0 += kPgThreads) {
        const int p = c0 + tid;
        const int is_free = p < p1 && st.refs[p] == 0;
        const int k = base + block_scan(is_free, sh, total);
        base += total;
        if (!is_free || k >= wanted) continue;
        int lo = 0, hi = st.S - 1;                   // smallest row with upto > k
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] > k) hi = mid;
            else lo = mid + 1;
        }
        const int keep = shared_tails ? wk.keeper[lo] : 0;
        if (!is_granted(lo, keep)) continue;
        const int len = st.lens[lo], held = pages_of(len, st.page);
        const int idx = k - (lo > 0 ? upto[lo - 1] : 0);
        st.refs[p] = 1;
        if (keep == 1 && idx == 0) {
            PageMove m;
            m.src = wk.tail[lo];
            m.dst = p;
            m.rows = len % st.page;
            st.moves[atomicAdd(st.count, 1)] = m;
        }
        st.table[lo * st.table_stride + held + idx - (keep == 1 ? 1 : 0)] = p;
    }
    cluster.sync();
    for (int s = gt; s < st.S; s += kAll)
        if (granted[s]) st.lens[s] += add[s];
}

// ---- fork --------------------------------------------------------------------------------------

__global__ void __cluster_dims__(kPgCluster, 1, 1) __launch_bounds__(kPgThreads)
page_fork_kernel(const PageState st, const int32_t* __restrict__ parents,
                 const int32_t* __restrict__ children, int n, int32_t* __restrict__ length,
                 uint8_t* __restrict__ done)
{
    cg::cluster_group cluster = cg::this_cluster();
    const int gt = static_cast<int>(cluster.block_rank()) * kPgThreads + threadIdx.x;
    constexpr int kAll = kPgCluster * kPgThreads;
    const int lane = threadIdx.x & 31, gw = gt >> 5;
    // 1. what every pair reads, before anything is written.  A warp per pair: the child has to be an
    //    empty row that no earlier pair names.
    for (int i = gw; i < n; i += kAll / 32) {
        const int p = parents[i], c = children[i];
        bool ok = p >= 0 && p < st.S && c >= 0 && c < st.S;
        bool twice = false;
        for (int j = lane; j < i; j += 32) twice |= children[j] == c;
        if (__any_sync(0xffffffffu, twice)) ok = false;
        int len = 0;
        if (ok) {
            len = st.lens[p];
            ok = st.lens[c] == 0 && len >= 0 && pages_of(len, st.page) <= st.W;
        }
        if (lane == 0) {
            if (!ok) page_report(st.status);
            length[i] = ok ? len : -1;
            done[i] = ok ? 1 : 0;
        }
    }
    cluster.sync();
    // 2. rows and counts.  A parent that is also somebody's (empty) child was read as empty above,
    //    so no row is read here while it is written.
    for (int i = gw; i < n; i += kAll / 32) {
        const int len = length[i];
        if (len < 0) continue;
        const int32_t* from = st.table + parents[i] * st.table_stride;
        int32_t* to = st.table + children[i] * st.table_stride;
        const int held = pages_of(len, st.page);
        for (int w = lane; w < held; w += 32) {
            const int id = from[w];
            to[w] = id;
            if (id < 0 || id >= st.P) page_report(st.status);
            else atomicAdd(&st.refs[id], 1);
        }
        if (lane == 0) st.lens[children[i]] = len;
    }
}

// ---- trim --------------------------------------------------------------------------------------

// A warp per named row; of a row that is named twice the first counts.
__global__ void __launch_bounds__(128)
page_trim_kernel(const PageState st, const int32_t* __restrict__ rows, const int32_t* __restrict__ keep, int n)
{
    const int lane = threadIdx.x & 31;
    for (int i = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < n; i += (gridDim.x * blockDim.x) >> 5) {
        const int s = rows[i], to = keep ? keep[i] : 0;
        bool twice = false;
        for (int j = lane; j < i; j += 32) twice |= rows[j] == s;
        if (__any_sync(0xffffffffu, twice)) continue;
        if (s < 0 || s >= st.S || to < 0) {
            if (lane == 0) page_report(st.status);
            continue;
        }
        const int len = st.lens[s];
        if (len <= to) continue;
        __syncwarp();
        const int held = min(pages_of(len, st.page), st.W);
        int32_t* row = st.table + s * st.table_stride;
        for (int w = pages_of(to, st.page) + lane; w < held; w += 32) {
            const int id = row[w];
            row[w] = -1;
            if (id < 0 || id >= st.P) page_report(st.status);
            else atomicSub(&st.refs[id], 1);
        }
        if (lane == 0) st.lens[s] = to;
    }
}

// ---- copy --------------------------------------------------------------------------------------

// Turns two lists of page ids into moves.  Of several pairs with one destination the last counts; a
// page that is read may not be written by another pair of the call (such a pair is left out and
// reported), so the moves are independent of one another.  `mark` [P] is scratch; only the entries
// that the lists name are touched.
__global__ void __cluster_dims__(kPgCluster, 1, 1) __launch_bounds__(kPgThreads)
page_copy_list_kernel(const PageState st, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
                      int n, int32_t* __restrict__ mark)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    const int gt = static_cast<int>(cluster.block_rank()) * kPgThreads + threadIdx.x;
    constexpr int kAll = kPgCluster * kPgThreads;
    auto inside = [&](int id) { return id >= 0 && id < st.P; };
    if (gt == 0) *st.count = 0;
    for (int i = gt; i < n; i += kAll) {
        const int a = src[i], b = dst[i];
        if (inside(a)) mark[a] = 0;
        if (inside(b)) mark[b] = 0;
    }
    cluster.sync();
    for (int i = gt; i < n; i += kAll) {
        const int a = src[i], b = dst[i];
        if (inside(a) && inside(b) && a != b) atomicMax(&mark[b], i + 1);
    }
    cluster.sync();
    for (int i = gt; i < n; i += kAll) {
        const int a = src[i], b = dst[i];
        if (!inside(a) || !inside(b) || (a != b && mark[a] != 0)) {
            page_report(st.status);
            continue;
        }
        if (a == b || mark[b] != i + 1) continue;
        PageMove m;
        m.src = a;
        m.dst = b;
        m.rows = st.page;
        st.moves[atomicAdd(st.count, 1)] = m;
    }
}

// ---- compact -----------------------------------------------------------------------------------

__global__ void __cluster_dims__(kPgCluster, 1, 1) __launch_bounds__(kPgThreads)
page_compact_kernel(const PageState st, int32_t* __restrict__ remap, int32_t* __restrict__ holes,
                    int32_t* __restrict__ live_out)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), tid = threadIdx.x;
    __shared__ int sh[33];
    __shared__ int sh_live, sh_holes, sh_movers;
    const int per = ((st.P + kPgCluster - 1) / kPgCluster + 3) & ~3;
    const int p0 = min(st.P, rank * per), p1 = min(st.P, p0 + per);
    int mine = 0, t;
    for (int p = p0 + tid; p < p1; p += kPgThreads) mine += st.refs[p] > 0;
    block_scan(mine, sh, t);
    if (tid == 0) sh_live = t;
    cluster.sync();
    int live = 0;
    for (int r = 0; r < kPgCluster; ++r) live += *cluster.map_shared_rank(&sh_live, r);
    int h = 0, m = 0;
    for (int p = p0 + tid; p < p1; p += kPgThreads) {
        const bool used = st.refs[p] > 0;
        h += p < live && !used;
        m += p >= live && used;
    }
    block_scan(h, sh, t);
    if (tid == 0) sh_holes = t;
    block_scan(m, sh, t);
    if (tid == 0) sh_movers = t;
    cluster.sync();
    int hole_base = 0, mover_base = 0, moves = 0;
    for (int r = 0; r < kPgCluster; ++r) {
        const int hr = *cluster.map_shared_rank(&sh_holes, r), mr = *cluster.map_shared_rank(&sh_movers, r);
        moves += mr;
        if (r < rank) { hole_base += hr; mover_base += mr; }
    }
    // the k-th free page below `live` takes the k-th used page from `live` on
    for (int c0 = p0; c0 < p1; c0 += kPgThreads) {
        const int p = c0 + tid;
        const bool used = p < p1 && st.refs[p] > 0;
        if (p < p1 && !(used && p >= live)) remap[p] = used ? p : -1;      // the moved ones follow below
        const int is_hole = p < p1 && p < live && !used, is_mover = used && p >= live;
        int hk, mk;
        const int a = block_scan(is_hole, sh, hk);
        if (is_hole) holes[hole_base + a] = p;
        const int b = block_scan(is_mover, sh, mk);
        if (is_mover) st.moves[mover_base + b].src = p;
        hole_base += hk;
        mover_base += mk;
    }
    cluster.sync();
    for (int k = rank * kPgThreads + tid; k < moves; k += kPgCluster * kPgThreads) {
        const int from = st.moves[k].src, to = holes[k];
        st.moves[k].dst = to;
        st.moves[k].rows = st.page;
        remap[from] = to;
        st.refs[to] = st.refs[from];
        st.refs[from] = 0;
    }
    if (rank == 0 && tid == 0) {
        *st.count = moves;
        *live_out = live;
    }
}

// An entry whose page nobody holds (counts and table disagree) would name another sequence's page from here
// on, or one that is handed out next: it is reported and becomes -1, which no operator follows.
__global__ void __launch_bounds__(256)
page_remap_kernel(const PageState st, const int32_t* remap)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
         i < static_cast<int64_t>(st.S) * st.W; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int s = static_cast<int>(i / st.W), w = static_cast<int>(i - static_cast<int64_t>(s) * st.W);
        if (w >= pages_of(st.lens[s], st.page)) continue;
        int32_t* e = st.table + s * st.table_stride + w;
        const int id = *e;
        const int to = id < 0 || id >= st.P ? -1 : remap[id];
        if (to < 0) page_report(st.status);
        if (to != id && id >= 0 && id < st.P) *e = to;
    }
}

// ---- moving the bytes --------------------------------------------------------------------------

struct PoolParams {
    uint8_t* k;
    uint8_t* v;
    int64_t layer_stride, page_stride;     // bytes
    int layers, row_bytes;                 // one token of one page
};

// A task is 16 KiB of one page of one layer of one pool: 256 threads, four 16-byte loads each in
// flight before the stores.  The list's length is known on the device only, so a fixed grid walks it.
constexpr int kMoveBytes = 16384;

// The list is written while this kernel is already resident, so its pointers are not __restrict__: loads that
// the compiler may take for those of a constant could be moved ahead of the wait.
__global__ void __launch_bounds__(256)
page_move_kernel(const PageMove* moves, const int32_t* count, const PoolParams pp, int page)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");       // started while the bookkeeping still runs
    const int pieces = (page * pp.row_bytes + kMoveBytes - 1) / kMoveBytes;
    const int64_t tasks = static_cast<int64_t>(*count) * pp.layers * 2 * pieces;
    for (int64_t i = blockIdx.x; i < tasks; i += gridDim.x) {
        int64_t rest = i;
        const int piece = static_cast<int>(rest % pieces);
        rest /= pieces;
        const int pool = static_cast<int>(rest & 1);
        rest >>= 1;
        const int layer = static_cast<int>(rest % pp.layers);
        const PageMove m = moves[rest / pp.layers];
        uint8_t* base = (pool ? pp.v : pp.k) + layer * pp.layer_stride + static_cast<int64_t>(piece) * kMoveBytes;
        const int bytes = min(kMoveBytes, m.rows * pp.row_bytes - piece * kMoveBytes);
        const uint8_t* src = base + m.src * pp.page_stride;
        uint8_t* dst = base + m.dst * pp.page_stride;
        uint4 buf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = (j * 256 + threadIdx.x) * 16;
            if (at < bytes) buf[j] = __ldcs(reinterpret_cast<const uint4*>(src + at));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = (j * 256 + threadIdx.x) * 16;
            if (at < bytes) __stcs(reinterpret_cast<uint4*>(dst + at), buf[j]);
        }
    }
}

// A launch that may start while the one before it on the stream still runs; its kernel waits for that one.
template <class... KArgs, class... Args>
static int launch_early(int64_t blocks, void (*kernel)(KArgs...), cudaStream_t s, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    DPK_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
    return DPK_OK;
}

// `most`: moves that the list can hold at most.  Many more blocks than fit the GPU copy faster than as
// many as fit (96 MB of pages by 4 layers and 2 pools, 786 MB read and written: 124 us with 40 blocks per
// SM, 131 with 8, 126 to 141 with bulk copies through shared memory), but each costs its start where the
// list is nearly empty, as it is for extend.
static int move_pages(const PageState& st, const PoolParams& pp, int64_t most, int per_sm, cudaStream_t s)
{
    const int pieces = (st.page * pp.row_bytes + kMoveBytes - 1) / kMoveBytes;
    int64_t blocks = most * pp.layers * 2 * pieces;
    const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
    if (blocks > cap) blocks = cap;
    if (blocks < 1) blocks = 1;
    return launch_early(blocks, page_move_kernel, s, st.moves, st.count, pp, st.page);
}

static int pool_params(PoolParams& pp, void* k, void* v, int layers, int64_t layer_stride, int64_t page_stride,
                       int P, int page, int row_elems)
{
    DPK_REQUIRE((k && v) || P == 0, "NULL tensor");          // a pool of nothing has no address
    DPK_REQUIRE(layers > 0 && row_elems > 0 && row_elems % 8 == 0, "a token's row must be a multiple of 8 elements");
    DPK_REQUIRE(page_stride % 8 == 0 && layer_stride % 8 == 0 && aligned16(k) && aligned16(v),
                "pools must be 16-byte aligned with strides of multiples of 8 elements");
    DPK_REQUIRE(page_stride >= static_cast<int64_t>(page) * row_elems, "page_stride is smaller than a page");
    DPK_REQUIRE(static_cast<int64_t>(page) * row_elems <= (1 << 28), "page too large");
    pp.k = static_cast<uint8_t*>(k);
    pp.v = static_cast<uint8_t*>(v);
    pp.layer_stride = layer_stride * 2;
    pp.page_stride = page_stride * 2;
    pp.layers = layers;
    pp.row_bytes = row_elems * 2;
    return DPK_OK;
}

static int page_state(PageState& st, int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int S,
                      int W, int P, int page)
{
    DPK_REQUIRE(S >= 0 && W >= 0 && P >= 0 && page > 0, "bad shape");
    DPK_REQUIRE((table || S == 0 || W == 0) && (lens || S == 0) && (refs || P == 0), "NULL tensor");
    DPK_REQUIRE(table_stride >= W, "table_stride is smaller than a row");
    DPK_REQUIRE(static_cast<int64_t>(W) * page < (1ll << 31), "a row of the table holds 2^31 tokens or more");
    DPK_REQUIRE(P <= (1 << 30) && S <= (1 << 24) && static_cast<int64_t>(S) * (W + 1) < (1ll << 31),
                "too many pages or sequences");
    st.table = table;
    st.table_stride = table_stride;
    st.lens = lens;
    st.refs = refs;
    st.S = S;
    st.W = W;
    st.P = P;
    st.page = page;
    st.count = nullptr;
    st.moves = nullptr;
    st.status = nullptr;
    return DPK_OK;
}

static int page_status(PageState& st)        // after every check of the arguments
{
    st.status = device_status_ptr();
    return st.status ? DPK_OK : fail(DPK_ERR_CUDA, "no status word on this device");
}

// workspace: [count, 3 pad][moves 3 * most][arrays]
static int32_t* take_moves(PageState& st, void* ws, int64_t most)
{
    int32_t* w = static_cast<int32_t*>(ws);
    st.count = w;
    st.moves = reinterpret_cast<PageMove*>(w + 4);
    return w + 4 + 3 * most;
}

}  // namespace dpk

using namespace dpk;

extern "C" {

size_t dpk_page_workspace_bytes(int S, int P, int n)
{
    if (S < 0 || P < 0 || n < 0) return 0;
    // extend: 7 S; fork: n; copy: 3 n + P; compact: 5 P (32-bit words)
    return (size_t(4) + 7 * size_t(S) + 4 * size_t(n) + 5 * size_t(P)) * sizeof(int32_t);
}

int dpk_page_extend(int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int S, int W, int P,
                    int page, const int32_t* add, uint8_t* granted, void* k, void* v, int layers,
                    int64_t layer_stride, int64_t page_stride, int row_elems, void* workspace,
                    size_t workspace_bytes, void* stream)
{
    PageState st;
    PoolParams pp;
    int rc = page_state(st, table, table_stride, lens, refs, S, W, P, page);
    if (rc) return rc;
    rc = pool_params(pp, k, v, layers, layer_stride, page_stride, P, page, row_elems);
    if (rc) return rc;
    if (S == 0) return DPK_OK;
    DPK_REQUIRE(add && granted, "NULL tensor");
    const size_t need = dpk_page_workspace_bytes(S, 0, 0);
    DPK_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    rc = page_status(st);
    if (rc) return rc;
    int32_t* w = take_moves(st, workspace, S);
    ExtendWork wk = {w, w + S, w + 2 * S};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    page_extend_kernel<<<kPgCluster, kPgThreads, 0, s>>>(st, wk, add, granted);
    DPK_CUDA(cudaGetLastError());
    return move_pages(st, pp, S, 8, s);
}

int dpk_page_fork(int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int S, int W, int P,
                  int page, const int32_t* parents, const int32_t* children, int n, uint8_t* done,
                  void* workspace, size_t workspace_bytes, void* stream)
{
    PageState st;
    int rc = page_state(st, table, table_stride, lens, refs, S, W, P, page);
    if (rc) return rc;
    DPK_REQUIRE(n >= 0, "bad shape");
    if (n == 0) return DPK_OK;
    DPK_REQUIRE(parents && children && done, "NULL tensor");
    const size_t need = dpk_page_workspace_bytes(0, 0, n);
    DPK_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    rc = page_status(st);
    if (rc) return rc;
    page_fork_kernel<<<kPgCluster, kPgThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        st, parents, children, n, static_cast<int32_t*>(workspace), done);
    DPK_CUDA(cudaGetLastError());
    return DPK_OK;
}

int dpk_page_trim(int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int S, int W, int P,
                  int page, const int32_t* rows, const int32_t* keep, int n, void* stream)
{
    PageState st;
    int rc = page_state(st, table, table_stride, lens, refs, S, W, P, page);
    if (rc) return rc;
    DPK_REQUIRE(n >= 0, "bad shape");
    if (n == 0) return DPK_OK;
    DPK_REQUIRE(rows, "NULL tensor");
    rc = page_status(st);
    if (rc) return rc;
    int blocks = (n + 3) / 4;
    if (blocks > sm_count() * 8) blocks = sm_count() * 8;
    page_trim_kernel<<<blocks, 128, 0, static_cast<cudaStream_t>(stream)>>>(st, rows, keep, n);
    DPK_CUDA(cudaGetLastError());
    return DPK_OK;
}

int dpk_page_copy(void* k, void* v, int layers, int64_t layer_stride, int64_t page_stride, int row_elems, int P,
                  int page, const int32_t* src, const int32_t* dst, int n, void* workspace,
                  size_t workspace_bytes, void* stream)
{
    PageState st;
    PoolParams pp;
    int32_t none = 0;            // no table here: the copy deals with page ids alone
    DPK_REQUIRE(P >= 0 && page > 0, "bad shape");
    int rc = page_state(st, &none, 0, &none, &none, 0, 0, P, page);
    if (rc) return rc;
    rc = pool_params(pp, k, v, layers, layer_stride, page_stride, P, page, row_elems);
    if (rc) return rc;
    DPK_REQUIRE(n >= 0, "bad shape");
    if (n == 0) return DPK_OK;
    DPK_REQUIRE(src && dst, "NULL tensor");
    const size_t need = dpk_page_workspace_bytes(0, P, n);
    DPK_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    rc = page_status(st);
    if (rc) return rc;
    st.table = st.lens = st.refs = nullptr;
    int32_t* mark = take_moves(st, workspace, n);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    page_copy_list_kernel<<<kPgCluster, kPgThreads, 0, s>>>(st, src, dst, n, mark);
    DPK_CUDA(cudaGetLastError());
    return move_pages(st, pp, n, 40, s);
}

int dpk_page_compact(void* k, void* v, int layers, int64_t layer_stride, int64_t page_stride, int row_elems,
                     int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int S, int W, int P,
                     int page, int32_t* live, void* workspace, size_t workspace_bytes, void* stream)
{
    PageState st;
    PoolParams pp;
    int rc = page_state(st, table, table_stride, lens, refs, S, W, P, page);
    if (rc) return rc;
    rc = pool_params(pp, k, v, layers, layer_stride, page_stride, P, page, row_elems);
    if (rc) return rc;
    DPK_REQUIRE(live, "NULL tensor");
    const size_t need = dpk_page_workspace_bytes(0, P, 0);
    DPK_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    rc = page_status(st);
    if (rc) return rc;
    int32_t* remap = take_moves(st, workspace, P);
    int32_t* holes = remap + P;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    page_compact_kernel<<<kPgCluster, kPgThreads, 0, s>>>(st, remap, holes, live);
    DPK_CUDA(cudaGetLastError());
    if (S > 0 && W > 0) {
        int64_t blocks = (static_cast<int64_t>(S) * W + 255) / 256;
        if (blocks > sm_count() * 8) blocks = sm_count() * 8;
        rc = launch_early(blocks, page_remap_kernel, s, st, remap);
        if (rc) return rc;
    }
    return move_pages(st, pp, P / 2 + 1, 40, s);
}

}  // extern "C"
