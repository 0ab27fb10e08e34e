// Attention of new tokens over a paged KV cache: C-ABI entry, work list, joining kernel and the
// warp-per-range kernel for few rows (sm_100a).  The kernel for chunks is in dpk_attn_paged_tc.cu.
//
// For new token i of sequence s (n_s of them, the last of its kv_len[s] tokens) and query head h:
//     o = sum_j softmax_j(scale q.k_j) v_j   over the keys j <= kv_len[s] - n_s + i   (causal)
//                                            or j < kv_len[s]                         (not causal)
// K and V are read through the page table; rows whose head group is routed out, and rows that see
// no key, are zero.
//
// Two to four launches: paged_rows_kernel lists the active rows (chunks with a mask), paged_plan_kernel
// cuts the work (dpk_attn_paged.cuh; lists of up to kPwTiles or kPtTiles tiles are made inside the
// attention kernel instead), an attention kernel runs it, paged_join_kernel joins the tiles that several
// workers shared and writes the zero rows.  Each is started while its predecessor still runs.
//
// Scores that are NaN or +inf, and rows that see -inf alone, give NaN, however the work was cut.
//
// The attention kernel here gives every WARP a range of 32-key units.  Its tile is 16 rows, so the
// Hq/Hk heads of up to 16 / (Hq/Hk) new tokens read every K/V byte once; K and V arrive through a
// private three-stage ring of cp.async (16-byte copies: a page may end anywhere inside a unit, and
// rows behind the last key are zero-filled, so whatever an unused row of a page holds is never
// multiplied).  It is bounded by HBM: 4 * D bytes per key against 16 MMA rows.
#define DPK_KERNEL_ID 13   // thousands digit of the device status word
#include "dpk_attn_paged_plan.cuh"

#include <math.h>

namespace dpk {

// ---- the work list -------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kPlanItems = 4096;        // (sequence, KV head) pairs whose tile numbers fit shared memory

// Active rows of every (sequence, KV head), in token order, and its tiles; used where tiles have many rows, so that
// none of them is spent on a routed-out (token, head).  A thread looks at 16 rows in a row.
__global__ void __launch_bounds__(1024) paged_rows_kernel(const PagedParams p)
{
    __shared__ int2 sh[32];
    paged_let_next_start();
    const int s = blockIdx.x, kvh = blockIdx.y;
    int tok0;
    const int total_rows = plan_new(p, s, tok0) * p.rep;
    int32_t* out = p.rows + (static_cast<int64_t>(kvh) * p.N + tok0) * p.rep;
    const int g0 = kvh * p.rep / p.hpg, h0 = kvh * p.rep - g0 * p.hpg;
    int carry = 0;
    for (int x0 = 0; x0 < total_rows; x0 += blockDim.x * 16) {
        const int x = x0 + threadIdx.x * 16;
        uint32_t on = 0;
        if (x < total_rows) {
            const int i = x / p.rep;
            int r = x - i * p.rep;
            int g = (kvh * p.rep + r) / p.hpg, h = kvh * p.rep + r - g * p.hpg;   // group and place in it
            const uint8_t* m = p.mask + static_cast<int64_t>(tok0 + i) * p.NG;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (x + k < total_rows && m[g] != 0) on |= 1u << k;
                if (++h == p.hpg) {
                    h = 0;
                    ++g;
                }
                if (++r == p.rep) {
                    r = 0;
                    g = g0;
                    h = h0;
                    m += p.NG;
                }
            }
        }
        int2 t;
        int at = carry + plan_scan(make_int2(__popc(on), 0), sh, t).x;
        for (; on; on &= on - 1) out[at++] = x + __ffs(on) - 1;
        carry += t.x;
    }
    if (threadIdx.x == 0) p.row_count[s * p.Hk + kvh] = carry;
    __syncthreads();
    PagedTile* slot = p.slot + plan_slot(p, s, kvh);
    for (int t = threadIdx.x; t * p.tile_rows < carry; t += blockDim.x) {
        PagedTile pt;
        if (plan_tile(p, s, kvh, t, carry, pt) == 0) pt.kv_end = 0;
        slot[t] = pt;
    }
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedParams p)
{
    __shared__ int2 sh[32];
    __shared__ int sh_first[kPlanItems];
    paged_let_next_start();
    if (p.rows) paged_wait_previous();
    int tiles, length;
    plan_work(p, p.tile, p.start, static_cast<int64_t>(p.S) * p.Hk <= kPlanItems ? sh_first : p.first_tile, sh, tiles,
              length);
    if (threadIdx.x == 0) {
        p.head->tiles = tiles;
        p.head->length = length;
        p.head->range = plan_range(p, tiles, length);
    }
}

// ---- attention, a range per warp ---------------------------------------------------------------

constexpr int kPwBN = 32;            // keys per unit
constexpr int kPwStages = 3;
constexpr int kPwWarps = 4;
constexpr int kPwRows = 16;

__device__ __forceinline__ void pw_ldsm_x4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void pw_ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
template <bool kBf16>
__device__ __forceinline__ void pw_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (kBf16) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
template <int D>
__device__ __forceinline__ uint32_t pw_off(int r, int c)
{
    return static_cast<uint32_t>(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

// Up to kPwTiles tiles by the host's bound, Hk * (N * rep / 16 + S) (a decode step of 15 sequences with 32
// query and 8 KV heads, of 16 with 16 and 8), the attention kernel makes the work list itself, every CTA for
// its own use in shared memory behind the rings: that saves a launch of a kernel that takes as long as a
// small step's attention (8 tiles: 11.4 us on the device instead of 12.5, 22.7 a call instead of 26.2).  A
// CTA of 128 threads takes longer over a long list than the launch does (128 tiles: the same on the
// device; 512: 262 us instead of 258).
constexpr int kPwTiles = 144;

template <int D, bool kBf16, bool kPlanHere>
__global__ void __launch_bounds__(kPwWarps * 32) paged_warp_kernel(const PagedParams p)
{
    constexpr int CH = D / 8, KS = D / 16, NT_S = kPwBN / 8, NT_O = D / 8;
    constexpr int TILE_B = kPwBN * D * 2;
    constexpr int WARP_B = kPwStages * 2 * TILE_B;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, t4 = lane & 3;
    const uint32_t pipe = smem_u32(smem + warp * WARP_B);

    int tiles, length, range;
    PagedTile* tile_of = p.tile;
    int32_t* start = p.start;
    paged_let_next_start();
    if constexpr (kPlanHere) {
        __shared__ int2 sh[32];
        tile_of = reinterpret_cast<PagedTile*>(smem + kPwWarps * WARP_B);
        start = reinterpret_cast<int32_t*>(tile_of + kPwTiles);
        plan_work(p, tile_of, start, start + kPwTiles + 1, sh, tiles, length);
        range = plan_range(p, tiles, length);
    } else {
        paged_wait_previous();
        tiles = p.head->tiles;
        length = p.head->length;
        range = p.head->range;
    }
    const int worker = blockIdx.x * kPwWarps + warp;
    if (static_cast<int64_t>(worker) * range >= length) {
        if (lane == 0 && worker < p.workers) p.border[worker].last_worker = -1;
        return;
    }
    const int u_begin = worker * range, u_end = min(length, u_begin + range);
    const int tile0 = paged_find_tile(p, tile_of, start, tiles, u_begin);

    // ---- loader: two units ahead of the arithmetic, across the ends of tiles -----------------
    int ld_tile = tile0 - 1, ld_j = 0, ld_n = 0;   // ld_j: the unit of ld_tile to be loaded next
    PagedTile lt;
    bool ld_more = true;
    // this lane's key of the unit: element offset of its row, -1 behind the last visible key
    auto key_row = [&]() -> int64_t {
        if (ld_j >= ld_n) {
            ++ld_tile;
            const int first = ld_tile < tiles ? start[ld_tile] : length;
            ld_more = first < u_end;
            if (!ld_more) return -1;
            lt = tile_of[ld_tile];
            ld_j = max(0, u_begin - first);
            ld_n = min((lt.kv_end + kPwBN - 1) / kPwBN, u_end - first);
        }
        const int key = ld_j * kPwBN + lane;
        if (key >= lt.kv_end) return -1;
        const int w = key / p.page;
        const int id = p.table[lt.seq * p.table_stride + w];
        if (id < 0 || id >= p.P) {
            atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
            return -1;
        }
        return id * p.page_stride + (key - w * p.page) * p.token_stride + lt.kvh * D;
    };
    int64_t my_row = key_row();
    auto load_unit = [&](int stage) {              // issues the copies of ld_unit, then looks up the next
        if (ld_more) {
            const uint32_t kdst = pipe + stage * 2 * TILE_B;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int x = i * 32 + lane, r = x / CH, c = x % CH;
                const int64_t row = __shfl_sync(0xffffffffu, my_row, r);
                const uint32_t n = row >= 0 ? 16u : 0u;
                const int64_t off = (row >= 0 ? row : 0) * 2 + c * 16;
                cp_async_16(kdst + pw_off<D>(r, c), p.K + off, n);
                cp_async_16(kdst + TILE_B + pw_off<D>(r, c), p.V + off, n);
            }
            ++ld_j;
            my_row = key_row();
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kPwStages - 1; ++s) load_unit(s);

    // ---- arithmetic ------------------------------------------------------------------------
    int stage = 0, border = -1;         // border: the tile that ends behind this warp's range
    for (int tile = tile0; tile < tiles && start[tile] < u_end; ++tile) {
        const PagedTile t = tile_of[tile];
        const int t_first = start[tile], t_units = (t.kv_end + kPwBN - 1) / kPwBN;
        const int j0 = max(0, u_begin - t_first), j1 = min(t_units, u_end - t_first);
        // rows gid and gid + 8 of this lane: token (or -1) and the last key they see
        int head0 = 0, head1 = 0;
        const int i0 = gid < t.rows ? paged_row(p, t, gid, head0) : -1;
        const int i1 = gid + 8 < t.rows ? paged_row(p, t, gid + 8, head1) : -1;
        const int lim0 = paged_last_key(p, t, i0), lim1 = paged_last_key(p, t, i1);
        uint32_t qf[KS][4];
        {
            const uint8_t* q0 = p.Q + ((t.tok0 + max(i0, 0)) * p.q_ts + static_cast<int64_t>(head0) * D) * 2 + t4 * 4;
            const uint8_t* q1 = p.Q + ((t.tok0 + max(i1, 0)) * p.q_ts + static_cast<int64_t>(head1) * D) * 2 + t4 * 4;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[ks][0] = i0 >= 0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 32) : 0u;
                qf[ks][1] = i1 >= 0 ? *reinterpret_cast<const uint32_t*>(q1 + ks * 32) : 0u;
                qf[ks][2] = i0 >= 0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 32 + 16) : 0u;
                qf[ks][3] = i1 >= 0 ? *reinterpret_cast<const uint32_t*>(q1 + ks * 32 + 16) : 0u;
            }
        }
        float o[NT_O][4];
#pragma unroll
        for (int j = 0; j < NT_O; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }
        float mx0 = -INFINITY, mx1 = -INFINITY, l0 = 0.f, l1 = 0.f;

        for (int j = j0; j < j1; ++j) {
            int fill = stage + kPwStages - 1;
            if (fill >= kPwStages) fill -= kPwStages;
            load_unit(fill);
            cp_async_wait<kPwStages - 1>();
            __syncwarp();
            const uint32_t kbase = pipe + stage * 2 * TILE_B, vbase = kbase + TILE_B;
            const int kv0 = j * kPwBN;
            float s[NT_S][4];
#pragma unroll
            for (int j = 0; j < NT_S; ++j) { s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int jp = 0; jp < NT_S / 2; ++jp) {
                    uint32_t kf[4];
                    const int r = jp * 16 + (lane & 7) + (lane >> 4) * 8;
                    pw_ldsm_x4(kbase + pw_off<D>(r, ks * 2 + ((lane >> 3) & 1)), kf);
                    pw_mma<kBf16>(s[2 * jp], qf[ks], kf[0], kf[1]);
                    pw_mma<kBf16>(s[2 * jp + 1], qf[ks], kf[2], kf[3]);
                }
            }
            if (kv0 + kPwBN - 1 > min(lim0, lim1)) {
#pragma unroll
                for (int j = 0; j < NT_S; ++j) {
                    const int k0 = kv0 + j * 8 + 2 * t4;
                    if (k0 > lim0) s[j][0] = -INFINITY;
                    if (k0 + 1 > lim0) s[j][1] = -INFINITY;
                    if (k0 > lim1) s[j][2] = -INFINITY;
                    if (k0 + 1 > lim1) s[j][3] = -INFINITY;
                }
            }
            float tm0 = -INFINITY, tm1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT_S; ++j) {
                tm0 = fmaxf(tm0, fmaxf(s[j][0], s[j][1]));
                tm1 = fmaxf(tm1, fmaxf(s[j][2], s[j][3]));
            }
            tm0 = fmaxf(tm0, __shfl_xor_sync(0xffffffffu, tm0, 1));
            tm0 = fmaxf(tm0, __shfl_xor_sync(0xffffffffu, tm0, 2));
            tm1 = fmaxf(tm1, __shfl_xor_sync(0xffffffffu, tm1, 1));
            tm1 = fmaxf(tm1, __shfl_xor_sync(0xffffffffu, tm1, 2));
            const float nm0 = fmaxf(mx0, tm0), nm1 = fmaxf(mx1, tm1);
            const float ref0 = nm0 == -INFINITY ? 0.f : nm0 * p.scale_log2;
            const float ref1 = nm1 == -INFINITY ? 0.f : nm1 * p.scale_log2;
            const float corr0 = paged_exp2(mx0 * p.scale_log2 - ref0);
            const float corr1 = paged_exp2(mx1 * p.scale_log2 - ref1);
            mx0 = nm0;
            mx1 = nm1;
            float rs0 = 0.f, rs1 = 0.f;
            // P enters the second product in V's 16 bits: one MMA takes both operands in one type, and the
            // remainder would be a second product.  Its sum is taken in 32 bits.  Against 64 bits the output is
            // off by 0.0023 (bf16; 64 sequences of up to 16384 keys) where P in 32 bits leaves 0.0017, the
            // rounding of the output.
            uint32_t pf[NT_S][2];
#pragma unroll
            for (int j = 0; j < NT_S; ++j) {
                const float p0 = paged_exp2(fmaf(s[j][0], p.scale_log2, -ref0));
                const float p1 = paged_exp2(fmaf(s[j][1], p.scale_log2, -ref0));
                const float p2 = paged_exp2(fmaf(s[j][2], p.scale_log2, -ref1));
                const float p3 = paged_exp2(fmaf(s[j][3], p.scale_log2, -ref1));
                rs0 += p0 + p1;
                rs1 += p2 + p3;
                pf[j][0] = pack_half2<kBf16>(p0, p1);
                pf[j][1] = pack_half2<kBf16>(p2, p3);
            }
            l0 = l0 * corr0 + rs0;
            l1 = l1 * corr1 + rs1;
#pragma unroll
            for (int j = 0; j < NT_O; ++j) {
                o[j][0] *= corr0; o[j][1] *= corr0;
                o[j][2] *= corr1; o[j][3] *= corr1;
            }
#pragma unroll
            for (int kk = 0; kk < kPwBN / 16; ++kk) {
                const uint32_t af[4] = {pf[2 * kk][0], pf[2 * kk][1], pf[2 * kk + 1][0], pf[2 * kk + 1][1]};
#pragma unroll
                for (int jp = 0; jp < NT_O / 2; ++jp) {
                    uint32_t vf[4];
                    const int r = kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
                    pw_ldsm_x4_trans(vbase + pw_off<D>(r, jp * 2 + (lane >> 4)), vf);
                    pw_mma<kBf16>(o[2 * jp], af, vf[0], vf[1]);
                    pw_mma<kBf16>(o[2 * jp + 1], af, vf[2], vf[3]);
                }
            }
            __syncwarp();                            // the stage is refilled by the next unit's copies
            if (++stage == kPwStages) stage = 0;
        }

        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if (j1 - j0 == t_units) {                            // the whole tile was this warp's
            const float inv0 = paged_inverse(lim0, l0), inv1 = paged_inverse(lim1, l1);
            uint8_t* d0 = p.O + ((static_cast<int64_t>(t.tok0 + max(i0, 0)) * p.Hq + head0) * D + 2 * t4) * 2;
            uint8_t* d1 = p.O + ((static_cast<int64_t>(t.tok0 + max(i1, 0)) * p.Hq + head1) * D + 2 * t4) * 2;
#pragma unroll
            for (int j = 0; j < NT_O; ++j) {
                if (i0 >= 0)
                    *reinterpret_cast<uint32_t*>(d0 + j * 16) = pack_half2<kBf16>(o[j][0] * inv0, o[j][1] * inv0);
                if (i1 >= 0)
                    *reinterpret_cast<uint32_t*>(d1 + j * 16) = pack_half2<kBf16>(o[j][2] * inv1, o[j][3] * inv1);
            }
        } else {
            if (j0 == 0) border = tile;
            const int64_t slot = (static_cast<int64_t>(worker) * 2 + (t_first > u_begin ? 1 : 0)) * kPwRows;
            float* d0 = p.part_o + (slot + gid) * D + 2 * t4;
            float* d1 = d0 + 8 * D;
#pragma unroll
            for (int j = 0; j < NT_O; ++j) {
                if (gid < t.rows) *reinterpret_cast<float2*>(d0 + j * 8) = make_float2(o[j][0], o[j][1]);
                if (gid + 8 < t.rows) *reinterpret_cast<float2*>(d1 + j * 8) = make_float2(o[j][2], o[j][3]);
            }
            if (t4 == 0) {
                float* ml = p.part_ml + (slot + gid) * 2;
                if (gid < t.rows) *reinterpret_cast<float2*>(ml) = make_float2(mx0, l0);
                if (gid + 8 < t.rows) *reinterpret_cast<float2*>(ml + 16) = make_float2(mx1, l1);
            }
        }
    }
    cp_async_wait<0>();
    if (lane == 0) paged_write_border(p, tile_of, start, worker, border, u_begin, range);
}

// ---- joining -----------------------------------------------------------------------------------

// The last join_blocks = workers * row_groups blocks join the tiles that several workers shared: block
// (w, g) takes a share of the rows of the tile that starts in worker w's range and ends behind it.
// Few parts: a warp joins kRows rows by itself, their loads in flight together; many parts of few
// rows: the block's four warps share the parts of each row.  The blocks before write the
// rows that no unit covers, a token per warp: routed out, without a visible key, and (clear_tail)
// of no sequence.  They need nothing of the attention kernel, so they do not wait for it.
struct JoinRow {
    float m, l;
};

template <int C>
__device__ __forceinline__ void join_add(JoinRow& s, float (&acc)[C], const float2& ml, const float (&x)[C], float scale_log2)
{
    if (ml.y == 0.f) return;               // no weight in this part; a sum that is NaN stays in, whatever its maximum
    const float top = fmaxf(s.m, ml.x);
    const float a = paged_exp2((s.m - top) * scale_log2), b = paged_exp2((ml.x - top) * scale_log2);
    s.l = s.l * a + ml.y * b;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = acc[c] * a + x[c] * b;
    s.m = top;
}

template <int C>
__device__ __forceinline__ void join_load(const PagedParams& p, int64_t slot, int D, int lane, float2& ml, float (&x)[C])
{
    ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
    const float* src = p.part_o + slot * D + lane * C;
#pragma unroll
    for (int c = 0; c < C; c += 2) *reinterpret_cast<float2*>(&x[c]) = *reinterpret_cast<const float2*>(src + c);
}

template <int D, bool kBf16, int kRows>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedParams p, int row_groups, int join_blocks)
{
    constexpr int C = D / 32;                                // columns of a lane
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ float sh_o[4][D];
    __shared__ float2 sh_ml[4];
    const int zero_blocks = gridDim.x - join_blocks;
    if (static_cast<int>(blockIdx.x) >= zero_blocks) {
        paged_wait_previous();
        const int block = blockIdx.x - zero_blocks;
        const int w0 = block / row_groups, group = block - w0 * row_groups;
        const PagedBorder border = p.border[w0];
        const PagedTile& t = border.tile;
        const int w1 = border.last_worker, slot0 = border.slot;
        if (w1 < 0) return;
        auto slot_of = [&](int w, int r) { return (static_cast<int64_t>(w) * 2 + (w == w0 ? slot0 : 0)) * p.tile_rows + r; };
        auto store = [&](int i, int head, const JoinRow& s, const float (&acc)[C]) {
            const float inv = paged_inverse(paged_last_key(p, t, i), s.l);
            uint8_t* out = p.O + ((static_cast<int64_t>(t.tok0 + i) * p.Hq + head) * D + lane * C) * 2;
#pragma unroll
            for (int c = 0; c < C; c += 2)
                *reinterpret_cast<uint32_t*>(out + c * 2) = pack_half2<kBf16>(acc[c] * inv, acc[c + 1] * inv);
        };
        // steps of either way: a warp takes kRows rows and two parts at a time, a block a row and 16 parts
        // and a barrier
        const int parts = w1 - w0 + 1, at_once = row_groups * 4 * kRows;
        const int by_warp = (t.rows + at_once - 1) / at_once * ((parts + 1) / 2);
        const int by_block = (t.rows + row_groups - 1) / row_groups * ((parts + 15) / 16 + 1);
        if (by_warp <= by_block) {
            for (int r = (group * 4 + warp) * kRows; r < t.rows; r += row_groups * 4 * kRows) {
                int i[kRows], head[kRows];
                JoinRow s[kRows];
                float acc[kRows][C];
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    i[k] = r + k < t.rows ? paged_row(p, t, r + k, head[k]) : -1;
                    s[k] = {-INFINITY, 0.f};
#pragma unroll
                    for (int c = 0; c < C; ++c) acc[k][c] = 0.f;
                }
                for (int w = w0; w <= w1; w += 2) {
                    float2 ml[2][kRows];
                    float x[2][kRows][C];
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int k = 0; k < kRows; ++k) {
                            ml[v][k] = make_float2(-INFINITY, 0.f);
                            if (i[k] >= 0 && w + v <= w1) join_load<C>(p, slot_of(w + v, r + k), D, lane, ml[v][k], x[v][k]);
                        }
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int k = 0; k < kRows; ++k) join_add<C>(s[k], acc[k], ml[v][k], x[v][k], p.scale_log2);
                }
#pragma unroll
                for (int k = 0; k < kRows; ++k)
                    if (i[k] >= 0) store(i[k], head[k], s[k], acc[k]);
            }
            return;
        }
        for (int r = group; r < t.rows; r += row_groups) {
            int head;
            const int i = paged_row(p, t, r, head);
            if (i < 0) continue;
            JoinRow s = {-INFINITY, 0.f};
            float acc[C];
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = 0.f;
            for (int w = w0 + warp; w <= w1; w += 16) {
                float2 ml[4];
                float x[4][C];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ml[k] = make_float2(-INFINITY, 0.f);
                    if (w + 4 * k <= w1) join_load<C>(p, slot_of(w + 4 * k, r), D, lane, ml[k], x[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) join_add<C>(s, acc, ml[k], x[k], p.scale_log2);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) sh_o[warp][lane * C + c] = acc[c];
            if (lane == 0) sh_ml[warp] = make_float2(s.m, s.l);
            __syncthreads();
            if (warp == 0) {
                for (int k = 1; k < 4; ++k) {
                    float x[C];
#pragma unroll
                    for (int c = 0; c < C; ++c) x[c] = sh_o[k][lane * C + c];
                    join_add<C>(s, acc, sh_ml[k], x, p.scale_log2);
                }
                store(i, head, s, acc);
            }
            __syncthreads();
        }
        return;
    }
    for (int t = blockIdx.x * 4 + warp; t < p.N; t += zero_blocks * 4) {
        int seen = -1;                                       // last key the token sees
        bool owned = false;                                  // some sequence's token
        if (p.S > 0 && t < p.qstart[p.S]) {
            int lo = 0, hi = p.S;                            // last sequence that starts at or before t
            while (hi - lo > 1) {
                const int step = (hi - lo + 31) / 32;
                const int at = lo + lane * step;
                const bool ok = lane == 0 || (at < hi && p.qstart[at] <= t);
                const int n = __popc(__ballot_sync(0xffffffffu, ok));
                hi = min(hi, lo + n * step);
                lo = lo + (n - 1) * step;
            }
            const int begin = p.qstart[lo], end = p.qstart[lo + 1], len = p.kv_lens[lo];
            owned = begin >= 0 && begin <= t && t < end && end <= p.N;       // those that plan_new accepts
            seen = len <= 0 || len > static_cast<int64_t>(p.W) * p.page ? -1
                   : p.causal ? min(len - 1, len - end + t) : len - 1;
        }
        if (!owned) {                                        // behind the last sequence, or a start makes no sense
            if (!p.clear_tail) continue;
            seen = -1;
        }
        if (seen >= 0 && !p.mask) continue;
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;     // lanes of a head's row, rows of a store
        uint8_t* out = p.O + static_cast<int64_t>(t) * p.Hq * D * 2;
        for (int h0 = 0; h0 < p.Hq; h0 += 32) {
            const int h = h0 + lane;
            uint32_t dead = __ballot_sync(0xffffffffu, h < p.Hq && (seen < 0 ||
                                          p.mask[static_cast<int64_t>(t) * p.NG + h / p.hpg] == 0));
            while (dead) {
                uint32_t mine = dead;
                for (int k = 0; k < lane / kLanes; ++k) mine &= mine - 1;
                if (mine)
                    *reinterpret_cast<uint4*>(out + ((h0 + __ffs(mine) - 1) * D + lane % kLanes * 8) * 2) =
                        make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) dead &= dead - 1;
            }
        }
    }
}

template <int D, bool kBf16>
static int launch_warp(const PagedParams& p, int used, bool plan_here, cudaStream_t s)
{
    constexpr int rings = kPwWarps * kPwStages * 2 * kPwBN * D * 2;
    constexpr int lists = kPwTiles * int(sizeof(PagedTile)) + (2 * kPwTiles + 1) * 4;
    const dim3 grid((used + kPwWarps - 1) / kPwWarps);
    if (plan_here) {
        DPK_CUDA(cudaFuncSetAttribute(paged_warp_kernel<D, kBf16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      rings + lists));
        paged_warp_kernel<D, kBf16, true><<<grid, kPwWarps * 32, rings + lists, s>>>(p);
        DPK_CUDA(cudaGetLastError());
    } else {
        DPK_CUDA(cudaFuncSetAttribute(paged_warp_kernel<D, kBf16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      rings));
        DPK_CUDA(paged_launch(paged_warp_kernel<D, kBf16, false>, grid, kPwWarps * 32, rings, s, p));
    }
    return DPK_OK;
}

int attn_paged_warp(const PagedParams& p, int D, int dtype, int used, bool plan_here, cudaStream_t s)
{
    if (D == 64)
        return dtype == DPK_BF16 ? launch_warp<64, true>(p, used, plan_here, s)
                                 : launch_warp<64, false>(p, used, plan_here, s);
    return dtype == DPK_BF16 ? launch_warp<128, true>(p, used, plan_here, s)
                             : launch_warp<128, false>(p, used, plan_here, s);
}

template <int D, bool kBf16>
static int launch_join(const PagedParams& p, int used, cudaStream_t s)
{
    int zero = (p.N + 3) / 4;
    const int cap = sm_count() * 8;
    if (zero > cap) zero = cap;
    if (p.tile_rows <= 16)
        DPK_CUDA(paged_launch(paged_join_kernel<D, kBf16, 1>, dim3(used * 4 + zero), 128, 0, s, p, 4, used * 4));
    else
        DPK_CUDA(paged_launch(paged_join_kernel<D, kBf16, 2>, dim3(used * 4 + zero), 128, 0, s, p, 4, used * 4));
    return DPK_OK;
}

// Which kernel, and how the work is cut, from what the host knows.
struct PagedShape {
    bool tc;
    int tile_rows, unit_keys, tile_gap, workers, min_range;
    int64_t max_tiles;
    bool plan_here;
    size_t off_start, off_tile, off_slot, off_first, off_rows, off_count, off_border, off_o, off_ml, bytes;
};

static PagedShape paged_shape(int64_t N, int S, int Hq, int Hk, int D, int max_query_len, bool has_mask, int sms)
{
    PagedShape g;
    const int rep = Hq / Hk;
    // up to 16 rows per sequence and KV head are one tile of the warp kernel; more of them would
    // read K and V once per 16 rows there
    g.tc = static_cast<int64_t>(max_query_len) * rep > kPwRows;
    g.tile_rows = g.tc ? 128 : kPwRows;
    g.unit_keys = g.tc ? 64 : kPwBN;
    g.workers = g.tc ? 2 * sms : sms * kPwWarps;
    g.tile_gap = g.tc ? 3 : 1;
    g.min_range = 2;
    g.max_tiles = int64_t(Hk) * ((N * rep) / g.tile_rows + S);
    const int here = g.tc ? kPtTiles : kPwTiles;
    g.plan_here = g.max_tiles <= here && int64_t(S) * Hk <= here;
    size_t at = 16;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 15) & ~size_t(15);
        return here;
    };
    g.off_tile = take(size_t(g.max_tiles) * sizeof(PagedTile));
    g.off_slot = take(g.tc && has_mask ? size_t(g.max_tiles) * sizeof(PagedTile) : 0);
    g.off_start = take(size_t(g.max_tiles + 1) * 4);
    g.off_first = take(size_t(S) * Hk * 4);
    g.off_rows = take(g.tc && has_mask ? size_t(Hk) * N * rep * 4 : 0);
    g.off_count = take(g.tc && has_mask ? size_t(S) * Hk * 4 : 0);
    g.off_border = take(size_t(g.workers) * sizeof(PagedBorder));
    g.off_o = take(size_t(g.workers) * 2 * g.tile_rows * D * 4 + 16);      // room to start on 32 bytes
    g.off_ml = take(size_t(g.workers) * 2 * g.tile_rows * 8);
    g.bytes = at;
    return g;
}

static bool paged_sizes_ok(int64_t N, int S, int Hq, int Hk, int D)
{
    return N >= 0 && N < (1ll << 31) && S >= 0 && Hq > 0 && Hk > 0 && D > 0 && Hq % Hk == 0;
}

}  // namespace dpk

using namespace dpk;

extern "C" {

size_t dpk_attn_paged_workspace_bytes(int64_t N, int S, int Hq, int Hk, int D, int max_query_len, int has_mask)
{
    if (!paged_sizes_ok(N, S, Hq, Hk, D)) return 0;
    return paged_shape(N, S, Hq, Hk, D, max_query_len, has_mask != 0, sm_total()).bytes;
}

int dpk_attn_paged(const void* Q, const void* K, const void* V, const int32_t* page_table,
                   const int32_t* kv_lens, const int32_t* query_start, const uint8_t* mask, void* O, int64_t N,
                   int S, int W, int P, int page_size, int Hq, int Hk, int D, int NG, float scale, int causal,
                   int dtype, int max_query_len, int clear_tail, int64_t q_token_stride, int64_t page_stride,
                   int64_t page_token_stride, int64_t table_stride, void* workspace, size_t workspace_bytes,
                   void* stream)
{
    // a pool without pages and a table without entries have no address; nothing reads them
    DPK_REQUIRE(Q && ((K && V) || P == 0) && O && (page_table || W == 0 || S == 0) && (kv_lens || S == 0) && query_start,
                "NULL tensor");
    DPK_REQUIRE(dtype == DPK_F16 || dtype == DPK_BF16, "dtype must be DPK_F16 or DPK_BF16");
    DPK_REQUIRE(N >= 0 && N < (1ll << 31) && S >= 0 && W >= 0 && P >= 0 && Hq > 0 && Hk > 0, "bad shape");
    DPK_REQUIRE(D == 64 || D == 128, "head_dim %d not supported (64 or 128)", D);
    DPK_REQUIRE(Hq % Hk == 0, "Hq=%d must be a multiple of Hk=%d", Hq, Hk);
    DPK_REQUIRE(!mask || (NG > 0 && Hq % NG == 0), "Hq=%d must be a multiple of NG=%d", Hq, NG);
    DPK_REQUIRE(Hq / Hk <= 128, "more than 128 query heads per KV head are not supported");
    DPK_REQUIRE(page_size > 0 && page_size % 8 == 0, "page_size %d must be a multiple of 8", page_size);
    DPK_REQUIRE(int64_t(W) * page_size < (1ll << 30), "a row of the table holds 2^30 tokens or more");
    DPK_REQUIRE(max_query_len >= 1, "max_query_len must be at least 1");
    // the running maximum is one of q.k, so the scale may not turn its order round; 0 * -inf is no score
    DPK_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
    const int64_t q_ts = q_token_stride ? q_token_stride : int64_t(Hq) * D;
    const int64_t kv_ts = page_token_stride ? page_token_stride : int64_t(Hk) * D;
    const int64_t ps = page_stride ? page_stride : page_size * kv_ts;
    const int64_t ts = table_stride ? table_stride : W;
    DPK_REQUIRE(q_ts >= int64_t(Hq) * D && kv_ts >= int64_t(Hk) * D && ts >= W,
                "strides must cover the heads of a token and the pages of a row");
    DPK_REQUIRE(q_ts % 8 == 0 && kv_ts % 8 == 0 && ps % 8 == 0, "strides must be multiples of 8 elements (16 bytes)");
    DPK_REQUIRE(aligned16(Q) && aligned16(K) && aligned16(V) && aligned16(O), "tensors must be 16-byte aligned");
    if (N == 0) return DPK_OK;
    const PagedShape g = paged_shape(N, S, Hq, Hk, D, max_query_len, mask != nullptr, sm_total());
    const int workers = g.workers / sm_total() * sm_count();      // SMs left free by dpk_set_sm_margin
    const int64_t most = g.max_tiles * ((int64_t(W) * page_size + g.unit_keys - 1) / g.unit_keys + g.tile_gap);
    // places are 32-bit, and a worker's range may end a range behind the line (plan_range: below 2^16, or an equal share)
    DPK_REQUIRE(most < (1ll << 31) - (1 << 16), "too much work for one call: %lld tiles of up to %lld keys",
                (long long)g.max_tiles, (long long)W * page_size);
    DPK_REQUIRE((g.max_tiles + 1) * g.workers < (1ll << 31), "too many tiles for one call");
    DPK_REQUIRE(int64_t(Hq) * N < (1ll << 31), "too many rows for one call");
    DPK_REQUIRE(workspace && workspace_bytes >= g.bytes, "workspace of %zu bytes needed, %zu given", g.bytes,
                workspace_bytes);
    DPK_REQUIRE(aligned16(workspace), "workspace must be 16-byte aligned");
    PagedParams p;
    p.Q = static_cast<const uint8_t*>(Q);
    p.K = static_cast<const uint8_t*>(P > 0 ? K : Q);          // tensor maps are made all the same
    p.V = static_cast<const uint8_t*>(P > 0 ? V : Q);
    p.O = static_cast<uint8_t*>(O);
    p.table = page_table;
    p.kv_lens = kv_lens;
    p.qstart = query_start;
    p.mask = mask;
    p.q_ts = q_ts; p.page_stride = ps; p.token_stride = kv_ts; p.table_stride = ts;
    p.N = static_cast<int>(N); p.S = S; p.P = P;
    p.W = P > 0 ? W : 0;                       // without a page no length can be right
    p.page = page_size;
    p.Hq = Hq; p.Hk = Hk; p.NG = mask ? NG : 1;
    p.rep = Hq / Hk;
    p.hpg = Hq / p.NG;
    p.causal = causal ? 1 : 0;
    p.clear_tail = clear_tail ? 1 : 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    p.head = reinterpret_cast<PagedHead*>(w);
    p.tile = reinterpret_cast<PagedTile*>(w + g.off_tile);
    p.slot = reinterpret_cast<PagedTile*>(w + g.off_slot);
    p.start = reinterpret_cast<int32_t*>(w + g.off_start);
    p.first_tile = reinterpret_cast<int32_t*>(w + g.off_first);
    p.rows = g.tc && mask ? reinterpret_cast<int32_t*>(w + g.off_rows) : nullptr;
    p.row_count = g.tc && mask ? reinterpret_cast<int32_t*>(w + g.off_count) : nullptr;
    p.border = reinterpret_cast<PagedBorder*>(w + g.off_border);
    p.part_o = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(w + g.off_o) + 31) & ~uintptr_t(31));
    p.part_ml = reinterpret_cast<float*>(w + g.off_ml);
    p.tile_rows = g.tile_rows; p.unit_keys = g.unit_keys; p.tile_gap = g.tile_gap;
    p.workers = workers; p.min_range = g.min_range;
    p.max_tiles = static_cast<int>(g.max_tiles);
    p.status = device_status_ptr();
    if (!p.status) return fail(DPK_ERR_CUDA, "no status word on this device");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // workers that can get work at all, as far as the host knows
    int64_t used = (most + g.min_range - 1) / g.min_range;
    if (used > workers) used = workers;
    if (used < 1) used = 1;
    const int plan_threads = int64_t(S) * Hk <= 256 && g.max_tiles <= 512 ? 256 : kPlanThreads;
    if (p.rows && S > 0) {
        DPK_REQUIRE(Hk <= 65535, "grid too large");
        const int64_t per_thread = (static_cast<int64_t>(max_query_len) * p.rep + 15) / 16;
        const int threads = per_thread >= 1024 ? 1024 : static_cast<int>((per_thread + 31) / 32 * 32);
        paged_rows_kernel<<<dim3(S, Hk), threads, 0, s>>>(p);
        DPK_CUDA(cudaGetLastError());
        if (!g.plan_here) DPK_CUDA(paged_launch(paged_plan_kernel, dim3(1), plan_threads, 0, s, p));
    } else if (!g.plan_here) {
        paged_plan_kernel<<<1, plan_threads, 0, s>>>(p);
        DPK_CUDA(cudaGetLastError());
    }
    const int rc = g.tc ? attn_paged_tc(p, D, dtype, static_cast<int>(used), g.plan_here, s)
                        : attn_paged_warp(p, D, dtype, static_cast<int>(used), g.plan_here, s);
    if (rc) return rc;
    if (D == 64) return dtype == DPK_BF16 ? launch_join<64, true>(p, (int)used, s) : launch_join<64, false>(p, (int)used, s);
    return dtype == DPK_BF16 ? launch_join<128, true>(p, (int)used, s) : launch_join<128, false>(p, (int)used, s);
}

}  // extern "C"
