// Attention of new tokens over a paged KV cache on tcgen05 tensor cores (sm_100a): chunks of tokens.
//
// A CTA is a worker of the work list (dpk_attn_paged.cuh): it walks its range of 64-key units, tile
// after tile.  A tile is 128 active (token, query head) rows of one sequence and one KV head, so the
// heads that share K and V share its loads too.  Per unit
//     S = Q K^T      UMMA 128 x 64 x D, both operands K-major in shared memory, S in TMEM (two buffers)
//     P = exp2(..)   four warps, one row per thread: running reference maximum and sum in registers,
//                    P in 16 bits back into TMEM over S
//     O += P V       UMMA 128 x D x 64, A = P from TMEM, V in its natural [key][d] layout
// O is rescaled only when a row's maximum has grown by more than 2^8.
//
// K and V arrive by TMA through a map [page][64-channel block][row of page][64] whose box is gcd(page_size,
// 64) rows of one or both blocks: a unit is put together from as many boxes as pages meet in it, each
// lane of the producer warp looking up and loading its own (one lane that issues all of them is slower:
// 721 us instead of 526 for 4096 tokens over 12288 in pages of 16, with a box per block).  The copy engine needs some 30 cycles
// a box whatever its size, so a box takes both blocks of a head where the operand can be read that way:
// always for V, whose product steps through the rows 16 at a time, and for K where the 8-row groups of a
// block stay equally spaced (boxes of 8 or of 64 rows): 494 us instead of 526 for those 4096 tokens in
// pages of 16, 530 instead of 717 in pages of 8, 457 in pages of 64.
// Boxes behind the tile's last visible key get a page number outside the map and arrive as zeros; rows
// of V behind it inside a box (whatever a page holds behind its sequence) are cleared in shared memory by
// the softmax warps before the product, since 0 * NaN would not be 0.  Their K needs nothing: those
// scores are replaced by -inf.
//
// Warp roles (192 threads): 0-3 softmax and epilogue, 4 producer, 5 UMMA issuer and TMEM owner.
// 96 KiB of shared memory and 256 TMEM columns: two CTAs share an SM and fill each other's gaps.
// All waits are bounded.
#define DPK_KERNEL_ID 14   // thousands digit of the device status word
#include "dpk_attn_paged_plan.cuh"
#include "dpk_attn_tc.cuh"

namespace dpk {

constexpr int kPtBM = 128, kPtBN = 64, kPtThreads = 192, kPtTmemCols = 256;
constexpr float kPtRescale = 8.0f;       // log2 units

template <int D>
struct PtSmem {
    static constexpr int kQ = kPtBM * D * 2, kKV = kPtBN * D * 2;
    static constexpr int kOffQ = 0, kOffK = kQ, kOffV = kOffK + 2 * kKV, kOffBar = kOffV + 2 * kKV;
    static constexpr int kOffPlan = kOffBar + 16 * 8 + 16;
    static constexpr int kTotal = kOffPlan;
    static constexpr int kTotalPlan = kOffPlan + kPtTiles * (int(sizeof(PagedTile)) + 8) + 4;
};

// 32 bytes, a whole sector, from one thread (32-byte aligned): a warp's rows lie far apart, and 16-byte stores
// would send each sector twice.
__device__ __forceinline__ void pt_store_sector(void* dst, const uint32_t (&w)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// kBox: rows of a box where that is known at compile time (64: one box a unit), else 0.
template <int D, bool kBf16, int kBox>
__global__ void __launch_bounds__(kPtThreads, 2)
paged_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const PagedParams p, const int box, const bool whole, const bool plan_here)
{
    using L = PtSmem<D>;
    constexpr int KBQ = D / 64;
    const int box_rows = kBox ? kBox : box;
    const bool k_whole = kBox == 64 || whole;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem + L::kOffQ;
    uint8_t* sK = smem + L::kOffK;
    uint8_t* sV = smem + L::kOffV;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    // one barrier per buffer, so that no role can complete two phases of one before the other looks
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;      // [2] each
    uint64_t* v_full = bars + 3;
    uint64_t* k_empty = bars + 5;
    uint64_t* v_empty = bars + 7;
    uint64_t* s_full = bars + 9;
    uint64_t* p_full = bars + 11;
    uint64_t* pv_done = bars + 13;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    paged_let_next_start();
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) {
            atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_SMEM_BASE);
            p.border[blockIdx.x].last_worker = -1;
        }
        return;
    }
    // what needs nothing of the work list is done while that is still being made
    if (warp == 4 && lane == 0) {
        mbar_init(q_full, 128);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 128);
            mbar_init(&pv_done[s], 1);
        }
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 5) tmem_alloc(tmem_slot, kPtTmemCols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_o = tmem_base + 128;

    paged_wait_previous();
    int tiles, length, range;
    const PagedTile* tile_of = p.tile;
    const int32_t* start = p.start;
    if (plan_here) {
        // a short list is made by every CTA for itself: a launch less (24 sequences of 5 tokens over 300: 24.2 us a
        // call instead of 27.3, 18.5 on the device instead of 20.2)
        __shared__ int2 sh[32];
        PagedTile* my_tiles = reinterpret_cast<PagedTile*>(smem + L::kOffPlan);
        int32_t* my_start = reinterpret_cast<int32_t*>(my_tiles + kPtTiles);
        plan_work(p, my_tiles, my_start, my_start + kPtTiles + 1, sh, tiles, length);
        range = plan_range(p, tiles, length);
        tile_of = my_tiles;
        start = my_start;
    } else {
        tiles = p.head->tiles;
        length = p.head->length;
        range = p.head->range;
    }
    const int worker = blockIdx.x;
    int u_begin = 0, u_end = 0, tile0 = tiles;
    if (static_cast<int64_t>(worker) * range < length) {
        u_begin = worker * range;
        u_end = min(length, u_begin + range);
        tile0 = paged_find_tile(p, tile_of, start, tiles, u_begin);
    }
    if (tile0 >= tiles || start[tile0] >= u_end) {    // nothing, or only places between tiles
        if (threadIdx.x == 0) p.border[worker].last_worker = -1;
    } else if (warp < 4) {
        // =================== softmax / epilogue: thread = row of the tile ==================
        const int row = warp * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
        const bool o_sectors = (reinterpret_cast<uintptr_t>(p.O) & 31u) == 0;
        bool alive = true;
        int it = 0;                                     // units done, over all tiles
        int border = -1;
        // Q rows into the swizzled K-major layout: every warp its own 32 rows (8 lanes per 128 bytes, four
        // rows per pass; the rows' places in Q are looked up once, by the lane that owns the row)
        auto load_q = [&](const PagedTile& t, int& tok, int& head) {
            head = 0;
            tok = row < t.rows ? paged_row(p, t, row, head) : -1;
            const int64_t mine = tok < 0 ? -1 : (static_cast<int64_t>(t.tok0 + tok) * p.q_ts + static_cast<int64_t>(head) * D) * 2;
            const int chunk = lane & 7;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int sub = (lane >> 3) + 4 * k, r = warp * 32 + sub;
                const int64_t at = __shfl_sync(0xffffffffu, mine, sub);
                const uint8_t* src = p.Q + (at < 0 ? 0 : at);
#pragma unroll
                for (int kb = 0; kb < KBQ; ++kb)
                    cp_async_16(smem_u32(sQ) + kb * (kPtBM * 128) + r * 128 + ((chunk ^ (r & 7)) << 4),
                                src + kb * 128 + chunk * 16, at >= 0 ? 16u : 0u);
            }
            cp_async_commit();
        };
        auto q_ready = [&]() {
            cp_async_wait<0>();
            fence_proxy_async_smem();
            mbar_arrive(q_full);
        };
        PagedTile t = tile_of[tile0], nt = t;
        int t_first = start[tile0];
        int tok, head, ntok = -1, nhead = 0;
        load_q(t, tok, head);
        q_ready();
        bool more = true;
        for (int tile = tile0; alive && more; ++tile) {
            const int t_units = (t.kv_end + kPtBN - 1) / kPtBN;
            const int j0 = max(0, u_begin - t_first), j1 = min(t_units, u_end - t_first);
            const int n_first = start[tile + 1];           // what the next tile needs, long before
            more = tile + 1 < tiles && n_first < u_end;
            if (more) nt = tile_of[tile + 1];
            const int lim = paged_last_key(p, t, tok);
            // the fewest keys that a row of the warp sees: its first row's (rows are in token order)
            const int lim_first = __shfl_sync(0xffffffffu, lim, 0);
            const bool idle = warp * 32 >= t.rows;      // none of this warp's rows exists

            float m_ref = -INFINITY, l_sum = 0.f;
            const int seg_it = it;
            for (int j = j0; j < j1; ++j, ++it) {
                const int sb = it & 1;
                const uint32_t ph = (it >> 1) & 1;
                const bool got = mbar_wait(&s_full[sb], ph, abort_flag, p.status, DPK_DEV_TIMEOUT_TMEM_FULL);
                if (!__all_sync(0xffffffffu, got)) { alive = false; break; }
                tc_fence_after_sync();
                // the scores of the tile's last unit are there, so nothing reads Q any more: the next
                // tile's rows come in while this unit is worked on
                if (j == j1 - 1 && more) load_q(nt, ntok, nhead);
                const int kv0 = j * kPtBN;
                if (kv0 + kPtBN > t.kv_end && t.kv_end % box_rows != 0) {
                    // rows of V behind the last visible key that arrived with their box
                    const bool ok = mbar_wait(&v_full[sb], ph, abort_flag, p.status, DPK_DEV_TIMEOUT_FULL);
                    if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
                    const int r0 = t.kv_end - kv0;
                    const int r1 = min(kPtBN, (r0 + box_rows - 1) / box_rows * box_rows);
                    uint8_t* v = sV + sb * L::kKV;
                    for (int x = threadIdx.x; x < (r1 - r0) * KBQ * 8; x += 128) {
                        const int r = r0 + x / (KBQ * 8), c = x % (KBQ * 8);
                        const int which = r / box_rows, in_box = r - which * box_rows;
                        *reinterpret_cast<uint4*>(v + (which * KBQ + (c >> 3)) * (box_rows * 128) + in_box * 128 +
                                                  (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                if (idle) {
                    tc_fence_before_sync();
                    mbar_arrive(&p_full[sb]);
                    continue;
                }
                const uint32_t ts = tmem_base + sb * kPtBN + lane_base;
                uint32_t sv[kPtBN];
                {
                    uint32_t a32[32], b32[32];
                    tmem_ld_32x32b_x32(ts, a32);
                    tmem_ld_32x32b_x32(ts + 32, b32);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) { sv[i] = a32[i]; sv[32 + i] = b32[i]; }
                }
                if (kv0 + kPtBN - 1 > lim_first) {
#pragma unroll
                    for (int i = 0; i < kPtBN; ++i)
                        if (kv0 + i > lim) sv[i] = __float_as_uint(-INFINITY);
                }
                float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
                for (int i = 0; i < kPtBN; i += 8) {
                    t0 = tc_max3(t0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                    t1 = tc_max3(t1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                    t2 = tc_max3(t2, __uint_as_float(sv[i + 4]), __uint_as_float(sv[i + 5]));
                    t3 = tc_max3(t3, __uint_as_float(sv[i + 6]), __uint_as_float(sv[i + 7]));
                }
                const float tmax = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                float alpha = 1.f;
                bool moved = false;
                if (tmax > -INFINITY) {
                    if (m_ref == -INFINITY) {
                        m_ref = tmax;                   // nothing accumulated yet for this row
                    } else if ((tmax - m_ref) * p.scale_log2 > kPtRescale) {
                        alpha = tc_exp2((m_ref - tmax) * p.scale_log2);
                        m_ref = tmax;
                        moved = true;
                    }
                }
                const float ref = m_ref == -INFINITY ? 0.f : m_ref * p.scale_log2;
                // P goes to the second product in V's 16 bits: one MMA takes both operands in one type, and the
                // remainder would be a second product.  The row sum is taken in 32 bits.  Against 64 bits the
                // output is off by 0.0023 (bf16; 4096 tokens over 12288) and 0.00029 (fp16; 5 tokens over 4091) where
                // P in 32 bits leaves 0.0017 and 0.00021, the rounding of the output.
                uint32_t pk[kPtBN / 2];
                const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
                const float2 nref2 = make_float2(-ref, -ref);
                float2 ra = make_float2(0.f, 0.f), rb = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < kPtBN; i += 4) {
                    const float2 a = __ffma2_rn(make_float2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])),
                                                sc2, nref2);
                    const float2 b = __ffma2_rn(make_float2(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])),
                                                sc2, nref2);
                    const float2 pa = make_float2(tc_exp2(a.x), tc_exp2(a.y));
                    const float2 pb = make_float2(tc_exp2(b.x), tc_exp2(b.y));
                    ra = __fadd2_rn(ra, pa);
                    rb = __fadd2_rn(rb, pb);
                    pk[i >> 1] = pack_half2<kBf16>(pa.x, pa.y);
                    pk[(i >> 1) + 1] = pack_half2<kBf16>(pb.x, pb.y);
                }
                l_sum = l_sum * alpha + ((ra.x + ra.y) + (rb.x + rb.y));
                if (it > seg_it && __any_sync(0xffffffffu, moved)) {
                    // O may only be rescaled once the previous P V has finished
                    const int pb = (it - 1) & 1;
                    const bool ok = mbar_wait(&pv_done[pb], ((it - 1) >> 1) & 1, abort_flag, p.status,
                                              DPK_DEV_TIMEOUT_TMEM_EMPTY);
                    if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        tmem_ld_32x32b_x32(tmem_o + lane_base + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                        tmem_st_32x32b_x32(tmem_o + lane_base + c, v);
                    }
                    tmem_st_wait();
                }
                tmem_st_p(ts, pk);
                tmem_st_wait();
                tc_fence_before_sync();
                mbar_arrive(&p_full[sb]);
            }
            if (!alive) break;
            if (more) q_ready();

            // ---- epilogue: the row, finished or as this worker's part ----------------------
            const int pb = (it - 1) & 1;
            const bool ok = mbar_wait(&pv_done[pb], ((it - 1) >> 1) & 1, abort_flag, p.status,
                                      DPK_DEV_TIMEOUT_TMEM_EMPTY);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after_sync();
            if (!idle) {
                const bool whole = j1 - j0 == t_units;
                const float inv = paged_inverse(lim, l_sum);
                const int64_t slot = (static_cast<int64_t>(worker) * 2 + (t_first > u_begin ? 1 : 0)) * kPtBM + row;
                uint8_t* out = p.O + (static_cast<int64_t>(t.tok0 + max(tok, 0)) * p.Hq + head) * (D * 2);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t v[32];
                    tmem_ld_32x32b_x32(tmem_o + lane_base + c, v);
                    tmem_ld_wait();
                    if (tok < 0) continue;
                    if (whole) {
#pragma unroll
                        for (int q2 = 0; q2 < 2; ++q2) {
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                w[i] = pack_half2<kBf16>(__uint_as_float(v[q2 * 16 + 2 * i]) * inv,
                                                         __uint_as_float(v[q2 * 16 + 2 * i + 1]) * inv);
                            if (o_sectors) {
                                pt_store_sector(out + (c + q2 * 16) * 2, w);
                            } else {
                                uint4* dst = reinterpret_cast<uint4*>(out + (c + q2 * 16) * 2);
                                dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
                                dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        }
                    } else {
                        float* dst = p.part_o + slot * D + c;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t w[8] = {v[q * 8], v[q * 8 + 1], v[q * 8 + 2], v[q * 8 + 3],
                                                   v[q * 8 + 4], v[q * 8 + 5], v[q * 8 + 6], v[q * 8 + 7]};
                            pt_store_sector(dst + q * 8, w);
                        }
                    }
                }
                if (!whole && tok >= 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m_ref, l_sum);
            }
            if (j0 == 0 && j1 < t_units) border = tile;
            tc_fence_before_sync();     // the next tile's first P V overwrites O after these reads
            t = nt;
            t_first = n_first;
            tok = ntok;
            head = nhead;
        }
        cp_async_wait<0>();
        if (threadIdx.x == 0) paged_write_border(p, tile_of, start, worker, border, u_begin, range);
    } else if (warp == 4) {
        // =================== producer ======================================================
        // lane (box, part of a head) looks up its piece of the next unit while this one is loaded, and
        // issues that piece's copy of K; the first lane of a box also issues that of V
        const int parts = k_whole ? 1 : KBQ;
        const int pieces = kPtBN / box_rows * parts;
        const int my_box = lane / parts, kb = lane % parts;
        const uint32_t at_k = k_whole ? my_box * (KBQ * box_rows * 128)
                                       : kb * (kPtBN * 128) + my_box * box_rows * 128;
        const uint32_t at_v = my_box * (KBQ * box_rows * 128);
        int tile = tile0 - 1, j_next = 0, j_end = 0;
        bool have = true;                               // there is a next unit
        PagedTile t, nt = tile_of[tile0];
        int n_first = start[tile0];
        int raw_page = 0, next_row = -1, next_col = 0;  // not looked at before it is needed; row -1: no key
        auto look_up = [&]() {
            next_row = -1;
            if (j_next >= j_end) {
                ++tile;
                have = tile < tiles && n_first < u_end;
                if (!have) return;
                t = nt;
                j_next = max(0, u_begin - n_first);
                j_end = min((t.kv_end + kPtBN - 1) / kPtBN, u_end - n_first);
                n_first = start[tile + 1];            // long before it is needed
                if (tile + 1 < tiles) nt = tile_of[tile + 1];
            }
            next_col = t.kvh * KBQ + kb;
            const int key = j_next * kPtBN + my_box * box_rows;
            ++j_next;
            if (lane >= pieces || key >= t.kv_end) return;
            const int w = key / p.page;
            raw_page = p.table[t.seq * p.table_stride + w];
            next_row = key - w * p.page;
        };
        look_up();
        int v_page = 0, v_row = 0, v_col = 0;           // the unit whose V is loaded next
        bool last = false;
        // K runs one unit ahead of V: it is needed one softmax earlier and released earlier
        for (int j = 0; !last; ++j) {
            int k_page = p.P, k_row = 0;                // a page outside the map reads as zeros
            const int k_col = next_col;
            last = !have;
            if (!last) {
                if (next_row >= 0) {
                    if (raw_page >= 0 && raw_page < p.P) {
                        k_page = raw_page;
                        k_row = next_row;
                    } else {
                        atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
                    }
                }
                look_up();
                const int s = j & 1;
                const bool ok = mbar_wait(&k_empty[s], ((j >> 1) & 1) ^ 1, abort_flag, p.status, DPK_DEV_TIMEOUT_EMPTY);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (lane == 0) mbar_arrive_expect_tx(&k_full[s], L::kKV);
                __syncwarp();
                if (lane < pieces) tma_load_4d(sK + s * L::kKV + at_k, &tmK, &k_full[s], 0, k_row, k_col, k_page);
            }
            if (j > 0) {
                const int s = (j - 1) & 1;
                const bool ok = mbar_wait(&v_empty[s], (((j - 1) >> 1) & 1) ^ 1, abort_flag, p.status,
                                          DPK_DEV_TIMEOUT_EMPTY);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (lane == 0) mbar_arrive_expect_tx(&v_full[s], L::kKV);
                __syncwarp();
                if (lane < pieces && kb == 0)
                    tma_load_4d(sV + s * L::kKV + at_v, &tmV, &v_full[s], 0, v_row, v_col, v_page);
            }
            v_page = k_page;
            v_row = k_row;
            v_col = k_col;
        }
    } else {
        // =================== UMMA issuer ===================================================
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc_f16(kBf16 ? 1 : 0, kPtBM, kPtBN);
            const uint32_t idesc_o = umma_idesc_f16(kBf16 ? 1 : 0, kPtBM, D) | (1u << 16);   // B is MN-major
            // distance of a head's 64-channel blocks of K; 8-row groups are 1024 bytes apart, but KBQ times
            // that in boxes of 8 rows that hold whole heads (the descriptors' stride, in 16 bytes)
            const uint32_t k_block = (k_whole ? box_rows : kPtBN) * 128;
            const uint64_t spread = static_cast<uint64_t>((KBQ - 1) * 1024 >> 4) << 32;
            const uint64_t k_spread = k_whole && box_rows == 8 ? spread : 0, v_spread = box_rows == 8 ? spread : 0;
            uint32_t v_step[kPtBN / 16];                // where every 16th row of V is
#pragma unroll
            for (int k = 0; k < kPtBN / 16; ++k)
                v_step[k] = (k * 16 / box_rows * KBQ * box_rows + k * 16 % box_rows) * 128;
            bool ok = true;
            int it = 0, seg = 0;
            int n_first = start[tile0], n_end = tile_of[tile0].kv_end;
            for (int tile = tile0; ok && tile < tiles && n_first < u_end; ++tile, ++seg) {
                const int len = min((n_end + kPtBN - 1) / kPtBN, u_end - n_first) - max(0, u_begin - n_first);
                n_first = start[tile + 1];            // long before it is needed
                if (tile + 1 < tiles) n_end = tile_of[tile + 1].kv_end;
                ok = mbar_wait(q_full, seg & 1, abort_flag, p.status, DPK_DEV_TIMEOUT_FULL);
                auto issue_s = [&](int i) -> bool {
                    const int s = i & 1;
                    if (!mbar_wait(&k_full[s], (i >> 1) & 1, abort_flag, p.status, DPK_DEV_TIMEOUT_FULL)) return false;
                    tc_fence_after_sync();
#pragma unroll
                    for (int kb = 0; kb < KBQ; ++kb) {
                        const uint64_t a = umma_desc_k_sw128(smem_u32(sQ) + kb * (kPtBM * 128));
                        const uint64_t b = umma_desc_k_sw128(smem_u32(sK) + s * L::kKV + kb * k_block) + k_spread;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16_ss(tmem_base + s * kPtBN, a + 2 * k, b + 2 * k, idesc_s, (kb | k) != 0 ? 1u : 0u);
                    }
                    umma_commit(&s_full[s]);
                    umma_commit(&k_empty[s]);
                    return true;
                };
                for (int j = 0; ok && j < 2 && j < len; ++j) ok = issue_s(it + j);
                for (int j = 0; ok && j < len; ++j, ++it) {
                    const int s = it & 1;
                    const uint32_t ph = (it >> 1) & 1;
                    ok = mbar_wait(&p_full[s], ph, abort_flag, p.status, DPK_DEV_TIMEOUT_FULL) &&
                         mbar_wait(&v_full[s], ph, abort_flag, p.status, DPK_DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after_sync();
#pragma unroll
                    for (int k = 0; k < kPtBN / 16; ++k) {
                        const uint64_t b = umma_desc_mn_sw128(smem_u32(sV) + s * L::kKV + v_step[k], box_rows * 128) + v_spread;
                        umma_f16_ts(tmem_o, tmem_base + s * kPtBN + k * 8, b, idesc_o, (j | k) != 0 ? 1u : 0u);
                    }
                    umma_commit(&pv_done[s]);
                    umma_commit(&v_empty[s]);
                    if (j + 2 < len) ok = issue_s(it + 2);
                }
            }
        }
    }

    // after a wait that ran out: let copies in flight land before the shared memory goes away
    if (*abort_flag) __nanosleep(2000000);
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 5) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kPtTmemCols);
    }
}

template <int D, bool kBf16, int kBox>
static int launch_tc_box(const PagedParams& p, int used, int box, bool plan_here, cudaStream_t s)
{
    const bool k_whole = D == 64 || box == 8 || box == 64;
    CUtensorMap tmK, tmV;
    const uint64_t cols = static_cast<uint64_t>(p.Hk) * D;
    int rc = make_tmap_paged_sw128(&tmK, p.K, cols, p.page, p.P, p.token_stride, p.page_stride, box, k_whole ? D / 64 : 1);
    if (rc) return rc;
    rc = make_tmap_paged_sw128(&tmV, p.V, cols, p.page, p.P, p.token_stride, p.page_stride, box, D / 64);
    if (rc) return rc;
    const int smem = plan_here ? PtSmem<D>::kTotalPlan : PtSmem<D>::kTotal;
    DPK_CUDA(cudaFuncSetAttribute(paged_tc_kernel<D, kBf16, kBox>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  PtSmem<D>::kTotalPlan));
    if (plan_here && !p.rows) {                         // the call's first kernel starts after all earlier work
        paged_tc_kernel<D, kBf16, kBox><<<used, kPtThreads, smem, s>>>(tmK, tmV, p, box, k_whole, plan_here);
        DPK_CUDA(cudaGetLastError());
    } else {
        DPK_CUDA(paged_launch(paged_tc_kernel<D, kBf16, kBox>, dim3(used), kPtThreads, smem, s, tmK, tmV, p, box,
                              k_whole, plan_here));
    }
    return DPK_OK;
}

template <int D, bool kBf16>
static int launch_tc(const PagedParams& p, int used, bool plan_here, cudaStream_t s)
{
    int box = 64;                                       // gcd(page, 64): page is a multiple of 8
    while (p.page % box) box >>= 1;
    return box == 64 ? launch_tc_box<D, kBf16, 64>(p, used, box, plan_here, s)
                     : launch_tc_box<D, kBf16, 0>(p, used, box, plan_here, s);
}

int attn_paged_tc(const PagedParams& p, int D, int dtype, int used, bool plan_here, cudaStream_t s)
{
    if (D == 64)
        return dtype == DPK_BF16 ? launch_tc<64, true>(p, used, plan_here, s) : launch_tc<64, false>(p, used, plan_here, s);
    return dtype == DPK_BF16 ? launch_tc<128, true>(p, used, plan_here, s) : launch_tc<128, false>(p, used, plan_here, s);
}

}  // namespace dpk
