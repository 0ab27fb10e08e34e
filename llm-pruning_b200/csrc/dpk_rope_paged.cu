// Rotary positions with several axes, fused with the write of k and v into a paged cache (sm_100a).
//
// A token has one position per axis (time, height, width, ...); rotary pair i turns by
//     angle = position[axis(i)][token] * inv_freq[i]
//     (a, b) -> (a cos - b sin, b cos + a sin)
// where (a, b) are channels (i, R/2 + i) ("half" pairing) or (2i, 2i + 1) ("neighbours"), R <= D the
// rotary width; channels from R on pass through.  The last tokens of every sequence are the new
// ones: token t of sequence s = new token i goes to cache position kv_len[s] - n_s + i, i.e. row
// (position % page_size) of page table[s][position / page_size].
//
// The angle is computed here instead of being read as cos/sin tables: the tables would be 2 * R/2
// values per token for arithmetic that the kernel has time for, and in 16 bits they would round the
// rotation twice.  A position of 10^6 in fp32 leaves the angle 0.06 rad off, so the product is taken
// in fp64, in turns, and only the fraction of a turn goes on in fp32 (sincospif: no large-argument
// path).  One pair's angle serves all heads of the token.
//
// HBM bound: q, k and v are read once and written once.
#define DPK_KERNEL_ID 15   // thousands digit of the device status word
#include "dpk_host.h"
#include "dpk_sm100.cuh"

namespace dpk {

constexpr int kRopeMaxAxes = 8;

struct RopePagedParams {
    const uint8_t* q;        // [N, Hq, D], token stride q_ts
    const uint8_t* k;        // [N, Hk, D], token stride kv_ts
    const uint8_t* v;        // NULL without a cache
    uint8_t* q_out;          // [N, Hq, D], token stride qo_ts; may be q
    uint8_t* k_out;          // [N, Hk, D] packed, without a cache; may be k
    uint8_t* k_pages;        // [P, page, Hk, D] or NULL
    uint8_t* v_pages;
    const void* positions;   // [axes, N] int32 or int64
    const float* inv_freq;   // [R/2]
    const int32_t* axis_map; // [R/2] or NULL: then `ends`
    const int32_t* table;    // [S, W]
    const int32_t* kv_lens;  // [S]
    const int32_t* qstart;   // [S + 1]
    const uint8_t* granted;  // [S] or NULL: 0 where the cache had no room for the new tokens
    int64_t q_ts, kv_ts, qo_ts, page_stride, token_stride, table_stride, axis_stride;   // elements
    int ends[kRopeMaxAxes];  // axis a serves the pairs below ends[a] that no earlier axis serves
    float scale;             // of cos and sin
    int N, S, W, P, page, Hq, Hk, D, R, axes, wide_positions;
    int* status;
};

__device__ __forceinline__ void rope_report(const RopePagedParams& p)
{
    atomicCAS(p.status, 0, 1000 * DPK_KERNEL_ID + DPK_DEV_BAD_INDEX);
}

template <bool kBf16>
__device__ __forceinline__ void turn_half(uint4& a, uint4& b, const float2* cs)
{
    uint32_t* x = &a.x;
    uint32_t* y = &b.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a0, a1, b0, b1;
        unpack_half2<kBf16>(x[j], a0, a1);
        unpack_half2<kBf16>(y[j], b0, b1);
        const float2 t0 = cs[2 * j], t1 = cs[2 * j + 1];
        x[j] = pack_half2<kBf16>(fmaf(a0, t0.x, -b0 * t0.y), fmaf(a1, t1.x, -b1 * t1.y));
        y[j] = pack_half2<kBf16>(fmaf(b0, t0.x, a0 * t0.y), fmaf(b1, t1.x, a1 * t1.y));
    }
}

template <bool kBf16>
__device__ __forceinline__ void turn_near(uint4& a, const float2* cs)
{
    uint32_t* x = &a.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a0, b0;
        unpack_half2<kBf16>(x[j], a0, b0);
        const float2 t = cs[j];
        x[j] = pack_half2<kBf16>(fmaf(a0, t.x, -b0 * t.y), fmaf(b0, t.x, a0 * t.y));
    }
}

constexpr int kRopeMaxPairs = 256;
constexpr int kRopeWarps = 4;
constexpr int kRopeFlight = 4;           // heads of a lane in flight

// A warp takes one token, or (few tokens) every `split`-th group of its heads.  A lane keeps one place
// c of a head -- 16 channels: the two halves of 8 pairs, or 16 in a row -- for all the heads it visits,
// so the 8 angles it needs stay in registers; a warp covers 32 / (D/16) heads per step.  Nothing is
// shared between warps: one warp's lookups and sines are hidden by the others' copies.  A CTA per
// token with a barrier between angles and copies measured 130 to 157 us where this takes 114 (16384
// tokens, 64 + 2 * 8 heads of 128: 5.9 TB/s; 2 heads in flight 117, 8 heads 128).  The bound of five CTAs per SM
// holds the kernel at 96 registers; with the 111 it takes otherwise four fit, and those 16384 tokens take 117 us instead
// of 113 replayed from a graph.
template <bool kBf16, bool kNear>
__global__ void __launch_bounds__(kRopeWarps * 32, 5) rope_paged_kernel(const RopePagedParams p, int split)
{
    __shared__ float2 sh_cs[kRopeWarps][kRopeMaxPairs];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float2* cs = sh_cs[warp];
    const int per_head = p.D / 16, rot = p.R / 16;       // places of a head, those that turn
    const int across = per_head < 32 ? per_head : 32;    // places of a head that a warp covers at once
    const int step = 32 / across;                        // heads per step
    const int heads = p.Hq + (p.v ? 2 : 1) * p.Hk;
    const int64_t jobs = static_cast<int64_t>(p.N) * split;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kRopeWarps;
    for (int64_t job = static_cast<int64_t>(blockIdx.x) * kRopeWarps + warp; job < jobs; job += warps) {
        const int t = static_cast<int>(job / split), part = static_cast<int>(job - static_cast<int64_t>(t) * split);
        // where the token's k and v go: element offset in the pools, -1 nowhere
        int64_t row = -1;
        if (p.v) {
            if (t >= p.qstart[p.S]) continue;            // behind the last sequence: left as it is
            int lo = 0, hi = p.S;                        // last sequence that starts at or before t
            while (hi - lo > 1) {
                const int width = (hi - lo + 31) / 32, at = lo + lane * width;
                const bool ok = lane == 0 || (at < hi && p.qstart[at] <= t);
                const int n = __popc(__ballot_sync(0xffffffffu, ok));
                hi = min(hi, lo + n * width);
                lo += (n - 1) * width;
            }
            // The place follows from the end of the sequence's new tokens, so a start that makes no sense would name
            // tokens that are cached already: only a sequence whose range is one has places.
            const int begin = p.qstart[lo], end = p.qstart[lo + 1], len = p.kv_lens[lo];
            const bool sound = begin >= 0 && begin <= t && t < end && end <= p.N &&
                               len <= static_cast<int64_t>(p.W) * p.page;
            // a refused sequence's length does not count its new tokens: the place would be a cached token's
            const bool refused = sound && p.granted && p.granted[lo] == 0;
            const int pos = len - end + t;
            const int w = pos / p.page;
            const int id = sound && !refused && pos >= 0 && w < p.W ? p.table[lo * p.table_stride + w] : -1;
            if (id >= 0 && id < p.P) row = id * p.page_stride + (pos - w * p.page) * p.token_stride;
            else if (lane == 0 && !refused) rope_report(p);      // q is turned all the same
        }
        __syncwarp();
        for (int i = lane; i < p.R / 2; i += 32) {
            int axis = 0;
            if (p.axis_map) {
                axis = p.axis_map[i];
                if (axis < 0 || axis >= p.axes) {
                    rope_report(p);
                    axis = 0;
                }
            } else {
                while (axis < p.axes - 1 && i >= p.ends[axis]) ++axis;
            }
            const int64_t at = axis * p.axis_stride + t;
            const double pos = p.wide_positions ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                                : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
            const double turns = pos * static_cast<double>(p.inv_freq[i]) * 0.15915494309189533577;
            float s, c;
            sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
            cs[i] = make_float2(c * p.scale, s * p.scale);
        }
        __syncwarp();
        for (int cb = 0; cb < per_head; cb += across) {
            const int c = cb + lane % across;
            const bool turns = c < rot, busy = lane < step * across && c < per_head;
            float2 mine[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) mine[k] = turns ? cs[c * 8 + k] : make_float2(1.f, 0.f);
            const int lo_at = !kNear && turns ? c * 16 : c * 32;
            const int hi_at = !kNear && turns ? p.R + c * 16 : c * 32 + 16;      // bytes: R/2 channels further
            const int first = part * step + lane / across, stride = split * step;
            for (int h0 = first; h0 < heads; h0 += kRopeFlight * stride) {
                uint4 lo[kRopeFlight], hi[kRopeFlight];
#pragma unroll
                for (int k = 0; k < kRopeFlight; ++k) {
                    const int head = h0 + k * stride;
                    if (!busy || head >= heads) continue;
                    const uint8_t* src;
                    if (head < p.Hq) src = p.q + (t * p.q_ts + static_cast<int64_t>(head) * p.D) * 2;
                    else if (head < p.Hq + p.Hk) src = p.k + (t * p.kv_ts + static_cast<int64_t>(head - p.Hq) * p.D) * 2;
                    else src = p.v + (t * p.kv_ts + static_cast<int64_t>(head - p.Hq - p.Hk) * p.D) * 2;
                    lo[k] = *reinterpret_cast<const uint4*>(src + lo_at);
                    hi[k] = *reinterpret_cast<const uint4*>(src + hi_at);
                }
#pragma unroll
                for (int k = 0; k < kRopeFlight; ++k) {
                    const int head = h0 + k * stride;
                    if (!busy || head >= heads) continue;
                    if (turns && head < p.Hq + p.Hk) {
                        if constexpr (kNear) {
                            turn_near<kBf16>(lo[k], mine);
                            turn_near<kBf16>(hi[k], mine + 4);
                        } else {
                            turn_half<kBf16>(lo[k], hi[k], mine);
                        }
                    }
                    uint8_t* dst;
                    if (head < p.Hq) {
                        dst = p.q_out + (t * p.qo_ts + static_cast<int64_t>(head) * p.D) * 2;
                    } else if (!p.v) {
                        dst = p.k_out + (static_cast<int64_t>(t) * p.Hk + head - p.Hq) * p.D * 2;
                    } else if (row < 0) {
                        continue;
                    } else if (head < p.Hq + p.Hk) {
                        dst = p.k_pages + (row + static_cast<int64_t>(head - p.Hq) * p.D) * 2;
                    } else {
                        dst = p.v_pages + (row + static_cast<int64_t>(head - p.Hq - p.Hk) * p.D) * 2;
                    }
                    *reinterpret_cast<uint4*>(dst + lo_at) = lo[k];
                    *reinterpret_cast<uint4*>(dst + hi_at) = hi[k];
                }
            }
        }
    }
    // starts that no token looked at: sequences without a row, a first start that is not 0
    if (p.v) {
        const int64_t all = static_cast<int64_t>(gridDim.x) * (kRopeWarps * 32);
        bool bad = false;
#pragma unroll 8
        for (int64_t s = static_cast<int64_t>(blockIdx.x) * (kRopeWarps * 32) + threadIdx.x; s < p.S; s += all) {
            const int begin = p.qstart[s], end = p.qstart[s + 1];
            bad |= begin < 0 || end < begin || end > p.N || (s == 0 && begin != 0);
        }
        if (bad) rope_report(p);
    }
}

template <bool kBf16, bool kNear>
static void launch_rope(const RopePagedParams& p, cudaStream_t s)
{
    // 20 warps fit an SM: fewer tokens than that are split by heads, down to one step a warp; more warps
    // than fit would only repeat the lookups (2200 tokens: 25 us unsplit, 31 split in two)
    const int per_head = p.D / 16, step = per_head < 32 ? 32 / per_head : 1;
    const int heads = p.Hq + (p.v ? 2 : 1) * p.Hk;
    const int64_t room = static_cast<int64_t>(sm_count()) * 20;
    int64_t split = room / p.N, most = (heads + step - 1) / step;
    if (split > most) split = most;
    if (split < 1) split = 1;
    const int64_t blocks = (p.N * split + kRopeWarps - 1) / kRopeWarps;
    rope_paged_kernel<kBf16, kNear><<<static_cast<unsigned>(blocks), kRopeWarps * 32, 0, s>>>(p, static_cast<int>(split));
}

}  // namespace dpk

using namespace dpk;

extern "C" {

int dpk_rope_append_paged(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                          int64_t q_token_stride, int64_t kv_token_stride, int64_t q_out_token_stride,
                          const void* positions, int64_t axis_stride, int positions_64, const float* inv_freq,
                          const int32_t* axis_map, const int32_t* sections, int axes, int rotary, int neighbours,
                          float scale, void* k_pages, void* v_pages, int64_t page_stride, int64_t page_token_stride,
                          const int32_t* table, int64_t table_stride, const int32_t* kv_lens,
                          const int32_t* query_start, int N, int S, int W, int P, int page_size, int Hq, int Hk,
                          int D, int dtype, void* stream)
{
    return dpk_rope_append_paged_granted(q, k, v, q_out, k_out, q_token_stride, kv_token_stride, q_out_token_stride,
                                         positions, axis_stride, positions_64, inv_freq, axis_map, sections, axes,
                                         rotary, neighbours, scale, k_pages, v_pages, page_stride, page_token_stride,
                                         table, table_stride, kv_lens, query_start, N, S, W, P, page_size, Hq, Hk, D,
                                         dtype, nullptr, stream);
}

int dpk_rope_append_paged_granted(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                                  int64_t q_token_stride, int64_t kv_token_stride, int64_t q_out_token_stride,
                                  const void* positions, int64_t axis_stride, int positions_64,
                                  const float* inv_freq, const int32_t* axis_map, const int32_t* sections, int axes,
                                  int rotary, int neighbours, float scale, void* k_pages, void* v_pages,
                                  int64_t page_stride, int64_t page_token_stride, const int32_t* table,
                                  int64_t table_stride, const int32_t* kv_lens, const int32_t* query_start, int N,
                                  int S, int W, int P, int page_size, int Hq, int Hk, int D, int dtype,
                                  const uint8_t* granted, void* stream)
{
    DPK_REQUIRE(q && k && q_out && positions && inv_freq, "NULL tensor");
    DPK_REQUIRE((k_pages == nullptr) == (v_pages == nullptr), "k_pages and v_pages go together");
    // a cache of no pages has no address, but a state: its tokens have no place, which is reported
    const bool cached = k_pages || (query_start && P == 0 && !k_out);
    DPK_REQUIRE(dtype == DPK_F16 || dtype == DPK_BF16, "dtype must be DPK_F16 or DPK_BF16");
    DPK_REQUIRE(N >= 0 && Hq > 0 && Hk > 0, "bad shape");
    DPK_REQUIRE(D > 0 && D % 16 == 0 && D <= 1024, "head_dim=%d must be a multiple of 16 up to 1024", D);
    DPK_REQUIRE(rotary > 0 && rotary % 16 == 0 && rotary <= D && rotary <= 2 * kRopeMaxPairs,
                "rotary width %d must be a multiple of 16, at most head_dim and %d", rotary, 2 * kRopeMaxPairs);
    DPK_REQUIRE(axes >= 1 && axes <= kRopeMaxAxes, "1 to %d axes are supported, got %d", kRopeMaxAxes, axes);
    DPK_REQUIRE(axes == 1 || axis_map || sections, "several axes need sections or an axis per pair");
    DPK_REQUIRE(q_token_stride >= int64_t(Hq) * D && q_out_token_stride >= int64_t(Hq) * D &&
                    kv_token_stride >= int64_t(Hk) * D && q_token_stride % 8 == 0 &&
                    q_out_token_stride % 8 == 0 && kv_token_stride % 8 == 0,
                "token strides must cover a token's heads and be multiples of 8 elements");
    DPK_REQUIRE(axes == 1 || axis_stride >= N, "positions of an axis overlap the next axis");
    RopePagedParams p;
    if (cached) {
        DPK_REQUIRE(v && (table || W == 0 || S == 0) && (kv_lens || S == 0) && query_start, "NULL tensor");
        DPK_REQUIRE(S >= 0 && W >= 0 && P >= 0 && page_size > 0 && table_stride >= W, "bad shape");
        DPK_REQUIRE(int64_t(W) * page_size < (1ll << 31), "a row of the table holds 2^31 tokens or more");
        DPK_REQUIRE(page_token_stride >= int64_t(Hk) * D && page_token_stride % 8 == 0 && page_stride % 8 == 0,
                    "page strides must cover a token's heads and be multiples of 8 elements");
        if (S == 0) return DPK_OK;
    } else {
        DPK_REQUIRE(k_out, "k_out is needed without a cache");
    }
    DPK_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_out) &&
                    aligned16(k_pages) && aligned16(v_pages), "tensors must be 16-byte aligned");
    int end = 0;
    for (int a = 0; a < kRopeMaxAxes; ++a) {
        if (sections && !axis_map && a < axes) {
            DPK_REQUIRE(sections[a] >= 0 && sections[a] <= rotary / 2, "bad section");
            end += sections[a];
        }
        p.ends[a] = sections && !axis_map ? end : rotary / 2;
    }
    DPK_REQUIRE(!sections || axis_map || end == rotary / 2, "sections sum to %d, the rotary width has %d pairs", end,
                rotary / 2);
    if (N == 0) return DPK_OK;
    p.q = static_cast<const uint8_t*>(q);
    p.k = static_cast<const uint8_t*>(k);
    p.v = cached ? static_cast<const uint8_t*>(v) : nullptr;
    p.q_out = static_cast<uint8_t*>(q_out);
    p.k_out = static_cast<uint8_t*>(k_out);
    p.k_pages = static_cast<uint8_t*>(k_pages);
    p.v_pages = static_cast<uint8_t*>(v_pages);
    p.positions = positions;
    p.inv_freq = inv_freq;
    p.axis_map = axis_map;
    p.table = table;
    p.kv_lens = kv_lens;
    p.qstart = query_start;
    p.granted = granted;
    p.q_ts = q_token_stride;
    p.kv_ts = kv_token_stride;
    p.qo_ts = q_out_token_stride;
    p.page_stride = page_stride;
    p.token_stride = page_token_stride;
    p.table_stride = table_stride;
    p.axis_stride = axis_stride;
    p.scale = scale;
    p.N = N; p.S = S; p.W = W; p.P = P; p.page = page_size;
    p.Hq = Hq; p.Hk = Hk; p.D = D; p.R = rotary; p.axes = axes;
    p.wide_positions = positions_64 ? 1 : 0;
    p.status = device_status_ptr();
    if (!p.status) return fail(DPK_ERR_CUDA, "no status word on this device");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == DPK_BF16) {
        if (neighbours) launch_rope<true, true>(p, s);
        else launch_rope<true, false>(p, s);
    } else {
        if (neighbours) launch_rope<false, true>(p, s);
        else launch_rope<false, false>(p, s);
    }
    DPK_CUDA(cudaGetLastError());
    return DPK_OK;
}

}  // extern "C"
