"""Paged-cache operators against plain 64-bit / integer implementations (oracle/paged_oracle.py).

Tolerances, per element.  With u half a unit in the last place of the type relative to the value:

* attention: the output is rounded once (u |o|), the weights p are rounded once before the second
  product (u sum p|v|; their sum is taken before); everything else is in 32 bits:
  scores and exponentials are off by less than 2^-13 of a weight here (scores of a few units,
  128 products of 2^-24 each, an exponential of 2^-22).
* rotation: one rounding (u |x|) and 32-bit sines, cosines and products (2^-20 of |a| + |b|).
* the smallest steps of fp16 below 2^-14 are absolute: 2^-25.
"""

import math
import random

import pytest
import torch

from oracle import paged_oracle as PO

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from dpk_b200 import build, ops
    build.build()
    return ops


@pytest.fixture(autouse=True)
def _status_clean(request, ops):
    yield
    if torch.cuda.is_available() and "gpu" in request.keywords:
        assert ops.device_status() == 0


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def make(new, cached, page, Hq, Hk, D, dtype, seed=0, spare=2, width=None, garbage=None):
    """A ragged batch whose pages are shuffled; what no token fills holds ``garbage``."""
    g = torch.Generator().manual_seed(seed)
    S = len(new)
    lens = [n + c for n, c in zip(new, cached)]
    used = [-(-n // page) for n in lens]
    P = sum(used) + spare
    order = torch.randperm(P, generator=g).tolist()
    W = width or max(max(used), 1)
    table = torch.full((S, W), -1, dtype=torch.int32)
    k = torch.randn(P, page, Hk, D, generator=g)
    v = torch.randn(P, page, Hk, D, generator=g)
    at = 0
    filled = torch.zeros(P, page, dtype=torch.bool)
    for s in range(S):
        ids = order[at:at + used[s]]
        at += used[s]
        table[s, :used[s]] = torch.tensor(ids, dtype=torch.int32)
        for j in range(lens[s]):
            filled[ids[j // page], j % page] = True
    if garbage is not None:
        k[~filled] = garbage
        v[~filled] = garbage
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], Hq, D, generator=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return dict(q=q.to(dtype), k=k.to(dtype), v=v.to(dtype), table=table, lens=i32(lens), start=i32(starts),
                gen=g)


def cuda(b):
    return {k: (t.cuda() if isinstance(t, torch.Tensor) else t) for k, t in b.items()}


def check_attention(got, b, mask=None, **kw):
    want, size = PO.attention(b["q"], b["k"].nan_to_num(0, 0, 0), b["v"].nan_to_num(0, 0, 0), b["table"],
                              b["lens"], b["start"], mask, **kw)
    u = u_of(b["q"].dtype)
    tol = u * want.abs() + (u + 2.0 ** -13) * size + 2.0 ** -25
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(9e9).max())} of the bound"


# ------------------------------------------------------------------------------ refusals (CPU)

def test_cpu_tensors_are_refused(ops):
    b = make([1, 1], [3, 0], 8, 2, 1, 64, BF)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_paged(b["q"], b["k"], b["v"], b["table"], b["lens"], b["start"])
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_axes(b["q"], b["q"], torch.zeros(2, dtype=torch.int64), torch.ones(32))
    refs = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.page_trim(b["table"], b["lens"], refs, b["lens"], page_size=8)


def test_c_entries_refuse_before_any_launch(ops):
    import ctypes

    from dpk_b200 import _native as N
    lib = N.load()
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255

    def attn(N_=4, S=2, W=4, P=8, page=16, Hq=8, Hk=2, D=128, NG=2, most=1, mask=p, ws=0, q_ts=0, ts=0, ps=0, sc=0.1):
        return lib.dpk_attn_paged(p, p, p, p, p, p, mask, p, N_, S, W, P, page, Hq, Hk, D, NG, sc, 1, N.BF16,
                                  most, 0, q_ts, ps, ts, 0, p, ws, None)
    for kw, word in ((dict(D=96), "head_dim"), (dict(Hq=7), "multiple of Hk"), (dict(NG=3), "multiple of NG"),
                     (dict(page=12), "page_size"), (dict(page=0), "page_size"), (dict(most=0), "max_query_len"),
                     (dict(Hq=258, Hk=2, mask=None), "128"), (dict(q_ts=8), "strides"), (dict(ts=257), "strides"),
                     (dict(W=1 << 28, page=8), "2\\^30"), (dict(sc=0.0), "scale"), (dict(sc=-1.0), "scale"),
                     (dict(sc=math.inf), "scale"), (dict(sc=math.nan), "scale"), (dict(), "workspace")):
        rc = attn(**kw)
        assert rc == N.ERR_INVALID, kw
        with pytest.raises(ValueError, match=word):
            N.check(rc)
    assert attn(N_=0) == N.OK

    def rope(axes=1, rotary=64, D=64, sections=None, amap=None, kp=p, page=16, W=4, k_out=None, ts=128):
        secs = (ctypes.c_int32 * len(sections))(*sections) if sections else None
        return lib.dpk_rope_append_paged(p, p, p, p, k_out, 256, 128, 256, p, 16, 1, p, amap, secs, axes, rotary, 0,
                                         1.0, kp, kp, 2048, ts, p, W, p, p, 4, 2, W, 8, page, 4, 2, D, N.BF16, None)
    for kw, word in ((dict(rotary=24), "rotary"), (dict(rotary=128), "rotary"), (dict(axes=3), "sections"),
                     (dict(axes=9, sections=[1] * 9), "axes"), (dict(axes=2, sections=[16, 15]), "sum"),
                     (dict(axes=2, sections=[33, -1]), "section"), (dict(D=72), "head_dim"),
                     (dict(kp=None), "k_out"), (dict(ts=64), "strides")):
        rc = rope(**kw)
        assert rc == N.ERR_INVALID, kw
        with pytest.raises(ValueError, match=word):
            N.check(rc)

    rc = lib.dpk_page_extend(p, 4, p, p, 2, 4, 8, 16, p, p, p, p, 1, 0, 2048, 128, p, 0, None)
    assert rc == N.ERR_INVALID and "workspace" in N.last_error()
    rc = lib.dpk_page_extend(p, 3, p, p, 2, 4, 8, 16, p, p, p, p, 1, 0, 2048, 128, p, 4096, None)
    assert rc == N.ERR_INVALID and "table_stride" in N.last_error()
    rc = lib.dpk_page_extend(p, 4096, p, p, 1 << 20, 4096, 8, 16, p, p, p, p, 1, 0, 2048, 128, p, 1 << 40, None)
    assert rc == N.ERR_INVALID and "too many" in N.last_error()
    rc = lib.dpk_page_fork(p, 4, p, p, 2, 4, 8, 0, p, p, 1, p, p, 4096, None)
    assert rc == N.ERR_INVALID
    rc = lib.dpk_page_copy(p, p, 1, 0, 104, 128, 8, 16, p, p, 1, p, 4096, None)
    assert rc == N.ERR_INVALID and "page_stride" in N.last_error()
    rc = lib.dpk_page_copy(p, p, 1, 0, 2048, 4, 8, 16, p, p, 1, p, 4096, None)
    assert rc == N.ERR_INVALID and "multiple of 8" in N.last_error()
    rc = lib.dpk_page_trim(None, 4, p, p, 2, 4, 8, 16, p, None, 1, None)
    assert rc == N.ERR_INVALID and "NULL" in N.last_error()
    rc = lib.dpk_page_compact(p, p, 1, 0, 2048, 128, p, 4, p, p, 2, 4, 8, 16, None, p, 4096, None)
    assert rc == N.ERR_INVALID and "NULL" in N.last_error()


def test_page_oracle_keeps_its_own_books():
    """Every page's count is the number of rows that hold it, whatever sequence of operators ran."""
    rng = random.Random(3)
    S, W, P, page = 12, 6, 40, 4
    st = PO.Pages([[-1] * W for _ in range(S)], [0] * S, [0] * P, page)
    for _ in range(300):
        act = rng.choice(["extend", "extend", "fork", "trim", "compact"])
        if act == "extend":
            st.extend([rng.choice([0, 0, 1, 3, 7, -1]) for _ in range(S)])
        elif act == "fork":
            n = rng.randint(1, 4)
            st.fork([rng.randrange(S) for _ in range(n)], [rng.randrange(S) for _ in range(n)])
        elif act == "trim":
            n = rng.randint(1, 4)
            st.trim([rng.randrange(S) for _ in range(n)], [rng.choice([0, 0, 2, 5, 9]) for _ in range(n)])
        else:
            st.compact()
        count = [0] * P
        for s in range(S):
            for j in range(st.held(s)):
                count[st.table[s][j]] += 1
        assert count == st.refs


# ------------------------------------------------------------------------------- attention (GPU)

ATTN = [
    # new, cached, page, Hq, Hk, D, NG, dtype
    ([1], [0], 8, 1, 1, 64, 0, BF),                        # one token, nothing cached
    ([1, 1, 1], [0, 7, 8], 8, 4, 2, 64, 2, FP),            # pages that end with the tokens, one before, one behind
    ([1] * 5, [31, 32, 33, 500, 63], 16, 8, 2, 128, 2, BF),
    ([1] * 3, [1000, 1, 130], 24, 32, 8, 128, 8, BF),      # pages of 24: several per unit, none aligned to it
    ([1, 2, 3], [300, 0, 17], 32, 6, 2, 64, 3, FP),        # groups that split a KV head's queries
    ([4, 4], [250, 90], 128, 16, 4, 128, 16, BF),          # a page larger than a unit, one head per group
    ([5, 1, 0, 9], [40, 700, 20, 0], 16, 12, 4, 128, 0, FP),   # a sequence without new tokens
    ([40, 3, 1], [100, 65, 2], 16, 8, 2, 64, 2, BF),
    ([129, 70], [0, 300], 16, 8, 8, 128, 8, BF),           # one query head per KV head
    ([130, 1, 33], [200, 513, 31], 64, 16, 2, 128, 2, FP), # eight per KV head
    ([257], [64], 8, 10, 2, 64, 5, BF),                    # five per KV head, groups across KV heads
    ([90], [20], 40, 4, 1, 128, 1, BF),                    # whole-token routing, pages of 40
    ([70, 30], [150, 77], 32, 8, 2, 128, 2, BF),           # boxes of 32 rows
    ([70, 30], [150, 77], 96, 8, 2, 128, 0, FP),           # boxes of 32 rows in pages of 96
    ([70, 30], [150, 77], 8, 8, 2, 128, 2, FP),            # boxes of 8 rows
    ([70, 30], [150, 77], 48, 8, 2, 128, 4, BF),           # boxes of 16 rows, three a page
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention_paged(ops, case, causal):
    new, cached, page, Hq, Hk, D, NG, dtype = ATTN[case]
    b = make(new, cached, page, Hq, Hk, D, dtype, seed=case)
    mask = None
    if NG:
        mask = torch.rand(b["q"].shape[0], NG, generator=b["gen"]) < 0.6
    d = cuda(b)
    for most in (max(new), None):
        got, meta = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"],
                                        None if mask is None else mask.cuda(), max_query_len=most,
                                        is_causal=causal)
        assert meta == {}
        check_attention(got, b, mask, causal=causal)
        if mask is not None:
            dead = ~mask.repeat_interleave(Hq // NG, 1)
            assert (got.cpu()[dead] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf")])
def test_attention_paged_ignores_what_no_token_fills(ops, garbage, most):
    b = make([1, 30, 2], [70, 9, 0], 16, 8, 2, 128, BF, seed=5, garbage=garbage)
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    check_attention(got, b)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
def test_attention_paged_rows_that_see_nothing(ops, most):
    # kv_lens smaller than the new tokens: the first ones see no key; one sequence has an empty cache
    b = make([6, 3, 2], [0, 20, 5], 16, 4, 2, 64, BF, seed=9)
    b["lens"][0] = 2
    b["lens"][2] = 0
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    check_attention(got, b)
    assert (got[:4] == 0).all() and (got[9:] == 0).all()
    off = torch.zeros(11, 2, dtype=torch.bool, device="cuda")      # everything routed out
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], off, max_query_len=most)
    assert (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 80])
def test_attention_paged_rows_behind_the_last_sequence(ops, most):
    b = make([3, 50], [30, 0], 16, 4, 2, 64, BF, seed=10)
    extra = torch.randn(9, 4, 64).to(BF)
    b["q"] = torch.cat([b["q"], extra])
    d = cuda(b)
    mine = torch.full((62, 4, 64), 7.0, dtype=BF, device="cuda")
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], O=mine, max_query_len=most)
    assert got is mine and (got[53:] == 7).all()
    new, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    assert (new[53:] == 0).all() and torch.equal(new[:53], got[:53])
    check_attention(new, b)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 40])
def test_attention_paged_strides(ops, most):
    """q as columns of a fused projection, K and V interleaved in one pool, a slice of a page table."""
    b = make([2, 33, 1], [70, 40, 300], 16, 8, 2, 128, BF, seed=11)
    d = cuda(b)
    fused = torch.randn(36, 8 * 128 + 512, device="cuda").to(BF)
    fused[:, 512:] = d["q"].flatten(1)
    q = fused[:, 512:].view(36, 8, 128)
    P = d["k"].shape[0]
    pool = torch.empty(P, 2, 16, 2, 128, dtype=BF, device="cuda")
    pool[:, 0], pool[:, 1] = d["k"], d["v"]
    wide = torch.full((3, 40), -7, dtype=torch.int32, device="cuda")
    W = d["table"].shape[1]
    wide[:, 5:5 + W] = d["table"]
    want, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    got, _ = ops.attention_paged(q, pool[:, 0], pool[:, 1], wide[:, 5:5 + W], d["lens"], d["start"],
                                 max_query_len=most)
    assert torch.equal(got, want)
    token_major = torch.empty(P, 16, 2, 2, 128, dtype=BF, device="cuda")
    token_major[:, :, 0], token_major[:, :, 1] = d["k"], d["v"]
    got, _ = ops.attention_paged(q, token_major[:, :, 0], token_major[:, :, 1], wide[:, 5:5 + W], d["lens"],
                                 d["start"], max_query_len=most)
    assert torch.equal(got, want)
    room = torch.zeros(36 * 8 * 128 + 8, dtype=BF, device="cuda")          # an output that starts on 16 bytes
    mine = room[8:].view(36, 8, 128)
    got, _ = ops.attention_paged(q, pool[:, 0], pool[:, 1], wide[:, 5:5 + W], d["lens"], d["start"], O=mine,
                                 max_query_len=most)
    assert got is mine and torch.equal(mine, want) and (room[:8] == 0).all()
    check_attention(want, b)


@pytest.mark.gpu
def test_attention_paged_row_offsets_beyond_32_bits(ops):
    """Two pages 4.4 GB apart in one pool of two-byte elements (2.2 * 2^30 elements)."""
    page, Hk, D = 16, 2, 128
    P = 2 ** 31 // (page * Hk * D) + 4
    k = torch.zeros(P, page, Hk, D, dtype=BF, device="cuda")
    v = torch.zeros(P, page, Hk, D, dtype=BF, device="cuda")
    b = make([3, 1], [20, 9], page, 4, Hk, D, BF, seed=12, spare=0)
    ids = torch.tensor([P - 1, 2, P - 3], dtype=torch.int64)
    k[ids.cuda()], v[ids.cuda()] = b["k"].cuda(), b["v"].cuda()
    table = torch.where(b["table"] >= 0, ids[b["table"].clamp(min=0).long()].int(), -1)
    d = cuda(b)
    for most in (1, 64):
        got, _ = ops.attention_paged(d["q"], k, v, table.cuda(), d["lens"], d["start"], max_query_len=most)
        check_attention(got, b)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 128])
def test_attention_paged_large_scores_and_scale(ops, most):
    b = make([60, 1], [3, 100], 16, 4, 2, 64, BF, seed=13)
    b["q"] *= 40                                       # nearly one-hot weights, scores of hundreds
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], scale=0.25,
                                 max_query_len=most)
    want, size = PO.attention(b["q"], b["k"], b["v"], b["table"], b["lens"], b["start"], scale=0.25)
    # scores up to ~ 40 * 64 * 0.25 = 640 units: 32 bits leave them 64 * 640 * 2^-24 off, and that is
    # how far a weight is off, relatively
    tol = u_of(BF) * (want.abs() + size) + (2.0 ** -13 + 2 * 64 * 640 * 2.0 ** -24) * size + 1e-6
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_attention_paged_same_bits_every_time_and_on_another_stream(ops):
    b = make([1] * 6, [3000, 17, 900, 64, 1, 2222], 16, 16, 4, 128, BF, seed=14)
    d = cuda(b)
    first, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=1)[0]
                for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert torch.equal(o, first)
    check_attention(first, b)


@pytest.mark.gpu
def test_attention_paged_reports_bad_pages(ops):
    b = make([1, 1], [40, 40], 16, 4, 2, 64, BF, seed=15)
    d = cuda(b)
    for bad in (-1, d["k"].shape[0], 2 ** 31 - 1):
        for most in (1, 64):
            t = d["table"].clone()
            t[1, 1] = bad
            got, _ = ops.attention_paged(d["q"], d["k"], d["v"], t, d["lens"], d["start"], max_query_len=most)
            assert ops.device_status() % 1000 == 105
            assert torch.isfinite(got[0]).all()
    # lengths and starts outside their range
    for lens, start in (([41, 10 ** 9], [0, 1, 2]), ([41, -5], [0, 1, 2]), ([41, 41], [0, 1, 900]), ([41, 41], [0, 2, 1])):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        ops.attention_paged(d["q"], d["k"], d["v"], d["table"], i32(lens), i32(start), max_query_len=1)
        assert ops.device_status() % 1000 == 105


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
def test_attention_paged_in_a_graph_follows_the_state(ops, most):
    """Captured once, replayed with other lengths, tables and tokens; two graphs side by side."""
    b = make([1] * 4, [70, 3, 200, 31], 16, 8, 2, 128, BF, seed=16, width=20)
    d = cuda(b)
    run = lambda: ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)[0]
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    c = make([1] * 4, [5, 130, 0, 64], 16, 8, 2, 128, BF, seed=17, width=20, spare=10)
    n = min(c["k"].shape[0], d["k"].shape[0])
    assert int(c["table"].max()) < d["k"].shape[0] or n == d["k"].shape[0]
    c["table"].clamp_(max=n - 1)
    d["k"][:n], d["v"][:n] = c["k"][:n].cuda(), c["v"][:n].cuda()
    d["q"].copy_(c["q"])
    d["lens"].copy_(c["lens"])
    d["table"].copy_(c["table"])
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    c["k"], c["v"] = d["k"].cpu(), d["v"].cpu()
    for _, out in graphs:
        check_attention(out, c)


@pytest.mark.gpu
def test_attention_paged_of_nothing_and_through_the_registry(ops):
    import dpk_b200
    b = make([1, 40], [30, 9], 16, 4, 2, 64, BF, seed=22)
    d = cuda(b)
    got, meta = dpk_b200.run_kernel("attention_paged", d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"])
    check_attention(got, b)
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    out, _ = ops.attention_paged(d["q"][:0], d["k"], d["v"], d["table"], d["lens"], none)
    assert out.shape == (0, 4, 64)
    out, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], none)
    assert (out == 0).all()                                # every token is behind the last sequence
    out, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"][:0], d["lens"][:0], none[:1])
    assert (out == 0).all()
    inv, pos = torch.ones(32, device="cuda"), torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    assert ops.rope_append_paged(d["q"][:0], d["q"][:0, :2], d["q"][:0, :2], pos, inv, d["k"], d["v"], d["table"],
                                 d["lens"], none).shape == (0, 4, 64)
    assert torch.equal(d["k"].cpu(), b["k"])


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
def test_attention_paged_beside_other_work(ops, most):
    """Two calls at once on two streams, and calls that leave SMs to others."""
    from dpk_b200 import _native as N
    bs = [make([30, 2, 1] * 4, [700, 3, 90] * 4, 16, 8, 2, 128, BF, seed=23 + i) for i in range(2)]
    ds = [cuda(b) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                d = ds[i]
                outs[i].append(ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"],
                                                   max_query_len=most)[0])
    torch.cuda.synchronize()
    for i, b in enumerate(bs):
        check_attention(outs[i][0], b)
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])
    N.check(N.load().dpk_set_sm_margin(100))
    try:
        d = ds[0]
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
        check_attention(got, bs[0])
    finally:
        N.check(N.load().dpk_set_sm_margin(0))


@pytest.mark.gpu
def test_attention_paged_many_tiles_per_worker_and_many_parts_per_tile(ops):
    """600 sequences of a few tokens (several tiles per worker), then one sequence and one KV head over a
    long cache (every worker has a part of the one tile)."""
    new = [1 + i % 3 for i in range(600)]
    b = make(new, [i * 7 % 90 for i in range(600)], 8, 4, 2, 64, FP, seed=25)
    d = cuda(b)
    for most in (1, 3, 40):
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
        check_attention(got, b)
    b = make([3], [40000], 32, 8, 1, 64, BF, seed=26)
    d = cuda(b)
    for most in (1, 3):
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
        check_attention(got, b)


def test_attention_paged_is_registered():
    import dpk_b200
    assert dpk_b200.get_kernel("attention_paged", arch="sm100").backend == "b200"


@pytest.mark.gpu
def test_attention_paged_starts_that_do_not_ascend_are_reported(ops):
    """Overlapping and backward sequences: nothing outside the tensors is touched, and the status says so."""
    b = make([200, 150, 100], [20, 30, 40], 16, 8, 2, 64, BF, seed=21)
    d = cuda(b)
    mask = (torch.rand(450, 2, generator=b["gen"]) < 0.7).cuda()
    guard = torch.full((452, 8, 64), 5.0, dtype=BF, device="cuda")
    for start in ([0, 300, 100, 450], [0, 450, 0, 450], [450, 0, 450, 450], [-3, 200, 350, 450], [0, 200, 451, 450]):
        st = torch.tensor(start, dtype=torch.int32, device="cuda")
        for m in (mask, None):
            for most in (1, 200):
                ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], st, m, O=guard[1:451],
                                    max_query_len=most)
                assert ops.device_status() % 1000 == 105
    assert (guard[0] == 5).all() and (guard[451] == 5).all()


# ------------------------------------------------------------------------------------ rope (GPU)

ROPE = [
    # new, cached, page, Hq, Hk, D, R, axes, interleaved, dtype
    ([1], [0], 8, 1, 1, 64, 64, 1, False, BF),
    ([1, 1, 1], [15, 16, 17], 16, 32, 8, 128, 128, 3, False, BF),
    ([40, 1, 7], [3, 90, 0], 24, 6, 2, 64, 32, 2, True, FP),
    ([70, 0, 5], [0, 8, 11], 32, 3, 3, 128, 64, 3, True, BF),
    ([33], [100], 8, 64, 8, 128, 128, 2, False, FP),
    ([5, 6], [1, 2], 16, 2, 1, 96, 48, 3, False, BF),
    ([9], [0], 16, 1, 1, 32, 16, 1, False, FP),
    ([3, 2], [5, 0], 8, 2, 1, 768, 512, 2, False, BF),      # a head wider than a warp covers at once
    ([3, 2], [5, 0], 8, 3, 1, 1024, 272, 1, True, FP),
]


def rope_case(case, seed=0, far=0):
    new, cached, page, Hq, Hk, D, R, axes, near, dtype = ROPE[case]
    b = make(new, cached, page, Hq, Hk, D, dtype, seed=seed + case)
    n, g = b["q"].shape[0], b["gen"]
    b["kn"] = torch.randn(n, Hk, D, generator=g).to(dtype)
    b["vn"] = torch.randn(n, Hk, D, generator=g).to(dtype)
    b["pos"] = torch.randint(0, 1000, (axes, n), generator=g) + far
    half = R // 2
    b["inv"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float()
    b["sections"] = [half // axes + (a < half % axes) for a in range(axes)]
    b["axis"] = [a for a, m in enumerate(b["sections"]) for _ in range(m)]
    return b, near


def check_rotated(got, x, b, near, axis=None, scale=1.0):
    want, size = PO.rotate(x, b["pos"], b["inv"], axis or b["axis"], near, scale)
    tol = u_of(x.dtype) * want.abs() + 2.0 ** -20 * size + 2.0 ** -25
    assert ((got.cpu().double() - want).abs() <= tol).all()


def check_pages_written(d, b, new_k, new_v, k0, v0):
    """Every new token's row holds its k and v; every other row of the pools is what it was."""
    page = b["k"].shape[1]
    k, v = k0.clone(), v0.clone()
    start, lens = b["start"].tolist(), b["lens"].tolist()
    for s in range(len(lens)):
        for t in range(start[s], start[s + 1]):
            pos = lens[s] - start[s + 1] + t
            k[b["table"][s, pos // page], pos % page] = new_k[t]
            v[b["table"][s, pos // page], pos % page] = new_v[t]
    assert torch.equal(d["k"].cpu(), k) and torch.equal(d["v"].cpu(), v)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0, 3 * 10 ** 6])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_rope_append_paged(ops, case, far):
    b, near = rope_case(case, far=far)
    d = cuda(b)
    args = (d["pos"], d["inv"], d["k"], d["v"], d["table"], d["lens"], d["start"])
    q = ops.rope_append_paged(d["q"], d["kn"], d["vn"], *args, sections=b["sections"], interleaved=near)
    check_rotated(q, b["q"], b, near)
    assert torch.equal(d["q"].cpu(), b["q"])                       # the input is left alone
    q2, k2 = ops.rope_axes(d["q"], d["kn"], d["pos"], d["inv"], b["sections"], interleaved=near)
    check_rotated(k2, b["kn"], b, near)
    assert torch.equal(q2, q)
    check_pages_written(d, b, k2.cpu(), b["vn"], b["k"], b["v"])
    # in place, 32-bit positions, an axis per pair
    qi = d["q"].clone()
    amap = torch.tensor(b["axis"], dtype=torch.int32, device="cuda")
    out = ops.rope_append_paged(qi, d["kn"], d["vn"], d["pos"].int(), *args[1:], axis_map=amap, interleaved=near,
                                q_out=qi)
    assert out is qi and torch.equal(qi, q)


@pytest.mark.gpu
def test_rope_axes_alternating_axes_scale_and_strides(ops):
    b, _ = rope_case(4)
    d = cuda(b)
    half = len(b["inv"])
    axis = [i % 2 for i in range(half)]
    fused = torch.cat([d["q"].flatten(1), d["kn"].flatten(1), d["vn"].flatten(1)], 1).contiguous()
    n = fused.shape[0]
    q = fused[:, :64 * 128].view(n, 64, 128)
    k = fused[:, 64 * 128:72 * 128].view(n, 8, 128)
    v = fused[:, 72 * 128:].view(n, 8, 128)
    amap = torch.tensor(axis, dtype=torch.int32, device="cuda")
    qr, kr = ops.rope_axes(q, k, d["pos"], d["inv"], axis_map=amap, attention_scale=1.25)
    check_rotated(qr, b["q"], b, False, axis, 1.25)
    check_rotated(kr, b["kn"], b, False, axis, 1.25)
    out = ops.rope_append_paged(q, k, v, d["pos"], d["inv"], d["k"], d["v"], d["table"], d["lens"], d["start"],
                                axis_map=amap, attention_scale=1.25, q_out=q)
    assert torch.equal(out, qr) and torch.equal(fused[:, :64 * 128], qr.flatten(1))
    check_pages_written(d, b, kr.cpu(), b["vn"], b["k"], b["v"])


@pytest.mark.gpu
def test_rope_append_paged_rows_behind_the_last_sequence_and_bad_pages(ops):
    b, near = rope_case(1)
    d = cuda(b)
    start = torch.tensor([0, 1, 2, 2], dtype=torch.int32, device="cuda")     # the third sequence has none
    q0 = torch.full_like(d["q"], 3.0)
    ops.rope_append_paged(d["q"], d["kn"], d["vn"], d["pos"], d["inv"], d["k"], d["v"], d["table"], d["lens"], start,
                          sections=b["sections"], q_out=q0)
    assert (q0[2:] == 3).all()
    check_rotated(q0[:2], b["q"][:2], dict(b, pos=b["pos"][:, :2]), near)
    page_before = b["k"].clone()
    for bad in (-1, d["k"].shape[0]):
        d["k"].copy_(page_before)
        t = d["table"].clone()
        t[0, :] = bad
        ops.rope_append_paged(d["q"], d["kn"], d["vn"], d["pos"], d["inv"], d["k"], d["v"], t, d["lens"], d["start"],
                              sections=b["sections"])
        assert ops.device_status() == 15105
        row = b["table"][0, 0]
        assert torch.equal(d["k"].cpu()[row], page_before[row])


# ----------------------------------------------------------------------------------- pages (GPU)

class Cache:
    """GPU state beside the oracle's integers and a CPU copy of the pools."""

    def __init__(self, S, W, P, page, layers=2, Hk=2, D=64, dtype=BF, seed=0, wide=False):
        g = torch.Generator().manual_seed(seed)
        shape = (layers, P, page, Hk, D)
        self.kc, self.vc = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
        if wide:                                    # K and V of a page side by side in one pool
            both = torch.empty((layers, P, 2) + shape[2:], dtype=dtype, device="cuda")
            self.k, self.v = both[:, :, 0], both[:, :, 1]
            self.k.copy_(self.kc)
            self.v.copy_(self.vc)
        else:
            self.k, self.v = self.kc.cuda(), self.vc.cuda()
        self.books = PO.Pages([[-1] * W for _ in range(S)], [0] * S, [0] * P, page)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table, self.lens = torch.full((S, W), -1, **i32), torch.zeros(S, **i32)
        # an odd offset: the counts need not be 16-byte aligned
        self.refs = torch.zeros(P + 3, **i32)[3:]
        self.page = page

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def extend(self, ops, add):
        granted = ops.page_extend(self.k, self.v, self.table, self.lens, self.refs, self.ints(add))
        want, moves = self.books.extend(add)
        assert granted.tolist() == want
        for a, b, rows in moves:
            self.kc[:, b, :rows], self.vc[:, b, :rows] = self.kc[:, a, :rows], self.vc[:, a, :rows]
        return moves

    def fork(self, ops, parents, children):
        done = ops.page_fork(self.table, self.lens, self.refs, self.ints(parents), self.ints(children), self.page)
        want = self.books.fork(parents, children)
        assert done.tolist() == want
        return want

    def trim(self, ops, rows, keep=None):
        ops.page_trim(self.table, self.lens, self.refs, self.ints(rows), None if keep is None else self.ints(keep),
                      page_size=self.page)
        self.books.trim(rows, keep or [0] * len(rows))

    def compact(self, ops):
        live = ops.page_compact(self.k, self.v, self.table, self.lens, self.refs)
        want, moves = self.books.compact()
        assert live.tolist() == [want]
        for a, b in moves:
            self.kc[:, b], self.vc[:, b] = self.kc[:, a], self.vc[:, a]

    def same(self):
        assert self.table.tolist() == self.books.table
        assert self.lens.tolist() == self.books.lens
        assert self.refs.tolist() == self.books.refs
        assert torch.equal(self.k.cpu(), self.kc) and torch.equal(self.v.cpu(), self.vc)


@pytest.mark.gpu
@pytest.mark.parametrize("seed,S,W,P,page,wide", [(0, 6, 5, 14, 8, False), (1, 40, 6, 90, 16, True),
                                                  (2, 300, 4, 500, 8, False), (3, 9, 30, 70, 24, False)])
def test_pages_any_sequence_of_operators(ops, seed, S, W, P, page, wide):
    rng = random.Random(seed)
    c = Cache(S, W, P, page, seed=seed, wide=wide)
    reported = False
    for step in range(60):
        act = rng.choice(["extend", "extend", "extend", "fork", "fork", "trim", "compact"])
        if act == "extend":
            c.extend(ops, [rng.choice([0, 0, 1, 1, page, 2 * page + 3, -1, 3]) for _ in range(S)])
        elif act == "fork":
            empty = [s for s in range(S) if c.books.lens[s] == 0]
            kids = rng.sample(empty, min(len(empty), rng.randint(1, 6)))
            if rng.random() < 0.3:
                kids += [rng.randrange(S)]
            if kids:
                done = c.fork(ops, [rng.randrange(S) for _ in kids], kids)
                if not all(done):
                    assert ops.device_status() == 16105
                    reported = True
        elif act == "trim":
            n = rng.randint(1, max(1, S // 3))
            rows = [rng.randrange(S) for _ in range(n)]
            c.trim(ops, rows, None if rng.random() < 0.4 else [rng.randrange(W * page) for _ in range(n)])
        else:
            c.compact(ops)
        if step % 5 == 4 or S < 50:
            c.same()
    c.same()
    assert reported or seed != 1


@pytest.mark.gpu
def test_page_extend_all_holders_of_a_tail_write(ops):
    c = Cache(5, 4, 12, 8)
    c.extend(ops, [11, 0, 0, 0, 3])
    c.fork(ops, [0, 0], [2, 1])
    moves = c.extend(ops, [1, 1, 1, 0, 1])           # 3 holders, 3 writers: two copies, the first keeps it
    assert len(moves) == 2
    c.same()
    c.fork(ops, [4], [3])
    moves = c.extend(ops, [0, 0, 0, 1, 0])           # one of two holders writes
    assert len(moves) == 1
    c.same()
    # the pages do not last for the second copy: then the first holder may not keep the page either
    c = Cache(3, 4, 3, 8)
    c.extend(ops, [3, 0, 0])
    c.fork(ops, [0, 0], [1, 2])
    assert c.extend(ops, [1, 1, 14]) and c.books.lens == [3, 4, 3]
    c.same()


@pytest.mark.gpu
def test_page_operators_of_nothing(ops):
    c = Cache(3, 2, 4, 8)
    c.extend(ops, [0, 0, 0])
    c.compact(ops)
    c.trim(ops, [])
    c.fork(ops, [], [])
    ops.page_copy(c.k, c.v, c.ints([]), c.ints([]))
    c.extend(ops, [17, 16, 1])                       # two of the table's entries suffice for 16 tokens, not 17
    assert c.books.lens == [0, 16, 1]
    c.trim(ops, [1, 1, 0], [9, 0, 5])
    c.same()


@pytest.mark.gpu
def test_page_copy(ops):
    g = torch.Generator().manual_seed(4)
    for L, P, page, Hk, D, n in ((1, 9, 8, 1, 64, 4), (3, 200, 16, 8, 128, 90), (2, 40, 128, 8, 128, 15)):
        k, v = torch.randn(L, P, page, Hk, D, generator=g).to(FP), torch.randn(L, P, page, Hk, D, generator=g).to(FP)
        ids = torch.randperm(P, generator=g)
        src, dst = ids[:n].int(), ids[n:2 * n].int()
        kg, vg = k.cuda(), v.cuda()
        ops.page_copy(kg, vg, src.cuda(), dst.cuda())
        k[:, dst.long()], v[:, dst.long()] = k[:, src.long()], v[:, src.long()]
        assert torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)
    # one destination twice (the last counts), a page onto itself, a chain (left out), ids out of range
    k = torch.arange(10, dtype=torch.float32).view(10, 1, 1, 1).expand(10, 8, 1, 8).to(FP).contiguous().cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    v = k.clone()
    ops.page_copy(k, v, i32([1, 2, 3]), i32([5, 5, 3]))
    assert ops.device_status() == 0
    assert k[:, 0, 0, 0].tolist() == [0, 1, 2, 3, 4, 2, 6, 7, 8, 9] and torch.equal(k, v)
    ops.page_copy(k, v, i32([1, 8, 0, 10, 4]), i32([8, 9, 10, 6, -1]))
    assert ops.device_status() == 16105
    assert k[:, 0, 0, 0].tolist() == [0, 1, 2, 3, 4, 2, 6, 7, 1, 9]


@pytest.mark.gpu
def test_page_operators_report_bad_ids(ops):
    c = Cache(4, 3, 8, 8)
    c.extend(ops, [9, 3, 0, 0])
    c.table[0, 1] = 99
    ops.page_fork(c.table, c.lens, c.refs, c.ints([0]), c.ints([2]), 8)
    assert ops.device_status() == 16105
    ops.page_trim(c.table, c.lens, c.refs, c.ints([0, 77, -1, 1]), c.ints([0, 0, 0, -3]), page_size=8)
    assert ops.device_status() == 16105
    assert c.lens.tolist() == [0, 3, 9, 0]
    done = ops.page_fork(c.table, c.lens, c.refs, c.ints([9, 1, 1]), c.ints([3, 4, -1]), 8)
    assert ops.device_status() == 16105 and done.tolist() == [False, False, False]


@pytest.mark.gpu
def test_page_extend_many_pages_and_rows(ops):
    """More sequences than the cluster has threads, more pages than one step of its scan."""
    S, P, page = 9000, 40000, 8
    g = torch.Generator().manual_seed(8)
    c = Cache(S, 4, P, page, layers=1, Hk=1, D=8)
    refs = (torch.rand(P, generator=g) < 0.4).int()
    c.refs.copy_(refs)
    c.books.refs = refs.tolist()
    add = torch.randint(0, 30, (S,), generator=g).tolist()
    c.extend(ops, add)
    assert c.table.tolist() == c.books.table and c.refs.tolist() == c.books.refs and c.lens.tolist() == c.books.lens


# ----------------------------------------------------------------- the operators together (GPU)

@pytest.mark.gpu
def test_serving_run_over_a_paged_cache(ops):
    """Prompts in chunks, single tokens, forks, drafts that are refused, sequences that end, a compacted
    pool -- with the attention of every step checked against keys and values kept per sequence."""
    from dpk_b200.wide import PagedKVCache

    g = torch.Generator().manual_seed(31)
    rng = random.Random(31)
    S, L, Hq, Hk, D, NG, page = 6, 2, 8, 2, 64, 4, 8
    cache = PagedKVCache(L, 90, page, Hk, D, S, 200, BF, "cuda")
    inv = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    kept = [[([], []) for _ in range(L)] for _ in range(S)]       # per row and layer: keys, values
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lens = lambda: [len(kept[s][0][0]) for s in range(S)]

    def step(add):
        granted = cache.extend(i32(add)).tolist()
        add = [a if ok else 0 for a, ok in zip(add, granted)]
        starts = [0]
        for a in add:
            starts.append(starts[-1] + a)
        n = starts[-1]
        if n == 0:
            return granted
        base = lens()
        pos = torch.tensor([[base[s] + i for s in range(S) for i in range(add[s])],
                            [rng.randrange(40) for _ in range(n)]]).cuda()
        for layer in range(L):
            q, k, v = (torch.randn(n, h, D, generator=g).to(BF).cuda() for h in (Hq, Hk, Hk))
            mask = torch.rand(n, NG, generator=g) < 0.7
            kr = ops.rope_axes(q, k, pos, inv, (20, 12))[1].cpu()
            qr = cache.rope_update(layer, q, k, v, pos, inv, i32(starts), sections=(20, 12))
            out = cache.attend(layer, qr, i32(starts), mask.to(BF).cuda(), max_query_len=max(add))
            for s in range(S):
                for i in range(add[s]):
                    kept[s][layer][0].append(kr[starts[s] + i])
                    kept[s][layer][1].append(v[starts[s] + i].cpu())
                if add[s] == 0:
                    continue
                ks, vs = (torch.stack(t)[None] for t in kept[s][layer])          # one page per sequence
                a, b = starts[s], starts[s + 1]
                one = dict(q=qr[a:b].cpu(), k=ks, v=vs, table=torch.zeros(1, 1, dtype=torch.int32),
                           lens=torch.tensor([ks.shape[1]]), start=torch.tensor([0, b - a]))
                check_attention(out[a:b], one, mask[a:b])
        assert cache.lengths.tolist() == lens()
        return granted

    def fork(parents, children):
        assert cache.fork(i32(parents), i32(children)).all()
        for p, c in zip(parents, children):
            kept[c] = [(list(k), list(v)) for k, v in kept[p]]

    def trim(rows, keep):
        cache.trim(i32(rows), i32(keep))
        for s, n in zip(rows, keep):
            for k, v in kept[s]:
                del k[n:], v[n:]

    assert all(step([20, 33, 0, 0, 8, 0]))
    assert all(step([17, 1, 0, 0, 1, 0]))                # a chunk beside single tokens
    fork([0, 1, 0], [2, 3, 5])
    assert all(step([1] * 6))                            # everybody writes: tails are copied
    assert all(step([4] * 6))                            # drafts ...
    trim([0, 2, 3], [lens()[0] - 4, lens()[2] - 3, 11])  # ... refused, one far into what it shares
    assert all(step([1] * 6))
    cache.free(i32([1]))
    kept[1] = [([], []) for _ in range(L)]
    live = cache.compact()
    assert int(live) == int((cache.ref_counts > 0).sum()) and (cache.ref_counts[int(live):] == 0).all()
    assert all(step([2, 50, 1, 1, 1, 1]))
    assert not all(step([100, 100, 100, 150, 150, 150]))  # more than the pool has
    step([1] * 6)
    cache.free(i32(list(range(S))))
    assert (cache.ref_counts == 0).all() and (cache.page_table == -1).all()


@pytest.mark.gpu
def test_decoder_layer_over_a_paged_cache(ops):
    """RoutedDecoderLayer.forward_cached: two sequences in chunks of many and of single tokens, against the
    oracle composition of each whole sequence with the masks that the layer decided."""
    from dpk_b200.layer import RoutedDecoderLayer
    from dpk_b200.wide import PagedKVCache
    from oracle import dpk_oracle as O

    g = torch.Generator().manual_seed(43)
    H, Hq, Hk, D, I, NGF, R = 256, 8, 2, 64, 1024, 8, 16
    r16 = lambda t: t.to(BF).float()
    rand = lambda *shape, std=1.0: r16(torch.randn(*shape, generator=g) * std)
    ws = {n: rand(*shp, std=0.05) for n, shp in dict(wq=(Hq * D, H), wk=(Hk * D, H), wv=(Hk * D, H),
                                                     wo=(H, Hq * D), wg=(I, H), wu=(I, H), wd=(H, I)).items()}
    router = lambda ng: (rand(R, H, std=H ** -0.5), rand(R, std=0.1), rand(2 * ng, R, std=R ** -0.5), rand(2 * ng, std=0.1))
    ra, rf = router(Hk), router(NGF)
    n1, n2 = r16(1 + 0.1 * torch.randn(H, generator=g)), r16(1 + 0.1 * torch.randn(H, generator=g))
    gpu = lambda t: t.to(BF).cuda()
    layer = RoutedDecoderLayer(*(gpu(ws[n]) for n in ("wq", "wk", "wv", "wo", "wg", "wu", "wd")), num_q_heads=Hq,
                               num_kv_heads=Hk, head_dim=D, attn_groups=Hk, ffn_groups=NGF, max_tokens=400)
    layer.set_front_end(tuple(map(gpu, ra)), tuple(map(gpu, rf)), gpu(n1), gpu(n2), 1e-5)
    cache = PagedKVCache(3, 60, 16, Hk, D, 2, 320, BF, "cuda")
    inv = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float()
    xs = [rand(190, H), rand(131, H)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    outs, masks = [[], []], [[], []]
    at = [0, 0]
    for add in ([150, 0], [30, 129], [1, 1], [9, 1]):
        assert cache.extend(i32(add)).all()
        x = torch.cat([xs[s][at[s]:at[s] + add[s]] for s in range(2)])
        pos = torch.tensor([at[s] + i for s in range(2) for i in range(add[s])])
        out, am, fm = layer.forward_cached(gpu(x), pos.cuda(), inv.cuda(), cache, 1, i32([0, add[0], sum(add)]),
                                           max_query_len=max(add), return_masks=True)
        for s in range(2):
            a = sum(add[:s])
            outs[s].append(out[a:a + add[s]].float().cpu())
            masks[s].append((am[a:a + add[s]].cpu(), fm[a:a + add[s]].cpu()))
            at[s] += add[s]
    for s in range(2):
        T = xs[s].shape[0]
        x, am, fm = xs[s][None], torch.cat([m[0] for m in masks[s]])[None], torch.cat([m[1] for m in masks[s]])[None]
        axis = [0] * (D // 2)
        pos = torch.arange(T)
        turn = lambda t: r16(PO.rotate(t, pos, inv, axis)[0].float())
        h = O.rms_norm(x.to(BF), n1, 1e-5).float()
        q = turn(r16(O.gemm_mn(h, ws["wq"], am)).view(T, Hq, D))[None]
        k = turn(r16(h @ ws["wk"].T).view(T, Hk, D))[None]
        v = r16(h @ ws["wv"].T).view(1, T, Hk, D)
        a = r16(O.attention_prefill(q, k, v, am)).view(1, T, Hq * D)
        x1 = r16(x + r16(O.gemm_k(a, ws["wo"], am)))
        h2 = O.rms_norm(x1.to(BF), n2, 1e-5).float()
        want = x1 + O.ffn_swiglu(h2, ws["wg"], ws["wu"], ws["wd"], fm, round_intermediate=BF)
        # the tolerance of the same chain without a cache (test_routed_decoder_layer_full_front_end)
        assert O.rel_err(torch.cat(outs[s])[None], want) <= 3e-2
    assert ops.device_status() == 0


@pytest.mark.gpu
def test_decode_step_in_one_graph(ops):
    """extend, rotary write and attention captured together: every replay is one more token."""
    from dpk_b200.wide import PagedKVCache

    g = torch.Generator().manual_seed(51)
    S, Hq, Hk, D, page = 3, 4, 2, 64, 8
    cache = PagedKVCache(1, 30, page, Hk, D, S, 64, BF, "cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    add, start = i32([1] * S), i32(list(range(S + 1)))
    q, k, v = (torch.zeros(S, h, D, dtype=BF, device="cuda") for h in (Hq, Hk, Hk))
    inv = torch.ones(D // 2, device="cuda")

    def step():
        cache.extend(add)
        qr = cache.rope_update(0, q, k, v, (cache.lengths - 1)[None], inv, start)
        return qr, cache.attend(0, qr, start, max_query_len=1)
    step()
    cache.free(i32(list(range(S))))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = step()
    keys, values = [[] for _ in range(S)], [[] for _ in range(S)]
    for n in range(1, 21):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == [n] * S
        kr = ops.rope_axes(q, k, torch.full((1, S), n - 1, device="cuda"), inv)[1].cpu()
        for s in range(S):
            keys[s].append(kr[s])
            values[s].append(v[s].cpu())
            one = dict(q=qr[s:s + 1].cpu(), k=torch.stack(keys[s])[None], v=torch.stack(values[s])[None],
                       table=torch.zeros(1, 1, dtype=torch.int32), lens=torch.tensor([n]), start=torch.tensor([0, 1]))
            check_attention(out[s:s + 1], one)
