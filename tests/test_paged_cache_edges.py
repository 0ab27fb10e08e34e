"""The paged-cache operators at the edges of what a call may hold: values that are no numbers, starts that make no
sense, sequences that got no room, counts that disagree with tables, tensors off their alignment, empty states,
buffers of captured steps, the rarer dispatch paths and pools beyond 2^31 elements.

Tolerances are those of ``test_paged_cache`` (64-bit and integer oracles, roundings counted per element)."""

import math

import pytest
import torch

from oracle import paged_oracle as PO
from test_paged_cache import BF, FP, Cache, check_attention, check_rotated, cuda, make, rope_case, u_of


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


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def poison(like, value):
    """Leaves ``value`` in memory that the allocator hands out again for tensors of this size."""
    held = [torch.full_like(like, value) for _ in range(4)]
    torch.cuda.synchronize()
    del held


# ------------------------------------------------------------------ values that are no numbers (GPU)

def check_not_numbers(got, b, mask=None, q=None):
    """NaN exactly where the 64-bit form has it; the other rows within the bounds of ``check_attention``."""
    q = b["q"] if q is None else q
    want, size = PO.attention(q, b["k"], b["v"], b["table"], b["lens"], b["start"], mask)
    got, lost = got.detach().cpu().double(), want.isnan()
    assert torch.equal(got.isnan(), lost)
    u = u_of(b["q"].dtype)
    tol = u * want.abs() + (u + 2.0 ** -13) * size + 2.0 ** -25
    assert ((got - want).abs() <= tol)[~lost].all()
    return lost


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
@pytest.mark.parametrize("cached", [20, 40000])      # a tile of one worker; a part of it with every worker
def test_attention_paged_nan_query(ops, cached, most):
    b = make([3], [cached], 32, 8, 2, 64, BF, seed=41)
    mask = torch.ones(3, 8, dtype=torch.bool)
    mask[2, 3] = False
    clean = b["q"].clone()
    clean[1, 5] = math.nan
    b["q"][1, 5] = b["q"][2, 3] = math.nan           # the second one is routed out
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], mask.cuda(),
                                 max_query_len=most)
    lost = check_not_numbers(got, b, mask, clean)
    assert lost[1, 5].all() and int(lost.sum()) == 64 and (got[2, 3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
@pytest.mark.parametrize("first,last", [(0, 6000), (17000, 17001), (12000, 40001)])
def test_attention_paged_nan_keys(ops, first, last, most):
    """A stretch of NaN keys over several workers' ranges, one key, and the keys up to the second token."""
    b = make([4], [40000], 32, 8, 2, 64, BF, seed=42)
    for pos in range(first, last):
        b["k"][b["table"][0, pos // 32], pos % 32, 0] = math.nan
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    lost = check_not_numbers(got, b)
    assert lost[:, :4].all() and not lost[:, 4:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
def test_attention_paged_nan_keys_up_to_a_workers_border(ops, most):
    """A stretch of NaN keys that ends after every unit in turn: with the first worker's range too."""
    b = make([4], [40000], 32, 8, 2, 64, BF, seed=42)
    d = cuda(b)
    for unit in range(60):
        d["k"][d["table"][0, unit].long(), :, 0] = math.nan
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
        lost = got.isnan()
        assert lost[:, :4].all() and not lost[:, 4:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
def test_attention_paged_nan_key_of_a_later_token(ops, most):
    b = make([4, 2], [30, 0], 16, 8, 2, 128, FP, seed=43)
    b["k"][b["table"][0, 32 // 16], 32 % 16, 1] = math.nan          # the third new token's
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    lost = check_not_numbers(got, b)
    assert lost[2:4, 4:].all() and int(lost.sum()) == 2 * 4 * 128


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 64])
@pytest.mark.parametrize("cached", [20, 40000])
def test_attention_paged_infinite_scores(ops, cached, most):
    """Scores of -inf alone leave no weights (NaN); beside a finite one they weigh nothing; +inf is NaN."""
    b = make([2], [cached], 32, 6, 3, 64, BF, seed=44)
    b["q"] = b["q"].abs() + 0.25
    b["k"][:, :, 0] = -math.inf
    b["k"][:, :, 1] = -math.inf
    b["k"][b["table"][0, 0], 5, 1] = 0.5
    b["k"][b["table"][0, 0], 7, 2] = math.inf
    d = cuda(b)
    got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
    lost = check_not_numbers(got, b)
    assert lost[:, :2].all() and not lost[:, 2:4].any() and lost[:, 4:].all()


# ------------------------------------------------------------------ starts that make no sense (GPU)

STARTS = [
    # starts, rows of q
    ([0, 5], 1),                # one sequence that ends behind the tensors
    ([2, 3, 5], 5),             # tokens before the first sequence
    ([-3, 2, 4], 4),
    ([0, 2, 9], 4),
    ([0, 4, 99], 4),            # the second sequence has no row at all
    ([0, 5, 3, 8], 8),          # backwards, and two sequences that overlap
    ([0, -1], 2),
    ([6, 2, 4], 6),
]


def owned(start, n):
    """Tokens that a sequence whose range makes sense names."""
    return {t for a, b in zip(start, start[1:]) if 0 <= a <= b <= n for t in range(a, b)}


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(STARTS)))
def test_rope_append_paged_bad_starts(ops, case):
    """Only the new tokens' places of sequences whose range makes sense are written, and the status says so."""
    start, n = STARTS[case]
    S, page, D = len(start) - 1, 8, 64
    lens = [20 + 3 * s for s in range(S)]
    b = make([0] * S, lens, page, 2, 2, D, BF, seed=45)
    g = b["gen"]
    q, k, v = (torch.randn(n, 2, D, generator=g).to(BF) for _ in range(3))
    pos = torch.arange(n)[None]
    inv = torch.ones(D // 2)
    d = cuda(b)
    dk, dv, dpos = k.cuda(), v.cuda(), pos.cuda()
    ops.rope_append_paged(q.cuda(), dk, dv, dpos, inv.cuda(), d["k"], d["v"], d["table"], d["lens"], i32(start))
    assert ops.device_status() == 15105
    kr = ops.rope_axes(q.cuda(), dk, dpos, inv.cuda())[1].cpu()
    free = torch.zeros(b["k"].shape[:2], dtype=torch.bool)
    for s, (a, e) in enumerate(zip(start, start[1:])):
        if not 0 <= a <= e <= n:
            continue
        for t in range(a, e):
            at = lens[s] - (e - t)
            place = (int(b["table"][s, at // page]), at % page)
            free[place] = True
            if sum(x <= t < y for x, y in zip(start, start[1:]) if 0 <= x <= y <= n) == 1 and start == sorted(start):
                assert torch.equal(d["k"][place].cpu(), kr[t]) and torch.equal(d["v"][place].cpu(), v[t])
    assert torch.equal(d["k"].cpu()[~free], b["k"][~free]) and torch.equal(d["v"].cpu()[~free], b["v"][~free])


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("most", [1, 64])
@pytest.mark.parametrize("case", range(len(STARTS)))
def test_attention_paged_bad_starts(ops, case, most, masked):
    """Rows that no sequence names are zero in a new output and left alone in a given one."""
    start, n = STARTS[case]
    S = len(start) - 1
    b = make([0] * S, [20 + 3 * s for s in range(S)], 8, 4, 2, 64, BF, seed=46)
    q = torch.randn(n, 4, 64, generator=b["gen"]).to(BF).cuda()
    mask = torch.ones(n, 2, dtype=torch.bool, device="cuda") if masked else None
    d = cuda(b)
    other = [t for t in range(n) if t not in owned(start, n)]
    poison(q, 7.0)
    got, _ = ops.attention_paged(q, d["k"], d["v"], d["table"], d["lens"], i32(start), mask, max_query_len=most)
    assert ops.device_status() % 1000 == 105
    assert (got[other] == 0).all() and torch.isfinite(got).all() and not (got == 7).any()
    mine = torch.full_like(q, 7.0)
    ops.attention_paged(q, d["k"], d["v"], d["table"], d["lens"], i32(start), mask, O=mine, max_query_len=most)
    assert ops.device_status() % 1000 == 105
    assert (mine[other] == 7).all()
    if start == sorted(start):
        mine[other] = 0
        assert torch.equal(mine, got)


# ------------------------------------------------------------------ sequences that got no room (GPU)

@pytest.mark.gpu
def test_rope_append_paged_leaves_refused_sequences_alone(ops):
    b, near = rope_case(1)
    d = cuda(b)
    granted = torch.tensor([True, False, True], device="cuda")
    q = ops.rope_append_paged(d["q"], d["kn"], d["vn"], d["pos"], d["inv"], d["k"], d["v"], d["table"], d["lens"],
                              d["start"], sections=b["sections"], granted=granted)
    check_rotated(q, b["q"], b, near)                 # the queries are turned all the same
    kr = ops.rope_axes(d["q"], d["kn"], d["pos"], d["inv"], b["sections"])[1].cpu()
    k, v = b["k"].clone(), b["v"].clone()
    for s in (0, 2):
        at = int(b["lens"][s]) - 1
        place = (int(b["table"][s, at // 16]), at % 16)
        k[place], v[place] = kr[s], b["vn"][s]
    assert torch.equal(d["k"].cpu(), k) and torch.equal(d["v"].cpu(), v)
    for bad in (granted.int(), granted[:2], granted.cpu()):
        with pytest.raises(ValueError):
            ops.rope_append_paged(d["q"], d["kn"], d["vn"], d["pos"], d["inv"], d["k"], d["v"], d["table"],
                                  d["lens"], d["start"], sections=b["sections"], granted=bad)


@pytest.mark.gpu
def test_decode_step_in_one_graph_with_a_pool_that_runs_out(ops):
    """A captured step brings a token for every row.  A refused row's tokens change nothing that is cached, not
    in pages that it shares either, and it goes on where it stopped once there is room."""
    from dpk_b200.wide import PagedKVCache

    g = torch.Generator().manual_seed(52)
    S, Hq, Hk, D, page = 4, 4, 2, 64, 8
    cache = PagedKVCache(1, 6, page, Hk, D, S, 64, BF, "cuda")
    add, start = i32([1] * S), i32(list(range(S + 1)))
    q, k, v = (torch.zeros(S, h, D, dtype=BF, device="cuda") for h in (Hq, Hk, Hk))
    inv = torch.ones(D // 2, device="cuda")

    def step():
        granted = cache.extend(add)
        qr = cache.rope_update(0, q, k, v, cache.lengths[None], inv, start)
        return granted, qr, cache.attend(0, qr, start, max_query_len=1)
    step()
    cache.free(i32(list(range(S))))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        granted, qr, out = step()
    keys, values = [[] for _ in range(S)], [[] for _ in range(S)]
    refused = 0

    def replay():
        nonlocal refused
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        lens, table, ok = cache.lengths.tolist(), cache.page_table.tolist(), granted.tolist()
        kr = ops.rope_axes(q, k, cache.lengths[None], inv)[1].cpu()
        for s in range(S):
            if ok[s]:
                keys[s].append(kr[s])
                values[s].append(v[s].cpu())
            refused += not ok[s]
            assert lens[s] == len(keys[s])
            for j in range(lens[s]):
                place = (0, table[s][j // page], j % page)
                assert torch.equal(cache.keys[place].cpu(), keys[s][j])
                assert torch.equal(cache.values[place].cpu(), values[s][j])
            if ok[s]:
                one = dict(q=qr[s:s + 1].cpu(), k=torch.stack(keys[s])[None], v=torch.stack(values[s])[None],
                           table=torch.zeros(1, 1, dtype=torch.int32), lens=torch.tensor([lens[s]]),
                           start=torch.tensor([0, 1]))
                check_attention(out[s:s + 1], one)

    for _ in range(14):                               # 4 rows of pages of 8 in a pool of 6
        replay()
    assert refused >= 4
    cache.free(i32([3]))                              # one page is free: row 2 takes it, and rows 0 and 3, which
    assert cache.fork(i32([0]), i32([3])).all()       # share a partly filled page, cannot write to it
    keys[3], values[3] = list(keys[0]), list(values[0])
    for _ in range(2):
        replay()
        assert granted.tolist() == [False, True, True, False]
    cache.free(i32([1]))
    keys[1], values[1] = [], []
    replay()
    assert granted.tolist() == [True] * 4


# ------------------------------------------------------------------ counts that disagree (GPU)

@pytest.mark.gpu
def test_page_compact_reports_entries_of_pages_that_nobody_holds(ops):
    from dpk_b200 import _native as N
    c = Cache(4, 3, 8, 8)
    c.extend(ops, [9, 3, 0, 0])                       # pages 0, 1 and 2
    c.trim(ops, [0])                                  # page 2 is the only one left
    c.table[2, 0], c.lens[2] = 6, 5                   # behind the pages that stay, held by nobody
    c.table[3, 0], c.lens[3] = 0, 5                   # the hole that page 2 moves to
    poison(torch.empty((N.load().dpk_page_workspace_bytes(0, 8, 0) + 3) // 4, dtype=torch.int32, device="cuda"), 3)
    live = ops.page_compact(c.k, c.v, c.table, c.lens, c.refs)
    assert ops.device_status() == 16105
    assert live.tolist() == [1] and c.refs.tolist() == [1] + [0] * 7
    assert c.table.tolist() == [[-1] * 3, [0, -1, -1], [-1] * 3, [-1] * 3]
    assert torch.equal(c.k[:, 0].cpu(), c.kc[:, 2]) and torch.equal(c.v[:, 0].cpu(), c.vc[:, 2])


# ------------------------------------------------------------------ alignment (GPU)

def shifted(t):
    """The same values, contiguous, one element off an aligned address."""
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    room[1:] = t.cuda().flatten()
    return room[1:].view(t.shape)


@pytest.mark.gpu
def test_paged_operators_take_unaligned_queries_keys_and_values(ops):
    b, near = rope_case(4)
    d = cuda(b)
    state = (d["k"], d["v"], d["table"], d["lens"], d["start"])
    q = ops.rope_append_paged(shifted(b["q"]), shifted(b["kn"]), shifted(b["vn"]), d["pos"], d["inv"], *state,
                              sections=b["sections"])
    check_rotated(q, b["q"], b, near)
    wrote = d["k"].clone(), d["v"].clone()
    q2, k2 = ops.rope_axes(shifted(b["q"]), shifted(b["kn"]), d["pos"], d["inv"], b["sections"])
    assert torch.equal(q2, q)
    # k and v of different strides, one of them off its alignment
    n = b["q"].shape[0]
    wide = torch.zeros(n, 8 * 128 + 64, dtype=FP, device="cuda")
    wide[:, :1024] = d["vn"].flatten(1)
    for x in (d["k"], d["v"]):
        x.zero_()
    for s, t in (("k", b["k"]), ("v", b["v"])):
        d[s].copy_(t)
    ops.rope_append_paged(d["q"], shifted(b["kn"]), wide[:, :1024].view(n, 8, 128), d["pos"], d["inv"], *state,
                          sections=b["sections"])
    assert torch.equal(d["k"], wrote[0]) and torch.equal(d["v"], wrote[1])
    at = b["lens"][0] - n
    assert torch.equal(d["k"][b["table"][0, at // 8].long(), at % 8], k2[0])
    a = make([3, 2], [30, 9], 16, 4, 2, 64, BF, seed=47)
    e = cuda(a)
    got, _ = ops.attention_paged(shifted(a["q"]), e["k"], e["v"], e["table"], e["lens"], e["start"])
    check_attention(got, a)


# ------------------------------------------------------------------ empty states (GPU)

@pytest.mark.gpu
@pytest.mark.parametrize("S,W,P", [(0, 4, 6), (3, 0, 6), (3, 4, 0), (0, 0, 0), (0, 4, 0), (3, 0, 0)])
def test_paged_operators_of_empty_states(ops, S, W, P):
    k = torch.zeros(2, P, 8, 2, 64, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    table = torch.full((S, W), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.zeros(P, dtype=torch.int32, device="cuda")
    none = i32([])
    granted = ops.page_extend(k, v, table, lens, refs, torch.zeros_like(lens))
    assert granted.dtype is torch.bool and granted.tolist() == [True] * S
    granted = ops.page_extend(k, v, table, lens, refs, torch.ones_like(lens))
    assert granted.tolist() == [False] * S and lens.tolist() == [0] * S
    assert ops.page_compact(k, v, table, lens, refs).tolist() == [0]
    ops.page_trim(table, lens, refs, torch.arange(S, dtype=torch.int32, device="cuda"), page_size=8)
    ops.page_trim(table, lens, refs, none, page_size=8)
    assert ops.page_fork(table, lens, refs, none, none, 8).shape == (0,)
    ops.page_copy(k, v, none, none)
    assert ops.device_status() == 0
    if P == 0:
        ops.page_copy(k, v, i32([0]), i32([1]))
        assert ops.device_status() == 16105
    if S == 0:
        ops.page_trim(table, lens, refs, i32([0]), page_size=8)
        assert ops.device_status() == 16105
        assert ops.page_fork(table, lens, refs, i32([0]), i32([1]), 8).tolist() == [False]
        assert ops.device_status() == 16105
    # no token is cached: every row sees nothing
    n = max(S, 1)
    start = i32(list(range(S + 1)))
    q = torch.ones(n, 4, 64, dtype=BF, device="cuda")
    for most in (1, 64):
        poison(q, 7.0)
        out, _ = ops.attention_paged(q, k[0], v[0], table, lens, start, max_query_len=most)
        assert (out == 0).all() and ops.device_status() == 0
    # a token without a place in the pages is reported, its query turned all the same
    pos, inv = torch.zeros(1, n, dtype=torch.int64, device="cuda"), torch.ones(32, device="cuda")
    out = ops.rope_append_paged(q, q[:, :2], q[:, :2], pos, inv, k[0], v[0], table, lens, start)
    if S:
        assert torch.equal(out, q) and ops.device_status() == 15105
        lens.fill_(5)                                  # lengths that the state cannot hold
        for most in (1, 64):
            out, _ = ops.attention_paged(q, k[0], v[0], table, lens, start, max_query_len=most)
            assert (out == 0).all() and ops.device_status() % 1000 == 105


# ------------------------------------------------------------------ a layer's captured steps (GPU)

def small_layer(seed=61, max_tokens=300):
    from dpk_b200.layer import RoutedDecoderLayer

    g = torch.Generator().manual_seed(seed)
    H, Hq, Hk, D, I, NGF, R = 256, 8, 2, 64, 1024, 8, 16
    rand = lambda *shape, std=0.05: (torch.randn(*shape, generator=g) * std).to(BF).cuda()
    layer = RoutedDecoderLayer(rand(Hq * D, H), rand(Hk * D, H), rand(Hk * D, H), rand(H, Hq * D), rand(I, H),
                               rand(I, H), rand(H, I), num_q_heads=Hq, num_kv_heads=Hk, head_dim=D, attn_groups=Hk,
                               ffn_groups=NGF, max_tokens=max_tokens)
    router = lambda ng: (rand(R, H), rand(R, std=0.1), rand(2 * ng, R, std=0.25), rand(2 * ng, std=0.1))
    layer.set_front_end(router(Hk), router(NGF), torch.ones(H, dtype=BF, device="cuda"),
                        torch.ones(H, dtype=BF, device="cuda"), 1e-5)
    return layer, g


def alike(layer, a, b):
    """Two outputs of ``layer`` on the same input.  Its down projection adds up to 8 parts of a sum to one 32-bit
    accumulator in any order, and the residual: 9 additions, each off by 2^-24 of what is summed at most, before
    one rounding to 16 bits.  (The output projection's two parts give the same bits in either order.)  What is summed
    is below sum_i |wd_i| |g_i| |u_i| with |silu(g) u| <= |g| |u|, |g| <= |wg_i| |h|, |u| <= |wu_i| |h|, and |h| = sqrt(256)
    of the normed input within its own rounding."""
    f = layer.ffn
    most = f.wd.float().abs() @ (f.wg.float().norm(dim=1) * f.wu.float().norm(dim=1)) * 256 * (1 + 2.0 ** -6)
    size = torch.maximum(a.float().abs(), b.float().abs())
    return bool(((a.float() - b.float()).abs() <= 2 * 9 * 2.0 ** -24 * (2 * most + size) + 2 * u_of(BF) * size).all())


def new_cache(rows=3):
    from dpk_b200.wide import PagedKVCache
    return PagedKVCache(1, 80, 16, 2, 64, rows, 320, BF, "cuda")


@pytest.mark.gpu
def test_forward_cached_captured_step_owns_its_buffers(ops):
    """A step captured for a few tokens, then a larger one that is not captured, then the captured one again:
    what the larger step left behind and what others allocated meanwhile stays as it is."""
    layer, g = small_layer()
    cache, twin = new_cache(), new_cache()
    inv = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    x1 = torch.randn(3, 256, generator=g).to(BF).cuda()
    x2 = torch.randn(280, 256, generator=g).to(BF).cuda()
    one, start1 = i32([1, 1, 1]), i32([0, 1, 2, 3])
    many, start2 = i32([200, 0, 80]), i32([0, 200, 200, 280])
    pos2 = torch.cat([torch.arange(200), torch.arange(80)]).cuda() + 1

    def step(c, x, add, start, pos, most):
        c.extend(add)
        return layer.forward_cached(x, c.lengths - 1 if pos is None else pos, inv, c, 0, start, max_query_len=most)
    step(twin, x1, one, start1, None, 1)              # loads what is loaded at first use
    twin.free(i32([0, 1, 2]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache, x1, one, start1, None, 1)
    graph.replay()
    a1 = out.clone()
    a2 = step(cache, x2, many, start2, pos2, 200)
    others = [torch.full((n,), 5.0, dtype=BF, device="cuda") for n in (3 * 768, 3 * 512, 4096, 280 * 768, 280 * 512)
              for _ in range(6)]
    graph.replay()
    a3 = out.clone()
    torch.cuda.synchronize()
    assert all((t == 5).all() for t in others)
    b1 = step(twin, x1, one, start1, None, 1)
    b2 = step(twin, x2, many, start2, pos2, 200)
    b3 = step(twin, x1, one, start1, None, 1)
    assert alike(layer, a1, b1) and alike(layer, a2, b2) and alike(layer, a3, b3)


@pytest.mark.gpu
def test_forward_cached_rows_behind_the_last_sequence(ops):
    """A padded step: the rows behind the last sequence get no attention, whatever memory held before."""
    layer, g = small_layer()
    inv = torch.ones(32, device="cuda")
    x = torch.randn(9, 256, generator=g).to(BF).cuda()
    pos = torch.zeros(9, dtype=torch.int64, device="cuda")
    outs = []
    for value in (math.nan, 3.0):
        cache = new_cache()
        cache.extend(i32([2, 0, 3]))
        for width in (9 * 512, 9 * 768):
            poison(torch.empty(width, dtype=BF, device="cuda"), value)
        if getattr(layer, "_attn_out", None) is not None:
            layer._attn_out.fill_(value)
        outs.append(layer.forward_cached(x, pos, inv, cache, 0, i32([0, 2, 2, 5]), max_query_len=3))
    assert torch.isfinite(outs[0]).all() and alike(layer, outs[0], outs[1])


@pytest.mark.gpu
def test_forward_cached_without_a_token(ops):
    layer, _ = small_layer()
    cache = new_cache()
    assert cache.extend(i32([0, 0, 0])).all()
    x, pos = torch.zeros(0, 256, dtype=BF, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    args = (x, pos, torch.ones(32, device="cuda"), cache, 0, i32([0, 0, 0, 0]))
    assert layer.forward_cached(*args).shape == (0, 256)
    for which in (True, "full"):
        out, am, fm = layer.forward_cached(*args, return_masks=which)
        assert out.shape == (0, 256) and am.shape == (0, 2) and fm.shape == (0, 8)
    assert (cache.ref_counts == 0).all()


# ------------------------------------------------------------------ bounds of arguments

@pytest.mark.gpu
def test_attention_paged_any_upper_bound_of_new_tokens(ops):
    b = make([3, 40], [30, 9], 16, 4, 2, 64, BF, seed=48)
    d = cuda(b)
    want, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=43)
    for most in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 40):
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"], max_query_len=most)
        assert torch.equal(got, want)


def test_attention_paged_refuses_work_near_the_end_of_32_bits(ops):
    """A worker's range ends at most a few ten thousand places behind the line's end, which has to fit too."""
    import ctypes

    from dpk_b200 import _native as N
    lib = N.load()
    buf = (ctypes.c_uint8 * 512)()
    p = (ctypes.addressof(buf) + 255) & ~255
    # 8 heads, S sequences of one token: 8 * (S + S // 16) tiles of W * 8 / 32 + 1 places
    S, W = 496, 4 * 509355                              # 4216 tiles of 509355 + 1 places: 2^31 - 39 thousand
    tiles = 8 * (S // 16 + S)
    places = tiles * ((W * 8 + 31) // 32 + 1)
    assert 2 ** 31 - 2 ** 16 <= places < 2 ** 31
    rc = lib.dpk_attn_paged(p, p, p, p, p, p, None, p, S, S, W, 8, 8, 8, 8, 64, 1, 0.1, 1, N.BF16, 1, 0, 0, 0, 0, 0, p, 0,
                            None)
    assert rc == N.ERR_INVALID and "too much work" in N.last_error()


# ------------------------------------------------------------------ rarer dispatch paths (GPU)

@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
def test_attention_paged_more_pairs_than_shared_memory_holds(ops, masked):
    """600 sequences of 8 KV heads: the tiles' numbers are in the workspace."""
    new = [1 + i % 2 for i in range(600)]
    b = make(new, [i * 5 % 23 for i in range(600)], 8, 8, 8, 64, BF, seed=49)
    mask = torch.rand(b["q"].shape[0], 4, generator=b["gen"]) < 0.6 if masked else None
    d = cuda(b)
    for most in (2, 40):
        got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"],
                                     None if mask is None else mask.cuda(), max_query_len=most)
        check_attention(got, b, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rep,D,dtype", [(17, 64, BF), (32, 128, FP), (128, 64, BF)])
def test_attention_paged_many_query_heads_per_kv_head(ops, rep, D, dtype, masked):
    """More rows a token than the warp kernel's tile has: single tokens go to the chunk kernel."""
    for new, cached in (([1, 1, 1], [70, 0, 333]), ([5, 1, 20], [9, 64, 200])):
        b = make(new, cached, 16, 2 * rep, 2, D, dtype, seed=50 + rep)
        mask = torch.rand(sum(new), 2 * rep, generator=b["gen"]) < 0.5 if masked else None
        d = cuda(b)
        for most in (1, max(new)):
            got, _ = ops.attention_paged(d["q"], d["k"], d["v"], d["table"], d["lens"], d["start"],
                                         None if mask is None else mask.cuda(), max_query_len=most)
            check_attention(got, b, mask)


# ------------------------------------------------------------------ pools beyond 2^31 elements (GPU)

@pytest.mark.gpu
def test_rope_and_pages_offsets_beyond_32_bits(ops):
    """Writes, copies and moves between pages 4.4 GB apart in one pool of two-byte elements."""
    page, Hk, D = 16, 2, 128
    P = 2 ** 31 // (page * Hk * D) + 8
    k = torch.zeros(P, page, Hk, D, dtype=BF, device="cuda")
    v = torch.zeros(P, page, Hk, D, dtype=BF, device="cuda")
    g = torch.Generator().manual_seed(62)
    q, kn, vn = (torch.randn(3, h, D, generator=g).to(BF).cuda() for h in (4, Hk, Hk))
    # three tokens: in the last page, in the first one, across the border of two far pages
    table, lens, start = i32([[P - 1, -1], [0, -1], [1, P - 3]]), i32([4, 9, 17]), i32([0, 1, 2, 3])
    pos = torch.arange(3, device="cuda")[None]
    inv = torch.ones(D // 2, device="cuda")
    ops.rope_append_paged(q, kn, vn, pos, inv, k, v, table, lens, start)
    kr = ops.rope_axes(q, kn, pos, inv)[1]
    places = [(P - 1, 3), (0, 8), (P - 3, 0)]
    for t, at in enumerate(places):
        assert torch.equal(k[at], kr[t]) and torch.equal(v[at], vn[t])
        k[at], v[at] = 0, 0
    assert not k.any() and not v.any()
    for at in places:
        k[at], v[at] = 1, 2
    ops.page_copy(k, v, i32([P - 1, 0]), i32([3, P - 2]))
    assert torch.equal(k[3], k[P - 1]) and torch.equal(v[P - 2], v[0]) and torch.equal(k[P - 2], k[0])
    for p in (3, P - 2):
        k[p], v[p] = 0, 0
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    refs[[P - 1, 0, 1, P - 3]] = 1
    lens = i32([4, 9, 17])
    live = ops.page_compact(k, v, table, lens, refs)
    assert live.tolist() == [4] and table.tolist() == [[3, -1], [0, -1], [1, 2]]
    for at in ((3, 3), (0, 8), (2, 0)):
        assert (k[at] == 1).all() and (v[at] == 2).all()
