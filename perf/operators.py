"""Measured cases of the paged-cache operators: attention of new tokens over a paged cache,
rotary positions with several axes written into the cache's pages, and the bookkeeping of the pages
(extend, fork, trim, copy, compact).

Every operator exists twice here: ``own = False`` computes it in elementary torch operations in 32
bits (64 for the angles of far positions), rounded once at the end; ``own = True`` makes the calls
that a user makes of ``dpk_b200.ops``.  ``exact`` computes it a third time, in 64 bits.

The calls (all lengths and tables are int32 tensors on the GPU and stay there):

* ``ops.attention_paged(Q [N,Hq,D], K_pages [P,page,Hk,D], V_pages, page_table [S,W], kv_lens [S],
  query_start [S+1], Mask [N,NG] bool or None, max_query_len=, is_causal=) -> (O [N,Hq,D], {})``
* ``ops.rope_append_paged(q, k, v, positions [A,N], inv_freq [R/2], K_pages, V_pages, page_table,
  kv_lens, query_start, sections=, interleaved=) -> rotated q``; the rotated k and v go to the last
  tokens of each sequence
* ``ops.page_extend / page_fork / page_trim / page_copy / page_compact``
"""

import math
import os
import sys

import torch

own = False

GOLDEN = 0.6180339887498949


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-pruning_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dpk_b200 import ops
    return ops


# ------------------------------------------------------------------------------------- the cases

def listed():
    heads = dict(q_heads=32, kv_heads=8, head_dim=128)          # this repository's attention shapes
    wide = dict(q_heads=64, kv_heads=8, head_dim=128)           # its 70B-shaped layer
    return [
        # one user's next token over a short conversation: the smallest call, latency only
        dict(name="attn decode 1x700", op="attention", seqs=1, new=1, cached=700, spread=0.0,
             groups=8, keep=4, page=16, dtype="bf16", causal=True, **heads),
        # a decode step of 64 users at many lengths, half of the head groups routed out
        dict(name="attn decode 64x16384", op="attention", seqs=64, new=1, cached=16384, spread=0.6,
             groups=8, keep=4, page=16, dtype="bf16", causal=True, **heads),
        # a few drafted tokens of every sequence checked at once, no routing, fp16
        dict(name="attn verify 16x5x4096", op="attention", seqs=16, new=5, cached=4091, spread=0.3,
             groups=0, keep=0, page=32, dtype="fp16", causal=True, **wide),
        # a step of a server: prompts in chunks beside single tokens, everything ragged
        dict(name="attn mixed 12x509x3000", op="attention", seqs=12, new=509, cached=3000, spread=1.0,
             groups=8, keep=6, page=16, dtype="bf16", causal=True, **wide),
        # a long prompt's chunk over what is cached of it
        dict(name="attn chunk 1x4096x12288", op="attention", seqs=1, new=4096, cached=12288, spread=0.0,
             groups=8, keep=4, page=64, dtype="bf16", causal=True, **heads),
        # rotary positions of one decode step: 64 sequences, one token each
        dict(name="rope decode 64", op="rope", seqs=64, new=1, cached=2000, spread=1.0, axes=3, page=16,
             pairing="half", rotary=128, dtype="bf16", **heads),
        # images in a prompt, odd token counts, rotation of neighbouring channels, fp16
        dict(name="rope images 3x1031", op="rope", seqs=3, new=1031, cached=77, spread=0.5, axes=2,
             page=16, pairing="neighbours", rotary=64, dtype="fp16", q_heads=16, kv_heads=16, head_dim=64),
        # a long video prompt of the 70B-shaped layer
        dict(name="rope video 4x4096", op="rope", seqs=4, new=4096, cached=100000, spread=0.0, axes=3,
             page=64, pairing="half", rotary=128, dtype="bf16", **wide),
        # one token more for each of 256 sequences: page tables and counts only, a few shared tails
        dict(name="pages extend 256", op="pages", act="extend", seqs=256, tokens=8000, pages=131072,
             page=16, layers=1, kv_heads=1, head_dim=64, dtype="bf16"),
        # a beam-search step: losers dropped, winners forked into their rows, everybody extended
        dict(name="pages beams 64x4", op="pages", act="beams", seqs=256, tokens=2000, pages=12288,
             page=16, layers=4, kv_heads=8, head_dim=128, dtype="bf16"),
        # pages of finished prompts copied for reuse
        dict(name="pages copy 1500", op="pages", act="copy", seqs=8, tokens=4000, pages=6000, page=16,
             layers=4, kv_heads=8, head_dim=128, dtype="fp16"),
        # a pool after many sequences came and went: the live pages moved together
        dict(name="pages compact 8192", op="pages", act="compact", seqs=60, tokens=1900, pages=8192,
             page=16, layers=4, kv_heads=8, head_dim=128, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rope", "pages"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    head_dim = rng.choice([64, 128, 128])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 3, 4, 5, 8])
        cached = _log(rng, 1, 16000)
        new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 4000)])
        # the plain form keeps every score of a sequence: bounds what a drawn case costs
        most = 1.5e9 / (new * (new + cached) * q_heads)
        if most < 1:
            cached = max(1, int(1.5e9 / (new * q_heads)) - new)
            most = 1
        seqs = min(_log(rng, 1, 64), max(1, int(most)))
        groups = rng.choice([0, 1, kv_heads, q_heads])
        return dict(op=op, seqs=seqs, new=new, cached=cached, spread=rng.choice([0.0, 0.3, 1.0]),
                    groups=groups, keep=max(1, groups * rng.choice([1, 2, 3]) // 4) if groups else 0,
                    page=page, dtype=dtype, causal=rng.random() < 0.8, q_heads=q_heads,
                    kv_heads=kv_heads, head_dim=head_dim)
    if op == "rope":
        kv_heads = rng.choice([1, 2, 4, 8])
        tokens = _log(rng, 1, 16384)
        seqs = min(tokens, _log(rng, 1, 128))
        return dict(op=op, seqs=seqs, new=max(1, tokens // seqs), cached=_log(rng, 1, 30000) // seqs + 1,
                    spread=rng.choice([0.0, 0.5, 1.0]), axes=rng.choice([1, 2, 3]), page=page,
                    pairing=rng.choice(["half", "neighbours"]),
                    rotary=rng.choice([head_dim, head_dim // 2]), dtype=dtype,
                    q_heads=kv_heads * rng.choice([1, 3, 4, 8]), kv_heads=kv_heads, head_dim=head_dim)
    act = rng.choice(["extend", "beams", "copy", "compact"])
    seqs = 4 * _log(rng, 1, 60)
    tokens = _log(rng, 10, 1800)
    need = seqs * (tokens // page + 3)
    pages = int(need * rng.uniform(1.1, 1.6)) + 8
    kv_heads = rng.choice([1, 2, 8])
    layers = max(1, min(4, int(1.2e9 / (pages * page * kv_heads * head_dim * 4))))
    return dict(op=op, act=act, seqs=seqs, tokens=tokens, pages=pages, page=page, layers=layers,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype)


# ------------------------------------------------------------------------------------ the inputs

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _ragged(most, spread, seqs, shift):
    """``seqs`` lengths of at most ``most``, spread below it without any randomness."""
    return [max(1, int(round(most * (1.0 - spread * math.modf((s + 1) * GOLDEN + shift)[0]))))
            for s in range(seqs)]


def _lengths(case):
    new = _ragged(case["new"], case["spread"], case["seqs"], 0.0)
    cached = _ragged(case["cached"], case["spread"], case["seqs"], 0.37)
    if case["seqs"] > 2 and case["spread"] >= 1.0:
        cached[1] = 0                                  # a prompt's first chunk
        new[2] = 1                                     # a single token beside the chunks
    return new, cached


def _fill(g, shape, dtype):
    """N(0,1) values, made in pieces so that the 32-bit draft of a large cache stays small."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda"))
    return t


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sequences(case, g):
    new, cached = _lengths(case)
    page = case["page"]
    width = max(-(-(n + c) // page) for n, c in zip(new, cached)) + 1
    used = [-(-(n + c) // page) for n, c in zip(new, cached)]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(table=table, kv_lens=_ints([n + c for n, c in zip(new, cached)]),
                query_start=_ints(starts), tokens=starts[-1], pages=pages, most_new=max(new),
                most_len=max(n + c for n, c in zip(new, cached)))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)
    dt = _dtype(case)
    if case["op"] == "pages":
        return _prepare_pages(case, g, dt)
    st = dict(case=case, **_sequences(case, g))
    n, hq, hk, d = st["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    st["q"] = _fill(g, (n, hq, d), dt)
    st["k_pages"] = _fill(g, (st["pages"], case["page"], hk, d), dt)
    st["v_pages"] = _fill(g, (st["pages"], case["page"], hk, d), dt)
    if case["op"] == "attention":
        st["mask"] = None
        if case["groups"]:
            scores = torch.rand((n, case["groups"]), generator=g, device="cuda")
            chosen = scores.topk(case["keep"], dim=1).indices
            st["mask"] = torch.zeros((n, case["groups"]), dtype=torch.bool, device="cuda")
            st["mask"].scatter_(1, chosen, True)
        return st
    st["k"] = _fill(g, (n, hk, d), dt)
    st["v"] = _fill(g, (n, hk, d), dt)
    half, axes = case["rotary"] // 2, case["axes"]
    st["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()
    # text, then frames of 24 x 36 patches: time, height and width count on from the cached tokens
    starts = st["query_start"].long()
    seq = torch.searchsorted(starts, torch.arange(n, device="cuda"), right=True) - 1
    i = torch.arange(n, device="cuda") - starts[seq]
    base = (st["kv_lens"].long() - (starts[1:] - starts[:-1]))[seq] + torch.randint(
        0, 4, (n,), generator=g, device="cuda")
    patch = (i - 16).clamp(min=0)
    text = i < 16
    rows = [torch.where(text, i, 16 + patch // 864), torch.where(text, i, 16 + patch // 36 % 24),
            torch.where(text, i, 16 + patch % 36)]
    st["positions"] = torch.stack([base + r for r in rows[:axes]])
    st["sections"] = tuple(half * (a + 1) // axes - half * a // axes for a in range(axes))
    return st


def _prepare_pages(case, g, dt):
    """A pool in the middle of its life, kept as ONE int32 buffer [table | lengths | counts] so that
    a pass can start from it with one small copy."""
    S, P, page = case["seqs"], case["pages"], case["page"]
    lens = _ragged(case["tokens"], 0.6, S, 0.11)
    if case["act"] == "beams":                       # the beams of a group are equally long
        lens = [lens[s // 4 * 4] for s in range(S)]
    width = -(-case["tokens"] // page) + 4
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    table = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(S):
        u = -(-lens[s] // page)
        first = 0
        if s % 4 and case["act"] in ("beams", "extend"):
            if case["act"] == "beams":               # a group shares all full pages but the last two
                first = max(0, lens[s] // page - 2)
            elif s % 16 == 1:                        # a forked sequence: shares its tail as well
                lens[s], u = lens[s - 1], -(-lens[s - 1] // page)
                first = u
            table[s, :first] = table[s // 4 * 4, :first]
        table[s, first:u] = order[at:at + u - first]
        at += u - first
    live = table[table >= 0].long()
    refs.index_add_(0, live, torch.ones_like(live, dtype=torch.int32))
    st = dict(case=case, S=S, P=P, width=width,
              master=torch.cat([table.flatten(), _ints(lens), refs]),
              k_pages=_fill(g, (case["layers"], P, page, case["kv_heads"], case["head_dim"]), dt),
              v_pages=_fill(g, (case["layers"], P, page, case["kv_heads"], case["head_dim"]), dt))
    st["work"] = st["master"].clone()
    act = case["act"]
    if act == "extend":
        st["add"] = torch.ones(S, dtype=torch.int32, device="cuda")
    elif act == "beams":
        # of every group of four, two random beams are dropped and the others forked into their rows
        order4 = torch.rand((S // 4, 4), generator=g, device="cuda").argsort(1).to(torch.int32)
        order4 += 4 * torch.arange(S // 4, device="cuda", dtype=torch.int32)[:, None]
        st["losers"] = order4[:, :2].contiguous().flatten()
        st["winners"] = order4[:, 2:].contiguous().flatten()
        st["add"] = torch.ones(S, dtype=torch.int32, device="cuda")
    elif act == "copy":
        n = min(max(1, P // 4), 1500)
        ids = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
        st["src"], st["dst"] = ids[:n].contiguous(), ids[n:2 * n].contiguous()
    return st


def _views(st):
    S, W = st["S"], st["width"]
    b = st["work"]
    return b[:S * W].view(S, W), b[S * W:S * W + S], b[S * W + S:]


# --------------------------------------------------------------------------------- the plain forms

def _plain_attention(st):
    c = st["case"]
    S, page, D = c["seqs"], c["page"], c["head_dim"]
    hk, rep = c["kv_heads"], c["q_heads"] // c["kv_heads"]
    n, L = st["most_new"], st["most_len"]
    starts = st["query_start"].long()
    new = starts[1:] - starts[:-1]
    lens = st["kv_lens"].long()
    dev = st["q"].device
    pages = st["table"][:, :-(-L // page)].clamp(min=0).long()
    k = st["k_pages"][pages].flatten(1, 2)[:, :L].float().permute(0, 2, 3, 1)      # [S,Hk,D,L]
    v = st["v_pages"][pages].flatten(1, 2)[:, :L].float().transpose(1, 2)          # [S,Hk,L,D]
    at = (starts[:-1, None] + torch.arange(n, device=dev)).clamp(max=st["tokens"] - 1)
    q = st["q"][at].float().view(S, n, hk, rep, D).permute(0, 2, 3, 1, 4).reshape(S, hk, rep * n, D)
    scores = (q @ k).view(S, hk, rep, n, L) * D ** -0.5
    key = torch.arange(L, device=dev)
    limit = lens[:, None].expand(S, n)
    if c["causal"]:
        limit = (lens - new)[:, None] + torch.arange(n, device=dev) + 1
    hidden = key >= torch.minimum(limit, lens[:, None])[..., None]                 # [S,n,L]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(S, hk, rep * n, L) @ v).view(S, hk, rep, n, D) / total.clamp(min=1e-38)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, n, c["q_heads"], D)
    tok = torch.arange(st["tokens"], device=dev)
    seq = torch.searchsorted(starts, tok, right=True) - 1
    o = o[seq, tok - starts[seq]]
    if st["mask"] is not None:
        keep = st["mask"].repeat_interleave(c["q_heads"] // c["groups"], dim=1)
        o = torch.where(keep[..., None], o, 0.0)
    return o.to(st["q"].dtype)


def _plain_rotate(x, cos, sin, rotary, neighbours):
    x = x.float()
    r, rest = x[..., :rotary], x[..., rotary:]
    if neighbours:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1)


def _plain_rope(st):
    c = st["case"]
    dt, dev, page = st["q"].dtype, st["q"].device, c["page"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=dev),
                                   torch.tensor(st["sections"], device=dev))
    angle = st["positions"].double()[axis].T * st["inv_freq"].double()              # [N, R/2]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    nb = c["pairing"] == "neighbours"
    q = _plain_rotate(st["q"], cos, sin, c["rotary"], nb).to(dt)
    k = _plain_rotate(st["k"], cos, sin, c["rotary"], nb).to(dt)
    starts = st["query_start"].long()
    tok = torch.arange(st["tokens"], device=dev)
    seq = torch.searchsorted(starts, tok, right=True) - 1
    place = st["kv_lens"].long()[seq] - starts[seq + 1] + tok
    pages = st["table"][seq, place // page].long()
    st["k_pages"][pages, place % page] = k
    st["v_pages"][pages, place % page] = st["v"]
    return q, st["k_pages"], st["v_pages"]


def _plain_extend(st, table, lens, refs, add):
    """Rows in order take the lowest free pages; a shared, partly filled last page is copied for
    everybody who writes to it but, where all its holders write, the first of them."""
    S, W, P, page = st["S"], st["width"], st["P"], st["case"]["page"]
    dev = table.device
    have, want = (lens + page - 1) // page, (lens + add + page - 1) // page
    row = torch.arange(S, device=dev)
    fits = (want <= W) & (add >= 0)
    tail = table[row, (have - 1).clamp(min=0).long()]
    writes = (add > 0) & fits & (lens % page != 0)
    shared = writes & (refs[tail.clamp(min=0).long()] > 1)
    same = (tail[:, None] == tail[None]) & shared[:, None] & shared[None]
    holders = same.sum(1)
    first = same.to(torch.int32).argmax(1) == row
    last = S - 1 - same.flip(1).to(torch.int32).argmax(1)
    keeps = shared & first & (holders == refs[tail.clamp(min=0).long()])
    copies = shared & ~keeps
    need = torch.where(fits, want - have, 0) + copies.int()
    upto = need.cumsum(0)
    free = (refs == 0).sum()
    granted = fits & ((need == 0) | (upto <= free))
    granted &= ~keeps | (upto[last] <= free)
    order = torch.sort((refs != 0).to(torch.int8), stable=True).indices.int()       # free pages first
    give = granted & (need > 0)
    copies &= granted
    base = upto - need
    # the copies' pages first, then the new ones
    col = torch.arange(W, device=dev)[None]
    fresh = give[:, None] & (col >= have[:, None]) & (col < want[:, None])
    rank = (base + copies.int())[:, None] + col - have[:, None]
    table.copy_(torch.where(fresh, order[rank.clamp(0, P - 1)], table))
    new_tail = order[base.clamp(max=P - 1).long()]
    spot = (col == (have - 1)[:, None]) & copies[:, None]
    table.copy_(torch.where(spot, new_tail[:, None], table))
    ranks = torch.arange(P, device=dev)
    owner = torch.searchsorted(upto, ranks, right=True).clamp(max=S - 1)
    refs.add_(torch.zeros_like(refs).scatter_(0, order.long(), ((ranks < upto[-1]) & give[owner]).int()))
    refs.index_add_(0, tail.clamp(min=0).long(), -copies.int())
    rows = torch.where(copies, lens % page, 0)
    for pool in (st["k_pages"], st["v_pages"]):
        old, new = pool[:, tail.clamp(min=0).long()], pool[:, new_tail.long()]
        moved = (torch.arange(page, device=dev)[None] < rows[:, None])[None, :, :, None, None]
        target = torch.where(copies, new_tail, P).long()
        keep = target < P
        pool[:, target[keep]] = torch.where(moved, old, new)[:, keep]
    lens.add_(torch.where(granted, add, 0))
    return granted


def _plain_pages(st):
    act, page, P, W = st["case"]["act"], st["case"]["page"], st["P"], st["width"]
    st["work"].copy_(st["master"])
    table, lens, refs = _views(st)
    out = [table, lens, refs, st["k_pages"], st["v_pages"]]
    col = torch.arange(W, device=table.device)[None]
    if act == "copy":
        for pool in (st["k_pages"], st["v_pages"]):
            pool[:, st["dst"].long()] = pool[:, st["src"].long()]
        return out[3:]
    if act == "extend":
        return out + [_plain_extend(st, table, lens, refs, st["add"])]
    if act == "beams":
        lose, win = st["losers"].long(), st["winners"].long()
        old = table[lose]
        held = (col < ((lens[lose] + page - 1) // page)[:, None]).int()
        refs.index_add_(0, old.clamp(min=0).long().flatten(), -held.flatten())
        table[lose] = -1
        lens[lose] = 0
        held = (col < ((lens[win] + page - 1) // page)[:, None]).int()
        refs.index_add_(0, table[win].clamp(min=0).long().flatten(), held.flatten())
        table[lose] = table[win]
        lens[lose] = lens[win]
        return out + [_plain_extend(st, table, lens, refs, st["add"])]
    live = (refs > 0).sum()
    order = torch.arange(P, device=table.device)
    hole, mover = (order < live) & (refs == 0), (order >= live) & (refs > 0)
    src, dst = mover.nonzero().flatten(), hole.nonzero().flatten()
    for pool in (st["k_pages"], st["v_pages"]):
        pool[:, dst] = pool[:, src]
    to = order.to(torch.int32)
    to[src] = dst.int()
    refs[dst] = refs[src]
    refs[src] = 0
    held = col < ((lens + page - 1) // page)[:, None]
    table.copy_(torch.where(held, to[table.clamp(min=0).long()], table))
    return out + [live.to(torch.int32).view(1)]


# --------------------------------------------------------------------------------- the calls

def _own_pages(st):
    ops = _ops()
    act, page = st["case"]["act"], st["case"]["page"]
    kp, vp = st["k_pages"], st["v_pages"]
    if act == "copy":
        ops.page_copy(kp, vp, st["src"], st["dst"])
        return [kp, vp]
    st["work"].copy_(st["master"])
    table, lens, refs = _views(st)
    out = [table, lens, refs, kp, vp]
    if act == "extend":
        return out + [ops.page_extend(kp, vp, table, lens, refs, st["add"])]
    if act == "beams":
        ops.page_trim(table, lens, refs, st["losers"], page_size=page)
        ops.page_fork(table, lens, refs, st["winners"], st["losers"], page_size=page)
        return out + [ops.page_extend(kp, vp, table, lens, refs, st["add"])]
    return out + [ops.page_compact(kp, vp, table, lens, refs)]


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        return _plain_attention(st) if op == "attention" else _plain_rope(st) if op == "rope" else _plain_pages(st)
    if op == "attention":
        return _ops().attention_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_lens"],
                                      st["query_start"], st["mask"], max_query_len=st["most_new"],
                                      is_causal=st["case"]["causal"])[0]
    if op == "rope":
        q = _ops().rope_append_paged(st["q"], st["k"], st["v"], st["positions"], st["inv_freq"],
                                     st["k_pages"], st["v_pages"], st["table"], st["kv_lens"],
                                     st["query_start"], sections=st["sections"],
                                     interleaved=st["case"]["pairing"] == "neighbours")
        return q, st["k_pages"], st["v_pages"]
    return _own_pages(st)


# ------------------------------------------------------------------------------- bytes and flops

def work(case):
    if case["op"] == "pages":
        S, page, W = case["seqs"], case["page"], -(-case["tokens"] // case["page"]) + 4
        one = page * case["kv_heads"] * case["head_dim"] * 2 * 2 * case["layers"]       # a page of K and V
        lens = _ragged(case["tokens"], 0.6, S, 0.11)
        if case["act"] == "copy":
            n = min(max(1, case["pages"] // 4), 1500)
            return dict(bytes=2 * n * one, flops=0)
        if case["act"] == "extend":
            # counts scanned for free pages, every length, and the shared tails copied
            return dict(bytes=4 * case["pages"] + 16 * S + (S // 16) * one, flops=0)
        if case["act"] == "beams":
            held = sum(-(-n // page) for n in lens) // 2
            return dict(bytes=4 * case["pages"] + 24 * held + S // 2 * one, flops=0)
        live = sum(-(-n // page) for n in lens)
        movers = live * max(0, case["pages"] - live) // case["pages"]
        return dict(bytes=8 * case["pages"] + 4 * S * W + 2 * movers * one, flops=0)
    new, cached = _lengths(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    n = sum(new)
    if case["op"] == "rope":
        # q read and written; k and v read and written once into the pages; positions
        return dict(bytes=2 * 2 * n * (hq + 2 * hk) * d + 8 * n * case["axes"],
                    flops=6 * n * (hq + hk) * case["rotary"] // 2)
    share = case["keep"] / case["groups"] if case["groups"] else 1.0
    heads_per_group = hq // case["groups"] if case["groups"] else hq
    kv, pairs = 0.0, 0
    for a, c in zip(new, cached):
        read = 1.0 - (1.0 - share) ** (a * max(1, (hq // hk) // heads_per_group))
        kv += read * (a + c) * hk * d * 2 * 2
        pairs += a * c + a * (a + 1) // 2 if case["causal"] else a * (a + c)
    return dict(bytes=int(kv + n * hq * d * 2 * (1 + share) + n * case["groups"]),
                flops=int(4 * d * hq * share * pairs))


# ------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["op"] == "pages":
        return None                                     # whole numbers and copies: nothing is rounded
    st = prepare(case, seed)
    starts, lens = st["query_start"].tolist(), st["kv_lens"].tolist()
    page, d = case["page"], case["head_dim"]
    if case["op"] == "attention":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        hk = case["kv_heads"]
        rep = case["q_heads"] // hk
        for s in range(case["seqs"]):
            a, b, L = starts[s], starts[s + 1], lens[s]
            ids = st["table"][s, :-(-L // page)].long()
            at = torch.arange(b - a, device="cuda")[:, None] + (L - (b - a))
            seen = torch.arange(L, device="cuda")[None] <= (at if case["causal"] else L)
            for h in range(hk):
                k = st["k_pages"][ids, :, h].reshape(-1, d)[:L].double()
                v = st["v_pages"][ids, :, h].reshape(-1, d)[:L].double()
                for r in range(h * rep, h * rep + rep):
                    z = st["q"][a:b, r].double() @ k.T / math.sqrt(d)
                    z = torch.where(seen, z, -math.inf)
                    out[a:b, r] = torch.softmax(z, -1) @ v
        if st["mask"] is not None:
            out *= torch.repeat_interleave(st["mask"].double(), case["q_heads"] // case["groups"], 1)[..., None]
        return out
    # a rotation is a product of complex numbers
    R = case["rotary"]
    which = [a for a, many in enumerate(st["sections"]) for _ in range(many)]
    turn = torch.polar(torch.ones((st["tokens"], R // 2), dtype=torch.float64, device="cuda"),
                       st["positions"].double()[which].T * st["inv_freq"].double())[:, None]

    def rotated(x):
        x = x.double()
        near = case["pairing"] == "neighbours"
        part = x[..., :R].unflatten(-1, (R // 2, 2)) if near else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
        z = z.flatten(-2) if near else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, x[..., R:]], -1)

    k, keys, values = rotated(st["k"]), st["k_pages"].double(), st["v_pages"].double()
    for s in range(case["seqs"]):
        a, b, L = starts[s], starts[s + 1], lens[s]
        at = torch.arange(L - (b - a), L, device="cuda")
        ids = st["table"][s].long()[at // page]
        keys[ids, at % page] = k[a:b]
        values[ids, at % page] = st["v"][a:b].double()
    return rotated(st["q"]), keys, values
