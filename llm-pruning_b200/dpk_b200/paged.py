"""Operators of the paged KV cache: attention of new tokens, rotary write, bookkeeping of pages.

Host side of the ``dpk_attn_paged`` / ``dpk_rope_append_paged`` / ``dpk_page_*`` entry points, with
the conventions of :mod:`dpk_b200.ops` (which re-exports everything here): CUDA tensors only,
current stream, ``ValueError`` for refused arguments, nothing read back to the host.

State of a cache (int32 tensors on the GPU): ``page_table [S,W]`` page ids, ``kv_lens [S]`` tokens
held (a step's new ones included), ``ref_counts [P]`` holders of a page, 0 = free.  A step names its
new tokens by ``query_start [S+1]``: those of sequence ``s`` are rows ``query_start[s] ..
query_start[s+1]-1`` of the packed q/k/v; the first start is 0, and a sequence whose range is none (it
runs backwards or leaves the tensors) is reported and has no tokens.  :class:`dpk_b200.wide.PagedKVCache` keeps the state.
No reference counterpart (its cache is contiguous, ``WIDE/wrapper/cache.py:10-60``); values outside
their range are reported through :func:`dpk_b200.ops.device_status` and never followed.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence, Tuple

import torch

from . import _native as N

_CODES = {torch.bfloat16: N.BF16, torch.float16: N.F16}


def _code(t: torch.Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"dpk_b200 kernels take float16 or bfloat16 tensors, got {t.dtype}")
    return code


def _on_gpu(*tensors: Optional[torch.Tensor]) -> int:
    """Index of the one CUDA device that holds all of them."""
    dev = tensors[0].get_device()
    if dev < 0:
        raise ValueError("dpk_b200 operators run on CUDA tensors only (no CPU fallback)")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            if t.get_device() < 0:
                raise ValueError("dpk_b200 operators run on CUDA tensors only (no CPU fallback)")
            raise ValueError("all tensors must be on the same device")
    return dev


def _call(dev: int, entry, *args) -> None:
    """One C entry point on the current stream of device ``dev``; entering the device is skipped where
    it is the current one already (it costs as much as a launch)."""
    if torch.cuda.current_device() == dev:
        rc = entry(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = entry(*args, _raw_stream(dev))
    if rc:
        N.check(rc)


def _ints(t: torch.Tensor, shape: tuple, name: str) -> torch.Tensor:
    """A contiguous int32 tensor of ``shape``."""
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}, got "
                         f"{t.dtype} {list(t.shape)}")
    return t


def _table(page_table: torch.Tensor) -> Tuple[int, int, int]:
    """``(S, W, stride)`` of a page table; its rows may be slices of a wider one."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("page_table must be a two-dimensional int32 tensor")
    S, W = page_table.shape
    stride = page_table.stride(0) if S > 1 else W
    if (W > 1 and page_table.stride(1) != 1) or stride < W:
        raise ValueError("the entries of a page_table row must be contiguous, and rows must not overlap")
    return S, W, stride


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor) -> Tuple[int, int, int, int, int, int]:
    """``(P, page_size, Hk, D, page_stride, token_stride)`` of one layer's pools."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("K_pages and V_pages must be alike, [pages, page_size, kv_heads, head_dim]")
    P, page, Hk, D = k_pages.shape
    if k_pages.stride() != v_pages.stride():
        raise ValueError("K_pages and V_pages must have the same strides")
    ps, ts, hs, es = k_pages.stride()
    if P <= 1:
        ps = page * ts
    if page == 1:
        ts = Hk * D
    if es != 1 or (Hk > 1 and hs != D) or ts < Hk * D or (P > 1 and ps < Hk * D):
        raise ValueError("the heads of a cached token must be contiguous")
    return P, page, Hk, D, ps, ts


def _token_rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """``t [N,heads,D]`` with the heads of a token back to back: the tensor (copied only if it does
    not fit) and its token stride in elements."""
    n, heads, D = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, heads * D
    ts = t.stride(0) if n > 1 else heads * D
    if not ((D == 1 or t.stride(2) == 1) and (heads == 1 or t.stride(1) == D) and ts >= heads * D
            and ts % 8 == 0 and t.data_ptr() % 16 == 0):
        t = t.clone(memory_format=torch.contiguous_format)       # of a contiguous one too: it starts off 16 bytes
        ts = heads * D
    return t, ts


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is None:                 # a torch build without CUDA, or without this shortcut
    def _raw_stream(dev: int) -> int:
        return torch.cuda.current_stream(dev).cuda_stream


def attention_paged(Q: torch.Tensor, K_pages: torch.Tensor, V_pages: torch.Tensor,
                    page_table: torch.Tensor, kv_lens: torch.Tensor, query_start: torch.Tensor,
                    Mask: Optional[torch.Tensor] = None, O: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, is_causal: Optional[bool] = True,
                    max_query_len: Optional[int] = None, kernel_version: Optional[int] = 0,
                    arch: Optional[str] = "sm100"):
    """Head-group-routed attention of the new tokens over a paged cache; returns ``(O [N,Hq,D], {})``
    like its siblings :func:`attention_prefill` and :func:`attention_decode`.

    ``Q [N,Hq,D]``: the new tokens of all sequences, back to back; ``K_pages, V_pages
    [P,page_size,Hk,D]`` already hold them (:func:`rope_append_paged`).  New token ``i`` of the ``n``
    new ones of sequence ``s`` sees keys ``j <= kv_lens[s] - n + i``, or with ``is_causal=False`` all
    ``kv_lens[s]`` of them.  ``Mask [N,NG]`` (non-zero = active) routes head groups as everywhere
    else; ``None`` keeps every head.  Rows that are routed out or see no key are zero.  Rows of no
    sequence (behind ``query_start[S]``) are zero in a new ``O`` and left alone in one that is passed in.

    ``max_query_len``: an upper bound of a sequence's new tokens, known to the host (default: N).
    It chooses between the kernel for a few tokens per sequence and the one for chunks, so give 1
    for a decode step; a larger sequence than it says is still computed, only slower.

    Head sizes 64 and 128, ``scale`` above zero.  Positions that hold no token may contain anything; what
    the new tokens themselves wrote as values has to be finite.  Rows that see a score of NaN or +inf, or
    scores of -inf alone, are NaN."""
    dev = _on_gpu(Q, K_pages, V_pages, page_table, kv_lens, query_start, Mask, O)
    code = _code(Q)
    if K_pages.dtype != Q.dtype:
        raise ValueError("Q and the pages must share one dtype")
    if Q.dim() != 3:
        raise ValueError("Q must be [tokens, heads, head_dim]")
    n, Hq, D = Q.shape
    P, page, Hk, Dk, ps, ts = _pool(K_pages, V_pages)
    if Dk != D:
        raise ValueError(f"head_dim of Q ({D}) and of the pages ({Dk}) differ")
    S, W, tstride = _table(page_table)
    _ints(kv_lens, (S,), "kv_lens")
    _ints(query_start, (S + 1,), "query_start")
    m8, NG = None, 1
    if Mask is not None:
        if Mask.dim() != 2 or Mask.shape[0] != n:
            raise ValueError(f"Mask must be [tokens, groups] with {n} tokens, got {list(Mask.shape)}")
        NG = Mask.shape[1]
        m8 = Mask if Mask.dtype in (torch.bool, torch.uint8) else Mask != 0
        if not m8.is_contiguous():
            m8 = m8.contiguous()
    Qc, q_ts = _token_rows(Q)
    clear = 0
    if O is None:
        O = torch.empty_like(Q) if Q.is_contiguous() else Q.new_empty((n, Hq, D))
        clear = 1
    elif O.shape != Q.shape or O.dtype != Q.dtype or not O.is_contiguous():
        raise ValueError("O must be contiguous with the shape and dtype of Q")
    most = n if max_query_len is None else int(max_query_len)
    if n and most < 1:
        raise ValueError("max_query_len must be at least 1")
    most = min(most, 2 ** 31 - 1)        # what the C argument holds
    if n == 0 or S == 0:                 # nothing to attend: every row is behind the last sequence
        if clear:
            O.zero_()
        return O, {}
    lib = N.load()
    with_mask = 0 if m8 is None else 1
    if torch.cuda.current_device() == dev:
        nbytes = _attention_workspace_bytes(dev, n, S, Hq, Hk, D, most, with_mask)
    else:
        with torch.cuda.device(dev):
            nbytes = _attention_workspace_bytes(dev, n, S, Hq, Hk, D, most, with_mask)
    ws = page_table.new_empty((nbytes + 3) // 4)
    _call(dev, lib.dpk_attn_paged,
          Qc.data_ptr(), K_pages.data_ptr(), V_pages.data_ptr(), page_table.data_ptr(), kv_lens.data_ptr(),
          query_start.data_ptr(), None if m8 is None else m8.data_ptr(), O.data_ptr(), n, S, W, P, page, Hq,
          Hk, D, NG, D ** -0.5 if scale is None else float(scale), 1 if is_causal else 0, code,
          most if most > 1 else 1, clear, q_ts, ps, ts, tstride, ws.data_ptr(), nbytes)
    return O, {}


@functools.lru_cache(maxsize=64)
def _host_ints(values: tuple):
    """A host array of C ints (never written to)."""
    return (ctypes.c_int32 * len(values))(*values)


def _rope(dev, q, k, v, positions, inv_freq, sections, axis_map, interleaved, attention_scale, q_out, cache,
          granted=None):
    code = _code(q)
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise ValueError("q, k and v must share one dtype")
    if q.dim() != 3 or k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [N,Hq,D] and k [N,Hk,D]")
    if v is not None and v.shape != k.shape:
        raise ValueError("k and v must have one shape")
    n, Hq, D = q.shape
    Hk = k.shape[1]
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[1] != n or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64 [axes,{n}], got {positions.dtype} "
                         f"{list(positions.shape)}")
    if n > 1 and positions.stride(1) != 1:
        positions = positions.contiguous()
    axes = positions.shape[0]
    axis_stride = positions.stride(0) if axes > 1 else n
    if axes > 1 and axis_stride < n:
        positions = positions.contiguous()
        axis_stride = n
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 vector")
    rotary = 2 * inv_freq.shape[0]
    secs = None
    if axis_map is not None:
        _ints(axis_map, (rotary // 2,), "axis_map")
    elif sections is not None:
        if len(sections) != axes:
            raise ValueError(f"{len(sections)} sections for {axes} axes")
        secs = _host_ints(tuple(map(int, sections)))
    elif axes > 1:
        raise ValueError("several axes need sections or axis_map")
    qc, q_ts = _token_rows(q)
    kc, kv_ts = _token_rows(k)
    vc = None
    if v is not None:
        vc, v_ts = _token_rows(v)
        if v_ts != kv_ts:
            kc, vc = kc.contiguous(), vc.contiguous()
            kv_ts = Hk * D
    if q_out is None:
        q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((n, Hq, D))
        qo_ts = Hq * D
    else:
        if q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must have the shape and dtype of q")
        same, qo_ts = _token_rows(q_out)
        if same is not q_out:
            raise ValueError("q_out: the heads of a token must be contiguous, 16-byte aligned")
    k_out = None
    if cache is None:
        k_out = k.new_empty((n, Hk, D))
        tail = (None, None, 0, 0, None, 0, None, None, n, 0, 0, 0, 0)
    else:
        k_pages, v_pages, page_table, kv_lens, query_start = cache
        if k_pages.dtype != q.dtype:
            raise ValueError("q and the pages must share one dtype")
        P, page, Hp, Dp, ps, ts = _pool(k_pages, v_pages)
        if (Hp, Dp) != (Hk, D):
            raise ValueError(f"pages of {Hp} heads of {Dp}, k of {Hk} heads of {D}")
        S, W, tstride = _table(page_table)
        _ints(kv_lens, (S,), "kv_lens")
        _ints(query_start, (S + 1,), "query_start")
        if granted is not None and (granted.dtype not in (torch.bool, torch.uint8) or granted.shape != (S,)
                                    or not granted.is_contiguous()):
            raise ValueError(f"granted must be a contiguous bool or uint8 tensor of shape [{S}], got "
                             f"{granted.dtype} {list(granted.shape)}")
        if S == 0:
            return q_out, None
        tail = (k_pages.data_ptr(), v_pages.data_ptr(), ps, ts, page_table.data_ptr(), tstride,
                kv_lens.data_ptr(), query_start.data_ptr(), n, S, W, P, page)
    if n == 0:
        return q_out, k_out
    _call(dev, N.load().dpk_rope_append_paged_granted,
          qc.data_ptr(), kc.data_ptr(), None if vc is None else vc.data_ptr(), q_out.data_ptr(),
          None if k_out is None else k_out.data_ptr(), q_ts, kv_ts, qo_ts, positions.data_ptr(), axis_stride,
          1 if positions.dtype is torch.int64 else 0, inv_freq.data_ptr(),
          None if axis_map is None else axis_map.data_ptr(), secs, axes, rotary, 1 if interleaved else 0,
          float(attention_scale), *tail, Hq, Hk, D, code, None if granted is None else granted.data_ptr())
    return q_out, k_out


def rope_append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                      inv_freq: torch.Tensor, K_pages: torch.Tensor, V_pages: torch.Tensor,
                      page_table: torch.Tensor, kv_lens: torch.Tensor, query_start: torch.Tensor,
                      sections: Optional[Sequence[int]] = None, axis_map: Optional[torch.Tensor] = None,
                      interleaved: bool = False, attention_scale: float = 1.0,
                      q_out: Optional[torch.Tensor] = None,
                      granted: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding with one or several position axes, and the write of the rotated ``k`` and of
    ``v`` into the pages of the new tokens; returns the rotated ``q [N,Hq,D]`` (in ``q_out``, which
    may be ``q`` itself).

    ``positions [axes,N]`` (or ``[N]``): a token's position on each axis, e.g. time, height and width
    of an image patch.  Rotary pair ``i`` turns by ``positions[axis(i)] * inv_freq[i]``; its axis
    comes from ``sections`` (the first ``sections[0]`` pairs belong to axis 0, ...) or pair by pair
    from ``axis_map`` (int32).  ``inv_freq`` (float32) has one entry per pair, so ``2 *
    len(inv_freq)`` of the head's channels turn and the others pass through.  A pair is channels
    ``(i, R/2+i)``, with ``interleaved`` channels ``(2i, 2i+1)``; ``attention_scale`` multiplies cos
    and sin.  A token's place in the cache is its place in the sequence (the last tokens of
    ``kv_lens[s]``), whatever its rotary positions.  Rows behind ``query_start[S]`` are not touched (in a
    new ``q`` they hold anything).  Counterpart of :func:`rope_append`; computed
    from positions, so far ones keep their exact angle.

    ``granted [S]`` (bool or uint8): what :func:`page_extend` returned for this step.  A refused sequence's
    length does not count its new tokens, so they have no place: with ``granted`` their ``k`` and ``v`` are
    left out, without it such a sequence must bring none."""
    dev = _on_gpu(q, k, v, positions, inv_freq, K_pages, V_pages, page_table, kv_lens, query_start, axis_map, q_out,
                  granted)
    return _rope(dev, q, k, v, positions, inv_freq, sections, axis_map, interleaved, attention_scale, q_out,
                 (K_pages, V_pages, page_table, kv_lens, query_start), granted)[0]


def rope_axes(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              sections: Optional[Sequence[int]] = None, axis_map: Optional[torch.Tensor] = None,
              interleaved: bool = False, attention_scale: float = 1.0):
    """The rotation of :func:`rope_append_paged` without a cache: ``(rotated q, rotated k)``."""
    dev = _on_gpu(q, k, positions, inv_freq, axis_map)
    return _rope(dev, q, k, None, positions, inv_freq, sections, axis_map, interleaved, attention_scale, None, None)


# ---------------------------------------------------------------------------------------- pages

def _state(page_table, kv_lens, ref_counts):
    S, W, stride = _table(page_table)
    _ints(kv_lens, (S,), "kv_lens")
    if ref_counts.dim() != 1:
        raise ValueError("ref_counts must be one-dimensional")
    P = ref_counts.shape[0]
    _ints(ref_counts, (P,), "ref_counts")
    return (page_table.data_ptr(), stride, kv_lens.data_ptr(), ref_counts.data_ptr(), S, W, P)


def _pools(k_pages, v_pages):
    """``(arguments of the C entry points, P, page_size)`` of pools ``[L,P,page,Hk,D]`` or ``[P,...]``."""
    if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.stride() != v_pages.stride():
        raise ValueError("K_pages and V_pages must be alike")
    if k_pages.dim() == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    if k_pages.dim() != 5 or k_pages.element_size() != 2:
        raise ValueError("pools must be 16-bit [layers, pages, page_size, kv_heads, head_dim]")
    L, P, page, Hk, D = k_pages.shape
    ls, ps, ts, hs, es = k_pages.stride()
    row = Hk * D
    if (es != 1 and D > 1) or (hs != D and Hk > 1) or (ts != row and page > 1):
        raise ValueError("a page must be contiguous")
    if P <= 1:
        ps = page * row
    if L <= 1:
        ls = 0
    return (k_pages.data_ptr(), v_pages.data_ptr(), L, ls, ps, row), P, page


@functools.lru_cache(maxsize=256)
def _page_workspace_bytes(S: int, P: int, n: int) -> int:
    return N.load().dpk_page_workspace_bytes(S, P, n)


@functools.lru_cache(maxsize=256)
def _attention_workspace_bytes(dev: int, *sizes: int) -> int:
    return N.load().dpk_attn_paged_workspace_bytes(*sizes)


def _workspace(S: int, P: int, n: int, like: torch.Tensor):
    nbytes = _page_workspace_bytes(S, P, n)
    return like.new_empty((nbytes + 3) // 4), nbytes


def _vector(t: torch.Tensor, name: str, n: Optional[int] = None) -> int:
    if t.dim() != 1:
        raise ValueError(f"{name} must be one-dimensional")
    _ints(t, (t.shape[0] if n is None else n,), name)
    return t.shape[0]


def page_extend(K_pages: torch.Tensor, V_pages: torch.Tensor, page_table: torch.Tensor,
                kv_lens: torch.Tensor, ref_counts: torch.Tensor, add: torch.Tensor) -> torch.Tensor:
    """Room for ``add [S]`` (int32) more tokens of each sequence: takes free pages (lowest first, by
    the sequences in row order), writes them into ``page_table`` and adds to ``kv_lens``.  A partly
    filled last page that other sequences hold too is copied, in all layers, before it is written to
    (where all its holders write, the first keeps it).  Returns ``granted [S]`` bool; a sequence that
    is not granted -- the free pages or its row of the table do not suffice -- is left as it was, and
    has no places for its new tokens: see ``granted`` of :func:`rope_append_paged`."""
    dev = _on_gpu(page_table, kv_lens, ref_counts, add, K_pages, V_pages)
    st = _state(page_table, kv_lens, ref_counts)
    pools, P, page = _pools(K_pages, V_pages)
    if P != st[6]:
        raise ValueError(f"ref_counts has {st[6]} entries, the pools have {P} pages")
    _vector(add, "add", st[4])
    granted = add.new_empty(st[4], dtype=torch.bool)
    ws, nbytes = _workspace(st[4], 0, 0, add)
    _call(dev, N.load().dpk_page_extend, *st, page, add.data_ptr(), granted.data_ptr(), *pools, ws.data_ptr(), nbytes)
    return granted


def page_fork(page_table: torch.Tensor, kv_lens: torch.Tensor, ref_counts: torch.Tensor,
              parents: torch.Tensor, children: torch.Tensor, page_size: int) -> torch.Tensor:
    """Rows ``children [n]`` become second holders of all pages of rows ``parents [n]``; nothing is
    copied (:func:`page_extend` does that when one of them writes).  A child has to be an empty row
    that no earlier pair names.  Returns ``done [n]`` bool."""
    dev = _on_gpu(page_table, kv_lens, ref_counts, parents, children)
    st = _state(page_table, kv_lens, ref_counts)
    n = _vector(parents, "parents")
    _vector(children, "children", n)
    done = parents.new_empty(n, dtype=torch.bool)
    ws, nbytes = _workspace(0, 0, n, parents)
    _call(dev, N.load().dpk_page_fork, *st, int(page_size), parents.data_ptr(), children.data_ptr(), n,
          done.data_ptr(), ws.data_ptr(), nbytes)
    return done


def page_trim(page_table: torch.Tensor, kv_lens: torch.Tensor, ref_counts: torch.Tensor,
              rows: torch.Tensor, keep: Optional[torch.Tensor] = None, *, page_size: int) -> None:
    """Cuts sequences ``rows [n]`` to their first ``keep [n]`` tokens and lets go of the pages behind;
    without ``keep`` the sequences are freed.  A ``keep`` of at least the length does nothing; of a row
    that is named twice the first counts."""
    dev = _on_gpu(page_table, kv_lens, ref_counts, rows, keep)
    st = _state(page_table, kv_lens, ref_counts)
    n = _vector(rows, "rows")
    if keep is not None:
        _vector(keep, "keep", n)
    _call(dev, N.load().dpk_page_trim, *st, int(page_size), rows.data_ptr(),
          None if keep is None else keep.data_ptr(), n)


def page_copy(K_pages: torch.Tensor, V_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Pages ``dst [n]`` become copies of pages ``src [n]`` in all layers of both pools.  Of several
    pairs with one destination the last counts; a pair whose source is another pair's destination
    is left out and reported (:func:`dpk_b200.ops.device_status`)."""
    dev = _on_gpu(K_pages, V_pages, src, dst)
    pools, P, page = _pools(K_pages, V_pages)
    n = _vector(src, "src")
    _vector(dst, "dst", n)
    ws, nbytes = _workspace(0, P, n, src)
    _call(dev, N.load().dpk_page_copy, *pools, P, page, src.data_ptr(), dst.data_ptr(), n, ws.data_ptr(), nbytes)


def page_compact(K_pages: torch.Tensor, V_pages: torch.Tensor, page_table: torch.Tensor,
                 kv_lens: torch.Tensor, ref_counts: torch.Tensor) -> torch.Tensor:
    """Moves the held pages to the front of the pools (each hole, in ascending order, takes the next
    held page behind), rewrites ``page_table`` and ``ref_counts``.  Returns their number, int32 ``[1]``:
    pages from there on are free.  An entry whose page nobody holds by the counts is reported and becomes -1."""
    dev = _on_gpu(page_table, kv_lens, ref_counts, K_pages, V_pages)
    st = _state(page_table, kv_lens, ref_counts)
    pools, P, page = _pools(K_pages, V_pages)
    if P != st[6]:
        raise ValueError(f"ref_counts has {st[6]} entries, the pools have {P} pages")
    live = kv_lens.new_empty(1)
    ws, nbytes = _workspace(0, P, 0, kv_lens)
    _call(dev, N.load().dpk_page_compact, *pools, *st, page, live.data_ptr(), ws.data_ptr(), nbytes)
    return live
