"""A paged KV cache on the gfx950 HIP kernels: attention of chunks of new
tokens over it, the write of their rows into it, the cached rows' attention
weights, and eviction by them.

The cached rows of a sequence lie in pages of ``page_size`` rows (a multiple
of 16) anywhere in a pool: row j of sequence b is row ``j % page_size`` of page
``block_table[b, j // page_size]``.  Pools are ``k_pages`` / ``v_pages``
``[pages, H_KV, page_size, D]`` and, with the graph bias, ``rk_pages``
``[pages, H_G, page_size, R]``, with any strides but a unit feature stride and
16-byte aligned rows.  A row whose page id is outside the pool is not there:
it is neither read nor written.  Sequences may share pages for reading.  Pools
that a call writes (``paged_append``, ``paged_evict``) hold no two rows in one
memory: expanded ones are refused.

The new tokens of a call are packed, as in ``flash_naylis_attn``'s varlen
mode: tokens ``[cu_seqlens_q[b], cu_seqlens_q[b + 1])`` belong to sequence b.
They are the last rows of its cache: ``seqlens_k[b]`` counts the rows in use,
theirs included.  One token a sequence is a decode step, a piece of a prompt a
prefill, and one call may hold both, and sequences without a token.  Rows
past those that the table has room for are not there: the append drops their
tokens, attention sees the rows before them, eviction takes the table's rows
for all.

A step of a server is ``paged_append`` (q and k normalised and rotated, k, v
and R_k into their pages), then ``flash_naylis_paged``; where the cache has
outgrown its budget, ``paged_evict`` by the ``key_weights`` that the attention
calls added up.

The reference's multi-token step against a cache runs PyTorch SDPA without
the bias, or fails with it (FNA2/attention_fna2.py:412-429, :445-473).  All
lengths and tables stay on the device: none of the three functions
synchronises (given device tensors), and each can be captured into a graph.  How
they run (parts, buffers) goes by the table's width, not by the lengths, which the
host does not know: a table not much wider than its sequences' pages serves them
best.  ``PageTable`` keeps its books on the host, and each of its methods waits for
the stream while it uploads them.  Forward only (no autograd).  There is no
fallback: without the HIP library, or off the GPU, the calls raise.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _capi

_DTYPES = {torch.bfloat16: _capi.FNA2_BF16, torch.float16: _capi.FNA2_F16}


def _gpu(t: torch.Tensor, name: str, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on the gfx950 HIP kernel: {name} must be on the GPU")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[T, heads, F] as the kernels read it: unit feature stride, 16-byte
    aligned rows, else a contiguous copy."""
    ok = (t.stride(2) == 1 and t.data_ptr() % 16 == 0
          and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0)
    return t if ok else t.contiguous()


def _t3(t: Optional[torch.Tensor]) -> _capi.Tensor:
    if t is None or t.numel() == 0:
        return _capi.empty_tensor()
    return _capi.Tensor(t.data_ptr(), 0, t.stride(0), t.stride(1))


def _pool(t: Optional[torch.Tensor]) -> _capi.Tensor:
    if t is None or t.numel() == 0:
        return _capi.empty_tensor()
    return _capi.Tensor(t.data_ptr(), t.stride(0), t.stride(2), t.stride(1))


def _ints(t: torch.Tensor, device) -> torch.Tensor:
    return t.to(device=device, dtype=torch.int32).contiguous()


def _f32(t: Optional[torch.Tensor], device) -> Optional[torch.Tensor]:
    return None if t is None else t.detach().to(device=device, dtype=torch.float32).contiguous()


def _written(t: torch.Tensor, name: str) -> None:
    """A tensor that a call writes in place, as ``copy_`` would."""
    assert not t.requires_grad, f"{name} is written in place and cannot require a gradient"
    if t.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError(f"{name}: an inference tensor is written in inference mode only")


def _written_pools(what: str, k_pages, v_pages, rk_pages) -> None:
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("rk_pages", rk_pages)):
        if t is not None:
            _written(t, name)
    assert k_pages.numel() == 0 or k_pages.data_ptr() != v_pages.data_ptr(), \
        f"{what}: k_pages and v_pages are one memory, and both are written"


def _bump(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _cache(what: str, k_pages, v_pages, block_table, seqlens_k, heads: int, rk_pages=None,
           heads_graph: int = 0):
    """(PagedCache, tensors kept alive) of a call's cache."""
    dev = k_pages.device
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("rk_pages", rk_pages)):
        if t is None:
            continue
        assert t.dim() == 4, f"{what}: {name} must be [pages, heads, page_size, features]"
        _gpu(t, name, what)
        assert t.device == dev, f"{what}: {name} is on another device"
        if t.numel() and not (t.stride(3) == 1 and t.data_ptr() % 16 == 0
                              and all(s % 8 == 0 for s in t.stride()[:3])):
            raise AssertionError(f"{what}: {name} needs a unit feature stride and 16-byte aligned "
                                 "rows (it is used in place, never copied)")
    assert k_pages.dtype in _DTYPES, f"{what}: k_pages must be bfloat16 or float16"
    assert v_pages.dtype == k_pages.dtype and v_pages.shape == k_pages.shape, \
        f"{what}: k_pages and v_pages must have one shape and dtype"
    pages, hkv, ps, D = k_pages.shape
    if rk_pages is not None:
        assert rk_pages.dtype == torch.bfloat16, f"{what}: rk_pages must be bfloat16"
        assert rk_pages.shape[0] == pages and rk_pages.shape[2] == ps, \
            f"{what}: rk_pages must have the pages of k_pages"
        assert rk_pages.shape[1] == heads_graph, f"{what}: rk_pages must hold the graph heads"
    assert block_table.dim() == 2, f"{what}: block_table must be [sequences, pages]"
    table = block_table.to(device=dev, dtype=torch.int32)
    if table.stride(1) != 1 and table.shape[1] > 1 or table.stride(0) < table.shape[1]:
        table = table.contiguous()
    lens = _ints(seqlens_k, dev)
    N = table.shape[0]
    assert lens.shape == (N,), f"{what}: seqlens_k must hold one length a sequence"
    c = _capi.PagedCache()
    c.dtype = _DTYPES[k_pages.dtype]
    c.batch, c.heads, c.heads_kv, c.heads_graph = N, int(heads), hkv, int(heads_graph)
    c.head_dim, c.rank = D, 0 if rk_pages is None else rk_pages.shape[3]
    c.num_pages, c.page_size, c.table_width = pages, ps, table.shape[1]
    c.block_table, c.table_stride = table.data_ptr(), table.stride(0)
    c.seqlens_k = lens.data_ptr()
    c.k_pages, c.v_pages, c.rk_pages = _pool(k_pages), _pool(v_pages), _pool(rk_pages)
    return c, (table, lens)


def _chunk(what: str, c: _capi.PagedCache, cu_seqlens_q, total: int, max_q: int, dev):
    cu = _ints(cu_seqlens_q, dev)
    assert cu.shape == (c.batch + 1,), f"{what}: cu_seqlens_q must hold one entry a sequence and one more"
    assert int(max_q) >= 0, f"{what}: max_seqlen_q must not be negative"
    c.total_q, c.max_seqlen_q = int(total), min(int(max_q), int(total))
    c.cu_seqlens_q = cu.data_ptr()
    return cu


def _stream(dev) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _new_rows(what, name, t, T, heads, feat, dtype, dev):
    assert t.dim() == 3 and tuple(t.shape) == (T, heads, feat), \
        f"{what}: {name} must be [{T}, {heads}, {feat}]"
    assert t.dtype == dtype, f"{what}: {name} must be {dtype}"
    _gpu(t, name, what)
    assert t.device == dev, f"{what}: {name} is on another device"
    return _rows(t.detach())


def flash_naylis_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       block_table: torch.Tensor, seqlens_k: torch.Tensor,
                       cu_seqlens_q: torch.Tensor, max_seqlen_q: int,
                       r_q: Optional[torch.Tensor] = None,
                       rk_pages: Optional[torch.Tensor] = None,
                       graph_scale: Optional[torch.Tensor] = None,
                       softmax_scale: Optional[float] = None, is_causal: bool = True,
                       key_weights: Optional[torch.Tensor] = None, return_lse: bool = False
                       ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of packed chunks of new tokens over a paged cache.

    q ``[T, H, D]`` (bf16 or fp16, as the pools), r_q ``[T, H_G, R]`` bf16,
    graph_scale ``[H_G]`` (the bias: r_q, rk_pages and graph_scale, or none of
    them).  ``max_seqlen_q`` is a hint of the longest chunk (it
    picks the kernels, not the result).  Causal: token i of a chunk of lq sees
    rows ``0 .. seqlens_k - lq + i``; not causal: all ``seqlens_k``.  Hidden rows
    do not reach a token's result, whatever they hold; a token that sees no row,
    and a token of no sequence, gives zeros.

    key_weights ``[N, H_KV, capacity]`` fp32, rows contiguous: every cached
    row's softmax weight, summed over the chunk's tokens and the query heads of
    the KV head, is added to it (rows at or past ``capacity`` are left out).

    Returns out ``[T, H, D]`` (and the fp32 LSE ``[T, H]``)."""
    what = "flash_naylis_paged"
    nat = _capi.native_or_none() if q.is_cuda else None
    if nat is not None:  # the native launch path (None: a call it leaves to the code below)
        done = nat.paged_attn(
            q, k_pages, v_pages, block_table, seqlens_k, cu_seqlens_q, int(max_seqlen_q), r_q,
            rk_pages, graph_scale,
            float(q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale),
            bool(is_causal), key_weights, return_lse)
        if done is not None:
            return done if return_lse else done[0]
    assert q.dim() == 3, f"{what}: q must be [T, H, D]"
    dev = k_pages.device
    T, H, D = q.shape
    H_G = R = 0
    if r_q is None:
        assert rk_pages is None and graph_scale is None, \
            f"{what}: rk_pages and graph_scale need r_q"
    else:
        assert rk_pages is not None and graph_scale is not None, \
            f"{what}: r_q needs rk_pages and graph_scale"
        assert r_q.dim() == 3, f"{what}: r_q must be [T, H_G, R]"
        H_G, R = r_q.shape[1], r_q.shape[2]
    c, keep = _cache(what, k_pages, v_pages, block_table, seqlens_k, H,
                     rk_pages if H_G else None, H_G)
    assert c.head_dim == D, f"{what}: q and the pools disagree on the head dimension"
    q = _new_rows(what, "q", q, T, H, D, k_pages.dtype, dev)
    cu = _chunk(what, c, cu_seqlens_q, T, max_seqlen_q, dev)
    a = _capi.PagedAttnArgs()
    gs = None
    if H_G:
        r_q = _new_rows(what, "r_q", r_q, T, H_G, R, torch.bfloat16, dev)
        assert R == c.rank, f"{what}: r_q and rk_pages disagree on the rank"
        gs = _f32(graph_scale, dev)
        assert gs.numel() == H_G, f"{what}: graph_scale must hold H_G values"
        a.r_q, a.graph_scale = _t3(r_q), gs.data_ptr()
    a.c = c
    a.causal = int(bool(is_causal))
    a.softmax_scale = float(softmax_scale) if softmax_scale is not None else D ** -0.5
    w = key_weights
    if w is not None:
        assert w.dim() == 3 and w.shape[:2] == (c.batch, c.heads_kv) and w.dtype == torch.float32, \
            f"{what}: key_weights must be [sequences, H_KV, capacity] float32"
        _gpu(w, "key_weights", what)
        assert w.device == dev and (w.stride(2) == 1 or w.shape[2] <= 1), \
            f"{what}: key_weights needs contiguous rows on the pools' device"
        _written(w, "key_weights")
    out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    lse = None
    if return_lse or w is not None:
        lse = torch.empty((H, T), dtype=torch.float32, device=dev).t()
        a.lse = _t3(lse)
    a.q, a.out = _t3(q), _t3(out)
    lib = _capi.lib()
    _capi.raise_for(lib.fna2_check_paged_attn(ctypes.byref(a)), what)
    wa = scores = None
    if w is not None:
        # (with room for the scores, where they save a second reading of K and
        # the memory is there)
        nbytes = lib.fna2_paged_scores_bytes(ctypes.byref(a))
        try:
            if nbytes:
                scores = torch.empty(nbytes, dtype=torch.uint8, device=dev)
                a.scores, a.scores_bytes = scores.data_ptr(), nbytes
        except torch.OutOfMemoryError:
            pass
        wa = _capi.PagedWeightsArgs()
        wa.attn = a
        wa.key_weights = w.data_ptr()
        wa.stride_b, wa.stride_h, wa.capacity = w.stride(0), w.stride(1), w.shape[2]
        _capi.raise_for(lib.fna2_check_paged_weights(ctypes.byref(wa)), what)
    if T > 0:
        nbytes = lib.fna2_paged_attn_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
        with torch.cuda.device(dev):
            _capi.raise_for(lib.fna2_paged_attn(ctypes.byref(a), _stream(dev)), what)
            if wa is not None:
                _capi.raise_for(lib.fna2_paged_weights(ctypes.byref(wa), _stream(dev)), what)
                _bump(w)
    del keep, cu, gs, scores
    return (out, lse) if return_lse else out


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, block_table: torch.Tensor, seqlens_k: torch.Tensor,
                 cu_seqlens_q: torch.Tensor, r_k: Optional[torch.Tensor] = None,
                 rk_pages: Optional[torch.Tensor] = None,
                 inv_freq: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None,
                 norm_q: Optional[torch.Tensor] = None, norm_k: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, position_shift: Optional[torch.Tensor] = None
                 ) -> torch.Tensor:
    """The new tokens' rows, in one launch: q ``[T, H, D]`` and k ``[T, H_KV,
    D]`` RMS-normalised by ``norm_q`` / ``norm_k`` ``[D]`` (each optional) and
    rotated by ``inv_freq`` ``[D / 2]`` (optional), k, v and r_k ``[T, H_G, R]``
    (bf16) written to their pages.  Returns the new q ``[T, H, D]``.

    The chain is evaluated in fp32 (the angle in fp64) and rounded once, as
    ``rope_varlen`` with a norm does.  A token's position is its cache row, or
    ``positions[t]`` (int32), plus ``position_shift[b]`` (int32 ``[N]``) of its
    sequence: after an eviction a sequence's rows and positions differ by a
    number.  ``seqlens_k`` counts the rows after the append.  Rows before 0 or
    past the table are not stored (no other row gives way to them); tokens of no
    sequence keep their q and store nothing.  Pages that are written may belong
    to one sequence only."""
    what = "paged_append"
    nat = _capi.native_or_none() if q.is_cuda else None
    if nat is not None:
        done = nat.paged_append(q, k, v, k_pages, v_pages, block_table, seqlens_k, cu_seqlens_q,
                                r_k, rk_pages, inv_freq, positions, norm_q, norm_k, float(eps),
                                position_shift)
        if done is not None:
            return done
    assert q.dim() == 3 and k.dim() == 3, f"{what}: q [T, H, D] and k [T, H_KV, D] expected"
    dev = k_pages.device
    T, H, D = q.shape
    H_G = R = 0
    if r_k is not None or rk_pages is not None:
        assert r_k is not None and rk_pages is not None, f"{what}: r_k and rk_pages go together"
        assert r_k.dim() == 3, f"{what}: r_k must be [T, H_G, R]"
        H_G, R = r_k.shape[1], r_k.shape[2]
    c, keep = _cache(what, k_pages, v_pages, block_table, seqlens_k, H, rk_pages if H_G else None,
                     H_G)
    dt = k_pages.dtype
    q = _new_rows(what, "q", q, T, H, c.head_dim, dt, dev)
    k = _new_rows(what, "k", k, T, c.heads_kv, c.head_dim, dt, dev)
    v = _new_rows(what, "v", v, T, c.heads_kv, c.head_dim, dt, dev)
    cu = _chunk(what, c, cu_seqlens_q, T, T, dev)
    a = _capi.PagedAppendArgs()
    if H_G:
        r_k = _new_rows(what, "r_k", r_k, T, H_G, R, torch.bfloat16, dev)
        assert R == c.rank, f"{what}: r_k and rk_pages disagree on the rank"
        a.r_k = _t3(r_k)
    a.c = c
    inv, wq, wk = _f32(inv_freq, dev), _f32(norm_q, dev), _f32(norm_k, dev)
    assert inv is None or inv.numel() == D // 2, f"{what}: inv_freq must hold head_dim / 2 frequencies"
    for n in (wq, wk):
        assert n is None or n.numel() == D, f"{what}: norm weights must hold head_dim values"
    pos = None
    if positions is not None:
        assert inv is not None, f"{what}: positions need inv_freq"
        pos = _ints(positions, dev)
        assert pos.shape == (T,), f"{what}: positions must hold one position a token"
    shift = None
    if position_shift is not None:
        assert inv is not None, f"{what}: position_shift needs inv_freq"
        shift = _ints(position_shift, dev)
        assert shift.shape == (c.batch,), f"{what}: position_shift must hold one number a sequence"
    _written_pools(what, k_pages, v_pages, rk_pages)
    out = torch.empty((T, H, D), dtype=dt, device=dev)
    a.q, a.k, a.v, a.q_out = _t3(q), _t3(k), _t3(v), _t3(out)
    a.positions = None if pos is None else pos.data_ptr()
    a.inv_freq = None if inv is None else inv.data_ptr()
    a.norm_q = None if wq is None else wq.data_ptr()
    a.norm_k = None if wk is None else wk.data_ptr()
    a.eps = float(eps)
    lib = _capi.lib()
    _capi.raise_for(lib.fna2_check_paged_append(ctypes.byref(a)), what)
    with torch.cuda.device(dev):
        _capi.raise_for(lib.fna2_paged_append_shifted(
            ctypes.byref(a), None if shift is None else shift.data_ptr(), _stream(dev)), what)
    _bump(k_pages, v_pages, rk_pages if H_G else None)
    del keep, cu
    return out


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                seqlens_k: torch.Tensor, key_weights: torch.Tensor, budget: int, recent: int = 0,
                first: int = 0, rk_pages: Optional[torch.Tensor] = None,
                heads: Optional[int] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Brings every sequence with more than ``budget`` cached rows back to
    ``budget``: each KV head keeps its first ``first`` and last ``recent`` rows
    and, between them, those of largest weight in ``key_weights`` ``[N, H_KV,
    capacity]`` (fp32; NaN above all others, equal weights: the lower row; rows
    at or past ``capacity`` weigh 0).  The kept rows move up in their order, in
    place, to be rows ``0 .. budget - 1``; R_k rows move with their KV head's
    (``heads``: the query heads, which say whose).  Rows past the new length
    keep what they held.  A sequence's pages may not be shared with another of
    the call.

    Returns (kept ``[N, H_KV, budget]`` int32, the rows kept, then -1;
    the new lengths ``[N]`` int32; the kept rows' weights ``[N, H_KV,
    capacity]``, then 0).  ``seqlens_k`` and ``key_weights`` are not written."""
    what = "paged_evict"
    dev = k_pages.device
    H_G = 0 if rk_pages is None else rk_pages.shape[1]
    if H_G:
        assert heads is not None, f"{what}: rk_pages needs heads, the number of query heads"
    nat = _capi.native_or_none() if k_pages.is_cuda else None
    if nat is not None:
        done = nat.paged_evict(k_pages, v_pages, block_table, seqlens_k, key_weights, int(budget),
                               int(recent), int(first), rk_pages,
                               int(heads if heads is not None else k_pages.shape[1]))
        if done is not None:
            return done
    c, keep = _cache(what, k_pages, v_pages, block_table, seqlens_k,
                     heads if heads is not None else k_pages.shape[1], rk_pages if H_G else None,
                     H_G)
    w = key_weights
    assert w.dim() == 3 and w.shape[:2] == (c.batch, c.heads_kv) and w.dtype == torch.float32, \
        f"{what}: key_weights must be [sequences, H_KV, capacity] float32"
    _gpu(w, "key_weights", what)
    assert w.device == dev, f"{what}: key_weights is on another device"
    if w.stride(2) != 1 and w.shape[2] > 1:
        w = w.contiguous()
    _written_pools(what, k_pages, v_pages, rk_pages)
    assert 0 <= int(budget) < 1 << 31 and 0 <= int(recent) and 0 <= int(first) and \
        int(recent) + int(first) <= int(budget), f"{what}: 0 <= first + recent <= budget expected"
    N, hkv = c.batch, c.heads_kv
    # (more rows than the table has room for are never kept)
    kept = torch.empty((N, hkv, int(budget)), dtype=torch.int32, device=dev)
    lens = torch.empty((N,), dtype=torch.int32, device=dev)
    w_out = torch.empty((N, hkv, w.shape[2]), dtype=torch.float32, device=dev)
    a = _capi.PagedEvictArgs()
    a.c = c
    a.budget, a.recent, a.first = int(budget), int(recent), int(first)
    a.key_weights = w.data_ptr() or None
    a.stride_b, a.stride_h, a.capacity = w.stride(0), w.stride(1), w.shape[2]
    a.weights_out = w_out.data_ptr() or None
    a.kept, a.new_lens = kept.data_ptr() or None, lens.data_ptr() or None
    lib = _capi.lib()
    _capi.raise_for(lib.fna2_check_paged_evict(ctypes.byref(a)), what)
    with torch.cuda.device(dev):
        _capi.raise_for(lib.fna2_paged_evict(ctypes.byref(a), _stream(dev)), what)
    _bump(k_pages, v_pages, rk_pages if H_G else None)
    del keep
    return kept, lens, w_out


class PageTable:
    """Which pages hold the rows of which sequence: one for all the layers of
    a model, whose pools (``PagedKVCache``) all have its pages.

    ``extend(counts)`` takes in the new tokens of a step; ``block_table``
    ``[sequences, max_pages]``, ``seqlens`` and ``position_shift``
    ``[sequences]`` and ``cu_seqlens_q`` (int32) then describe them for every
    layer.  These are on the device and written in place, so that captured
    graphs read the step at hand (of as many tokens as the captured one).
    ``max_seqlen_q`` and ``total_q`` are numbers.  A token's position is its row
    plus its sequence's ``position_shift``, the rows that ``truncate`` took away
    before it; ``positions`` are those of the step's tokens one by one, a tensor
    of this step only.  The bookkeeping is the host's: nothing is read back from
    the device, but each upload (one, and the block table where pages changed)
    waits for the stream's earlier work."""

    def __init__(self, sequences: int, num_pages: int, page_size: int = 64,
                 max_pages: Optional[int] = None, device=None):
        assert page_size > 0 and page_size % 16 == 0, "page_size must be a multiple of 16"
        assert sequences >= 0 and num_pages >= 0
        self.page_size, self.num_pages = int(page_size), int(num_pages)
        self.width = int(num_pages if max_pages is None else max_pages)
        self.rows = [0] * sequences       # rows in use
        self.next_position = [0] * sequences
        self.pages = [[] for _ in range(sequences)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._host = torch.full((sequences, self.width), -1, dtype=torch.int32)
        self.block_table = self._host.to(device)
        self._cu = [0] * (sequences + 1)
        # [seqlens | position_shift | cu_seqlens_q], uploaded in one copy
        self._step = torch.zeros(3 * sequences + 1, dtype=torch.int32, device=device)
        self.seqlens, self.position_shift, self.cu_seqlens_q = self._step.split(
            [sequences, sequences, sequences + 1])
        self.max_seqlen_q = self.total_q = 0
        self._positions: Optional[Sequence[int]] = None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def positions(self) -> Optional[torch.Tensor]:
        """[total_q] int32: the positions of the last ``extend``'s tokens, a new
        tensor; None: a token's row, in every sequence."""
        if self._positions is None:
            return None
        return torch.tensor(self._positions, dtype=torch.int32, device=self.seqlens.device)

    def token_positions(self, tokens: int, cu_seqlens_q: Optional[torch.Tensor] = None
                        ) -> torch.Tensor:
        """[tokens] positions of a step's packed tokens, formed on the device from
        what this table keeps there, so that a captured step forms its own anew.
        (Tokens of no sequence: any number.)"""
        row = torch.arange(tokens, device=self.seqlens.device)
        if not self.rows:
            return row
        cu = self.cu_seqlens_q if cu_seqlens_q is None else _ints(cu_seqlens_q, row.device)
        b = torch.searchsorted(cu[1:], row.to(cu.dtype), right=True).clamp(max=len(self.rows) - 1)
        return row - cu[b + 1] + self.seqlens[b] + self.position_shift[b]

    def _upload(self, table: bool) -> None:
        shift = [p - r for r, p in zip(self.rows, self.next_position)]
        self._step.copy_(torch.tensor(self.rows + shift + self._cu, dtype=torch.int32))
        if table:
            self.block_table.copy_(self._host)

    def _give_back(self, b: int, keep: int) -> bool:
        if len(self.pages[b]) <= keep:
            return False
        self._free += reversed(self.pages[b][keep:])
        del self.pages[b][keep:]
        self._host[b, keep:] = -1
        return True

    def extend(self, counts: Sequence[int]) -> None:
        """counts[b] new tokens for sequence b (0: none this step).  Raises
        ValueError, with nothing changed, where the pages do not suffice."""
        counts = [int(c) for c in counts]
        assert len(counts) == len(self.rows) and all(c >= 0 for c in counts), \
            "one count for each sequence"
        ps = self.page_size
        need = [-(-(r + c) // ps) for r, c in zip(self.rows, counts)]
        more = [max(n - len(p), 0) for n, p in zip(need, self.pages)]
        if max(need, default=0) > self.width:
            raise ValueError(f"PageTable full: a sequence needs {max(need)} pages, "
                             f"its table holds {self.width}")
        if sum(more) > len(self._free):
            raise ValueError(f"PageTable full: {sum(more)} pages needed, {len(self._free)} free")
        for b, m in enumerate(more):
            for _ in range(m):
                self._host[b, len(self.pages[b])] = self._free[-1]
                self.pages[b].append(self._free.pop())
        cu, pos = [0], []
        moved = self.rows != self.next_position
        for b, c in enumerate(counts):
            cu.append(cu[-1] + c)
            if moved:
                pos += range(self.next_position[b], self.next_position[b] + c)
            self.rows[b] += c
            self.next_position[b] += c
        self._cu = cu
        self.total_q, self.max_seqlen_q = cu[-1], max(counts, default=0)
        self._positions = pos if moved else None
        self._upload(any(more))

    def truncate(self, budget: int) -> None:
        """After every layer's ``PagedKVCache.evict(budget)``: no sequence has
        more than ``budget`` rows, and the pages behind them are free.  The
        positions of the tokens to come go on counting."""
        self.rows = [min(r, int(budget)) for r in self.rows]
        freed = [self._give_back(b, -(-r // self.page_size)) for b, r in enumerate(self.rows)]
        self._upload(any(freed))

    def release(self, b: int) -> None:
        """Sequence b is done: its pages are free, and its place for another."""
        self.rows[b] = self.next_position[b] = 0
        self._give_back(b, 0)
        self._upload(True)


class PagedKVCache:
    """One layer's pools on the pages of a ``PageTable``: a ``past_kv`` of
    ``NaylisAttention`` that serves many sequences of differing lengths, prompts
    in pieces and single tokens in one call.

    ``k``, ``v`` ``[pages, H_KV, page_size, D]``, ``r_k`` ``[pages, H_G,
    page_size, R]`` (bf16) for a layer with graph heads.  With ``weigh`` the
    layer's calls add up each cached row's attention weight (``key_weights``
    ``[sequences, H_KV, max_pages * page_size]``), by which ``evict`` goes."""

    def __init__(self, table: PageTable, k: torch.Tensor, v: torch.Tensor,
                 r_k: Optional[torch.Tensor] = None, key_weights: Optional[torch.Tensor] = None):
        assert k.shape == v.shape and k.dim() == 4 and k.shape[0] == table.num_pages and \
            k.shape[2] == table.page_size, "k and v must be [pages, H_KV, page_size, D]"
        assert r_k is None or (r_k.dim() == 4 and r_k.shape[0] == k.shape[0]
                               and r_k.shape[2] == k.shape[2]), \
            "r_k must be [pages, H_G, page_size, R]"
        self.table, self.k, self.v, self.r_k, self.key_weights = table, k, v, r_k, key_weights

    @classmethod
    def empty(cls, table: PageTable, n_kv_heads: int, head_dim: int, graph_heads: int = 0,
              rank: int = 0, dtype=torch.bfloat16, weigh: bool = False) -> "PagedKVCache":
        dev, ps = table.block_table.device, table.page_size
        mk = lambda h, f, dt: torch.zeros(table.num_pages, h, ps, f, dtype=dt, device=dev)
        w = torch.zeros(len(table.rows), n_kv_heads, table.width * ps, device=dev) if weigh else None
        return cls(table, mk(n_kv_heads, head_dim, dtype), mk(n_kv_heads, head_dim, dtype),
                   mk(graph_heads, rank, torch.bfloat16) if graph_heads > 0 else None, w)

    def evict(self, budget: int, recent: int = 0, first: int = 0,
              heads: Optional[int] = None) -> torch.Tensor:
        """``paged_evict`` of this layer by its ``key_weights`` (``heads``: the
        layer's query heads, needed with ``r_k``); returns the rows kept.  When
        every layer has done so, ``PageTable.truncate(budget)``."""
        assert self.key_weights is not None, "evict: this cache does not weigh its rows"
        t = self.table
        kept, _, w = paged_evict(self.k, self.v, t.block_table, t.seqlens, self.key_weights,
                                 budget, recent, first, self.r_k, heads)
        self.key_weights.copy_(w)
        return kept

    def forget(self, b: int) -> None:
        """Sequence b's place is for another: its weights start at 0 (after
        ``PageTable.release(b)``, in every layer)."""
        if self.key_weights is not None:
            self.key_weights[b].zero_()
