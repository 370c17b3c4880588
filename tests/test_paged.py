"""The paged cache (fna2_paged_attn, _weights, _append, _evict) against
``oracle.paged_oracle``.

CPU: the C ABI's validation and struct layouts, the Python entry points'
refusals, the oracle against the attention oracle and torch.
GPU: every operator over small sizes where it can go wrong, and runs of them
together.

Tolerances, with h = eps / 2 of the output type (bf16 2^-8, fp16 2^-11):
* out: its own rounding, h |out|, and P's, h times the same average of |V|
  (P is rounded to the type at most once, relatively), plus 2e-4 of that
  average for fp32 scores: |S| sums 128 products of order one, whose fp32 sum is
  off by at most 128 * 2^-24 * sum |q_i k_i| scale < 1e-4 for the draws here,
  and exp and the sums add a few 2^-24.
* LSE: 1e-4 by the same sum; weights: relatively 2e-4 (S and LSE).
* append: h |y| and 1e-5 for the fp32 chain (values of order one).
* eviction: equal.
"""
import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from fna2_amd import _capi, paged
from oracle import fna2_oracle as O
from oracle import paged_oracle as PO

ROOT = Path(__file__).resolve().parents[1]
FAKE = 1 << 20
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def lib():
    return _capi.lib()


# ── building caches ──────────────────────────────────────────────────────────

class Case:
    """A cache in pages that lie in no order, and a chunk of new tokens."""

    def __init__(self, lq, lk, H, HKV, HG, D, R, ps, dtype=torch.bfloat16, seed=0, device="cpu",
                 layout="phrd", spare=3, width=None, tail=0, head=0):
        g = torch.Generator().manual_seed(seed)
        N = len(lk)
        used = [-(-n // ps) for n in lk]
        width = max(used + [1]) + 1 if width is None else width
        P = sum(used) + spare
        perm = torch.randperm(P, generator=g).to(torch.int32)
        table = torch.full((N, width), -1, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = perm[at:at + u]
            at += u
        cu = [head]
        for n in lq:
            cu.append(cu[-1] + n)
        T = cu[-1] + tail
        randn = lambda *s, std=1.0: torch.randn(*s, generator=g) * std

        def pool(heads, feat, dt, std=1.0):
            if layout == "prhd":  # rows of all heads together
                return (randn(P, ps, heads, feat, std=std)).to(dt).to(device).transpose(1, 2)
            return randn(P, heads, ps, feat, std=std).to(dt).to(device)

        to = lambda t: t.to(device)
        self.N, self.T, self.H, self.HKV, self.HG, self.D, self.R, self.ps = N, T, H, HKV, HG, D, R, ps
        self.lq, self.lk, self.used, self.P, self.width = lq, lk, used, P, width
        self.k, self.v = pool(HKV, D, dtype), pool(HKV, D, dtype)
        self.rk = pool(HG, R, torch.bfloat16, R ** -0.5) if HG else None
        self.table, self.lens = to(table), to(torch.tensor(lk, dtype=torch.int32))
        self.cu = to(torch.tensor(cu, dtype=torch.int32))
        self.q = to(randn(T, H, D).to(dtype))
        self.rq = to(randn(T, HG, R, std=R ** -0.5).bfloat16()) if HG else None
        self.gs = to(1 + randn(HG)) if HG else None
        self.kn, self.vn = to(randn(T, HKV, D).to(dtype)), to(randn(T, HKV, D).to(dtype))
        self.rkn = to(randn(T, HG, R).bfloat16()) if HG else None
        self.max_q = max(lq + [0])
        self.dtype, self.device = dtype, device

    def attend(self, hint=None, **kw):
        return paged.flash_naylis_paged(self.q, self.k, self.v, self.table, self.lens, self.cu,
                                        self.max_q if hint is None else hint, r_q=self.rq,
                                        rk_pages=self.rk, graph_scale=self.gs, **kw)

    def oracle(self, scale=None, causal=True):
        return PO.attend(self.q, self.k, self.v, self.table, self.lens, self.cu, self.rq, self.rk,
                         self.gs, scale, causal)

    def slot(self, b, j):
        return int(self.table[b, j // self.ps]), j % self.ps


def close_out(c, got, ref, mag):
    got = got.double().cpu().numpy()
    h = HALF[c.dtype]
    lim = h * np.abs(ref) + (h + 2e-4) * mag + 1e-7
    bad = ~(np.abs(got - ref) <= lim)
    assert not bad.any(), f"{bad.sum()} of {bad.size}: worst {np.nanmax(np.abs(got - ref) / lim):.2f} of the bound"


def check_attend(c, scale=None, causal=True, hint=None, weights=True):
    ref, lse, w, mag = c.oracle(scale, causal)
    acc = torch.rand(c.N, c.HKV, c.width * c.ps, generator=torch.Generator().manual_seed(1)).to(c.device)
    before = acc.double().cpu().numpy()
    out, got_lse = c.attend(hint, softmax_scale=scale, is_causal=causal, return_lse=True,
                            key_weights=acc if weights else None)
    torch.cuda.synchronize()
    close_out(c, out, ref, mag)
    got_lse = got_lse.double().cpu().numpy()
    assert (np.isneginf(got_lse) == np.isneginf(lse)).all()
    fin = np.isfinite(lse)
    assert np.abs(got_lse[fin] - lse[fin]).max(initial=0) <= 1e-4
    if weights:
        got = acc.double().cpu().numpy()
        assert (np.abs(got - (before + w)) <= 2e-4 * w + 2.0 ** -23 * (before + w)).all()
    return out


# ── CPU ──────────────────────────────────────────────────────────────────────

def _cache_args(**over):
    c = _capi.PagedCache()
    c.dtype, c.batch, c.total_q, c.max_seqlen_q = 1, 4, 40, 16
    c.heads, c.heads_kv, c.heads_graph, c.head_dim, c.rank = 16, 4, 12, 128, 32
    c.num_pages, c.page_size, c.table_width = 50, 64, 8
    c.block_table, c.table_stride = FAKE, 8
    c.seqlens_k = c.cu_seqlens_q = FAKE
    c.k_pages = c.v_pages = _capi.Tensor(FAKE, 4 * 64 * 128, 128, 64 * 128)
    c.rk_pages = _capi.Tensor(FAKE, 12 * 64 * 32, 32, 64 * 32)
    for k, v in over.items():
        setattr(c, k, v)
    return c


_ATTN = ("causal", "softmax_scale", "q", "r_q", "graph_scale", "out", "lse", "workspace",
         "workspace_bytes")


def _attn(**over):
    a = _capi.PagedAttnArgs()
    a.c = _cache_args(**{k: v for k, v in over.items() if k not in _ATTN})
    a.causal, a.softmax_scale = 1, 0.088
    a.q = a.out = _capi.Tensor(FAKE, 0, 16 * 128, 128)
    a.r_q = _capi.Tensor(FAKE, 0, 12 * 32, 32)
    a.graph_scale = FAKE
    a.lse = _capi.Tensor(FAKE, 0, 1, 40)
    for k, v in over.items():
        if k in _ATTN:
            setattr(a, k, v)
    return a


def _st(code):
    return _capi.STATUS[code]


NO = _capi.empty_tensor()


@pytest.mark.parametrize("over,code", [
    (dict(), "FNA2_OK"),
    (dict(dtype=2), "FNA2_OK"),
    (dict(dtype=3), "FNA2_E_DTYPE"),
    (dict(head_dim=96), "FNA2_E_HEAD_DIM"),
    (dict(heads_kv=3), "FNA2_E_HEADS"),
    (dict(heads=64, heads_kv=1, heads_graph=0), "FNA2_OK"),  # groups past 32 columns are split
    (dict(heads=16, heads_kv=1, rank=64, rk_pages=_capi.Tensor(FAKE, 12 * 64 * 64, 64, 64 * 64)),
     "FNA2_OK"),                                             # ... and ranks past one tile
    (dict(rank=64), "FNA2_E_STRIDE"),                        # rows that overlap
    (dict(heads_graph=17), "FNA2_E_HEADS"),
    (dict(rank=12), "FNA2_E_RANK"),
    (dict(rank=72), "FNA2_E_RANK"),
    (dict(heads_graph=0, rank=12, r_q=NO, graph_scale=None, rk_pages=NO), "FNA2_OK"),
    (dict(page_size=24), "FNA2_E_SHAPE"),
    (dict(page_size=0), "FNA2_E_SHAPE"),
    (dict(page_size=48), "FNA2_OK"),
    (dict(batch=-1), "FNA2_E_SHAPE"),
    (dict(total_q=-1), "FNA2_E_SHAPE"),
    (dict(max_seqlen_q=-1), "FNA2_E_SHAPE"),
    (dict(num_pages=-1), "FNA2_E_SHAPE"),
    (dict(table_width=1 << 25, table_stride=1 << 25), "FNA2_E_SHAPE"),  # past 2^30 rows
    (dict(table_stride=7), "FNA2_E_STRIDE"),
    (dict(block_table=None), "FNA2_E_NULL"),
    (dict(seqlens_k=None), "FNA2_E_SEQLENS"),
    (dict(cu_seqlens_q=None), "FNA2_E_SEQLENS"),
    (dict(k_pages=NO), "FNA2_E_NULL"),
    (dict(rk_pages=NO), "FNA2_E_NULL"),
    (dict(num_pages=0, k_pages=NO, v_pages=NO, rk_pages=NO), "FNA2_OK"),
    (dict(table_width=0, block_table=None), "FNA2_OK"),
    (dict(k_pages=_capi.Tensor(FAKE + 8, 4 * 64 * 128, 128, 64 * 128)), "FNA2_E_STRIDE"),
    (dict(k_pages=_capi.Tensor(FAKE, 4 * 64 * 128, 0, 64 * 128)), "FNA2_E_STRIDE"),
    (dict(v_pages=_capi.Tensor(FAKE, 4 * 64 * 128, 132, 64 * 128)), "FNA2_E_STRIDE"),
    (dict(v_pages=_capi.Tensor(FAKE, 0, 1 << 27, 128)), "FNA2_E_SHAPE"),
    (dict(rk_pages=_capi.Tensor(FAKE, 0, 32, 1 << 30)), "FNA2_E_SHAPE"),
    (dict(softmax_scale=float("inf")), "FNA2_E_SCALE"),
    (dict(q=NO), "FNA2_E_NULL"),
    (dict(out=NO), "FNA2_E_NULL"),
    (dict(r_q=NO), "FNA2_E_NULL"),
    (dict(graph_scale=None), "FNA2_E_NULL"),
    (dict(lse=_capi.Tensor(FAKE + 2, 0, 1, 40)), "FNA2_E_STRIDE"),
    (dict(lse=NO), "FNA2_OK"),
    (dict(total_q=0, q=NO, out=NO, r_q=NO, cu_seqlens_q=None), "FNA2_OK"),
    (dict(batch=0, seqlens_k=None, block_table=None), "FNA2_OK"),
])
def test_check_paged_attn_codes(lib, over, code):
    a = _attn(**over)
    assert _st(lib.fna2_check_paged_attn(ctypes.byref(a))) == code
    assert (lib.fna2_paged_attn_workspace_bytes(ctypes.byref(a)) > 0) == \
        (code == "FNA2_OK" and a.c.total_q > 0)


def test_check_paged_weights_codes(lib):
    def code(**over):
        w = _capi.PagedWeightsArgs()
        w.attn = _attn(**over.pop("attn", {}))
        w.key_weights, w.stride_b, w.stride_h, w.capacity = FAKE, 4 * 512, 512, 512
        for k, v in over.items():
            setattr(w, k, v)
        return _st(lib.fna2_check_paged_weights(ctypes.byref(w)))
    assert code() == "FNA2_OK"
    assert code(attn=dict(out=NO)) == "FNA2_OK"  # out is not used
    assert code(attn=dict(lse=NO)) == "FNA2_E_NULL"
    assert code(attn=dict(head_dim=32)) == "FNA2_E_HEAD_DIM"
    assert code(key_weights=None) == "FNA2_E_NULL"
    assert code(key_weights=FAKE + 2) == "FNA2_E_STRIDE"
    assert code(capacity=-1) == "FNA2_E_SHAPE"
    assert code(stride_h=500) == "FNA2_E_STRIDE"  # heads that share rows
    assert code(stride_b=0) == "FNA2_E_STRIDE"
    assert code(capacity=0, key_weights=None) == "FNA2_OK"


def test_check_paged_scores(lib):
    """The scores' size: columns by rows where few columns serve a row, else 0;
    a buffer that is too small or not aligned is refused."""
    import ctypes
    size = lambda a: lib.fna2_paged_scores_bytes(ctypes.byref(a))
    one = _attn(max_seqlen_q=1)
    assert size(one) == 4 * 4 * (8 * 64) * 4 * 4  # sequences, KV heads, rows, columns, bytes
    assert size(_attn(max_seqlen_q=8)) == 0 and size(_attn(max_seqlen_q=16)) == 0
    assert size(_attn(max_seqlen_q=1, table_width=1 << 20, table_stride=1 << 20)) == 0
    assert size(_attn(max_seqlen_q=1, table_width=0)) == 0
    for over, want in ((dict(scores=FAKE, scores_bytes=size(one)), "FNA2_OK"),
                       (dict(scores=FAKE, scores_bytes=size(one) - 1), "FNA2_E_WORKSPACE"),
                       (dict(scores=FAKE + 8, scores_bytes=size(one)), "FNA2_E_WORKSPACE")):
        a = _attn(max_seqlen_q=1)
        for k, v in over.items():
            setattr(a, k, v)
        assert _st(lib.fna2_check_paged_attn(ctypes.byref(a))) == want


def test_check_paged_append_codes(lib):
    def code(**over):
        a = _capi.PagedAppendArgs()
        names = ("q", "k", "v", "r_k", "q_out", "positions", "inv_freq", "norm_q", "norm_k", "eps")
        a.c = _cache_args(**{k: v for k, v in over.items() if k not in names})
        a.q = a.q_out = _capi.Tensor(FAKE, 0, 16 * 128, 128)
        a.k = a.v = _capi.Tensor(FAKE, 0, 4 * 128, 128)
        a.r_k = _capi.Tensor(FAKE, 0, 12 * 32, 32)
        a.norm_q = a.norm_k = a.inv_freq = FAKE
        a.eps = 1e-6
        for k, v in over.items():
            if k in names:
                setattr(a, k, v)
        return _st(lib.fna2_check_paged_append(ctypes.byref(a)))
    assert code() == "FNA2_OK"
    assert code(norm_q=None, norm_k=None, inv_freq=None) == "FNA2_OK"
    assert code(eps=float("nan")) == "FNA2_E_SCALE"
    assert code(norm_k=FAKE + 1) == "FNA2_E_STRIDE"
    assert code(positions=FAKE + 2) == "FNA2_E_STRIDE"
    assert code(k=NO) == "FNA2_E_NULL"
    assert code(r_k=NO) == "FNA2_E_NULL"
    assert code(q_out=_capi.Tensor(FAKE, 0, 16 * 128 + 4, 128)) == "FNA2_E_STRIDE"
    assert code(cu_seqlens_q=None) == "FNA2_E_SEQLENS"
    assert code(total_q=0, q=NO, k=NO, v=NO) == "FNA2_OK"


def test_check_paged_evict_codes(lib):
    def code(**over):
        a = _capi.PagedEvictArgs()
        names = ("budget", "recent", "first", "key_weights", "stride_b", "stride_h", "capacity",
                 "weights_out", "kept", "new_lens")
        a.c = _cache_args(cu_seqlens_q=None, **{k: v for k, v in over.items() if k not in names})
        a.budget, a.recent, a.first, a.capacity = 100, 20, 4, 512
        a.key_weights, a.weights_out, a.kept, a.new_lens = FAKE, 2 * FAKE, FAKE, FAKE
        a.stride_b, a.stride_h = 2048, 512
        for k, v in over.items():
            if k in names:
                setattr(a, k, v)
        return _st(lib.fna2_check_paged_evict(ctypes.byref(a)))
    assert code() == "FNA2_OK"
    assert code(budget=23) == "FNA2_E_SHAPE"
    assert code(budget=24) == "FNA2_OK"
    assert code(first=-1) == "FNA2_E_SHAPE"
    assert code(recent=2 ** 31 - 1, budget=2 ** 30) == "FNA2_E_SHAPE"
    assert code(kept=None) == "FNA2_E_NULL"
    assert code(new_lens=None) == "FNA2_E_NULL"
    assert code(weights_out=None) == "FNA2_E_NULL"
    assert code(weights_out=FAKE) == "FNA2_E_ALIAS"
    assert code(capacity=0, key_weights=None, weights_out=None) == "FNA2_OK"
    assert code(batch=0, kept=None, new_lens=None) == "FNA2_OK"


def test_paged_struct_layout_matches_header(tmp_path):
    structs = {"fna2_paged_cache": _capi.PagedCache, "fna2_paged_attn_args": _capi.PagedAttnArgs,
               "fna2_paged_weights_args": _capi.PagedWeightsArgs,
               "fna2_paged_append_args": _capi.PagedAppendArgs,
               "fna2_paged_evict_args": _capi.PagedEvictArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fna2.h"', "int main(void){"]
    for st, cls in structs.items():
        lines.append(f'printf("{st} size %zu\\n", sizeof({st}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{st} {f} %zu\\n", offsetof({st}, {f}));')
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        st, f, n = line.split()
        cls = structs[st]
        assert int(n) == (ctypes.sizeof(cls) if f == "size" else getattr(cls, f).offset), line


def test_python_refusals_off_gpu():
    c = Case([2], [20], 4, 2, 3, 64, 8, 16)
    w = torch.zeros(1, 2, 48)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        c.attend()
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        paged.paged_evict(c.k, c.v, c.table, c.lens, w, 10)
    with pytest.raises(AssertionError, match="heads"):
        paged.paged_evict(c.k, c.v, c.table, c.lens, w, 10, rk_pages=c.rk)


def test_oracle_attend_is_the_attention_oracle():
    """One contiguous page table: the last tokens of the dense causal forward."""
    c = Case([5], [37], 4, 2, 3, 64, 16, 16)
    out, lse, w, _ = c.oracle()
    rows = lambda p: torch.stack([p[c.slot(0, j)[0], :, c.slot(0, j)[1]] for j in range(37)])
    k, v, rk = rows(c.k), rows(c.v), rows(c.rk)
    q = torch.cat([torch.zeros(32, 4, 64, dtype=c.dtype), c.q])
    rq = torch.cat([torch.zeros(32, 3, 16, dtype=torch.bfloat16), c.rq])
    t = lambda x: x.transpose(0, 1)[None]
    ref, ref_lse = O.forward(t(q), t(k), t(v), t(rq), t(rk), c.gs, 64 ** -0.5, True)
    assert np.abs(ref[0].transpose(1, 0, 2)[32:] - out).max() < 1e-12
    assert np.abs(ref_lse[0].T[32:] - lse).max() < 1e-12
    assert abs(w.sum() - 5 * 4) < 1e-4  # every (token, head)'s weights sum to one


def test_oracle_planted_mistakes_show():
    """The bounds tell a chunk off by one row, and heads that share a KV head
    mixed up, from the right result."""
    c = Case([5, 1], [37, 20], 4, 2, 0, 64, 0, 16)
    ref, _, _, mag = c.oracle()
    bad = PO.attend(c.q, c.k, c.v, c.table, c.lens - 1, c.cu)[0]
    swapped = PO.attend(c.q[:, [0, 2, 1, 3]], c.k, c.v, c.table, c.lens, c.cu)[0][:, [0, 2, 1, 3]]
    for wrong in (bad, swapped):
        with pytest.raises(AssertionError):
            close_out(c, torch.from_numpy(wrong), ref, mag)


def test_oracle_evict_against_sorting():
    c = Case([0], [50], 4, 2, 4, 64, 8, 16)
    w = torch.rand(1, 2, 64)
    w[0, 0, 10:20] = 0.5
    w[0, 1, 7] = float("nan")
    kept, lens, wo, kp, vp, rkp = PO.evict(c.k, c.v, c.table, c.lens, w, 30, 5, 2, c.rk, 4)
    assert lens.tolist() == [30]
    for kv in range(2):
        x = torch.nan_to_num(w[0, kv, 2:45], nan=9.0)
        order = torch.sort(x, descending=True, stable=True).indices[:23] + 2
        rows = sorted(order.tolist() + [0, 1] + list(range(45, 50)))
        assert kept[0, kv].tolist() == rows
        for r, j in enumerate(rows):
            (pd, do), (ps, po) = c.slot(0, r), c.slot(0, j)
            assert (kp[pd, kv, do] == c.k[ps, kv, po].double().numpy()).all()
            for h in (2 * kv, 2 * kv + 1):
                assert (rkp[pd, h, do] == c.rk[ps, h, po].double().numpy()).all()


# ── GPU: attention ───────────────────────────────────────────────────────────

BF, FP = torch.bfloat16, torch.float16
ATTEND = [
    # lq, lk, H, HKV, HG, D, R, ps, dtype
    ([1], [1], 4, 4, 4, 64, 16, 16, BF),
    ([1, 1, 1], [300, 1, 77], 8, 2, 6, 128, 32, 32, BF),     # decode, vanilla heads in a group
    ([1, 1], [97, 33], 4, 4, 4, 64, 16, 16, FP),
    ([1, 1], [130, 64], 16, 2, 0, 128, 0, 48, BF),           # group 8, no graph heads
    ([1, 1], [200, 31], 8, 2, 3, 128, 24, 16, FP),           # rank 24: 3 chunks a head
    ([1, 1], [90, 40], 32, 1, 20, 64, 64, 16, BF),           # ranks of a group past one tile
    ([1, 2], [70, 40], 64, 1, 0, 64, 0, 16, BF),             # a group past 32 columns
    ([1, 1], [90, 17], 6, 2, 4, 128, 8, 16, BF),             # group 3
    ([5, 3, 0, 1], [64, 63, 40, 0], 8, 2, 8, 128, 16, 16, BF),   # drafted tokens, idle, empty
    ([4, 9], [2, 9], 4, 2, 4, 64, 32, 16, BF),               # more tokens than rows: rows that see none
    ([0, 0], [30, 0], 4, 2, 4, 64, 32, 16, BF),              # no token at all
    ([33, 31], [33, 140], 4, 4, 4, 128, 32, 32, BF),         # whole prompt, piece of one
    ([70], [130], 4, 2, 2, 64, 64, 16, FP),
    ([130, 1, 2], [131, 200, 40], 4, 1, 3, 128, 40, 64, BF), # a piece beside decoding sequences
    ([150], [400], 2, 2, 2, 64, 8, 256, BF),
    ([129], [129], 3, 3, 0, 128, 0, 16, FP),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"q{c[0]}-k{c[1]}-h{c[2]}.{c[3]}.{c[4]}")
def test_attend(gpu, case, causal):
    check_attend(Case(*case, seed=3, device=gpu), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.1, 0.0, 2.0])
@pytest.mark.parametrize("lq", [1, 40])
def test_attend_scales(gpu, scale, lq):
    check_attend(Case([lq, 1], [90, 55], 4, 2, 3, 64, 16, 16, device=gpu), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [0, 1, 7, 64, 10 ** 6])
def test_attend_does_not_depend_on_the_hint(gpu, hint):
    check_attend(Case([37, 1, 4], [90, 55, 4], 4, 2, 4, 128, 16, 16, device=gpu), hint=hint)


@pytest.mark.gpu
def test_attend_more_sequences_than_a_wave_has_lanes(gpu):
    n = 150
    lk = [(i * 37) % 50 for i in range(n)]
    lq = [min(k, (i * 7) % 3) for i, k in enumerate(lk)]
    check_attend(Case(lq, lk, 2, 1, 2, 64, 8, 16, device=gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 6, 40, 300])
def test_attend_long_cache_is_split(gpu, lq):
    """A long cache is cut into runs that the merge joins: against torch in
    fp64 (the oracle's loops are slow here)."""
    c = Case([lq, 1], [5001, 777], 4, 2, 3, 128, 32, 64, device=gpu, seed=5)
    out, lse = c.attend(return_lse=True)
    again = c.attend()
    assert torch.equal(out, again)
    t = 0
    for b, (m, n) in enumerate(zip(c.lq, c.lk)):
        ids = c.table[b, :-(-n // c.ps)].long()
        rows = lambda p, h: p[ids, h].reshape(-1, p.shape[3])[:n].double()
        hide = torch.arange(n, device=gpu)[None] > n - m + torch.arange(m, device=gpu)[:, None]
        for h in range(4):
            s = c.q[t:t + m, h].double() @ rows(c.k, h // 2).t() * 128 ** -0.5
            if h < 3:
                s = s + c.gs[h].double() * (c.rq[t:t + m, h].double() @ rows(c.rk, h).t())
            s[hide] = -math.inf
            p = torch.softmax(s, -1)
            V = rows(c.v, h // 2)
            ref, mag = p @ V, p @ V.abs()
            lim = HALF[c.dtype] * ref.abs() + (HALF[c.dtype] + 2e-4) * mag
            assert ((out[t:t + m, h].double() - ref).abs() <= lim).all()
            assert (lse[t:t + m, h].double() - torch.logsumexp(s, -1)).abs().max() <= 1e-4
        t += m


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq", [[1, 1], [5, 3], [40, 33]])
def test_hidden_rows_never_reach_a_result(gpu, lq, dtype):
    """NaN and infinities behind a sequence's last row, in pages that no table
    names, and in the K and V of later tokens."""
    c = Case(lq, [75, 61], 4, 2, 4, 128, 16, 32, dtype, device=gpu)
    base = check_attend(c)
    named = {c.slot(b, j) for b in range(2) for j in range(c.lk[b])}
    odd = [float("nan"), float("inf"), -float("inf")]
    for p in range(c.P):
        for r in range(c.ps):
            if (p, r) not in named:
                c.k[p, :, r], c.v[p, :, r], c.rk[p, :, r] = odd[r % 3], odd[(r + 1) % 3], odd[p % 3]
    assert torch.equal(c.attend(), base)
    if lq == [1, 1]:
        return
    # the last token's rows: every earlier token's result stays as it was
    for b in range(2):
        p, r = c.slot(b, c.lk[b] - 1)
        c.k[p, :, r], c.v[p, :, r, ::2] = float("nan"), float("inf")
        c.v[p, :, r, 1::2], c.rk[p, :, r] = float("nan"), float("nan")
    got = c.attend()
    for b in range(2):
        t0, t1 = int(c.cu[b]), int(c.cu[b + 1])
        assert torch.equal(got[t0:t1 - 1], base[t0:t1 - 1])
        assert not torch.isfinite(got[t1 - 1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("H,HKV,HG,R", [(4, 4, 4, 8), (6, 2, 4, 8), (4, 2, 4, 24), (32, 1, 20, 64),
                                        (40, 1, 0, 0)])
@pytest.mark.parametrize("lq", [[1, 1], [5, 3], [40, 33]])
def test_weights_past_garbage(gpu, lq, H, HKV, HG, R):
    """The rows' weights with NaN in every row that is no sequence's, behind odd
    numbers of rank chunks and in pages next to the used ones."""
    c = Case(lq, [75, 61], H, HKV, HG, 64, R, 16, device=gpu)
    ref = torch.zeros(2, HKV, c.width * 16, device=gpu)
    c.attend(key_weights=ref)
    check_attend(c)
    named = torch.zeros(c.P, 16, dtype=torch.bool)
    for b in range(2):
        for j in range(c.lk[b]):
            named[c.slot(b, j)] = True
    hole = ~named.to(gpu)
    for pool in (c.k, c.v, c.rk):
        if pool is not None:
            pool.masked_fill_(hole[:, None, :, None], float("nan"))
    acc = torch.zeros_like(ref)
    c.attend(key_weights=acc)
    assert torch.equal(acc, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", [c for c in ATTEND if max(c[0]) <= 9],
                         ids=lambda c: f"q{c[0]}-k{c[1]}-h{c[2]}.{c[3]}.{c[4]}")
def test_weights_without_the_scores(gpu, lib, monkeypatch, case, causal):
    """The rows' weights from K, where the attention left no scores: right, and
    past garbage (NaN in the rows that are no sequence's) the same bits."""
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    monkeypatch.setattr(lib, "fna2_paged_scores_bytes", lambda a: 0)
    c = Case(*case, seed=3, device=gpu)
    check_attend(c, causal=causal)
    ref = torch.zeros(c.N, c.HKV, c.width * c.ps, device=gpu)
    c.attend(key_weights=ref, is_causal=causal)
    named = torch.zeros(c.P, c.ps, dtype=torch.bool)
    for b in range(c.N):
        for j in range(c.lk[b]):
            named[c.slot(b, j)] = True
    hole = ~named.to(gpu)
    for pool in (c.k, c.v, c.rk):
        if pool is not None:
            pool.masked_fill_(hole[:, None, :, None], float("nan"))
    acc = torch.zeros_like(ref)
    c.attend(key_weights=acc, is_causal=causal)
    assert torch.equal(acc, ref)


@pytest.mark.gpu
def test_weights_where_the_scores_do_not_fit(gpu, lib, monkeypatch):
    """No memory for the scores: the weights come from K."""
    c = Case([1, 1], [300, 77], 8, 2, 6, 128, 32, 32, device=gpu)
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    refused, empty = [], torch.empty

    def full(*size, **kw):
        if kw.get("dtype") is torch.uint8 and not refused:
            refused.append(size)
            raise torch.OutOfMemoryError("full")
        return empty(*size, **kw)

    monkeypatch.setattr(torch, "empty", full)
    check_attend(c)
    # (N, HKV, rows, columns, bytes)
    assert refused == [(2 * 2 * c.width * c.ps * 4 * 4,)]


@pytest.mark.gpu
def test_scores_serve_the_short_chunks_only(gpu):
    """A hint below the longest chunk: the sequences that one tile holds take
    the scores, the others K; long caches in several runs."""
    check_attend(Case([1, 7, 0, 2], [700, 400, 90, 33], 8, 4, 5, 64, 16, 16, device=gpu), hint=1)
    check_attend(Case([3, 40, 2], [500, 300, 2], 4, 2, 0, 128, 0, 32, FP, device=gpu), hint=3)


@pytest.mark.gpu
@pytest.mark.parametrize("D,R", [(64, 0), (64, 16), (128, 64), (128, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_under_a_wide_table(gpu, causal, D, R):
    """Tables that hold thousands of rows: larger blocks of keys."""
    check_attend(Case([40, 133], [300, 400], 8, 4, 7 if R else 0, D, R, 256, device=gpu, width=70),
                 causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[1, 1], [40, 9]])
def test_infinite_values_stay_infinite(gpu, lq):
    c = Case(lq, [75, 61], 4, 2, 0, 64, 0, 16, device=gpu)
    p, r = c.slot(0, 3)
    c.v[p, :, r, 5] = float("inf")
    out = c.attend()
    n = lq[0]
    assert (out[:n, :, 5] == float("inf")).all()
    out[:n, :, 5] = 0
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[1, 1], [20, 36]])
def test_pages_that_are_not_there(gpu, lq):
    """Ids outside the pool, inside the lengths: their rows are not seen."""
    c = Case(lq, [150, 90], 4, 2, 3, 128, 16, 16, device=gpu)
    c.table[0, 2], c.table[0, 5], c.table[1, 0] = -1, c.P, 2 ** 31 - 1
    check_attend(c)
    c.table[1] = -7  # none of a sequence's
    check_attend(c)


@pytest.mark.gpu
def test_shared_pages_and_wider_tables(gpu):
    """Two sequences that share a prefix's pages; a table that is a view of a
    wider one; lengths past the table are cut to it."""
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    c.table[1, :3] = c.table[0, :3]
    check_attend(c)
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    wide = torch.full((2, 40), 10 ** 9, dtype=torch.int32, device=gpu)
    wide[:, 3:3 + c.width] = c.table
    ref = c.attend()
    c.table = wide[:, 3:3 + c.width]
    assert torch.equal(c.attend(), ref)
    c.lens[1] = 10 ** 8
    check_attend(c)
    c.lens[0] = -5
    check_attend(c)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[1, 1], [36, 5]])
def test_strided_operands(gpu, lq):
    """Pools with a page's rows of all heads together, q and r_q column views
    of one projection: the same bits."""
    a = Case(lq, [150, 90], 4, 2, 3, 64, 16, 32, device=gpu)
    ref = a.attend()
    tr = lambda p: p.transpose(1, 2).contiguous().transpose(1, 2)
    a.k, a.v, a.rk = tr(a.k), tr(a.v), tr(a.rk)
    assert a.k.stride(2) == 2 * 64
    y = torch.zeros(a.T, 4 * 64 + 3 * 16 + 8, dtype=BF, device=gpu)
    y[:, :256], y[:, 256:304] = a.q.reshape(a.T, -1), a.rq.reshape(a.T, -1)
    a.q, a.rq = y[:, :256].view(a.T, 4, 64), y[:, 256:304].view(a.T, 3, 16)
    assert torch.equal(a.attend(), ref)
    a.q = torch.nn.functional.pad(a.q, (1, 0))[..., 1:]  # rows that are not 16-byte aligned
    assert torch.equal(a.attend(), ref)


@pytest.mark.gpu
def test_tokens_of_no_sequence(gpu):
    """Tokens before the first sequence and behind the last: zeros, LSE -inf."""
    for lq in ([2, 1], [40, 0]):
        c = Case(lq, [50, 30], 4, 2, 2, 64, 8, 16, device=gpu, head=2, tail=3)
        check_attend(c)
    c = Case([], [], 4, 2, 2, 64, 8, 16, device=gpu, tail=3)
    out, lse = c.attend(return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.gpu
def test_weights_capacity(gpu):
    """Rows at or past the capacity have no weight; nothing else is written."""
    c = Case([3, 40], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    _, _, w, _ = c.oracle()
    buf = torch.zeros(2, 2, 100, device=gpu)
    acc = buf[:, :, 10:43]
    c.attend(key_weights=acc)
    got = buf.double().cpu().numpy()
    assert (got[:, :, :10] == 0).all() and (got[:, :, 43:] == 0).all()
    assert np.allclose(got[:, :, 10:43], w[:, :, :33], rtol=2e-4, atol=1e-7)
    first = acc.clone()
    c.attend(key_weights=acc)
    assert torch.allclose(acc, 2 * first, rtol=1e-6)


@pytest.mark.gpu
def test_attend_refusals(gpu):
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    ok = dict(r_q=c.rq, rk_pages=c.rk, graph_scale=c.gs)
    args = [c.q, c.k, c.v, c.table, c.lens, c.cu, 3]

    def bad(i, x, **kw):
        a = list(args)
        if i is not None:
            a[i] = x
        with pytest.raises((AssertionError, RuntimeError)):
            paged.flash_naylis_paged(*a, **{**ok, **kw})

    bad(0, c.q.half())
    bad(0, c.q[:, :3])
    bad(0, c.q[..., :32])
    bad(0, c.q.cpu())
    bad(1, c.k[:, :, :8])
    bad(1, c.k.float())
    bad(2, c.v[1:])
    bad(3, c.table[:1])
    bad(4, c.lens[:1])
    bad(5, c.cu[:2])
    bad(6, -1)
    bad(None, None, rk_pages=None)
    bad(None, None, graph_scale=None)
    bad(None, None, graph_scale=c.gs[:2])
    bad(None, None, rk_pages=c.rk[:, :3])
    bad(None, None, softmax_scale=float("nan"))
    bad(None, None, key_weights=torch.zeros(2, 2, 10, dtype=torch.float64, device=gpu))
    bad(None, None, key_weights=torch.zeros(2, 3, 10, device=gpu))
    bad(None, None, key_weights=torch.zeros(2, 1, 10, device=gpu).expand(2, 2, 10))
    bad(None, None, key_weights=torch.zeros(2, 2, 10, device=gpu, requires_grad=True))
    w = torch.zeros(2, 2, 10, device=gpu)
    v0 = w._version
    paged.flash_naylis_paged(*args, **ok, key_weights=w)
    assert w._version > v0


# ── GPU: append ──────────────────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("norm,rope,given", [(True, True, False), (True, False, False),
                                             (False, True, True), (False, False, False),
                                             (True, True, True)])
@pytest.mark.parametrize("case", [
    ([1, 1, 1], [40, 1, 17], 4, 2, 3, 64, 8, 16, BF),
    ([5, 0, 33], [40, 9, 33], 8, 8, 0, 128, 0, 48, FP),
    ([3, 6], [2, 90], 6, 2, 6, 128, 40, 32, BF),  # rows before 0
    ([19, 4], [400, 30], 5, 5, 2, 64, 64, 16, FP),
])
def test_append(gpu, case, norm, rope, given):
    c = Case(*case, seed=7, device=gpu, head=1, tail=2)
    g = torch.Generator().manual_seed(2)
    D = c.D
    w = (lambda: (1 + 0.2 * torch.randn(D, generator=g)).to(gpu)) if norm else lambda: None
    wq, wk = w(), w()
    inv = 10000.0 ** (-torch.arange(0, D, 2).float() / D) if rope else None
    pos = torch.randint(0, 200000, (c.T,), generator=g).to(torch.int32) if given else None
    up = lambda t: None if t is None else t.to(gpu)
    if c.lq[0] == 5:
        c.table[2, 0] = -1  # not there: not stored
    ref = PO.append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk, inv, pos, wq, wk)
    got = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk,
                             up(inv), up(pos), wq, wk)
    for name, a, b in (("q", got, ref[0]), ("k", c.k, ref[1]), ("v", c.v, ref[2]),
                       ("rk", c.rk, ref[3])):
        if b is None:
            continue
        a = a.double().cpu().numpy()
        if name in ("v", "rk") or not (norm or rope):
            assert (a == b).all(), name
        else:
            assert (np.abs(a - b) <= HALF[c.dtype] * np.abs(b) + 1e-5).all(), name


@pytest.mark.gpu
def test_append_reads_projections_in_place(gpu):
    c = Case([7, 2], [50, 20], 4, 2, 3, 64, 16, 16, device=gpu)
    import copy
    d = copy.copy(c)
    d.k, d.v, d.rk = c.k.clone(), c.v.clone(), c.rk.clone()
    y = torch.cat([c.q.reshape(9, -1), c.kn.reshape(9, -1), c.vn.reshape(9, -1), c.rkn.reshape(9, -1)], 1)
    cut = lambda a, h, f: y[:, a:a + h * f].view(9, h, f)
    inv = 10000.0 ** (-torch.arange(0, 64, 2, device=gpu).float() / 64)
    v0 = d.k._version
    a = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk, inv)
    b = paged.paged_append(cut(0, 4, 64), cut(256, 2, 64), cut(384, 2, 64), d.k, d.v, c.table,
                           c.lens, c.cu, cut(512, 3, 16), d.rk, inv)
    assert d.k._version > v0
    for x, z in ((a, b), (c.k, d.k), (c.v, d.v), (c.rk, d.rk)):
        assert torch.equal(x, z)


@pytest.mark.gpu
def test_append_refusals(gpu):
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    inv = torch.ones(32, device=gpu)
    base = [c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu]

    def bad(i, x, **kw):
        a = list(base)
        if i is not None:
            a[i] = x
        with pytest.raises((AssertionError, RuntimeError)):
            paged.paged_append(*a, **{**dict(r_k=c.rkn, rk_pages=c.rk, inv_freq=inv), **kw})

    bad(0, c.q.half())
    bad(1, c.kn[:2])
    bad(2, c.vn[:, :1])
    bad(2, c.vn.cpu())
    bad(None, None, r_k=None)
    bad(None, None, rk_pages=None)
    bad(None, None, inv_freq=inv[:30])
    bad(None, None, norm_q=inv)
    bad(None, None, positions=torch.zeros(3, dtype=torch.int32, device=gpu))
    bad(None, None, inv_freq=None, positions=torch.zeros(4, dtype=torch.int32, device=gpu))
    bad(None, None, eps=float("inf"), norm_q=torch.ones(64, device=gpu))
    bad(3, c.k.clone().requires_grad_())


# ── GPU: eviction ────────────────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("budget,recent,first", [(30, 5, 2), (30, 0, 0), (16, 16, 0), (8, 4, 4),
                                                 (0, 0, 0), (49, 1, 1), (1000, 3, 1)])
@pytest.mark.parametrize("case", [
    ([50, 31, 0, 16], 4, 2, 4, 64, 8, 16, BF),
    ([200, 8, 333], 8, 2, 5, 128, 40, 48, FP),
    ([90], 3, 3, 0, 64, 0, 256, BF),
])
def test_evict(gpu, case, budget, recent, first):
    c = Case([0] * len(case[0]), *case, device=gpu, seed=11)
    g = torch.Generator().manual_seed(4)
    cap = c.width * c.ps
    w = torch.randn(c.N, c.HKV, cap, generator=g)
    w[:, :, ::5] = 0.0
    w[:, :, 1::7] = -0.0
    w[0, 0, 9], w[0, 0, 11], w[0, 0, 13] = float("inf"), float("nan"), -float("inf")
    ref = PO.evict(c.k, c.v, c.table, c.lens, w, budget, recent, first, c.rk, c.H)
    w = w.to(gpu)
    w0 = w.clone()
    got = paged.paged_evict(c.k, c.v, c.table, c.lens, w, budget, recent, first, c.rk, c.H)
    assert torch.equal(w.nan_to_num(7), w0.nan_to_num(7))
    assert (got[0].cpu().numpy() == ref[0]).all()
    assert (got[1].cpu().numpy() == ref[1]).all()
    assert np.array_equal(got[2].cpu().numpy(), ref[2], equal_nan=True)
    for a, b in ((c.k, ref[3]), (c.v, ref[4]), (c.rk, ref[5])):
        if b is not None:
            assert (a.double().cpu().numpy() == b).all()


@pytest.mark.gpu
def test_evict_long_and_odd(gpu):
    """More rows than a pass of the selection, equal weights across passes, a
    capacity below the length, pages that are not there, strided weights."""
    c = Case([0, 0], [2999, 1500], 2, 2, 2, 64, 24, 64, device=gpu, seed=12)
    c.table[0, 3], c.table[0, 20] = -1, c.P + 4
    g = torch.Generator().manual_seed(4)
    w = torch.randint(0, 12, (2, 2, 2 * 2500), generator=g).float()[:, :, ::2]
    ref = PO.evict(c.k, c.v, c.table, c.lens, w, 1111, 77, 3, c.rk, 2)
    got = paged.paged_evict(c.k, c.v, c.table, c.lens, w.to(gpu), 1111, 77, 3, c.rk, 2)
    for a, b in zip(got + (c.k, c.v, c.rk), ref):
        assert (a.double().cpu().numpy() == b).all()


@pytest.mark.gpu
def test_evict_refusals(gpu):
    c = Case([0], [70], 4, 2, 4, 64, 16, 16, device=gpu)
    w = torch.zeros(1, 2, 80, device=gpu)

    def bad(*a, **kw):
        with pytest.raises((AssertionError, RuntimeError)):
            paged.paged_evict(c.k, c.v, c.table, c.lens, *a, **kw)

    bad(w, -1)
    bad(w, 10, 8, 3)
    bad(w, 10, -1, 0)
    bad(w.double(), 10)
    bad(w[:, :1], 10)
    bad(w.cpu(), 10)
    bad(w, 10, rk_pages=c.rk)           # whose rows?
    bad(w, 10, rk_pages=c.rk, heads=3)  # fewer than the graph heads
    bad(w, 10, rk_pages=c.rk.half(), heads=4)


# ── GPU: the two launch paths ────────────────────────────────────────────────

@pytest.mark.gpu
def test_native_and_python_launchers_agree(gpu, monkeypatch):
    nat = _capi.native()
    c = Case([3, 40, 0], [70, 80, 9], 4, 2, 3, 64, 16, 16, device=gpu, tail=1)
    w = torch.rand(3, 2, c.width * 16, device=gpu)
    inv = torch.rand(32, device=gpu)
    pos = torch.arange(c.T, dtype=torch.int32, device=gpu)
    pools = [c.k.clone(), c.v.clone(), c.rk.clone()]

    def calls():
        for a, b in zip((c.k, c.v, c.rk), pools):
            a.copy_(b)
        acc = w.clone()
        q = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk,
                               inv.double(), pos, inv.repeat(2), None)
        out, lse = c.attend(return_lse=True, key_weights=acc)
        ev = paged.paged_evict(c.k, c.v, c.table, c.lens, acc, 35, 5, 1, c.rk, 4)
        return (q, out, lse, acc, *ev, c.k.clone(), c.v.clone(), c.rk.clone())

    assert nat.paged_attn(c.q, c.k, c.v, c.table, c.lens, c.cu, 40, c.rq, c.rk, c.gs, 0.1, True,
                          w.clone(), True) is not None
    assert nat.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk, inv,
                            pos, None, None, 0.0) is not None
    assert nat.paged_evict(c.k, c.v, c.table, c.lens, w, 35, 5, 1, c.rk, 4) is not None
    # left to the Python launchers: lengths on the CPU or in 64 bits, strided features
    assert nat.paged_attn(c.q, c.k, c.v, c.table, c.lens.cpu(), c.cu, 40, c.rq, c.rk, c.gs, 0.1,
                          True, None, True) is None
    assert nat.paged_attn(c.q, c.k, c.v, c.table, c.lens, c.cu.long(), 40, c.rq, c.rk, c.gs, 0.1,
                          True, None, True) is None
    assert nat.paged_evict(c.k, c.v, c.table, c.lens, w, 3, 5, 1, c.rk, 4) is None
    a = calls()
    odd = c.attend()
    c.lens, c.cu = c.lens.cpu(), c.cu.long()
    assert torch.equal(odd, c.attend())
    c.lens, c.cu = c.lens.to(gpu), c.cu.int()
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    for x, y in zip(a, calls()):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_inference_tensors(gpu):
    """As torch's own in-place calls: written in inference mode only."""
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    with torch.inference_mode():
        k, v, rk = c.k.clone(), c.v.clone(), c.rk.clone()
        paged.paged_append(c.q, c.kn, c.vn, k, v, c.table, c.lens, c.cu, c.rkn, rk)
        w = torch.zeros(2, 2, 96, device=gpu)
        c.attend(key_weights=w)
    with pytest.raises(RuntimeError):
        paged.paged_append(c.q, c.kn, c.vn, k, v, c.table, c.lens, c.cu, c.rkn, rk)
    with pytest.raises(RuntimeError):
        c.attend(key_weights=w)
    with pytest.raises(RuntimeError):
        paged.paged_evict(k, v, c.table, c.lens, w, 10)


# ── GPU: as they are used ────────────────────────────────────────────────────

def _serve(c, steps, gpu, budget=None):
    """Decode `steps` tokens for every sequence: append, attend (weighing),
    evict past the budget.  Returns outputs and the oracle's."""
    inv = 10000.0 ** (-torch.arange(0, c.D, 2, device=gpu).float() / c.D)
    wq = torch.ones(c.D, device=gpu)
    w = torch.zeros(c.N, c.HKV, c.width * c.ps, device=gpu)
    pos = c.lens.clone()
    cu = torch.arange(c.N + 1, dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(9)
    for _ in range(steps):
        new = lambda h, f, dt: torch.randn(c.N, h, f, generator=g).to(dt).to(gpu)
        q, k, v = new(c.H, c.D, c.dtype), new(c.HKV, c.D, c.dtype), new(c.HKV, c.D, c.dtype)
        rq, rk = new(c.HG, c.R, BF) * 0.3, new(c.HG, c.R, BF)
        c.lens += 1
        before = PO.append(q, k, v, c.k, c.v, c.table, c.lens, cu, rk, c.rk, inv, pos, wq, wq)
        q = paged.paged_append(q, k, v, c.k, c.v, c.table, c.lens, cu, rk, c.rk, inv, pos, wq, wq)
        for a, b in ((q, before[0]), (c.k, before[1]), (c.v, before[2]), (c.rk, before[3])):
            assert (np.abs(a.double().cpu().numpy() - b) <= HALF[c.dtype] * np.abs(b) + 1e-5).all()
        pos += 1
        ref, _, dw, mag = PO.attend(q, c.k, c.v, c.table, c.lens, cu, rq, c.rk, c.gs)
        w0 = w.double().cpu().numpy()
        out = paged.flash_naylis_paged(q, c.k, c.v, c.table, c.lens, cu, 1, r_q=rq, rk_pages=c.rk,
                                       graph_scale=c.gs, key_weights=w)
        close_out(c, out, ref, mag)
        assert np.allclose(w.double().cpu().numpy(), w0 + dw, rtol=2e-4, atol=1e-7)
        if budget:
            want = PO.evict(c.k, c.v, c.table, c.lens, w, budget, 4, 1, c.rk, c.H)
            kept, lens, w = paged.paged_evict(c.k, c.v, c.table, c.lens, w, budget, 4, 1, c.rk, c.H)
            for a, b in zip((kept, lens, w, c.k, c.v, c.rk), want):
                assert (a.double().cpu().numpy() == b).all()
            c.lens = lens
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_serving_steps_with_eviction(gpu, dtype):
    c = Case([1, 1, 1], [30, 12, 33], 4, 2, 3, 64, 8, 16, dtype, device=gpu, width=4)
    for b in range(3):  # pages for the rows to come
        for j in range(c.width):
            if int(c.table[b, j]) < 0:
                c.table[b, j] = c.P + 50
    grow = 12 - sum(c.used)
    extra = torch.randn(grow, 2, 16, 64).to(dtype).to(gpu)
    c.k, c.v = torch.cat([c.k, extra]), torch.cat([c.v, extra])
    c.rk = torch.cat([c.rk, torch.randn(grow, 3, 16, 8).bfloat16().to(gpu)])
    missing = [(b, j) for b in range(3) for j in range(c.width) if int(c.table[b, j]) >= c.P]
    for i, (b, j) in enumerate(missing):
        c.table[b, j] = c.P + i
    assert len(missing) <= c.k.shape[0] - c.P
    _serve(c, 6, gpu, budget=32)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[1, 1], [3, 0], [40, 3]])
def test_caches_without_rows(gpu, lq):
    """Lengths of zero, tables of no width, pools of no page: outputs 0, LSE
    -inf, weights and pools as they were."""
    def nothing(c):
        acc = torch.rand(2, 2, 48, device=gpu)
        before = acc.clone()
        out, lse = c.attend(return_lse=True, key_weights=acc)
        assert (out == 0).all() and (lse == -math.inf).all() and torch.equal(acc, before)
        k = c.k.clone()
        q = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk)
        assert torch.equal(q, c.q) and torch.equal(c.k, k)
        kept, lens, w = paged.paged_evict(c.k, c.v, c.table, c.lens, acc, 4, 1, 1, c.rk, 4)
        assert torch.equal(c.k, k) and kept.shape == (2, 2, 4) and w.shape == acc.shape
        return lens

    make = lambda: Case(lq, [0, 0], 4, 2, 3, 64, 8, 16, device=gpu)
    assert (nothing(make()) == 0).all()
    c = make()
    c.lens += 60
    c.table = c.table[:, :0]
    assert (nothing(c) == 0).all()
    c = make()
    c.lens += 20
    c.k, c.v, c.rk = c.k[:0], c.v[:0], c.rk[:0]
    assert (nothing(c) == 4).all()


@pytest.mark.gpu
def test_two_calls_at_once(gpu):
    """Calls on two streams: each has a workspace of its own."""
    a = Case([1, 1], [3000, 900], 4, 2, 3, 64, 16, 16, device=gpu, seed=1)
    b = Case([90, 2], [2000, 700], 4, 2, 3, 64, 16, 16, device=gpu, seed=2)
    want = [x.attend(return_lse=True) for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, (x, s) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(s):
                got[i].append(x.attend(return_lse=True))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[0], o) and torch.equal(w[1], l) for o, l in g)


@pytest.mark.gpu
def test_other_streams_and_graphs(gpu):
    """A step on a stream of its own, captured into a graph and replayed on
    new inputs and lengths, with eager work between the replays."""
    c = Case([3, 1], [40, 70], 4, 2, 4, 64, 16, 16, device=gpu)
    inv = 10000.0 ** (-torch.arange(0, 64, 2, device=gpu).float() / 64)
    w = torch.zeros(2, 2, c.width * c.ps, device=gpu)

    def step(acc, lens):
        q = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, lens, c.cu, c.rkn, c.rk, inv)
        out = paged.flash_naylis_paged(q, c.k, c.v, c.table, lens, c.cu, 3, r_q=c.rq,
                                       rk_pages=c.rk, graph_scale=c.gs, key_weights=acc)
        return out, paged.paged_evict(c.k.clone(), c.v.clone(), c.table, lens, acc, 35, 5, 1)

    ref_w = w.clone()
    ref, ev = step(ref_w, c.lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        own = w.clone()
        out, ev2 = step(own, c.lens)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, ref) and torch.equal(own, ref_w)
    assert all(torch.equal(a, b) for a, b in zip(ev, ev2))
    graph = torch.cuda.CUDAGraph()
    lens = c.lens.clone()
    with torch.cuda.graph(graph):
        out, ev2 = step(w, lens)
    for i in range(4):
        w.zero_()
        lens.copy_(c.lens - i)
        c.q.mul_(0.75)
        acc = torch.zeros_like(w)
        want, ev = step(acc, lens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, acc), i
        assert all(torch.equal(a, b) for a, b in zip(ev, ev2)), i


# ── Positions that run ahead of the rows ─────────────────────────────────────

def test_check_paged_append_position_shift(lib):
    a = _capi.PagedAppendArgs()
    a.c = _cache_args(heads_graph=0)
    a.q = a.q_out = _capi.Tensor(FAKE, 0, 16 * 128, 128)
    a.k = a.v = _capi.Tensor(FAKE, 0, 4 * 128, 128)
    a.inv_freq, a.eps = FAKE, 1e-6
    # (refused before anything is asked of a device)
    assert _st(lib.fna2_paged_append_shifted(ctypes.byref(a), FAKE + 2, None)) == "FNA2_E_STRIDE"
    a.c.total_q = 0
    assert _st(lib.fna2_paged_append_shifted(ctypes.byref(a), FAKE + 4, None)) == "FNA2_OK"
    assert _st(lib.fna2_paged_append_shifted(ctypes.byref(a), None, None)) == "FNA2_OK"


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("lq", [[1, 1, 1], [5, 0, 33]])
def test_append_position_shift(gpu, monkeypatch, lq, given, native):
    """A sequence's positions are its rows (or the positions given) plus a number."""
    if not native:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    c = Case(lq, [40, 9, 33], 4, 2, 3, 128, 8, 16, FP, seed=7, device=gpu, head=1, tail=2)
    g = torch.Generator().manual_seed(2)
    inv = 10000.0 ** (-torch.arange(0, 128, 2).float() / 128)
    shift = torch.tensor([100000, 0, 77], dtype=torch.int32)
    pos = torch.randint(0, 5000, (c.T,), generator=g).to(torch.int32) if given else None
    w = 1 + 0.2 * torch.randn(128, generator=g)
    ref = PO.append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk, inv, pos, w, w,
                    position_shift=shift)
    w = w.to(gpu)
    got = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk,
                             inv.to(gpu), None if pos is None else pos.to(gpu), w, w,
                             position_shift=shift.to(gpu) if native else shift)
    for a, b in ((got, ref[0]), (c.k, ref[1])):
        a = a.double().cpu().numpy()
        assert (np.abs(a - b) <= HALF[FP] * np.abs(b) + 1e-5).all()
    with pytest.raises(AssertionError, match="position_shift"):
        paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, inv_freq=inv.to(gpu),
                           position_shift=shift[:2].to(gpu))
    with pytest.raises(AssertionError, match="position_shift"):
        paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu,
                           position_shift=shift.to(gpu))


# ── A chunk that outgrows its table ──────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[100, 30], [70, 10 ** 8], [2 ** 31 - 1, 64]])
def test_append_past_the_table(gpu, lens):
    """A chunk that outgrows its table: the tokens whose rows the table holds are
    stored at those rows, the others are not, and no older row is touched."""
    c = Case([50, 20], [64, 64], 4, 2, 3, 64, 16, 16, device=gpu, width=4, seed=6)
    c.lens = torch.tensor(lens, dtype=torch.int32, device=gpu)
    before = c.k.clone(), c.v.clone(), c.rk.clone()
    ref = PO.append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk)
    q = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, c.rkn, c.rk)
    for a, b in zip((q, c.k, c.v, c.rk), ref):
        assert (a.double().cpu().numpy() == b).all()
    for b, m in enumerate(c.lq):
        for j in range(min(max(lens[b] - m, 0), 64)):
            p, r = c.slot(b, j)
            for pool, old in zip((c.k, c.v, c.rk), before):
                assert torch.equal(pool[p, :, r], old[p, :, r]), (b, j)


@pytest.mark.gpu
def test_append_past_the_table_keeps_positions(gpu):
    """... and each token is rotated for its own row, stored or not."""
    c = Case([50, 20], [64, 64], 4, 2, 0, 64, 0, 16, device=gpu, width=4, seed=6)
    c.lens = torch.tensor([100, 70], dtype=torch.int32, device=gpu)
    inv = 10000.0 ** (-torch.arange(0, 64, 2).float() / 64)
    ref = PO.append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, inv_freq=inv)
    q = paged.paged_append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu, inv_freq=inv.to(gpu))
    for a, b in zip((q, c.k, c.v), ref):
        a = a.double().cpu().numpy()
        assert (np.abs(a - b) <= HALF[c.dtype] * np.abs(b) + 1e-5).all()


def test_oracle_append_past_the_table():
    """Row by row: token i of m belongs to row lens - m + i, and is stored where
    the table has that row."""
    c = Case([50], [64], 2, 1, 0, 64, 0, 16, width=4)
    c.lens[0] = 100
    _, kp, vp, _ = PO.append(c.q, c.kn, c.vn, c.k, c.v, c.table, c.lens, c.cu)
    for j in range(64):
        p, r = c.slot(0, j)
        want = c.kn[j - 50] if j >= 50 else c.k[p, :, r]
        assert (kp[p, :, r] == want.double().numpy()).all()


# ── Infinities ───────────────────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scores", [True, False])
@pytest.mark.parametrize("lq", [[1, 1], [5, 3], [40, 33]])
@pytest.mark.parametrize("H,HKV,HG,R", [(4, 2, 3, 16), (4, 4, 4, 8), (6, 2, 0, 0)])
def test_weights_of_rows_with_infinite_keys(gpu, lib, monkeypatch, H, HKV, HG, R, lq, scores, causal):
    """A visible row whose score is minus infinity for every token and head weighs
    0: rows of a tile that no token fills do not add to it."""
    if not scores:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
        monkeypatch.setattr(lib, "fna2_paged_scores_bytes", lambda a: 0)
    c = Case(lq, [75, 61], H, HKV, HG, 64, R, 16, device=gpu, seed=9)
    c.q[:, :, 5] = -c.q[:, :, 5].abs() - 0.25
    for b in range(2):
        for j in (0, 2):
            p, r = c.slot(b, j)
            c.k[p, :, r, 5] = float("inf")
    check_attend(c, causal=causal)


def _odd_rank_rows(c, value):
    """R_k of graph head 1 holds `value` in one feature of a visible row of each
    sequence; R_q's feature and the scale are such that an infinity times them
    is minus infinity: head 1 gives the row no weight, the others are as ever."""
    c.rq[:, 1, 3] = -c.rq[:, 1, 3].abs() - 0.25
    c.gs[1] = 1.5
    for b in range(c.N):
        p, r = c.slot(b, min(2, c.lk[b] - c.lq[b]))
        c.rk[p, 1, r, 3] = value


@pytest.mark.gpu
@pytest.mark.parametrize("scores", [True, False])
@pytest.mark.parametrize("hint", [None, 1, 10 ** 6])
@pytest.mark.parametrize("lq", [[1, 1], [5, 3], [40, 33]])
@pytest.mark.parametrize("H,HKV,HG,D,R", [(4, 1, 3, 64, 8), (8, 2, 6, 128, 16), (12, 4, 12, 64, 24),
                                          (32, 1, 20, 64, 64)])
def test_infinite_ranks_stay_with_their_head(gpu, lib, monkeypatch, H, HKV, HG, D, R, lq, hint, scores):
    """Heads share a column tile with their ranks side by side; a row's infinity in
    one head's R_k reaches neither the other graph heads' results nor the vanilla
    heads', nor the rows' weights, whatever the kernel."""
    if not scores:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
        monkeypatch.setattr(lib, "fna2_paged_scores_bytes", lambda a: 0)
    c = Case(lq, [75, 61], H, HKV, HG, D, R, 16, device=gpu, seed=8)
    _odd_rank_rows(c, float("inf"))
    check_attend(c, hint=hint)


@pytest.mark.gpu
@pytest.mark.parametrize("hint", [None, 1, 10 ** 6])
@pytest.mark.parametrize("lq", [[1, 1], [5, 3], [40, 33]])
def test_nan_ranks_stay_with_their_head(gpu, lq, hint):
    c = Case(lq, [75, 61], 4, 1, 3, 64, 16, 16, device=gpu, seed=8)
    _odd_rank_rows(c, float("nan"))
    ref, lse, _, mag = c.oracle()
    out, got = c.attend(hint, return_lse=True)
    assert torch.isnan(out[:, 1]).all()
    for x in (ref, lse, mag):
        x[:, 1] = 0.0
    out[:, 1], got[:, 1] = 0.0, 0.0
    close_out(c, out, ref, mag)
    assert np.abs(got.double().cpu().numpy() - lse).max() <= 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_a_bias_without_its_queries_is_refused(gpu, monkeypatch, native):
    """R_k pages or a graph scale without R_q: an attention without the bias would
    not be what was asked for."""
    if not native:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    args = (c.q, c.k, c.v, c.table, c.lens, c.cu, 3)
    for kw in (dict(rk_pages=c.rk, graph_scale=c.gs), dict(rk_pages=c.rk), dict(graph_scale=c.gs)):
        with pytest.raises(AssertionError, match="r_q"):
            paged.flash_naylis_paged(*args, **kw)
    paged.flash_naylis_paged(*args)


# ── Rows that share memory ───────────────────────────────────────────────────

def test_check_written_rows_do_not_overlap(lib):
    """What a call writes, the pools of append and evict and the weights, has no two
    rows in one memory; pools that are only read may."""
    T = _capi.Tensor

    def codes(**over):
        ap, ev = _capi.PagedAppendArgs(), _capi.PagedEvictArgs()
        ap.c, ev.c = _cache_args(**over), _cache_args(**over)
        ap.q = ap.q_out = T(FAKE, 0, 16 * 128, 128)
        ap.k = ap.v = T(FAKE, 0, 4 * 128, 128)
        ap.r_k = T(FAKE, 0, 12 * 32, 32)
        ev.budget, ev.capacity, ev.stride_b, ev.stride_h = 100, 512, 2048, 512
        ev.key_weights, ev.weights_out, ev.kept, ev.new_lens = FAKE, 2 * FAKE, FAKE, FAKE
        return [_st(f(ctypes.byref(a))) for f, a in ((lib.fna2_check_paged_append, ap),
                                                     (lib.fna2_check_paged_evict, ev),
                                                     (lib.fna2_check_paged_attn, _attn(**over)))]
    fine, shared = ["FNA2_OK"] * 3, ["FNA2_E_STRIDE", "FNA2_E_STRIDE", "FNA2_OK"]
    assert codes() == fine
    assert codes(k_pages=T(FAKE, 64 * 4 * 128, 4 * 128, 128)) == fine      # rows of all heads together
    assert codes(k_pages=T(FAKE, 64 * 128, 128, 50 * 64 * 128)) == fine    # heads outermost
    assert codes(v_pages=T(FAKE, 2 * 4 * 64 * 128, 2 * 128, 2 * 64 * 128)) == fine  # K and V by turns
    assert codes(k_pages=T(FAKE, 0, 128, 64 * 128)) == shared              # one page, many times
    assert codes(v_pages=T(FAKE, 4 * 64 * 128, 128, 0)) == shared          # one head for all
    assert codes(v_pages=T(FAKE, 64 * 128, 128, 64 * 128)) == shared       # pages that overlap
    assert codes(rk_pages=T(FAKE, 12 * 64 * 32, 32, 63 * 32)) == shared
    assert codes(rk_pages=T(FAKE, 11 * 64 * 32, 32, 64 * 32)) == shared
    assert codes(v_pages=T(FAKE, 0, 128, 64 * 128), num_pages=1) == fine

    w = _capi.PagedWeightsArgs()
    w.attn, w.key_weights, w.capacity = _attn(), FAKE, 512
    for (w.stride_b, w.stride_h), want in (((2048, 512), "FNA2_OK"), ((512, 2048), "FNA2_OK"),
                                           ((512, 512), "FNA2_E_STRIDE"), ((1024, 512), "FNA2_E_STRIDE"),
                                           ((512, 1536), "FNA2_E_STRIDE"), ((2047, 512), "FNA2_E_STRIDE")):
        assert _st(lib.fna2_check_paged_weights(ctypes.byref(w))) == want, (w.stride_b, w.stride_h)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_pools_that_share_memory_are_read_only(gpu, monkeypatch, native):
    if not native:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    c = Case([3, 1], [70, 80], 4, 2, 4, 64, 16, 16, device=gpu)
    w = torch.zeros(2, 2, 96, device=gpu)
    v = c.v.clone()
    for k_pages, v_pages in ((c.k, c.k), (c.k[:1].expand_as(c.k), c.v), (c.k, c.v[:, :1].expand_as(c.v))):
        with pytest.raises((AssertionError, RuntimeError)):
            paged.paged_append(c.q, c.kn, c.vn, k_pages, v_pages, c.table, c.lens, c.cu)
        with pytest.raises((AssertionError, RuntimeError)):
            paged.paged_evict(k_pages, v_pages, c.table, c.lens, w, 10)
    assert torch.equal(c.v, v)
    # read, they are what they show
    c.v = c.v[:, :1].expand_as(c.v)
    check_attend(c)
    c.k = c.v
    check_attend(c)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", [True, False])
@pytest.mark.parametrize("dtype,H,HKV,HG,D,R,lq", [(FP, 4, 1, 3, 128, 32, [1, 4]), (BF, 6, 2, 4, 64, 8, [3, 1]),
                                                   (FP, 8, 2, 8, 64, 40, [9, 2]), (BF, 16, 2, 16, 128, 64, [2, 1])])
def test_infinite_ranks_in_a_split_cache(gpu, lib, monkeypatch, dtype, H, HKV, HG, D, R, lq, scores):
    """... and where runs cut the tile: only the run that holds the row is done again,
    and its part joins the others'."""
    if not scores:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
        monkeypatch.setattr(lib, "fna2_paged_scores_bytes", lambda a: 0)
    c = Case(lq, [900, 400], H, HKV, HG, D, R, 48, dtype, device=gpu, seed=10)
    _odd_rank_rows(c, float("inf"))
    for j in (500, 333):
        p, r = c.slot(0, j)
        c.rk[p, 1, r, 3] = float("inf")
    check_attend(c)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[100, 30], [65, 10 ** 8], [2 ** 31 - 1, 64], [114, 70]])
@pytest.mark.parametrize("lq", [[1, 1], [3, 5], [50, 20], [90, 1], [50, 300]])
@pytest.mark.parametrize("H,HKV,HG,R", [(4, 2, 3, 16), (4, 1, 4, 64), (3, 3, 0, 0)])
def test_attend_past_the_table(gpu, H, HKV, HG, R, lq, lens, causal):
    """A chunk that has outgrown its table: a token sees the table's rows up to its
    own row, which the table need not have."""
    c = Case(lq, [64, 64], H, HKV, HG, 64, R, 16, device=gpu, width=4, seed=6)
    c.lens = torch.tensor(lens, dtype=torch.int32, device=gpu)
    check_attend(c, causal=causal)


@pytest.mark.gpu
def test_a_chunk_past_its_table_is_the_wider_tables(gpu):
    """Append and attention of a chunk whose last rows the table does not have: its
    first tokens' results are those of a table with room for all."""
    for lq in (20, 90):
        wide = Case([lq], [64 + lq], 4, 2, 3, 64, 16, 16, device=gpu, seed=3)
        inv = 10000.0 ** (-torch.arange(0, 64, 2, device=gpu).float() / 64)
        room = (64 + lq // 2) // 16 * 16  # rows that the narrow table has
        out = []
        for table in (wide.table, wide.table[:, :room // 16]):
            k, v, rk = wide.k.clone(), wide.v.clone(), wide.rk.clone()
            q = paged.paged_append(wide.q, wide.kn, wide.vn, k, v, table, wide.lens, wide.cu,
                                   wide.rkn, rk, inv)
            y = paged.flash_naylis_paged(q, k, v, table, wide.lens, wide.cu, lq, r_q=wide.rq,
                                         rk_pages=rk, graph_scale=wide.gs)
            out.append((q, y[:room - 64]))
        assert torch.equal(out[0][0], out[1][0])
        h = HALF[BF]
        a, b = (y.double() for _, y in out)
        # (parts may be cut elsewhere: two roundings of the output, and of P)
        assert ((a - b).abs() <= 2 * h * a.abs() + 2 * h * wide.v.double().abs().max()).all()


def test_check_paged_token_count(lib):
    """A full table of 2^30 rows and the tokens behind it still count in 32 bits."""
    for total, want in (((1 << 30) - 256, "FNA2_OK"), ((1 << 30) - 255, "FNA2_E_SHAPE")):
        a = _attn(total_q=total, max_seqlen_q=total, table_width=1 << 24, table_stride=1 << 24)
        assert _st(lib.fna2_check_paged_attn(ctypes.byref(a))) == want
