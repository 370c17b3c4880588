"""Attention over a paged cache whose groups of sequences share their first
rows (fna2_paged_shared) against ``oracle.paged_oracle``, which knows nothing
of groups.

CPU: the C ABI's validation and struct layout, refusals.  GPU: groups of every
kind, over small sizes where they can go wrong.

Tolerances as in ``test_paged``: the output's rounding and P's, h = eps / 2 of
the type each, the second times the same average of |V|, and 2e-4 of that for
fp32 scores; LSE 1e-4, weights 2e-4 relatively.  A token's parts are joined in
fp32, a few 2^-24 of the sums.
"""
import ctypes
import gc
import subprocess

import numpy as np
import pytest
import torch

from fna2_amd import _capi, paged
from tests.test_paged import FAKE, ROOT, Case, _attn, _st, check_attend


class SharedCase(Case):
    """groups: (sequences, rows whose pages they share, rows said to be
    shared) in order; `apart`: sequences ahead of the first group."""

    def __init__(self, lq, lk, *sizes, groups, apart=0, **kw):
        super().__init__(lq, lk, *sizes, **kw)
        cg, rows, b = [apart], [], apart
        for n, pages_rows, said in groups:
            p = pages_rows // self.ps
            for i in range(b + 1, b + n):
                self.table[i, :p] = self.table[b, :p]
            b += n
            cg.append(b)
            rows.append(said)
        self.cg = torch.tensor(cg, dtype=torch.int32, device=self.device)
        self.rows = torch.tensor(rows, dtype=torch.int32, device=self.device)

    def attend(self, hint=None, **kw):
        return paged.flash_naylis_shared(self.q, self.k, self.v, self.table, self.lens, self.cu,
                                         self.max_q if hint is None else hint, self.cg, self.rows,
                                         r_q=self.rq, rk_pages=self.rk, graph_scale=self.gs, **kw)


# ── CPU ──────────────────────────────────────────────────────────────────────

def _shared(**over):
    a = _capi.PagedSharedArgs()
    a.attn = _attn(**{k: v for k, v in over.items() if k not in ("groups", "cu_groups", "shared_rows")})
    a.groups, a.cu_groups, a.shared_rows = 2, FAKE, FAKE
    for k in ("groups", "cu_groups", "shared_rows"):
        if k in over:
            setattr(a, k, over[k])
    return a


@pytest.mark.parametrize("over,code", [
    (dict(), "FNA2_OK"),
    (dict(groups=0, cu_groups=None, shared_rows=None), "FNA2_OK"),
    (dict(groups=-1), "FNA2_E_SHAPE"),
    (dict(groups=1 << 21), "FNA2_E_SHAPE"),
    (dict(cu_groups=None), "FNA2_E_SEQLENS"),
    (dict(shared_rows=None), "FNA2_E_SEQLENS"),
    (dict(head_dim=96), "FNA2_E_HEAD_DIM"),
    (dict(softmax_scale=float("nan")), "FNA2_E_SCALE"),
    (dict(out=_capi.empty_tensor()), "FNA2_E_NULL"),
])
def test_check(over, code):
    lib = _capi.lib()
    a = _shared(**over)
    assert _st(lib.fna2_check_paged_shared(ctypes.byref(a))) == code
    if code != "FNA2_OK":
        assert lib.fna2_paged_shared_workspace_bytes(ctypes.byref(a)) == 0
        assert _st(lib.fna2_paged_shared(ctypes.byref(a), None)) == code
    else:
        assert lib.fna2_paged_shared_workspace_bytes(ctypes.byref(a)) > 0
    assert _st(lib.fna2_check_paged_shared(None)) == "FNA2_E_NULL"


def test_workspace_is_checked_before_any_launch():
    lib = _capi.lib()
    a = _shared()
    if not torch.cuda.is_available():
        pytest.skip("the device comes first")
    assert _st(lib.fna2_paged_shared(ctypes.byref(a), None)) == "FNA2_E_WORKSPACE"


def test_struct_layout_matches_header(tmp_path):
    cls = _capi.PagedSharedArgs
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "fna2.h"', "int main(void){",
             'printf("%zu\\n", sizeof(fna2_paged_shared_args));']
    lines += [f'printf("%zu\\n", offsetof(fna2_paged_shared_args, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


@pytest.mark.parametrize("change", [
    dict(cg=None), dict(rows=None), dict(cg=torch.zeros(2, dtype=torch.int32)),
    dict(rows=torch.zeros(2, 2, dtype=torch.int32)),
])
def test_refusals(change, monkeypatch):
    c = SharedCase([1, 1], [40, 40], 4, 2, 4, 64, 16, 16, groups=[(1, 32, 32), (1, 32, 32)])
    for k, v in change.items():
        setattr(c, k, v)
    monkeypatch.setattr(paged, "_gpu", lambda *a: None)  # (the shapes are looked at on the CPU)
    with pytest.raises(AssertionError):
        c.attend()


def test_needs_the_gpu():
    c = SharedCase([1, 1], [40, 40], 4, 2, 4, 64, 16, 16, groups=[(2, 32, 32)])
    with pytest.raises(RuntimeError, match="GPU"):
        c.attend()


# ── GPU ──────────────────────────────────────────────────────────────────────

gpu = pytest.mark.gpu

CASES = {
    # name: (lq, lk, H, HKV, HG, D, R, ps), groups, further arguments
    "decode": (([1] * 3, [150, 137, 170], 8, 4, 4, 64, 32, 16), [(3, 112, 112)], {}),
    "two_groups": (([1, 2, 1, 1, 3], [300, 290, 289, 200, 199], 8, 4, 8, 64, 32, 16),
                   [(3, 256, 256), (2, 160, 160)], {}),
    "beside_others": (([1, 1, 1, 1], [90, 200, 210, 70], 4, 4, 4, 64, 8, 16), [(2, 160, 160)],
                      dict(apart=1)),
    "no_rows_of_its_own_page": (([1, 1], [97, 97], 4, 2, 4, 64, 16, 48), [(2, 96, 96)], {}),
    "chunk_from_the_prefix_on": (([40, 33, 5], [136, 129, 101], 4, 2, 4, 64, 16, 32),
                                 [(3, 96, 96)], {}),
    # what is said to be shared runs into a chunk, or past the rows: cut
    "said_too_many": (([20, 1], [100, 130], 4, 2, 4, 64, 16, 16), [(2, 96, 96)], {}),
    "said_past_the_end": (([1, 1], [100, 100], 4, 2, 2, 64, 16, 16), [(2, 96, 1 << 30)], {}),
    "said_odd": (([1, 1, 1], [100, 120, 140], 4, 2, 2, 64, 16, 16), [(3, 96, 95)], {}),
    "said_none": (([1, 1], [100, 120], 4, 2, 2, 64, 16, 16), [(2, 96, 0)], {}),
    "said_less_than_none": (([1, 1], [100, 120], 4, 2, 2, 64, 16, 16), [(2, 96, -64)], {}),
    "short": (([1, 1], [3, 1], 4, 2, 2, 64, 16, 16), [(2, 0, 16)], {}),
    "without_tokens": (([0, 1, 0, 2], [100, 90, 4, 70], 4, 2, 4, 64, 16, 16), [(4, 64, 64)], {}),
    "one_with_tokens": (([0, 3], [100, 90], 4, 2, 4, 64, 16, 16), [(2, 64, 64)], {}),
    "no_rows": (([1, 1], [0, 100], 4, 2, 4, 64, 16, 16), [(2, 0, 64)], {}),
    "heads_3": (([1, 4], [200, 203], 12, 4, 12, 128, 32, 64), [(2, 192, 192)], {}),
    "heads_8": (([2, 1], [150, 140], 16, 2, 9, 128, 24, 48), [(2, 96, 96)], {}),
    "heads_2": (([1, 7], [150, 147], 4, 2, 4, 128, 64, 16), [(2, 128, 128)], {}),
    "no_ranks": (([1, 9], [150, 149], 12, 4, 0, 128, 0, 16), [(2, 128, 128)], {}),
    "no_ranks_d64": (([1, 9], [150, 149], 6, 2, 0, 64, 0, 16), [(2, 128, 128)], {}),
    "fp16": (([5, 4, 5, 3], [250, 249, 180, 170], 16, 4, 12, 128, 24, 48),
             [(2, 240, 240), (2, 144, 144)], dict(dtype=torch.float16)),
    "many_tokens": (([70, 64, 31], [390, 384, 351], 4, 1, 4, 64, 32, 64), [(3, 320, 320)], {}),
    "many_tokens_d128": (([129, 100], [390, 361], 2, 2, 2, 128, 64, 64), [(2, 256, 256)], {}),
    # enough shared rows to be worth it for many tokens
    "many_tokens_long": (([70, 64, 31], [1670, 1664, 1631], 4, 1, 4, 64, 32, 64),
                         [(3, 1600, 1600)], {}),
    "many_tokens_long_d128": (([150, 3, 100], [1500, 1353, 1450], 2, 2, 2, 128, 64, 64),
                              [(3, 1344, 1344)], {}),
    "many_sequences_long": (([2] * 70, [270 + i % 23 for i in range(70)], 2, 1, 2, 64, 8, 16),
                            [(30, 256, 256), (40, 240, 250)], {}),
    "few_tokens_each": (([3] * 40, [300 + i % 7 for i in range(40)], 8, 2, 8, 64, 32, 16),
                        [(40, 256, 256)], {}),
    "heads_5": (([1, 6], [300, 305], 10, 2, 7, 64, 16, 16), [(2, 288, 288)], {}),
    "heads_3_many": (([150, 60], [480, 390], 6, 2, 6, 128, 32, 64), [(2, 320, 320)], {}),
    "loose_tokens": (([1, 1], [150, 150], 4, 2, 4, 64, 16, 16), [(2, 128, 128)],
                     dict(head=37, tail=40)),
    "rows_of_heads": (([1, 2], [150, 150], 4, 2, 4, 64, 16, 16), [(2, 128, 128)],
                      dict(layout="prhd")),
    "many_groups": (([1] * 160, [70 + i % 23 for i in range(160)], 2, 1, 2, 64, 8, 16),
                    [(2, 64, 64)] * 80, {}),
    "many_sequences": (([1] * 130, [70 + i % 23 for i in range(130)], 2, 1, 2, 64, 8, 16),
                       [(130, 64, 64)], {}),
    # (more than a workgroup has threads)
    "more_sequences": (([1] * 1100, [134 + i % 23 for i in range(1100)], 2, 1, 2, 64, 8, 16),
                       [(3, 128, 128), (1050, 128, 112), (40, 96, 96)], dict(apart=5)),
    "more_groups": (([1] * 1080, [70 + i % 23 for i in range(1080)], 2, 1, 2, 64, 8, 16),
                    [(1, 0, 64)] * 1000 + [(2, 64, 64)] * 40, {}),
}


def make(name, **kw):
    sizes, groups, more = CASES[name]
    return SharedCase(*sizes, groups=groups, device="cuda", **more, **kw)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("name", CASES)
def test_against_the_oracle(name, causal):
    print(name, causal, flush=True)
    check_attend(make(name), causal=causal)


LONG = [n for n, (_, groups, _) in CASES.items()
        if len(groups) < 3 and any(pages and said for _, pages, said in groups) and "long" not in n]


@gpu
@pytest.mark.parametrize("name", LONG)
def test_long_shared_rows_against_the_oracle(name):
    """The same with 3840 shared rows more, which are worth sharing for any of
    these tokens; whole pages and key steps, so that what lies behind stays."""
    print(name, flush=True)
    (lq, lk, *rest), groups, more = CASES[name]
    shared = range(more.get("apart", 0), more.get("apart", 0) + sum(g[0] for g in groups))
    lk = [n + 3840 * (b in shared) for b, n in enumerate(lk)]
    groups = [(n, pages + 3840, said + 3840 * (said > 0)) for n, pages, said in groups]
    check_attend(SharedCase(lq, lk, *rest, groups=groups, device="cuda", **more))


@gpu
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales(scale):
    check_attend(make("two_groups"), scale=scale)


@gpu
@pytest.mark.parametrize("causal", [True, False])
def test_past_the_table(causal):
    c = SharedCase([1, 2, 1], [112, 100, 105], 4, 2, 4, 64, 16, 16, groups=[(3, 112, 1000)],
                   device="cuda", width=7)
    c.lens[0], c.lens[1] = 200, 113  # more rows than the table has room for
    check_attend(c, causal=causal)


@gpu
def test_without_groups():
    c = make("decode")
    c.cg, c.rows = c.cg[:1], c.rows[:0]
    check_attend(c)


@gpu
def test_without_sequences():
    c = SharedCase([], [], 4, 2, 4, 64, 16, 16, groups=[], device="cuda", tail=3)
    assert (c.attend() == 0).all()
    c.cg, c.rows = torch.zeros(2, dtype=torch.int32, device="cuda"), c.lens.new_ones(1)
    assert (c.attend() == 0).all()


@gpu
def test_pages_that_are_not_there():
    c = make("two_groups")
    c.table[:3, 3] = -1
    c.table[4, 12] = 10 ** 6
    check_attend(c)


@gpu
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_hidden_rows_do_not_matter(what):
    """A later token's V, and rows behind the sequence."""
    c = make("chunk_from_the_prefix_on")
    ref = c.attend()
    for b, row in ((0, 135), (1, 128), (2, 100)):
        page, off = c.slot(b, row)
        c.v[page, :, off] = what
        c.v[page, :, off + 1:] = what
        c.k[page, :, off + 1:] = what
    out = c.attend()
    last = [39, 72, 77]
    keep = [t for t in range(78) if t not in last]
    assert torch.equal(out[keep], ref[keep])
    assert not torch.isfinite(out[last]).any()


@gpu
def test_an_infinite_shared_row_reaches_every_token():
    c = make("two_groups")
    page, off = c.slot(0, 5)
    c.v[page, 1, off, 3] = float("inf")
    out = c.attend()
    group = slice(0, 4)  # the tokens of the first group
    assert torch.isposinf(out[group, 2:4, 3]).all()
    out[group, 2:4, 3] = 0
    assert torch.isfinite(out).all()


@gpu
def test_the_same_every_time_and_on_another_stream():
    c = make("many_tokens")
    first = c.attend()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = c.attend()
    stream.synchronize()
    assert torch.equal(first, again)
    plain = paged.flash_naylis_paged(c.q, c.k, c.v, c.table, c.lens, c.cu, c.max_q, r_q=c.rq,
                                     rk_pages=c.rk, graph_scale=c.gs)
    assert (first.float() - plain.float()).abs().max() < 0.05


@gpu
def test_python_launcher_gives_the_same(monkeypatch):
    c = make("fp16")
    first, lse = c.attend(return_lse=True)
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    again, lse2 = c.attend(return_lse=True)
    assert torch.equal(first, again) and torch.equal(lse, lse2)


@gpu
def test_captured_step_follows_lengths_and_groups():
    c = make("two_groups")
    c.attend()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend()
    for cut in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.attend())
        c.lens -= 17
        c.rows -= 32
        if cut == 1:
            c.cg[1] = 2  # the third sequence into the second group: it shares nothing with it
            c.rows[1] = 0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, c.attend())


@gpu
def test_two_captured_graphs_share_nothing():
    a, b = make("decode"), make("two_groups")
    want = a.attend(), b.attend()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        oa = a.attend()
    with torch.cuda.graph(gb):
        ob = b.attend()
    for _ in range(3):
        ga.replay(), gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa, want[0]) and torch.equal(ob, want[1])


@gpu
def test_pools_past_32_bits():
    """The same pages at the end of pools of more than 2^31 elements."""
    c = make("two_groups")
    want = c.attend()
    n, P = c.k.shape[0], 2 ** 31 // c.k[0].numel() + 1
    for name in ("k", "v", "rk"):
        old = getattr(c, name)
        big = torch.empty((P + n, *old.shape[1:]), dtype=old.dtype, device="cuda")
        big[P:] = old
        setattr(c, name, big)
    c.table = torch.where(c.table >= 0, c.table + P, c.table)
    assert c.k.numel() > 2 ** 31 and torch.equal(c.attend(), want)


@gpu
def test_strided_inputs():
    c = make("fp16")
    want = c.attend()
    wide = torch.zeros(c.T, 3, c.H, c.D, dtype=c.dtype, device="cuda")
    wide[:, 1] = c.q
    c.q = wide[:, 1]
    odd = torch.zeros(c.T, c.HG, c.R + 4, dtype=torch.bfloat16, device="cuda")
    odd[:, :, 4:] = c.rq
    c.rq = odd[:, :, 4:]
    c.cg, c.rows = c.cg.long(), c.rows.cpu()
    assert torch.equal(c.attend(), want)


# Chunks that flash_naylis_paged serves with P in two parts (one column tile holds them)
SHORT = ["decode", "two_groups", "beside_others", "without_tokens", "heads_3", "heads_8", "no_ranks",
         "fp16", "few_tokens_each", "many_sequences_long", "more_sequences", "loose_tokens"]


def rounding(c, ref):
    """Root mean square of what the output's own rounding leaves."""
    own = torch.from_numpy(ref).to(c.dtype).double().numpy() - ref
    return np.sqrt((own ** 2).mean())


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("name", SHORT)
def test_short_chunks_are_as_precise_as_without_groups(name, causal):
    """P in two parts is off by 2^-16 of each p (bf16) or less, the scores by some 1e-5: against
    the output's rounding, which is off by 2^-9 / sqrt(3) = 1.1e-3 (bf16) or 1.4e-4 (fp16) of the
    value on average, both add less than 1% to the root of the mean square (1.1 allowed).  P in
    one part is off by as much again as the output: 1.4 times."""
    print(name, causal, flush=True)
    c = make(name)
    ref = c.oracle(causal=causal)[0]
    err = np.sqrt(((c.attend(is_causal=causal).double().cpu().numpy() - ref) ** 2).mean())
    assert err <= 1.1 * rounding(c, ref)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", [-12, 12])
@pytest.mark.parametrize("row", [5, 113])
def test_an_infinite_row_stays_infinite(row, score, dtype):
    """A first row, which is shared, or an own one, that weighs e^-12 (fp16 holds 2^-24 = e^-16.6)
    of the others, or that most of the weight is on, where p is 1 and its second part nothing: as
    without groups."""
    c = SharedCase([1] * 3, [150, 137, 170], 4, 2, 0, 64, 0, 16, groups=[(3, 112, 112)], dtype=dtype,
                   device="cuda")
    c.q[:] = c.q[:1, :1]
    for b in (range(1) if row < 112 else range(3)):
        page, off = c.slot(b, row)
        c.k[page, :, off] = score * 8 * c.q[0, 0] / c.q[0, 0].float().square().sum()
        c.v[page, 1, off, 3] = float("inf")
    for out in (c.attend(), paged.flash_naylis_paged(c.q, c.k, c.v, c.table, c.lens, c.cu, 1)):
        assert torch.isposinf(out[:, 2:, 3]).all()
        out[:, 2:, 3] = 0
        assert torch.isfinite(out).all()


def limited(c):
    """The call with memory for flash_naylis_paged, but not for the shared rows' parts."""
    plain = lambda: paged.flash_naylis_paged(c.q, c.k, c.v, c.table, c.lens, c.cu, c.max_q, r_q=c.rq,
                                             rk_pages=c.rk, graph_scale=c.gs, return_lse=True)
    want = [t.cpu() for t in plain()]
    total = torch.cuda.get_device_properties(0).total_memory
    limit = lambda nbytes: torch.cuda.set_per_process_memory_fraction(nbytes / total)
    peaks, held = [], []
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    try:
        # what other tests left between their tensors is taken first
        limit(torch.cuda.memory_reserved())
        size = 1 << 32
        while size >= 1 << 21:
            try:
                held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            except torch.OutOfMemoryError:
                size >>= 1
        limit(total)
        for call in (plain, lambda: c.attend(return_lse=True)):
            torch.cuda.reset_peak_memory_stats()
            call()
            torch.cuda.synchronize()
            peaks.append(torch.cuda.max_memory_reserved())
            torch.cuda.empty_cache()
        assert peaks[1] > peaks[0] + (8 << 20)
        limit(sum(peaks) / 2)
        return [t.cpu() for t in c.attend(return_lse=True)], want
    finally:
        limit(total)


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_without_the_memory_each_sequence_by_itself(native, monkeypatch):
    """The shared rows' parts take 8 bytes a token, head and feature; without them the call is
    flash_naylis_paged's."""
    if not native:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    c = SharedCase([60] * 64, [140 + i % 9 for i in range(64)], 16, 4, 16, 128, 32, 16,
                   groups=[(64, 64, 64)], device="cuda")
    got, want = limited(c)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.undo()
    c.max_q = 1 << 20  # (and with no limit, again)
    assert (c.attend().cpu().float() - want[0].float()).abs().max() < 0.05
