"""DevicePageTable, and NaylisAttention that serves from it: sequences that share a
prefix, steps captured whole, rotary positions in other layouts.

Books are whole numbers, equal to PageTable's.  A layer's outputs from pages are
compared with its own forward over whole sequences: both compute the same products of bf16
values and may round six things between to other neighbours (the rotated q and k, P, its
parts' join, the attention's output and the layer's), each by at most 2^-8 of the value:
6 * 2^-8 of the output's norm.
"""
import math

import pytest
import torch

from fna2_amd.attention_fna2 import NaylisAttention, RotaryPositionalEmbedding
from fna2_amd import paged
from fna2_amd.paged import DevicePageTable, PagedKVCache, PagedStep, PageTable
from tests.helpers import rel_norm

gpu_test = pytest.mark.gpu
TOL = 6 * 2.0 ** -8
EXTENDED = [dict(rope=dict(rotary_dim=32)), dict(rope=dict(interleaved=True)),
            dict(rope=dict(rotary_dim=24)),
            dict(rope=dict(rotary_dim=40, interleaved=True, scaling="yarn", factor=4.0,
                           original_max_len=64)),
            dict(rope=dict(scaling="linear", factor=2.0), use_qk_norm=False)]


# ── CPU ──────────────────────────────────────────────────────────────────────

def test_rotary_module_by_the_formula():
    r = RotaryPositionalEmbedding(16, rotary_dim=8, interleaved=True, scaling="linear", factor=2.0)
    assert r.extended and r.inv_freq.shape == (4,)
    q = torch.randn(2, 3, 5, 16, dtype=torch.float64)
    y, _ = r(q, q, position_offset=7)
    for s in range(5):
        for i in range(4):
            a = (7 + s) * 10000.0 ** (-2 * i / 8) / 2
            u, v = q[..., s, 2 * i], q[..., s, 2 * i + 1]
            c, si = torch.tensor(a).double().cos(), torch.tensor(a).double().sin()
            assert torch.allclose(y[..., s, 2 * i], u * c - v * si, atol=1e-5)
            assert torch.allclose(y[..., s, 2 * i + 1], v * c + u * si, atol=1e-5)
    assert torch.equal(y[..., 8:], q[..., 8:])


def test_rotary_module_plain_and_refusals():
    assert not RotaryPositionalEmbedding(16).extended
    assert not RotaryPositionalEmbedding(16, rotary_dim=16).extended
    for bad in (dict(rotary_dim=7), dict(rotary_dim=18), dict(rotary_dim=0),
                dict(scaling="more"), dict(interleaved=True, use_yarn=True)):
        with pytest.raises(ValueError):
            RotaryPositionalEmbedding(16, **bad)
    m = NaylisAttention(128, 2, rel_rank=8).rotate_by(rotary_dim=32, interleaved=True)
    assert m.rope.inv_freq.shape == (16,) and m.rope.interleaved
    with pytest.raises(ValueError):
        NaylisAttention(128, 2, use_rope=False).rotate_by(32)


def test_table_refusals():
    with pytest.raises(AssertionError):
        DevicePageTable(1, 4, page_size=24, device="cpu")
    t = DevicePageTable(3, 8, page_size=16, device="cpu")
    with pytest.raises(AssertionError):
        t.extend(torch.ones(3, dtype=torch.int32))  # a bound of the tokens is missing
    with pytest.raises(AssertionError):
        t.share(0, [0, 1], 32)
    with pytest.raises(AssertionError):
        t.share(0, [1, 1], 32)
    with pytest.raises(AssertionError):
        t.share(0, [1], 16 * 9)
    assert t.share(0, [1], 15) == 0 and t.cu_groups is None
    for call in (lambda: t.share(0, [-3], 16), lambda: t.share(-1, [0], 16), lambda: t.release(3),
                 lambda: t.share(0, [1], 16)):  # (which has no rows)
        with pytest.raises(ValueError):
            call()
    t._lent[0] = {1}
    with pytest.raises(ValueError, match="share rows"):
        t.truncate(8)
    with pytest.raises(ValueError, match="share rows"):
        PagedKVCache.empty(t, 1, 64, weigh=True).evict(8)
    with pytest.raises(ValueError, match="shared by"):
        t.release(0)
    with pytest.raises(RuntimeError, match="GPU"):
        t.extend([1, 1, 1])


# ── GPU: the books ───────────────────────────────────────────────────────────

def same(d, h):
    assert d.block_table.tolist() == h.block_table.tolist()
    assert d.seqlens.tolist() == h.seqlens.tolist()
    assert d.cu_seqlens_q.tolist() == h.cu_seqlens_q.tolist()
    assert d.position_shift.tolist() == h.position_shift.tolist()
    n = d.free_count.item()
    assert d.free_pages.tolist()[:n] == h._free


@gpu_test
def test_the_same_books_as_the_hosts(gpu):
    d = DevicePageTable(4, 30, page_size=16, max_pages=9, device=gpu)
    h = PageTable(4, 30, page_size=16, max_pages=9, device=gpu)
    same(d, h)
    for step in ([37, 0, 5, 1], [1, 60, 1, 1], "truncate 20", [3, 1, 0, 2], "release 1",
                 [1, 16, 1, 1], "truncate 8", "release 0", [50, 1, 1, 1]):
        if isinstance(step, str):
            what, n = step.split()
            for t in (d, h):
                getattr(t, what)(int(n))
        else:
            d.extend(step)
            h.extend(step)
            d.check()
            assert d.total_q == h.total_q and d.max_seqlen_q == h.max_seqlen_q
            want = h.positions if h.positions is not None else h.token_positions(h.total_q)
            assert d.positions.tolist() == want.tolist()
            assert d.token_positions(d.total_q).tolist() == want.tolist()
        same(d, h) if not isinstance(step, str) else None


@gpu_test
def test_full_table_and_rollback(gpu):
    t = DevicePageTable(2, 4, page_size=16, device=gpu)
    t.extend([20, 20])
    before = t.block_table.tolist()
    t.extend([20, 1])
    with pytest.raises(ValueError, match="1 pages"):
        t.check()
    assert t.block_table.tolist() == before and t.seqlens.tolist() == [20, 20]
    assert t.cu_seqlens_q.tolist() == [0, 0, 0] and (t.slots == -1).all()
    t.extend(torch.tensor([5, 1], dtype=torch.int32, device=gpu), total_q=7, max_seqlen_q=5)
    t.check()
    assert t.sequences.tolist() == [0] * 5 + [1, -1] and t.max_seqlen_q == 5
    t.rollback(torch.tensor([22, 100], dtype=torch.int32, device=gpu))
    assert t.seqlens.tolist() == [22, 21] and t.position_shift.tolist() == [0, 0]
    t.extend([1, 1])
    assert t.positions.tolist() == [22, 21]
    with pytest.raises(ValueError, match="more than 1 tokens"):
        t.extend(torch.tensor([1, 1], dtype=torch.int32, device=gpu), total_q=1)
        t.check()
    with pytest.raises(ValueError, match="outgrows"):
        t.extend([100, 0])
        t.check()


@gpu_test
def test_shared_pages_go_back_once(gpu):
    t = DevicePageTable(4, 20, page_size=16, device=gpu)
    t.extend([70, 0, 0, 0])
    assert t.share(0, [1, 3], 65) == 64
    assert t.cu_groups.tolist() == [0, 2, 3, 4, 4] and t.shared_rows.tolist() == [64, 0, 0, 0]
    assert t.seqlens.tolist() == [70, 64, 0, 64] and t.free_count.item() == 15
    t.extend([1, 20, 1, 1])
    assert t.positions.tolist() == [70, *range(64, 84), 0, 64] and t.free_count.item() == 11
    t.rollback(torch.tensor([71, 40, 1, 100], dtype=torch.int32, device=gpu))
    # (shared rows stay, or the next token's row would lie on a page that is another's too)
    assert t.borrowed.tolist() == [0, 4, 0, 4] and t.free_count.item() == 13
    assert t.seqlens.tolist() == [71, 64, 1, 65]
    with pytest.raises(ValueError, match=r"shared by \[1, 3\]"):
        t.release(0)
    t.release(1)
    assert t.free_count.item() == 13 and t.seqlens.tolist() == [71, 0, 1, 65]
    assert t.shared_rows.tolist() == [0, 0, 0, 0]
    t.release(0, 3)
    t.release(2)
    assert t.free_count.item() == 20 and sorted(t.free_pages.tolist()) == list(range(20))
    assert (t.block_table == -1).all()


@gpu_test
def test_shared_rows_stay(gpu):
    t = DevicePageTable(4, 20, page_size=16, device=gpu)
    t.extend([40, 0, 5, 0])
    for lender, borrowers, rows in ((0, [2], 16), (0, [1], 48), (3, [1], 16)):
        with pytest.raises(ValueError, match="rows"):
            t.share(lender, borrowers, rows)
    assert not t.shares and t.share(0, [1], 40) == 32 and t.shares
    t.extend([0, 20, 0, 0])
    assert t.share(1, [3], 48) == 48  # two pages of the first's, one of the second's
    assert t.cu_groups.tolist() == [0, 2, 3, 4, 4] and t.held.tolist() == [32, 48, 0, 48]
    t.rollback(torch.zeros(4, dtype=torch.int32, device=gpu))
    assert t.seqlens.tolist() == [32, 48, 0, 48] and t.free_count.item() == 17
    for b in (0, 1):
        with pytest.raises(ValueError, match="shared by"):
            t.release(b)
    t.release(3)
    assert t.held.tolist() == [32, 32, 0, 0]
    t.rollback(torch.zeros(4, dtype=torch.int32, device=gpu))
    assert t.seqlens.tolist() == [32, 32, 0, 0] and t.free_count.item() == 18
    t.release(1)
    assert t.held.tolist() == [0] * 4 and not t.shares
    t.truncate(16)
    assert t.seqlens.tolist() == [16, 0, 0, 0] and t.position_shift.tolist() == [16, 0, 0, 0]
    t.release(0)
    assert sorted(t.free_pages.tolist()) == list(range(20)) and t.free_count.item() == 20


# ── GPU: a layer on it ───────────────────────────────────────────────────────

def layer(gpu, rope=None, **kw):
    torch.manual_seed(0)
    m = NaylisAttention(512, 8, n_kv_heads=2, max_seq_len=256, **{**dict(rel_rank=16), **kw})
    with torch.no_grad():
        if m.graph_scale is not None:
            m.graph_scale.normal_(1.0, 0.5)
            m.rel_q_proj.weight.normal_(std=0.05)
            m.rel_k_proj.weight.normal_(std=0.05)
        if m.q_norm is not None:
            m.q_norm.weight.uniform_(0.5, 1.5)
            m.k_norm.weight.uniform_(0.5, 1.5)
    if rope:
        m.rotate_by(**rope)
    return m.to(gpu).bfloat16().eval()


def cache(m, t, **kw):
    return PagedKVCache.empty(t, m.n_kv_heads, m.head_dim, m.graph_heads, m.rel_rank, **kw)


class Served:
    """Three users behind one prompt: a lender, its prompt taken in, then shared."""

    def __init__(self, m, gpu, prompt=100, steps=((5, 30, 1), (1, 1, 1), (1, 0, 2)), ps=16):
        g = torch.Generator().manual_seed(1)
        self.m, self.steps = m, steps
        self.prompt = torch.randn(prompt, 512, generator=g).bfloat16().to(gpu)
        rows = prompt // ps * ps
        # each user's tokens: what of the prompt is on no whole page, then its own
        self.own = [torch.cat((self.prompt[rows:], torch.randn(sum(s[b] for s in steps), 512,
                                                               generator=g).bfloat16().to(gpu)))
                    for b in range(3)]
        self.table = DevicePageTable(4, 60, page_size=ps, device=gpu)
        self.cache = cache(m, self.table)
        self.table.extend([prompt, 0, 0, 0])
        m(self.prompt, past_kv=self.cache)
        assert self.table.share(0, [1, 2, 3], prompt) == rows
        self.rows, self.at = rows, [0, 0, 0]

    def take(self, counts):
        x = [o[a:a + c] for o, a, c in zip(self.own, self.at, counts)]
        self.at = [a + c for a, c in zip(self.at, counts)]
        return torch.cat(x)

    def run(self):
        out = [[], [], []]
        first = [len(o) - sum(s[b] for s in self.steps) + self.steps[0][b] for b, o in enumerate(self.own)]
        for counts in (first, *self.steps[1:]):
            self.table.extend([0, *counts])
            y, _ = self.m(self.take(counts), past_kv=self.cache, use_kv_cache=True)
            for b, part in enumerate(y.split(list(counts))):
                out[b].append(part)
        self.table.check()
        return [torch.cat(o) for o in out]

    def whole(self):
        """The users' own rows of the layer's forward over whole sequences."""
        out = []
        for o in self.own:
            x = torch.cat((self.prompt[:self.rows], o))
            y, _ = self.m(x, cu_seqlens_q=torch.tensor([0, len(x)], dtype=torch.int32, device=x.device),
                          max_seqlen_q=len(x), max_seqlen_k=len(x))
            out.append(y[self.rows:])
        return out


@gpu_test
@pytest.mark.parametrize("kw", [dict(), dict(vanilla_heads=3), *EXTENDED])
def test_users_behind_one_prompt(gpu, kw):
    with torch.no_grad():
        s = Served(layer(gpu, **kw), gpu)
        for got, want in zip(s.run(), s.whole()):
            assert rel_norm(got, want) <= TOL


@gpu_test
@pytest.mark.parametrize("kw", EXTENDED)
def test_other_rotary_layouts_on_every_path(gpu, kw):
    """Dense, packed, decoding against both caches, and paged by the host's table."""
    m = layer(gpu, **kw)
    x = torch.randn(2, 50, 512, device=gpu).bfloat16()
    with torch.no_grad():
        dense, _ = m(x)
        cu = torch.tensor([0, 50, 100], dtype=torch.int32, device=gpu)
        packed, _ = m(x.view(100, 512), cu_seqlens_q=cu, max_seqlen_q=50, max_seqlen_k=50)
        assert rel_norm(packed.view(2, 50, 512), dense) <= TOL
        t = PageTable(2, 20, page_size=16, device=gpu)
        c = cache(m, t)
        parts = []
        for a, b in ((0, 33), (33, 34), (34, 50)):
            t.extend([b - a, b - a])
            parts.append(m(x[:, a:b], past_kv=c)[0])
        assert rel_norm(torch.cat(parts, 1), dense) <= TOL
    # the kernel's rotation against the module's own formula, as the decode step has it
    q = torch.randn(100, 8, 64, device=gpu)
    k = torch.randn(100, 2, 64, device=gpu)
    a = m.rope.forward_varlen(q, k, cu)
    for i in (0, 1):
        rows = lambda y: y[50 * i:50 * i + 50].transpose(0, 1)[None]
        b = m.rope(rows(q), rows(k))
        for y, z in zip(a, b):
            assert (rows(y) - z).abs().max() <= 1e-5


@gpu_test
def test_decoding_in_another_layout(gpu):
    from fna2_amd.attention_fna2 import StaticKVCache
    m = layer(gpu, dict(rotary_dim=32, interleaved=True), decode_graph_bias=True)
    x = torch.randn(2, 20, 512, device=gpu).bfloat16()
    with torch.no_grad():
        dense, _ = m(x)
        static = StaticKVCache.empty(2, 2, 32, 64, 8, 16, device=gpu)
        _, past = m(x[:, :19], use_kv_cache=True)
        y, _ = m(x[:, 19:], past_kv=past)
        assert rel_norm(y, dense[:, 19:]) <= TOL
        m(x[:, :19], past_kv=static, use_kv_cache=True)
        y, _ = m(x[:, 19:], past_kv=static)
        assert rel_norm(y, dense[:, 19:]) <= TOL


@gpu_test
@pytest.mark.parametrize("kw", EXTENDED)
def test_training_in_another_layout(gpu, kw):
    """The layer's gradients with the kernel's rotation and with the formula's, by autograd."""
    m = layer(gpu, **kw).train()
    x = torch.randn(70, 512, device=gpu).bfloat16()
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=gpu)
    dy = torch.randn(70, 512, device=gpu).bfloat16()

    def grads():
        xs = x.clone().requires_grad_()
        y, _ = m(xs, cu_seqlens_q=cu, max_seqlen_q=40, max_seqlen_k=40)
        m.zero_grad()
        y.backward(dy)
        return [xs.grad] + [p.grad.clone() for p in m.parameters() if p.grad is not None]

    mine = grads()

    def formula(q, k, cu_seqlens, norm_q=None, norm_k=None, eps=1e-6, grad_slab=None):
        def one(y, w):
            y = y.float()
            if w is not None:
                y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
            parts = [m.rope._turn(p.transpose(0, 1), 0).transpose(0, 1) for p in y.split([30, 40])]
            return torch.cat(parts).to(q.dtype)
        return one(q, norm_q), one(k, norm_k)

    m.rope.forward_varlen = formula
    want = grads()
    assert len(mine) == len(want)
    for a, b in zip(mine, want):
        # q and k (and their gradients) round to neighbours: 2^-8 each, through the
        # products of the attention's and the projection's backward
        assert rel_norm(a, b) <= 8 * 2.0 ** -8


@gpu_test
def test_replaced_norms_with_another_layout(gpu):
    m = layer(gpu, dict(rotary_dim=32, interleaved=True))
    with torch.no_grad():
        want = Served(m, gpu).run()
        m.q_norm.register_forward_hook(lambda mod, i, o: o)
        for a, b in zip(Served(m, gpu).run(), want):
            assert rel_norm(a, b) <= TOL


@gpu_test
def test_replaced_rope_needs_the_hosts_table(gpu):
    m = layer(gpu)
    m.rope.register_forward_hook(lambda mod, i, o: o)
    t = DevicePageTable(1, 4, page_size=16, device=gpu)
    t.extend([3])
    with pytest.raises(RuntimeError, match="PageTable"), torch.no_grad():
        m(torch.randn(3, 512, device=gpu).bfloat16(), past_kv=cache(m, t))


@gpu_test
@pytest.mark.parametrize("kw", [dict(), dict(rope=dict(rotary_dim=32, interleaved=True))])
def test_a_step_captured_whole(gpu, kw):
    """Books, rotation, append and attention in one graph, replayed step after step."""
    m = layer(gpu, **kw)
    with torch.no_grad():
        eager, graphed = Served(m, gpu), Served(m, gpu)
        first = [9, 34, 5]
        for s in (eager, graphed):
            s.table.extend([0, *first])
            m(s.take(first), past_kv=s.cache)
        x = torch.randn(3, 512, device=gpu).bfloat16()
        counts = torch.tensor([0, 1, 1, 1], dtype=torch.int32, device=gpu)

        def step(s):
            s.table.extend(counts, total_q=3, max_seqlen_q=1)
            return m(x, past_kv=s.cache)[0]

        warm = Served(m, gpu)
        warm.table.extend([0, *first])
        step(warm)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step(graphed)
        for i in range(25):  # (past a page's end)
            x.normal_()
            counts[2] = i % 2  # (one sequence pauses: the step then has a token too many)
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            assert torch.equal(graphed.table.block_table, eager.table.block_table)
            assert torch.equal(graphed.table.seqlens, eager.table.seqlens)
        eager.table.check()
        graphed.table.check()


@gpu_test
def test_a_captured_step_outlives_its_sharing(gpu):
    """Captured while rows are shared and replayed after the last borrower's release, and the
    other way round."""
    m = layer(gpu)
    with torch.no_grad():
        for shared in (True, False):
            s = Served(m, gpu)
            if not shared:
                s.table.release(1, 2, 3)
                s.table.extend([0, 20, 20, 20])
                m(torch.randn(60, 512, device=gpu).bfloat16(), past_kv=s.cache)
            x = torch.randn(3, 512, device=gpu).bfloat16()
            step = lambda: m(x, past_kv=s.cache)[0]
            s.table.extend([0, 1, 1, 1])
            assert s.table.shares == shared
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = step()
            for i in range(3):
                if i == 1 and shared:
                    s.table.release(1, 2, 3)
                elif i == 1:
                    s.table.release(1, 2, 3)
                    assert s.table.share(0, [1, 2, 3], 96) == 96
                s.table.extend([0, 1, 1, 1])
                x.normal_()
                graph.replay()
                torch.cuda.synchronize()
                assert rel_norm(y, step()) <= TOL


@gpu_test
def test_a_full_table_changes_nothing(gpu):
    m = layer(gpu)
    t = DevicePageTable(2, 3, page_size=16, device=gpu)
    c = cache(m, t)
    x = torch.randn(40, 512, device=gpu).bfloat16()
    with torch.no_grad():
        t.extend([16, 16])
        m(x[:32], past_kv=c)
        before = c.k.clone()
        t.extend([20, 20])
        y, _ = m(x, past_kv=c)
    assert torch.equal(c.k, before) and t.status.item() == 3
    with pytest.raises(ValueError):
        t.check()


@gpu_test
def test_weights_of_shared_rows(gpu):
    """key_weights of a step that shares rows: as without."""
    m = layer(gpu)
    with torch.no_grad():
        got = []
        for shared in (True, False):
            s = Served(m, gpu)
            s.cache.key_weights = torch.zeros(4, 2, s.table.width * 16, device=gpu)
            if not shared:
                s.table.cu_groups = None
            s.run()
            got.append(s.cache.key_weights)
        assert (got[0] - got[1]).abs().max() <= 2e-2 and got[0].sum() > 0


def plain_extend(table, seqlens, counts, free_pages, free_count, page_size, total_q, shift=None):
    """paged_extend's step in plain Python (pages apart), on the CPU."""
    c, lens, T = counts.tolist(), seqlens.tolist(), total_q
    pos = [n + i for n, k in zip(lens, c) for i in range(k)]
    of = [b for b, k in enumerate(c) for _ in range(k)]
    ints = lambda x, n: torch.tensor(x + [-1] * (n - len(x)), dtype=torch.int32)
    cu = [sum(c[:b]) for b in range(len(c) + 1)]
    return PagedStep(ints(cu, len(cu)), ints([n + k for n, k in zip(lens, c)], len(c)),
                     free_count.clone(), ints(pos, T).long(), ints(of, T), ints(pos, T),
                     torch.zeros(1, dtype=torch.int32))


def test_a_steps_numbers_stay_where_they_are(monkeypatch):
    """What a captured layer reads of a step lies where it lay in the step that was captured,
    whatever steps came between."""
    monkeypatch.setattr(paged, "paged_extend", plain_extend)
    t = DevicePageTable(3, 8, page_size=16, device="cpu")
    with torch.inference_mode():
        t.extend([1, 1, 1])
    seen = {n: getattr(t, n) for n in ("slots", "sequences", "positions", "seqlens",
                                       "cu_seqlens_q", "status", "block_table", "position_shift")}
    for counts in ([40, 0, 3], [0, 0, 0], [1, 0, 0], [0, 1, 1], [2, 1, 1]):
        t.extend(counts)
        n = sum(counts)
        assert t.total_q == n and t.positions.shape == t.slots.shape == t.sequences.shape == (n,)
    t.extend([0, 2, 1])
    for n, x in seen.items():
        y = getattr(t, n)
        assert x.data_ptr() == y.data_ptr() and torch.equal(x, y)
    assert seen["positions"].tolist() == [3, 4, 6] and seen["sequences"].tolist() == [1, 1, 2]


@gpu_test
@pytest.mark.parametrize("kw", EXTENDED)
@pytest.mark.parametrize("inside", [False, True])
def test_a_captured_layer_in_another_layout_follows_the_table(gpu, kw, inside):
    """Captured with its extend outside the graph (or inside it), and replayed after steps of
    other sizes: the rows that it appends, and their angles, are the step's at hand."""
    m = layer(gpu, **kw)
    with torch.no_grad():
        eager, graphed = Served(m, gpu), Served(m, gpu)
        counts = torch.tensor([0, 1, 1, 1], dtype=torch.int32, device=gpu)
        x = torch.randn(3, 512, device=gpu).bfloat16()

        def take(s):
            s.table.extend(counts, total_q=3, max_seqlen_q=1)

        def step(s):
            return m(x, past_kv=s.cache)[0]

        for s in (eager, graphed):
            take(s)
            step(s)
        torch.cuda.synchronize()
        take(eager)
        graph = torch.cuda.CUDAGraph()
        if inside:
            with torch.cuda.graph(graph):
                take(graphed)
                y = step(graphed)
        else:
            take(graphed)
            with torch.cuda.graph(graph):
                y = step(graphed)
        for i in range(5):
            if i > 0:
                take(eager)
                if not inside:
                    take(graphed)
            x.normal_()
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            used = graphed.table.block_table.flatten().unique()[1:].long()
            assert torch.equal(graphed.cache.k[used], eager.cache.k[used])
            other = torch.randn(40 + 7 * i, 512, device=gpu).bfloat16()
            for s in (eager, graphed):  # (a step of another size between the replays)
                s.table.extend([0, 9 + i, 30 + 6 * i, 1])
                m(other, past_kv=s.cache)
            junk = [torch.full((n,), 1 << 20, dtype=torch.int32, device=gpu) for n in (3, 4, 8) * 20]
            del junk
        eager.table.check()
        graphed.table.check()


def test_rollback_reaches_the_caches_that_weigh(monkeypatch):
    """Every cache on the table, copies with theirs, none that has gone; rows that stay keep what
    they have."""
    import copy
    import pickle

    def trim(table, lens, keep, free, count, ps, borrowed=None):
        return torch.minimum(lens, keep), count.clone()

    monkeypatch.setattr(paged, "paged_trim", trim)
    t = DevicePageTable(2, 4, page_size=16, device="cpu")
    caches = [PagedKVCache.empty(t, 2, 64, weigh=w) for w in (True, False, True)]
    t.seqlens += torch.tensor([20, 9], dtype=torch.int32)
    for c in caches[::2]:
        c.key_weights += 1
    other = copy.deepcopy(caches[0])
    again = pickle.loads(pickle.dumps(caches[0]))
    assert other.table is not t and again.table is not t
    t.rollback(torch.tensor([17, 30], dtype=torch.int32))
    for c in caches[::2]:
        assert (c.key_weights[0, :, :17] == 1).all() and (c.key_weights[1, :, :9] == 1).all()
        assert c.key_weights.sum() == 2 * (17 + 9)
    for c in (other, again):
        assert (c.key_weights == 1).all()
        c.table.rollback(torch.tensor([0, 3], dtype=torch.int32))
        assert c.key_weights.sum() == 2 * 3
    assert caches[0].key_weights.sum() == 2 * (17 + 9)
    del caches[1:]
    assert len(paged._CACHES[t]) == 1


@gpu_test
@pytest.mark.parametrize("captured", [False, True])
def test_rows_that_were_rolled_back_weigh_nothing(gpu, captured):
    """Refused tokens' rows start again from no weight, as in a cache that never saw them."""
    m = layer(gpu)
    x = torch.randn(29, 512, device=gpu).bfloat16()
    accepted, drafted, after = (torch.randn(n, 512, device=gpu).bfloat16() for n in (1, 6, 5))
    with torch.no_grad():
        caches = []
        for drafts in (True, False):
            t = DevicePageTable(2, 20, page_size=16, max_pages=5, device=gpu)
            c = cache(m, t, weigh=True)
            t.extend([20, 9])
            m(x, past_kv=c)
            if drafts:  # four tokens of the first sequence, three of the second: one stays
                t.extend([4, 3])
                m(torch.cat((accepted, drafted)), past_kv=c)
                keep = torch.tensor([21, 9], dtype=torch.int32, device=gpu)
                if captured:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        t.rollback(keep)
                    for _ in range(3):
                        graph.replay()
                else:
                    t.rollback(keep)
                assert t.seqlens.tolist() == [21, 9]
                assert (c.key_weights[0, :, 21:] == 0).all() and (c.key_weights[1, :, 9:] == 0).all()
                assert (c.key_weights[0, :, :21] > 0).all() and (c.key_weights[1, :, :9] > 0).all()
            else:
                t.extend([1, 0])
                m(accepted, past_kv=c)
            t.extend([2, 3])
            m(after, past_kv=c)
            caches.append(c)
    a, b = (c.key_weights for c in caches)
    # (the same queries over rows that round to neighbours; sums over a KV head's four heads)
    assert (a[0, :, 21:] - b[0, :, 21:]).abs().max() <= 4 * 2.0 ** -6
    assert (a[1, :, 9:] - b[1, :, 9:]).abs().max() <= 4 * 2.0 ** -6
    assert (a[0, :, 21:23] > 0).all() and (a[1, :, 9:12] > 0).all()


def far_angles(rope, pos):
    return pos * rope.inv_freq.double().cpu()


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to(torch.bfloat16).float(), lambda m: m.cpu()])
@pytest.mark.parametrize("scaling", ["linear", "yarn"])
def test_scaled_frequencies_stay_in_32_bits(cast, scaling):
    """Whatever the layer is cast to, before or after rotate_by, the angles of far positions are
    those of the formula, rounded to fp32 once: off by 2^-24 of the angle."""
    factor, length, rd = 8.0, 4096, 64
    i = torch.arange(rd // 2, dtype=torch.float64)
    inv = 10000.0 ** (-2 * i / rd)
    if scaling == "linear":
        want = inv / factor
    else:  # by the turns over the original length: more than 32 kept, fewer than 1 divided
        pair = lambda turns: rd * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
        low, high = math.floor(pair(32.0)), math.ceil(pair(1.0))
        ramp = ((i - low) / (high - low)).clamp(0, 1)
        want = inv * (1 - ramp) + inv / factor * ramp
    how = dict(rotary_dim=rd, scaling=scaling, factor=factor, original_max_len=length)
    make = lambda: NaylisAttention(256, 2, rel_rank=8)
    for m in (cast(make().rotate_by(**how)), cast(make()).rotate_by(**how)):
        assert m.rope.inv_freq.dtype == torch.float32
        for pos in (1000, 30000, 10 ** 6):
            assert ((far_angles(m.rope, pos) - pos * want).abs() <= 2.0 ** -24 * pos * want + 1e-12).all()
        assert m.q_proj.weight.dtype == cast(make()).q_proj.weight.dtype


def test_a_checkpoint_does_not_change_the_frequencies():
    """inv_freq is of the layer's arguments: a plain layer's, or one's of another width, that a
    checkpoint holds, is left; the other parameters load."""
    make = lambda **how: NaylisAttention(256, 2, rel_rank=8).rotate_by(**how) if how else \
        NaylisAttention(256, 2, rel_rank=8)
    how = dict(rotary_dim=64, interleaved=True, scaling="yarn", factor=8.0, original_max_len=4096)
    plain, other = make(), make(rotary_dim=32)
    assert "rope.inv_freq" in plain.state_dict() and "rope.inv_freq" not in other.state_dict()
    older = dict(other.state_dict())
    older["rope.inv_freq"] = other.rope.inv_freq.clone()
    for saved in (plain.state_dict(), other.state_dict(), older):
        for assign in (False, True):
            m = make(**how)
            want = m.rope.inv_freq.clone()
            assert m.load_state_dict(saved, assign=assign) == ([], [])
            assert torch.equal(m.rope.inv_freq, want) and m.rope.factor > 1
            assert torch.equal(m.q_proj.weight, saved["q_proj.weight"])
    with pytest.raises(RuntimeError, match="q_nothing"):
        m.load_state_dict({**plain.state_dict(), "q_nothing": torch.ones(1)})
    with pytest.raises(RuntimeError, match="rope.nothing"):
        m.load_state_dict({**plain.state_dict(), "rope.nothing": torch.ones(1)})
    with torch.device("meta"):
        m = make(**how)
    assert m.rope.inv_freq.is_meta
    m.to_empty(device="cpu")
    assert torch.equal(m.rope.inv_freq, want) and m.rope.inv_freq.dtype == torch.float32
    m.to_empty(device="cpu")
    assert torch.equal(m.rope.inv_freq, want)


def test_a_plain_layers_frequencies_go_with_it():
    m = NaylisAttention(256, 2, rel_rank=8)
    assert m.bfloat16().rope.inv_freq.dtype == torch.bfloat16
    assert m.load_state_dict(NaylisAttention(256, 2, rel_rank=8).state_dict()) == ([], [])


def test_rotate_by_does_not_take_a_yarn_stretch_away():
    """A layer built with use_yarn scales its scores by yarn_scale too, which another rotation
    would drop unseen."""
    m = NaylisAttention(256, 2, rel_rank=8, use_yarn=True, yarn_scale=4.0)
    scale, rope = m._attn_scale(), m.rope
    for how in (dict(rotary_dim=64), dict(scaling="yarn", factor=4.0), dict()):
        with pytest.raises(ValueError, match="use_yarn"):
            m.rotate_by(**how)
    assert m.rope is rope and m._attn_scale() == scale
