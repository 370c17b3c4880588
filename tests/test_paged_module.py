"""PageTable, PagedKVCache and NaylisAttention on them.

CPU: the page table's bookkeeping.  GPU: a layer that serves prompts in pieces
and single tokens from pages against its own forward over whole sequences, with
the page table's steps captured into a graph, and with eviction.

Tolerance of the layer comparison: both sides compute the same products of bf16
values and may round five things between to other neighbours (the rotated q
and k, P, the attention's output and the layer's), each by at most 2^-8 of the
value: 5 * 2^-8 of the output's norm.
"""
import pytest
import torch

from fna2_amd import _capi
from fna2_amd.paged import PagedKVCache, PageTable

from tests.helpers import rel_norm


def test_page_table_counts_rows_and_pages():
    t = PageTable(3, 10, page_size=16, max_pages=5)
    t.extend([20, 0, 16])
    assert t.rows == [20, 0, 16] and [len(p) for p in t.pages] == [2, 0, 1]
    assert t.cu_seqlens_q.tolist() == [0, 20, 20, 36] and t.max_seqlen_q == 20 and t.total_q == 36
    assert t.seqlens.tolist() == [20, 0, 16] and t.positions is None and t.free_pages == 7
    named = [p for row in t.block_table.tolist() for p in row if p >= 0]
    assert len(set(named)) == 3 and sorted(named) == sorted(sum(t.pages, []))
    t.extend([1, 1, 1])
    assert [len(p) for p in t.pages] == [2, 1, 2] and t.free_pages == 5
    before = (list(t.rows), [list(p) for p in t.pages], t.block_table.tolist())
    with pytest.raises(ValueError, match="table holds 5"):
        t.extend([80, 0, 0])
    with pytest.raises(ValueError, match="5 free"):
        t.extend([50, 40, 30])
    assert before == (list(t.rows), [list(p) for p in t.pages], t.block_table.tolist())
    with pytest.raises(AssertionError):
        t.extend([1, 1])
    with pytest.raises(AssertionError):
        t.extend([1, -1, 0])


def test_page_table_truncate_and_release():
    t = PageTable(2, 6, page_size=16)
    t.extend([50, 10])
    data = t.block_table.data_ptr()
    t.truncate(20)
    assert t.rows == [20, 10] and [len(p) for p in t.pages] == [2, 1] and t.free_pages == 3
    assert (t.block_table[0, 2:] == -1).all() and t.seqlens.tolist() == [20, 10]
    t.extend([2, 1])
    # rows and positions differ from now on
    assert t.positions.tolist() == [50, 51, 10] and t.seqlens.tolist() == [22, 11]
    t.release(0)
    assert t.rows == [0, 11] and t.free_pages == 5 and (t.block_table[0] == -1).all()
    t.extend([3, 1])
    assert t.positions is None or t.positions.tolist() == [0, 1, 2, 11]
    assert t.block_table.data_ptr() == data  # written in place
    with pytest.raises(AssertionError):
        PageTable(1, 4, page_size=24)


def test_cache_shapes_are_checked():
    t = PageTable(2, 6, page_size=16)
    c = PagedKVCache.empty(t, 2, 64, graph_heads=3, rank=8, weigh=True)
    assert c.k.shape == (6, 2, 16, 64) and c.r_k.shape == (6, 3, 16, 8)
    assert c.key_weights.shape == (2, 2, 96)
    with pytest.raises(AssertionError):
        PagedKVCache(t, c.k[:5], c.v[:5])
    with pytest.raises(AssertionError):
        PagedKVCache(t, c.k, c.v, c.r_k[:, :, :8])
    with pytest.raises(AssertionError):
        PagedKVCache.empty(t, 2, 64).evict(10)


def test_module_without_the_kernels_raises():
    from fna2_amd.attention_fna2 import NaylisAttention
    m = NaylisAttention(128, 2, rel_rank=8, use_fna2=False)
    t = PageTable(1, 4, page_size=16)
    t.extend([3])
    with pytest.raises(RuntimeError):
        m(torch.zeros(3, 128), past_kv=PagedKVCache.empty(t, 2, 64, 2, 8))


# ── GPU ──────────────────────────────────────────────────────────────────────

def _layer(gpu, dtype=torch.bfloat16, **kw):
    from fna2_amd.attention_fna2 import NaylisAttention
    torch.manual_seed(0)
    m = NaylisAttention(512, 8, n_kv_heads=2, max_seq_len=256, **{**dict(rel_rank=16), **kw})
    if m.graph_scale is not None:
        with torch.no_grad():
            m.graph_scale.normal_(1.0, 0.5)
            m.rel_q_proj.weight.normal_(std=0.05)
            m.rel_k_proj.weight.normal_(std=0.05)
    return m.to(gpu).to(dtype).eval()


def _cache(m, t, **kw):
    return PagedKVCache.empty(t, m.n_kv_heads, m.head_dim, m.graph_heads, m.rel_rank, **kw)


STEPS = [[37, 0, 5], [40, 70, 1], [1, 1, 1], [1, 0, 1], [0, 3, 33], [1, 1, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(vanilla_heads=3), dict(vanilla_heads=7),
                                dict(use_qk_norm=False), dict(use_rope=False)])
def test_pieces_and_tokens_equal_the_whole_sequences(gpu, kw):
    m = _layer(gpu, **kw)
    t = PageTable(3, 40, page_size=16, device=gpu)
    c = _cache(m, t)
    total = [sum(s[b] for s in STEPS) for b in range(3)]
    xs = [torch.randn(n, 512, device=gpu).bfloat16() for n in total]
    got, at = [[] for _ in total], [0, 0, 0]
    with torch.no_grad():
        for s in STEPS:
            t.extend(s)
            x = torch.cat([xs[b][at[b]:at[b] + s[b]] for b in range(3)])
            y, back = m(x, past_kv=c, use_kv_cache=True)
            assert back is c
            for b, part in enumerate(torch.split(y, s)):
                got[b].append(part)
                at[b] += s[b]
        cu = torch.tensor([0, total[0], total[0] + total[1], sum(total)], dtype=torch.int32, device=gpu)
        ref, _ = m(torch.cat(xs), cu_seqlens_q=cu, max_seqlen_q=max(total))
    out = torch.cat([torch.cat(g) for g in got])
    assert rel_norm(out, ref.double().cpu().numpy()) < 5 * 2.0 ** -8
    assert t.seqlens.tolist() == total


@pytest.mark.gpu
def test_tokens_as_a_batch_and_wrong_calls(gpu):
    m = _layer(gpu)
    t = PageTable(2, 20, page_size=16, device=gpu)
    c, d = _cache(m, t), _cache(m, t)
    x = torch.randn(2, 3, 512, device=gpu).bfloat16()
    t.extend([3, 3])
    with torch.no_grad():
        y, none = m(x, past_kv=c)
        z, _ = m(x.view(6, 512), past_kv=d)
    assert none is None and y.shape == (2, 3, 512) and torch.equal(y.view(6, 512), z)
    with pytest.raises(ValueError):
        m(x[:, :2], past_kv=c)
    with pytest.raises(ValueError):
        m(x, past_kv=PagedKVCache.empty(t, 2, 64))
    with pytest.raises(RuntimeError):
        m(x, mask=torch.ones(3, 3, dtype=torch.bool, device=gpu), past_kv=c)


@pytest.mark.gpu
def test_a_decode_step_as_a_graph(gpu):
    """One captured step, replayed while the page table moves on under it, with
    eager steps of a second cache between."""
    m = _layer(gpu)
    t = PageTable(2, 40, page_size=16, device=gpu)
    a, b = _cache(m, t, weigh=True), _cache(m, t, weigh=True)
    x0 = torch.randn(2, 12, 512, device=gpu).bfloat16()
    with torch.no_grad():
        t.extend([12, 12])
        for c in (a, b):
            m(x0, past_kv=c)
        t.extend([1, 1])
        x = torch.randn(2, 1, 512, device=gpu).bfloat16()
        for _ in range(2):  # (the same rows again: nothing changes but the weights)
            m(x, past_kv=a)
        m(x, past_kv=b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = m(x, past_kv=a)
        for i in range(20):  # over a page's end
            t.extend([1, 1])
            x.copy_(torch.randn(2, 1, 512, device=gpu).bfloat16())
            want, _ = m(x, past_kv=b)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), i
    assert torch.equal(a.k, b.k) and torch.equal(a.r_k, b.r_k)


@pytest.mark.gpu
def test_two_layers_with_eviction(gpu):
    """Decoding with a budget: every layer evicts by its own weights, the table
    is cut once, positions go on counting; what is evicted last is what the
    weights say, and the outputs stay those of the rows that were kept."""
    layers = [_layer(gpu), _layer(gpu, vanilla_heads=4)]
    t = PageTable(2, 12, page_size=16, device=gpu)
    cs = [_cache(m, t, weigh=True) for m in layers]
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        t.extend([60, 41])
        x = torch.randn(101, 512, generator=g).bfloat16().to(gpu)
        for m, c in zip(layers, cs):
            x = x + m(x, past_kv=c)[0]
        for m, c in zip(layers, cs):
            # every token's weights sum to one for each query head
            assert torch.allclose(c.key_weights.sum(-1).sum(-1),
                                  torch.tensor([60. * 8, 41. * 8], device=gpu), rtol=1e-4)
            kept = c.evict(48, recent=8, first=2, heads=8)
            assert kept.shape == (2, 2, 48) and (kept[1, :, 41:] == -1).all()
            assert (kept[0, :, :2] == torch.tensor([0, 1], device=gpu)).all()
            assert (kept[0, :, -8:] == torch.arange(52, 60, device=gpu)).all()
            assert (c.key_weights[0, :, 48:] == 0).all()
        t.truncate(48)
        assert t.rows == [48, 41] and t.free_pages == 12 - 3 - 3
        for _ in range(9):
            t.extend([1, 1])
            x = torch.randn(2, 512, generator=g).bfloat16().to(gpu)
            for m, c in zip(layers, cs):
                x = x + m(x, past_kv=c)[0]
                assert torch.isfinite(x).all()
        assert t.next_position == [69, 50] and t.rows == [57, 50]
        t.release(1)
        for c in cs:
            c.forget(1)
            assert (c.key_weights[1] == 0).all()


# ── Positions that run ahead of the rows ─────────────────────────────────────

def test_page_table_writes_a_step_in_place():
    """What a captured step reads keeps its place through every call, and the
    positions of tokens are rows plus the shift."""
    t = PageTable(3, 12, page_size=16, max_pages=6)
    names = ("block_table", "seqlens", "position_shift", "cu_seqlens_q")
    held = {n: getattr(t, n) for n in names}
    place = {n: x.data_ptr() for n, x in held.items()}
    t.extend([50, 10, 0])
    assert t.position_shift.tolist() == [0, 0, 0]
    t.truncate(20)
    assert t.position_shift.tolist() == [30, 0, 0] and t.cu_seqlens_q.tolist() == [0, 50, 60, 60]
    t.extend([2, 1, 3])
    assert t.position_shift.tolist() == [30, 0, 0] and t.seqlens.tolist() == [22, 11, 3]
    assert t.positions.tolist() == [50, 51, 10, 0, 1, 2]
    t.truncate(8)
    assert t.position_shift.tolist() == [44, 3, 0]
    t.extend([1, 1, 1])
    assert t.positions.tolist() == [52, 11, 3] and t.cu_seqlens_q.tolist() == [0, 1, 2, 3]
    t.release(0)
    assert t.position_shift.tolist() == [0, 3, 0] and t.seqlens.tolist() == [0, 9, 4]
    for n in names:
        assert getattr(t, n) is held[n] and held[n].data_ptr() == place[n]


@pytest.mark.gpu
@pytest.mark.parametrize("when", ["before", "after"])
@pytest.mark.parametrize("kw", [dict(), dict(use_rope=False)])
def test_a_graph_follows_the_table_through_eviction(gpu, kw, when):
    """A step captured before any eviction, or after one, replayed while more
    follow: positions go on counting past the rows, as in eager steps of a second
    cache."""
    m = _layer(gpu, **kw)
    t = PageTable(2, 40, page_size=16, device=gpu)
    a, b = _cache(m, t, weigh=True), _cache(m, t, weigh=True)
    g = torch.Generator().manual_seed(2)
    x0 = torch.randn(2, 40, 512, generator=g).bfloat16().to(gpu)

    def evict(budget):
        b.key_weights.copy_(a.key_weights)
        kept = [c.evict(budget, recent=4, first=1, heads=8) for c in (a, b)]
        assert torch.equal(*kept)
        t.truncate(budget)

    with torch.no_grad():
        t.extend([40, 40])
        for c in (a, b):
            m(x0, past_kv=c)
        if when == "after":
            evict(33)
        t.extend([1, 1])
        x = torch.randn(2, 1, 512, generator=g).bfloat16().to(gpu)
        for _ in range(2):  # (the same rows again: nothing changes but the weights)
            m(x, past_kv=a)
        m(x, past_kv=b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = m(x, past_kv=a)
        for i in range(24):
            if i % 6 == 3:
                evict(32 - i // 2)
            t.extend([1, 1])
            x.copy_(torch.randn(2, 1, 512, generator=g).bfloat16())
            want, _ = m(x, past_kv=b)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), i
            assert torch.equal(a.k, b.k), i


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_steps_after_an_eviction(gpu, graph):
    """The rows that were kept are the cache's, each new token's key is rotated
    for its position (not its row), and a step's output is the attention of its
    query, so rotated, over them.

    Keys: half a step and 1e-5 for the fp32 chain.  Outputs: the rotated q, P, the
    attention's output and the layer's, each by at most 2^-8 of the value."""
    from oracle import paged_oracle as PO
    m = _layer(gpu)
    t = PageTable(2, 12, page_size=16, device=gpu)
    c = _cache(m, t, weigh=True)
    g = torch.Generator().manual_seed(4)
    inv = m.rope.inv_freq.double().cpu().numpy()
    f64 = lambda y: y.detach().double().cpu().numpy()
    rows = lambda pool, b: torch.stack([pool[t.pages[b][j // 16], :, j % 16] for j in range(t.rows[b])])
    x = torch.zeros(2, 512, dtype=torch.bfloat16, device=gpu)
    with torch.no_grad():
        t.extend([60, 41])
        m(torch.randn(101, 512, generator=g).bfloat16().to(gpu), past_kv=c)
        t.extend([1, 1])
        x.copy_(torch.randn(2, 512, generator=g).bfloat16())
        m(x, past_kv=c)
        if graph:
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg):
                yg, _ = m(x, past_kv=c)
        before = [[rows(p, b) for p in (c.k, c.v, c.r_k)] for b in range(2)]
        kept = c.evict(48, recent=8, first=2, heads=8)
        t.truncate(48)
        for b in range(2):
            n = t.rows[b]
            for p, old in zip((c.k, c.v), before[b]):
                for h in range(2):
                    assert torch.equal(rows(p, b)[:, h], old[kept[b, h, :n].long(), h])
            for h in range(8):
                assert torch.equal(rows(c.r_k, b)[:, h], before[b][2][kept[b, h // 4, :n].long(), h])
        for step in range(4):
            t.extend([1, 1])
            x.copy_(torch.randn(2, 512, generator=g).bfloat16())
            if graph:
                cg.replay()
                y = yg
            else:
                y, _ = m(x, past_kv=c)
            q, k, _, r_q, _ = m._project(x)
            pos = [61 + step, 42 + step]
            assert t.positions.tolist() == pos
            qs = []
            for b in range(2):
                want = PO.norm_rope(f64(k[b]), f64(m.k_norm.weight), pos[b], inv, m.k_norm.eps)
                got = f64(rows(c.k, b)[-1])
                assert (abs(got - want) <= 2.0 ** -8 * abs(want) + 1e-5).all(), (step, b)
                qs.append(PO.norm_rope(f64(q[b]), f64(m.q_norm.weight), pos[b], inv, m.q_norm.eps))
            out = PO.attend(torch.stack([torch.from_numpy(z) for z in qs]), c.k, c.v, t.block_table,
                            t.seqlens, t.cu_seqlens_q, r_q, c.r_k, m.graph_scale)[0]
            ref = out.reshape(2, 512) @ f64(m.out_proj.weight).T
            assert rel_norm(y, ref) < 4 * 2.0 ** -8, step


def test_positions_of_packed_tokens():
    t = PageTable(3, 12, page_size=16, max_pages=6)
    t.extend([50, 10, 0])
    t.truncate(20)
    t.extend([2, 0, 3])
    assert t.token_positions(5).tolist() == t.positions.tolist() == [50, 51, 0, 1, 2]
    # tokens of no sequence before and behind
    cu = torch.tensor([2, 4, 4, 7])
    assert t.token_positions(9, cu)[2:7].tolist() == [50, 51, 0, 1, 2]
    assert t.token_positions(0).shape == (0,)
    assert PageTable(0, 4, page_size=16).token_positions(3).shape == (3,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotation_at_positions_is_the_tables(dtype):
    """Row by row the same bits, at positions that the type rounds as well."""
    from fna2_amd.attention_fna2 import RotaryPositionalEmbedding
    rope = RotaryPositionalEmbedding(64)
    _rows_are_the_tables(rope, torch.device("cpu"), dtype)


def _rows_are_the_tables(rope, device, dtype):
    table = rope._table(3001, device, dtype)
    pos = torch.tensor([0, 1, 255, 256, 257, 1000, 1001, 2049, 3000, 5], device=device)
    for ids in (pos, pos.int()):
        for a, b in zip(rope._at(ids, dtype), table):
            assert torch.equal(a, b[pos])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotation_at_positions_is_the_tables_on_the_gpu(gpu, dtype):
    from fna2_amd.attention_fna2 import RotaryPositionalEmbedding
    _rows_are_the_tables(RotaryPositionalEmbedding(64).to(gpu), gpu, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(use_qk_norm=False), dict()])
def test_a_graph_at_positions_past_its_capture(gpu, kw):
    """A step captured early and replayed far past it, with evictions, and with
    the layer's own table growing between."""
    m = _layer(gpu, **kw)
    t = PageTable(2, 40, page_size=16, device=gpu)
    a, b = _cache(m, t, weigh=True), _cache(m, t, weigh=True)
    g = torch.Generator().manual_seed(3)
    x0 = torch.randn(12, 512, generator=g).bfloat16().to(gpu)
    with torch.no_grad():
        t.extend([7, 5])
        for c in (a, b):
            m(x0, past_kv=c)
        t.extend([1, 1])
        x = torch.randn(2, 512, generator=g).bfloat16().to(gpu)
        for _ in range(2):
            m(x, past_kv=a)
        m(x, past_kv=b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = m(x, past_kv=a)
        for i in range(60):
            if i % 25 == 20:
                b.key_weights.copy_(a.key_weights)
                for c in (a, b):
                    c.evict(16, recent=4, first=1, heads=8)
                t.truncate(16)
            if i % 20 == 10:
                m.rope._table(100 + 10 * i, gpu, torch.bfloat16)
            t.extend([1, 1])
            x.copy_(torch.randn(2, 512, generator=g).bfloat16())
            want, _ = m(x, past_kv=b)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), i
            assert torch.equal(a.k, b.k), i


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(use_qk_norm=False), dict()])
def test_a_padded_step(gpu, kw):
    """cu_seqlens_q of the caller's, with tokens of no sequence around the
    others, after an eviction: what the step without them gives.

    The projections of differing numbers of rows may round to other neighbours
    (2^-7), and after them the rotation (2^-8, without a norm three times): in 5 of 55
    rows a cache, a third of 2^-7 + 6 * 2^-8 of its norm."""
    m = _layer(gpu, **kw)
    t = PageTable(2, 40, page_size=16, device=gpu)
    a, b = _cache(m, t, weigh=True), _cache(m, t, weigh=True)
    g = torch.Generator().manual_seed(3)
    x0 = torch.randn(80, 512, generator=g).bfloat16().to(gpu)
    with torch.no_grad():
        t.extend([50, 30])
        for c in (a, b):
            m(x0, past_kv=c)
            c.evict(25, heads=8)
        t.truncate(25)
        t.extend([1, 4])
        x = torch.randn(9, 512, generator=g).bfloat16().to(gpu)
        want, _ = m(x[2:7], past_kv=a)
        cu = torch.tensor([2, 3, 7], dtype=torch.int32, device=gpu)
        got, _ = m(x, past_kv=b, cu_seqlens_q=cu)
    assert rel_norm(got[2:7], want.double().cpu().numpy()) < 5 * 2.0 ** -8
    assert rel_norm(b.k, a.k.double().cpu().numpy()) < 8 / 3 * 2.0 ** -8


# ── Activations of another type than the cache's ─────────────────────────────

def _prompt_and_steps(m, gpu, x, splits, **kw):
    """x [T, E] served as one sequence in pieces: (outputs, the cache, its table)."""
    t = PageTable(1, x.shape[0] // 16 + 2, page_size=16, device=gpu)
    c = _cache(m, t, **kw)
    out, at = [], 0
    with torch.no_grad():
        for n in splits:
            t.extend([n])
            out.append(m(x[at:at + n], past_kv=c)[0])
            at += n
    return torch.cat(out), c, t


def _rows_of(c, n, pool):
    ids = c.table.block_table[0, : -(-n // c.table.page_size)].long()
    return pool[ids].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:n]


@pytest.mark.gpu
@pytest.mark.parametrize("cached", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [True, False])
def test_an_fp32_layer_on_pages(gpu, norm, cached):
    """fp32 activations are normalised and rotated in fp32 and rounded once, to
    the cache's type: the cached keys are within half a step of the definition, and
    (bf16) the layer gives what its own forward does, also far along.

    Keys: 1e-5 on top for the fp32 chain of values of order one.  Without a norm the
    angles are the fp32 products that the layer's table holds."""
    m = _layer(gpu, torch.float32, use_qk_norm=norm)
    g = torch.Generator().manual_seed(5)
    if norm:
        with torch.no_grad():
            m.k_norm.weight.copy_(1 + 0.2 * torch.randn(64, generator=g))
    n = 1100
    x = torch.randn(n, 512, generator=g).to(gpu)
    y, c, _ = _prompt_and_steps(m, gpu, x, [1000, 98, 1, 1], dtype=cached)
    assert y.dtype == torch.float32
    with torch.no_grad():
        k = torch.cat([m._project(p)[1] for p in torch.split(x, [1000, 98, 1, 1])]).double().cpu()
        ref, _ = m(x, cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=gpu), max_seqlen_q=n)
    if norm:
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + m.k_norm.eps) * m.k_norm.weight.double().cpu()
        ang = torch.outer(torch.arange(n).double(), m.rope.inv_freq.double().cpu())
    else:
        ang = torch.outer(torch.arange(n).float(), m.rope.inv_freq.float().cpu()).double()
    a, b = k.chunk(2, -1)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    want = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    got = _rows_of(c, n, c.k).double().cpu()
    half = torch.finfo(cached).eps / 2
    assert ((got - want).abs() <= half * want.abs() + 1e-5).all()
    if cached == torch.bfloat16:
        # (the rotated q and k, P and the attention's output, each half a step)
        assert rel_norm(y, ref.double().cpu().numpy()) < 4 * 2.0 ** -8


# ── Hooked and replaced modules ──────────────────────────────────────────────

def _twice(mod, args, out):
    return tuple(2 * o for o in out) if isinstance(out, tuple) else 2 * out


def _same(mod, args, out):
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("rope", [True, False])
def test_hooked_and_replaced_norms_are_called(gpu, rope):
    """A hook on k_norm, or a class of its own in its place, takes part as in
    the layer's other steps: twice its output is what weights of twice the size give."""
    from fna2_amd.attention_fna2 import RMSNorm

    class Twice(RMSNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    x = torch.randn(70, 512, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    run = lambda m: _prompt_and_steps(m, gpu, x, [60, 9, 1])[0]
    hooked, replaced, doubled, plain = (_layer(gpu, use_rope=rope) for _ in range(4))
    hooked.k_norm.register_forward_hook(_twice)
    own = Twice(64).to(gpu).bfloat16()
    own.load_state_dict(replaced.k_norm.state_dict())
    replaced.k_norm = own
    doubled.k_norm.register_forward_hook(_same)
    with torch.no_grad():
        doubled.k_norm.weight.mul_(2)
    want = run(doubled)
    assert torch.equal(run(hooked), want) and torch.equal(run(replaced), want)
    assert not torch.equal(run(plain), want)


@pytest.mark.gpu
def test_hooked_and_replaced_rotations_are_called(gpu):
    from fna2_amd.attention_fna2 import RotaryPositionalEmbedding

    class Twice(RotaryPositionalEmbedding):
        def forward(self, q, k, position_offset=0):
            q, k = super().forward(q, k, position_offset)
            return 2 * q, 2 * k

    x = torch.randn(70, 512, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    run = lambda m: _prompt_and_steps(m, gpu, x, [60, 9, 1])[0]
    hooked, replaced, doubled, plain = (_layer(gpu, use_qk_norm=False) for _ in range(4))
    hooked.rope.register_forward_hook(_twice)
    replaced.rope = Twice(64, 256).to(gpu).bfloat16()
    replaced.rope.inv_freq = hooked.rope.inv_freq.clone()
    with torch.no_grad():
        doubled.q_proj.weight.mul_(2)
        doubled.k_proj.weight.mul_(2)
    want = run(doubled)
    assert torch.equal(run(hooked), want) and torch.equal(run(replaced), want)
    assert not torch.equal(run(plain), want)


@pytest.mark.gpu
def test_a_hooked_rotation_after_an_eviction(gpu):
    """Its positions are the tokens', not their rows; a step of it is not captured."""
    hooked, plain = _layer(gpu, use_qk_norm=False), _layer(gpu, use_qk_norm=False)
    seen = []
    hooked.rope.register_forward_hook(
        lambda mod, args, kw, out: seen.append(kw["position_offset"]), with_kwargs=True)
    g = torch.Generator().manual_seed(6)
    t = PageTable(2, 12, page_size=16, device=gpu)
    caches = [_cache(m, t, weigh=True) for m in (hooked, plain)]
    x0 = torch.randn(70, 512, generator=g).bfloat16().to(gpu)
    x = torch.randn(7, 512, generator=g).bfloat16().to(gpu)
    cu = torch.tensor([1, 3, 6], dtype=torch.int32, device=gpu)
    with torch.no_grad():
        t.extend([40, 30])
        got = [m(x0, past_kv=c)[0] for m, c in zip((hooked, plain), caches)]
        assert torch.equal(*got) and seen == [0, 0]
        caches[1].key_weights.copy_(caches[0].key_weights)
        for c in caches:
            c.evict(20, heads=8)
        t.truncate(20)
        t.extend([2, 3])
        got = [m(x, past_kv=c, cu_seqlens_q=cu)[0] for m, c in zip((hooked, plain), caches)]
        assert torch.equal(*got) and seen[2:] == [40, 30]
        assert torch.equal(caches[0].k, caches[1].k)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(graph):
                hooked(x, past_kv=caches[0], cu_seqlens_q=cu)
    torch.cuda.synchronize()
