"""The books of a paged cache on the GPU (fna2_paged_extend, _trim, _groups)
against the same in Python: whole numbers, equal.
"""
import ctypes
import subprocess

import pytest
import torch

from fna2_amd import _capi, paged
from fna2_amd.paged import PageTable, paged_extend, paged_groups, paged_trim
from tests.test_paged import FAKE, ROOT, _st

gpu = pytest.mark.gpu
i32 = torch.int32


def extend_ref(table, lens, counts, free, nfree, ps, T, shift):
    table, N, W = [list(r) for r in table], len(lens), len(table[0]) if table else 0
    counts, rows = [max(c, 0) for c in counts], [max(n, 0) for n in lens]
    need = [-(-(n + c) // ps) for n, c in zip(rows, counts)]
    more = [a - -(-n // ps) for a, n in zip(need, rows)]
    status = 0
    if any(n > W and c > 0 for n, c in zip(need, counts)):
        status = -1
    elif sum(counts) > T:
        status = -2
    elif sum(more) > nfree:
        status = sum(more) - nfree
    if status:
        return table, [0] * (N + 1), list(lens), nfree, [-1] * T, [-1] * T, [0] * T, status
    at = nfree
    cu, slots, seq, pos = [0], [], [], []
    for b in range(N):
        for j in range(need[b] - more[b], need[b]):
            at -= 1
            table[b][j] = free[at]
        for i in range(counts[b]):
            row = rows[b] + i
            page = table[b][row // ps]
            slots.append(-1 if page < 0 else page * ps + row % ps)
            seq.append(b)
            pos.append(row + (shift[b] if shift else 0))
        cu.append(cu[-1] + counts[b])
    left = T - len(seq)
    return (table, cu, [n + c for n, c in zip(rows, counts)], at, slots + [-1] * left,
            seq + [-1] * left, pos + [0] * left, 0)


def trim_ref(table, lens, keep, free, nfree, ps, borrowed):
    table, free, out = [list(r) for r in table], list(free), []
    for b, n in enumerate(lens):
        rows = max(n, 0)
        k = min(rows, max(keep[b], 0))
        for j in range(min(-(-rows // ps), len(table[b])) - 1, -(-k // ps) - 1, -1):
            if j >= (borrowed[b] if borrowed else 0) and nfree < len(free):
                free[nfree] = table[b][j]
                nfree += 1
            table[b][j] = -1
        out.append(k if k < rows else n)
    return table, free, out, nfree


def groups_ref(table, ps):
    N = len(table)
    common = [0] * N
    for b in range(1, N):
        for x, y in zip(table[b], table[b - 1]):
            if x != y or x < 0:
                break
            common[b] += 1
    cu, rows = [], []
    for b in range(N):
        if common[b] == 0:
            cu.append(b)
            rows.append(0)
        else:
            rows[-1] = min(rows[-1] or 1 << 30, common[b] * ps)
    return cu + [N] * (N + 1 - len(cu)), rows + [0] * (N - len(rows))


class Books:
    def __init__(self, lens, width, ps, spare, seed=0, cap=None):
        g = torch.Generator().manual_seed(seed)
        have = [min(-(-max(n, 0) // ps), width) for n in lens]
        P = sum(have) + spare
        perm = torch.randperm(P, generator=g).tolist()
        self.table, at = [[-1] * width for _ in lens], 0
        for b, h in enumerate(have):
            self.table[b][:h] = perm[at:at + h]
            at += h
        self.free = perm[at:] + [-7] * ((P if cap is None else cap) - spare)
        self.nfree, self.lens, self.ps = spare, lens, ps

    def tensors(self):
        t = lambda x: torch.tensor(x, dtype=i32, device="cuda")
        table = torch.full((len(self.lens), len(self.table[0]) + 3 if self.table else 3), -9, dtype=i32,
                           device="cuda")[:, :-3]  # rows of a wider tensor
        if self.table:
            table.copy_(t(self.table))
        return table, t(self.lens), t(self.free), t([self.nfree])


def check_extend(b, counts, T=None, shift=None):
    T = sum(max(c, 0) for c in counts) if T is None else T
    table, lens, free, nfree = b.tensors()
    t = lambda x: None if x is None else torch.tensor(x, dtype=i32, device="cuda")
    before = free.clone(), lens.clone()
    want = extend_ref(b.table, b.lens, counts, b.free, b.nfree, b.ps, T, shift)
    for _ in range(2):  # (a repeated call gives the same again)
        x = paged_extend(table, lens, t(counts), free, nfree, b.ps, T, t(shift))
        torch.cuda.synchronize()
        got = (table.tolist(), x.cu_seqlens_q.tolist(), x.seqlens.tolist(), x.free_count.item(),
               x.slots.tolist(), x.sequences.tolist(), x.positions.tolist(), x.status.item())
        assert got == want
    assert torch.equal(free, before[0]) and torch.equal(lens, before[1])
    assert x.slots.dtype == torch.int64
    return x


EXTENDS = {
    "one_token_each": ([5, 16, 31, 0], 4, 16, [1, 1, 1, 1], 9),
    "prompts": ([0, 0, 0], 40, 16, [100, 1, 333], 60),
    "some_without": ([7, 0, 64, 3], 8, 16, [0, 0, 5, 0], 3),
    "exactly_the_pages_there_are": ([16, 16], 4, 16, [16, 17], 3),
    "a_page_missing": ([16, 16], 4, 16, [16, 17], 2),
    "none_there": ([0, 0, 0], 4, 16, [1, 1, 40], 0),
    "past_the_table": ([60, 3], 4, 16, [5, 1], 9),
    "to_the_tables_end": ([60, 3], 4, 16, [4, 1], 9),
    "already_past_it": ([100, 3], 4, 16, [0, 1], 9),
    "below_nothing": ([-5, 3], 4, 16, [3, -4], 9),
    "one": ([0], 1, 48, [48], 1),
    "no_width": ([0, 0], 0, 16, [0, 0], 2),
}


@gpu
@pytest.mark.parametrize("name", EXTENDS)
def test_extend(name):
    lens, width, ps, counts, spare = EXTENDS[name]
    check_extend(Books(lens, width, ps, spare), counts)


@gpu
def test_extend_more_room_and_too_little():
    b = Books([5, 20, 40], 6, 16, 9)
    check_extend(b, [3, 0, 9], T=40, shift=[100, -3, 0])
    check_extend(b, [3, 0, 9], T=11)
    check_extend(b, [3, 0, 9], T=0)
    check_extend(b, [0, 0, 0], T=0)
    check_extend(b, [0, 0, 0], T=5)


@gpu
@pytest.mark.parametrize("N,most,ps", [(4095, 3, 16), (4096, 2, 32), (4097, 3, 16), (9000, 2, 48),
                                       (64, 2000, 16), (1, 5000, 64), (3, 1500, 256)])
def test_extend_sizes(N, most, ps):
    """More sequences than one scan holds, more tokens than one workgroup's."""
    g = torch.Generator().manual_seed(N)
    counts = torch.randint(0, most + 1, (N,), generator=g).tolist()
    lens = torch.randint(0, 3 * ps, (N,), generator=g).tolist()
    width = 4 + most // ps
    spare = sum(-(-(n + c) // ps) - -(-n // ps) for n, c in zip(lens, counts)) + 2
    check_extend(Books(lens, width, ps, spare), counts, shift=list(range(N)))


@gpu
def test_extend_stack_counts_that_are_wrong():
    """A count past the stack, or below 0, is cut to it."""
    b = Books([5], 6, 16, 2)
    table, lens, free, _ = b.tensors()
    c = torch.tensor([60], dtype=i32, device="cuda")
    x = paged_extend(table, lens, c, free, torch.tensor([10 ** 6], dtype=i32, device="cuda"), 16, 60)
    assert x.status.item() == 4 - len(b.free)  # 5 pages for 65 rows, one is there
    x = paged_extend(table, lens, c, free, torch.tensor([-3], dtype=i32, device="cuda"), 16, 60)
    assert x.status.item() == 4 and x.free_count.item() == 0
    assert table.tolist() == b.table


@gpu
@pytest.mark.parametrize("borrowed", [None, [0, 2, 1, 9]])
@pytest.mark.parametrize("keep", [[0, 0, 0, 0], [100, 17, 5, -1], [64, 64, 64, 64], [1, 33, 0, 48]])
def test_trim(keep, borrowed):
    b = Books([64, 70, 5, 47], 6, 16, 3)
    check_trim(b, keep, borrowed)


def check_trim(b, keep, borrowed=None):
    table, lens, free, nfree = b.tensors()
    t = lambda x: None if x is None else torch.tensor(x, dtype=i32, device="cuda")
    want = trim_ref(b.table, b.lens, keep, b.free, b.nfree, b.ps, borrowed)
    new_lens, count = paged_trim(table, lens, t(keep), free, nfree, b.ps, t(borrowed))
    torch.cuda.synchronize()
    assert (table.tolist(), free.tolist(), new_lens.tolist(), count.item()) == want


@gpu
def test_trim_edges():
    check_trim(Books([100, -4, 0], 4, 16, 1), [0, 0, 3])          # more rows than the table has
    check_trim(Books([64, 64], 4, 16, 3, cap=6), [0, 0])          # a stack without the room
    check_trim(Books([], 0, 16, 3), [])
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 200, (5000,), generator=g).tolist()
    keep = torch.randint(-5, 200, (5000,), generator=g).tolist()
    check_trim(Books(lens, 13, 16, 7), keep)


@gpu
def test_groups():
    P = lambda rows: check_groups(rows, 48)
    P([[1, 2, 3], [1, 2, 4], [1, 2, 5], [6, 2, 3]])
    P([[1, 2, 3], [1, 2, 3]])
    P([[1, 2, 3], [1, 2, 9], [1, 8, 9]])          # the least of the pairs
    P([[1, 2, -1], [1, 2, -1], [-1, -1, -1], [-1, -1, -1]])
    P([[5]])
    P([[1, 2], [3, 4], [1, 2]])                   # not neighbours
    g = torch.Generator().manual_seed(1)
    wide = torch.randint(0, 1000, (1, 300), generator=g).repeat(40, 1)
    for b in range(1, 40):
        wide[b, int(torch.randint(0, 301, (1,), generator=g)):] += 1000 * b
    P(wide.tolist())
    many = torch.randint(0, 2, (9001, 3), generator=g)
    P(many.tolist())


def check_groups(rows, ps):
    cu, shared = paged_groups(torch.tensor(rows, dtype=i32, device="cuda"), ps)
    assert (cu.tolist(), shared.tolist()) == groups_ref(rows, ps)


@gpu
def test_groups_of_nothing():
    cu, rows = paged_groups(torch.zeros(0, 4, dtype=i32, device="cuda"), 16)
    assert cu.tolist() == [0] and rows.tolist() == []
    cu, rows = paged_groups(torch.zeros(3, 0, dtype=i32, device="cuda"), 16)
    assert cu.tolist() == [0, 1, 2, 3] and rows.tolist() == [0, 0, 0]


@gpu
def test_python_launchers_give_the_same(monkeypatch):
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    check_extend(Books([5, 20, 40], 6, 16, 9), [3, 0, 9], T=40, shift=[100, -3, 0])
    check_trim(Books([64, 70, 5, 47], 6, 16, 3), [100, 17, 5, -1], [0, 2, 1, 9])
    check_groups([[1, 2, 3], [1, 2, 4], [1, 2, 5], [6, 2, 3]], 48)


@gpu
def test_captured_steps_go_on():
    """A loop of one captured step, fed its own results."""
    N, ps = 5, 16
    b = Books([10, 15, 16, 0, 31], 8, ps, 20)
    table, lens, free, nfree = b.tensors()
    counts = torch.ones(N, dtype=i32, device="cuda")
    paged_extend(table.clone(), lens, counts, free, nfree, ps, N)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = paged_extend(table, lens, counts, free, nfree, ps, N)
        lens.copy_(x.seqlens)
        nfree.copy_(x.free_count)
    state = (b.table, b.lens, b.nfree)
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        want = extend_ref(state[0], state[1], [1] * N, b.free, state[2], ps, N, None)
        assert (table.tolist(), lens.tolist(), nfree.item(), x.slots.tolist()) == \
            (want[0], want[2], want[3], want[4])
        state = (want[0], want[2], want[3])


# ── CPU ──────────────────────────────────────────────────────────────────────

def _books(**over):
    b = _capi.PagedBooks()
    b.batch, b.table_width, b.page_size, b.capacity = 4, 8, 16, 30
    b.block_table, b.table_stride = FAKE, 8
    b.seqlens = b.free_pages = b.free_count = FAKE
    for k, v in over.items():
        setattr(b, k, v)
    return b


def _filled(cls, **over):
    a = cls()
    a.b = _books(**{k: v for k, v in over.items() if hasattr(_capi.PagedBooks, k)})
    for n, t in cls._fields_:
        if n != "b":
            setattr(a, n, 7 if t is ctypes.c_int32 else 2 * FAKE)
    for k, v in over.items():
        if not hasattr(_capi.PagedBooks, k):
            setattr(a, k, v)
    return a


COMMON = [
    (dict(), "FNA2_OK"),
    (dict(batch=-1), "FNA2_E_SHAPE"),
    (dict(page_size=24), "FNA2_E_SHAPE"),
    (dict(page_size=0), "FNA2_E_SHAPE"),
    (dict(table_width=1 << 27), "FNA2_E_SHAPE"),
    (dict(table_stride=7), "FNA2_E_STRIDE"),
    (dict(block_table=None), "FNA2_E_NULL"),
    (dict(batch=1, table_stride=0), "FNA2_OK"),
]


@pytest.mark.parametrize("over,code", COMMON + [
    (dict(seqlens=None), "FNA2_E_SEQLENS"),
    (dict(free_count=None), "FNA2_E_NULL"),
    (dict(free_pages=None), "FNA2_E_NULL"),
    (dict(capacity=0, free_pages=None), "FNA2_OK"),
    (dict(capacity=-1), "FNA2_E_SHAPE"),
    (dict(total_q=-1), "FNA2_E_SHAPE"),
    (dict(counts=None), "FNA2_E_NULL"),
    (dict(slots=None), "FNA2_E_NULL"),
    (dict(slots=None, sequences=None, positions=None, total_q=0), "FNA2_OK"),
    (dict(position_shift=None), "FNA2_OK"),
    (dict(new_lens=FAKE), "FNA2_E_ALIAS"),
    (dict(new_free_count=FAKE), "FNA2_E_ALIAS"),
    (dict(status=None), "FNA2_E_NULL"),
])
def test_check_extend(over, code):
    a = _filled(_capi.PagedExtendArgs, **over)
    assert _st(_capi.lib().fna2_check_paged_extend(ctypes.byref(a))) == code


@pytest.mark.parametrize("over,code", COMMON + [
    (dict(keep=None), "FNA2_E_NULL"), (dict(borrowed=None), "FNA2_OK"),
    (dict(new_free_count=None), "FNA2_E_NULL"), (dict(new_lens=FAKE), "FNA2_OK"),
    (dict(new_free_count=FAKE), "FNA2_OK"),
])
def test_check_trim(over, code):
    a = _filled(_capi.PagedTrimArgs, **over)
    assert _st(_capi.lib().fna2_check_paged_trim(ctypes.byref(a))) == code


@pytest.mark.parametrize("over,code", COMMON + [
    (dict(seqlens=None, free_pages=None, free_count=None), "FNA2_OK"),
    (dict(cu_groups=None), "FNA2_E_NULL"), (dict(workspace=None), "FNA2_E_NULL"),
])
def test_check_groups(over, code):
    a = _filled(_capi.PagedGroupsArgs, **over)
    assert _st(_capi.lib().fna2_check_paged_groups(ctypes.byref(a))) == code


def test_struct_layout_matches_header(tmp_path):
    pairs = (("fna2_paged_books", _capi.PagedBooks), ("fna2_paged_extend_args", _capi.PagedExtendArgs),
             ("fna2_paged_trim_args", _capi.PagedTrimArgs),
             ("fna2_paged_groups_args", _capi.PagedGroupsArgs))
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "fna2.h"', "int main(void){"]
    want = []
    for st, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({st}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({st}, {f}));')
            want.append(getattr(cls, f).offset)
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == want


def test_needs_the_gpu():
    t = torch.zeros(2, 3, dtype=i32)
    v = torch.zeros(2, dtype=i32)
    for call in (lambda: paged_extend(t, v, v, v, v[:1], 16, 4),
                 lambda: paged_trim(t, v, v, v, v[:1], 16), lambda: paged_groups(t, 16)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.parametrize("change", [
    dict(block_table=torch.zeros(2, 3)), dict(block_table=torch.zeros(6, dtype=i32)),
    dict(block_table=torch.zeros(3, 2, dtype=i32).t()), dict(seqlens=torch.zeros(3, dtype=i32)),
    dict(counts=torch.zeros(1, dtype=i32)), dict(free_pages=torch.zeros(4)), dict(counts=None),
    dict(free_count=torch.zeros(2, dtype=i32)), dict(total_q=-1),
    dict(position_shift=torch.zeros(3, dtype=i32)),
])
def test_refusals(change, monkeypatch):
    monkeypatch.setattr(paged, "_gpu", lambda *a: None)  # (shapes are looked at on the CPU)
    a = dict(block_table=torch.zeros(2, 3, dtype=i32), seqlens=torch.zeros(2, dtype=i32),
             counts=torch.zeros(2, dtype=i32), free_pages=torch.zeros(4, dtype=i32),
             free_count=torch.zeros(1, dtype=i32), page_size=16, total_q=4)
    a.update(change)
    with pytest.raises(AssertionError):
        paged_extend(**a)
