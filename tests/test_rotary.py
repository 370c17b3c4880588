"""Rotary positions in both layouts, over part of the head, scaled, at given
positions (fna2_rotary, ``rotary_embed``) against the formula in 64 bits.

Tolerances, h = eps / 2 of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24):
* forward: h |y| for the store, and for the fp32 chain 4e-6 (|u| + |v|) s of the
  pair (u, v): the angle, at most pi, is rounded to 2^-24 pi = 1.9e-7, cos and sin by
  2 units, 2.4e-7; a norm's sum of squares is off by 22 roundings at most (16 values of a
  lane, 6 steps over lanes), 7e-7 after the square root; some six products
  and sums, 3.6e-7: 1.7e-6 in all, twice that allowed.
* dx: h |dx| and 8e-6 of r (|w g| + |x| r^2 mean |x w g|), the two sums and twice
  the products; without a norm as forward.
* dw: fp32 sums of T * heads terms in chains of at most some 200 (tokens and heads of
  a wave, waves, workgroups): 2e-5 sum |g x r|, and the rounding to the weights' type.
* A store in fp16 below its smallest normal value, 2^-14, where the step stays 2^-24, is off
  by half of that, 2^-25 = 3e-8, however small the value.
"""
import ctypes
import subprocess

import numpy as np
import pytest
import torch

from fna2_amd import _capi, rope
from fna2_amd.rope import rotary_embed, rotary_frequencies

from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
FAKE = 1 << 20
EPS = 1e-6
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
gpu = pytest.mark.gpu


# ── the formula in 64 bits ───────────────────────────────────────────────────

def spread(x, rd, inter):
    """(u, v) of every rotated pair."""
    return (x[..., 0:rd:2], x[..., 1:rd:2]) if inter else (x[..., :rd // 2], x[..., rd // 2:rd])


def join(u, v, x, rd, inter):
    y = x.clone()
    if inter:
        y[..., 0:rd:2], y[..., 1:rd:2] = u, v
    else:
        y[..., :rd // 2], y[..., rd // 2:rd] = u, v
    return y


def turned(x, pos, inv, inter, scale, sign=1):
    rd = 2 * len(inv)
    a = pos.double()[:, None, None] * inv.double()
    c, s = torch.cos(a) * scale, torch.sin(a) * scale * sign
    u, v = spread(x, rd, inter)
    return join(u * c - v * s, v * c + u * s, x, rd, inter)


def normed(x, w):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def pair_mag(x, inv, inter, scale):
    """|u| + |v| of a feature's pair, times the scale."""
    rd = 2 * len(inv)
    u, v = spread(x.abs(), rd, inter)
    return join(*[(u + v) * abs(scale)] * 2, x.abs(), rd, inter)


def grads(x, w, dy, pos, inv, inter, scale):
    """(dx, dw, magnitudes of both)."""
    g = turned(dy, pos, inv, inter, scale, -1)
    gm = pair_mag(dy, inv, inter, scale)
    if w is None:
        return g, None, gm, None
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    dx = r * (w * g - x * r * r * (x * w * g).mean(-1, keepdim=True))
    mag = r * ((w * gm).abs() + x.abs() * r * r * (x * w * gm).abs().mean(-1, keepdim=True))
    return dx, (g * x * r).sum((0, 1)), mag, (gm * x * r).abs().sum((0, 1))


def positions_of(cu, T):
    pos, inside = torch.zeros(T, dtype=torch.long), torch.zeros(T, dtype=torch.bool)
    for a, b in zip(cu, cu[1:]):
        pos[a:b], inside[a:b] = torch.arange(b - a), True
    return pos, inside


class Case:
    def __init__(self, T, H, HKV, D, rd, inter, dtype, norm=(True, True), scale=1.0, cu=None,
                 far=1000, seed=0, device="cuda", wide=0, wdtype=None):
        g = torch.Generator().manual_seed(seed)
        randn = lambda *n: torch.randn(*n, generator=g)
        self.T, self.H, self.HKV, self.D, self.rd, self.inter = T, H, HKV, D, rd, inter
        self.scale, self.dtype = scale, dtype
        y = randn(T, (H + HKV) * D + wide).to(dtype).to(device)
        self.q = y[:, :H * D].view(T, H, D)
        self.k = y[:, H * D:(H + HKV) * D].view(T, HKV, D)
        w = lambda on: (1 + 0.2 * randn(D)).to(wdtype or dtype).to(device) if on else None
        self.wq, self.wk = w(norm[0]), w(norm[1])
        self.inv = (10000.0 ** (-torch.arange(0, rd, 2) / rd)).float().to(device)
        self.dyq, self.dyk = randn(T, H, D).to(dtype).to(device), randn(T, HKV, D).to(dtype).to(device)
        if cu is None:
            self.pos, self.cu = torch.randint(0, far, (T,), generator=g, dtype=torch.int32), None
            self.at, self.inside = self.pos.long(), torch.ones(T, dtype=torch.bool)
            self.pos = self.pos.to(device)
        else:
            self.pos, self.cu = None, torch.tensor(cu, dtype=torch.int32, device=device)
            self.at, self.inside = positions_of(cu, T)

    def args(self):
        return dict(positions=self.pos, cu_seqlens=self.cu, interleaved=self.inter,
                    scale=self.scale, norm_q=self.wq, norm_k=self.wk, eps=EPS)

    def run(self):
        return rotary_embed(self.q, self.k, self.inv, **self.args())


def d64(t):
    return None if t is None else t.detach().double().cpu()


def within(name, got, ref, lim):
    bad = ~((d64(got) - ref).abs() <= lim)
    worst = ((d64(got) - ref).abs() / lim).max() if bad.any() else 0
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst {worst:.2f} of the bound"


def check_forward(c):
    ins = c.inside[:, None, None]
    for name, got, x, w in zip("qk", c.run(), (c.q, c.k), (c.wq, c.wk)):
        n = normed(d64(x), d64(w))
        ref = torch.where(ins, turned(n, c.at, d64(c.inv), c.inter, c.scale), d64(x))
        mag = pair_mag(n, c.inv, c.inter, c.scale)
        assert got.dtype == c.dtype and got.is_contiguous()
        within(name, got, ref, torch.where(ins, HALF[c.dtype] * ref.abs() + 4e-6 * mag, 0.0)
               + STEP[c.dtype] + 1e-9)


def check_backward(c):
    leaves = [t for t in (c.q, c.k, c.wq, c.wk) if t is not None]
    for t in leaves:
        t.requires_grad_()
    out = c.run()
    got = iter(torch.autograd.grad(out, leaves, (c.dyq, c.dyk)))
    dq, dk = next(got), next(got)
    dwq, dwk = (next(got) if w is not None else None for w in (c.wq, c.wk))
    ins = c.inside[:, None, None]
    for name, gx, gw, x, w, dy in (("q", dq, dwq, c.q, c.wq, c.dyq), ("k", dk, dwk, c.k, c.wk, c.dyk)):
        inside = lambda t: torch.where(ins, t, 0.0)
        dx, dw, mag, wmag = grads(d64(x), d64(w), inside(d64(dy)), c.at, d64(c.inv), c.inter, c.scale)
        ref = torch.where(ins, dx, d64(dy))
        within("d" + name, gx, ref, HALF[c.dtype] * ref.abs() + 8e-6 * inside(mag)
               + STEP[c.dtype] + 1e-9)
        if w is not None:
            assert gw.dtype == w.dtype
            within("dw" + name, gw, dw, HALF[w.dtype] * dw.abs() + 2e-5 * wmag + STEP[w.dtype] + 1e-9)
    for t in leaves:
        t.requires_grad_(False)


SHAPES = [
    # T, H, HKV, D, rd
    (1, 1, 1, 16, 2), (5, 3, 1, 16, 16), (7, 2, 2, 32, 24), (33, 8, 2, 64, 64), (19, 4, 2, 64, 16),
    (66, 6, 3, 128, 128), (21, 5, 1, 128, 96), (9, 2, 1, 256, 64), (3, 2, 2, 512, 512),
    (40, 32, 8, 128, 32), (13, 9, 9, 64, 22), (11, 3, 2, 128, 2), (17, 2, 1, 128, 126),
    (6, 40, 40, 64, 48),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, inter, dtype):
    print(shape, inter, dtype, flush=True)
    for norm in ((False, False), (True, True), (True, False), (False, True)):
        check_forward(Case(*shape, inter, dtype, norm, scale=1.25, wide=8))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, inter, dtype):
    print(shape, inter, dtype, flush=True)
    for norm in ((False, False), (True, True), (True, False), (False, True)):
        check_backward(Case(*shape, inter, dtype, norm, scale=0.75, wide=8))


@gpu
@pytest.mark.parametrize("inter,rd", [(False, 64), (True, 40), (False, 24)])
@pytest.mark.parametrize("T,cu", [
    (50, [0, 17, 17, 50]), (50, [3, 20, 41]), (50, [0]), (50, [9, 9]), (1, [0, 1]),
    (1100, [0, 1, 2, 700, 1099]), (4200, [7, 4000, 4150]), (12500, [0, 12500]),
])
def test_packed_sequences(T, cu, inter, rd):
    print(T, cu, inter, rd, flush=True)
    c = Case(T, 2, 1, 64, rd, inter, torch.bfloat16, cu=cu, wide=8)
    check_forward(c)
    check_backward(c)


@gpu
@pytest.mark.parametrize("T", [1024, 1025, 4097, 12289])
def test_token_counts(T):
    """Where the kernels take more tokens a wave."""
    c = Case(T, 4, 1, 64, 32, True, torch.float32, far=5000)
    check_forward(c)
    check_backward(c)


@gpu
@pytest.mark.parametrize("cu", [None, [3, 100, 100, 505]])
@pytest.mark.parametrize("heads", [(8, 8), (19, 1), (1, 13)])
@pytest.mark.parametrize("T", [511, 512, 513])
def test_token_counts_of_shared_tokens(T, heads, cu):
    """Where the waves of a workgroup share a token's rows in the backward, and no longer do."""
    check_backward(Case(T, *heads, 256, 64, True, torch.bfloat16, far=5000, cu=cu))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_far_and_negative_positions(dtype):
    c = Case(64, 2, 1, 64, 64, False, dtype, norm=(False, False), far=2 ** 31 - 1)
    c.pos[::3] *= -1
    c.at = c.pos.long().cpu()
    check_forward(c)


@gpu
def test_differences():
    """The gradients against central differences of the formula."""
    c = Case(9, 3, 2, 32, 20, True, torch.float32, scale=1.3)
    leaves = [c.q, c.k, c.wq, c.wk]
    c.q, c.k = c.q.contiguous(), c.k.contiguous()
    leaves = [t.requires_grad_() for t in (c.q, c.k, c.wq, c.wk)]
    got = torch.autograd.grad(c.run(), leaves, (c.dyq, c.dyk))

    def loss(q, k, wq, wk):
        y = [turned(normed(x, w), c.at, d64(c.inv), c.inter, c.scale) for x, w in ((q, wq), (k, wk))]
        return (y[0] * d64(c.dyq)).sum() + (y[1] * d64(c.dyk)).sum()

    g = torch.Generator().manual_seed(3)
    base = [d64(t) for t in leaves]
    for i in range(4):
        step = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * step, base[i] - 1e-5 * step
        diff = (loss(*up) - loss(*down)) / 2e-5
        # the sum's terms are each right to 1e-5 of gradients of order one; the
        # differences are to 1e-10 of the third derivative
        mine = (d64(got[i]) * step).sum()
        assert abs(mine - diff) <= 1e-5 * (d64(got[i]).abs() * step.abs()).sum() + 1e-6


@gpu
def test_the_whole_head_in_halves_is_rope_varlen():
    """... with a norm, where both round once (a different reduction of the angle:
    fp32 there, which positions below 64 leave within 4e-6)."""
    c = Case(64, 4, 2, 64, 64, False, torch.float32, cu=[0, 30, 64])
    a = c.run()
    b = rope.rope_varlen(c.q, c.k, c.cu, c.inv, c.wq, c.wk, EPS)
    for x, y in zip(a, b):
        assert (x - y).abs().max() < 1e-4


@gpu
def test_features_behind_the_rotated_ones_are_not_touched():
    """An infinity or a NaN there stays where it is; elsewhere it stays in its pair."""
    for inter, rd in ((False, 32), (True, 24), (False, 24)):
        c = Case(6, 2, 1, 64, rd, inter, torch.bfloat16, norm=(False, False))
        c.q[2, 1, 50] = float("inf")
        c.q[3, 0, 63] = float("nan")
        y, _ = c.run()
        assert torch.isposinf(y[2, 1, 50]) and torch.isnan(y[3, 0, 63])
        y[2, 1, 50] = y[3, 0, 63] = 0
        assert torch.isfinite(y).all()
        assert torch.equal(y[:, :, rd:][:2], c.q[:, :, rd:][:2])


@gpu
def test_empty():
    c = Case(0, 2, 1, 64, 32, True, torch.bfloat16)
    q, k = c.run()
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    leaves = [t.requires_grad_() for t in (c.q, c.k, c.wq, c.wk)]
    got = torch.autograd.grad(c.run(), leaves, (c.dyq, c.dyk))
    assert (got[2] == 0).all() and (got[3] == 0).all()


@gpu
def test_python_launcher_gives_the_same(monkeypatch):
    c = Case(77, 4, 2, 64, 24, False, torch.bfloat16, wide=8)
    leaves = [t.requires_grad_() for t in (c.q, c.k, c.wq, c.wk)]

    def both():
        y = c.run()
        return (*y, *torch.autograd.grad(y, leaves, (c.dyq, c.dyk)))

    a = both()
    monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    for x, y in zip(a, both()):
        assert torch.equal(x, y)


@gpu
def test_other_strides_dtypes_and_streams():
    c = Case(30, 4, 2, 64, 40, True, torch.float16, wide=8)
    want = c.run()
    c.pos, c.inv = c.pos.long(), c.inv.double()
    c.q = torch.cat((c.q.new_zeros(30, 4, 3), c.q), -1)[..., 3:]  # rows off 16 bytes
    c.k = c.k.transpose(0, 1).contiguous().transpose(0, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = c.run()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("wdtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
def test_norm_weights_of_another_type(wdtype):
    c = Case(40, 4, 2, 64, 32, True, torch.bfloat16, wdtype=wdtype)
    HALF[torch.float64] = STEP[torch.float64] = 2.0 ** -24  # (rounded to fp32 on the way)
    check_forward(c)
    check_backward(c)
    c.wk = c.wk.to(torch.float32)
    check_backward(c)


@gpu
def test_rows_past_32_bits():
    """The last tokens of a call of more than 2^31 elements, forward and backward, as by themselves."""
    c = Case(48, 8, 2, 512, 96, True, torch.bfloat16)
    T = 2 ** 31 // (8 * 512) + 100

    def long(t):
        y = torch.zeros(T, *t.shape[1:], dtype=t.dtype, device="cuda")
        y[-48:] = t
        return y

    want = (*rope.rotary_embed_raw(c.q, c.k, c.inv, **c.args()),
            *rope.rotary_embed_bwd(c.dyq, c.dyk, c.q, c.k, c.inv, **c.args())[:2])
    c.q, c.k, c.dyq, c.dyk, c.pos = (long(t) for t in (c.q, c.k, c.dyq, c.dyk, c.pos))
    assert c.q.numel() > 2 ** 31
    for a, b in zip(rope.rotary_embed_raw(c.q, c.k, c.inv, **c.args()), want[:2]):
        assert torch.equal(a[-48:], b)
    for a, b in zip(rope.rotary_embed_bwd(c.dyq, c.dyk, c.q, c.k, c.inv, **c.args()), want[2:]):
        assert torch.equal(a[-48:], b)


@gpu
def test_captured():
    c = Case(70, 4, 2, 128, 64, True, torch.bfloat16)
    c.run()
    raw = lambda: (*rope.rotary_embed_raw(c.q, c.k, c.inv, **c.args()), *rope.rotary_embed_bwd(
        c.dyq, c.dyk, c.q, c.k, c.inv, **c.args()))
    raw()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = raw()
    for i in range(3):
        c.pos += 11
        c.q.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, raw()))


@gpu
def test_gradients_of_expanded_and_unused_outputs():
    c = Case(12, 4, 2, 64, 32, True, torch.float32)
    q = c.q.contiguous().requires_grad_()
    y, _ = rotary_embed(q, c.k, c.inv, **c.args())
    y.sum().backward()
    c.dyq = torch.ones_like(y)
    dx, _, mag, _ = grads(d64(q), d64(c.wq), d64(c.dyq), c.at, d64(c.inv), True, 1.0)
    within("dq", q.grad, dx, HALF[c.dtype] * dx.abs() + 8e-6 * mag)


class _Slab:  # (as a GradSlab without room: the Python node's path)
    def block(self, i, layout):
        return None


@gpu
@pytest.mark.parametrize("slab", [None, _Slab()])
def test_second_derivatives_are_refused(slab):
    c = Case(12, 4, 2, 64, 32, True, torch.float32)
    q = c.q.clone().requires_grad_()
    y, z = rotary_embed(q, c.k, c.inv, **c.args(), grad_slab=slab)
    (g,) = torch.autograd.grad((y.square().sum() + z.sum()), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q, retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@gpu
@pytest.mark.parametrize("slab", [None, _Slab()])
def test_captured_training(slab):
    c = Case(70, 4, 2, 64, 32, True, torch.bfloat16)
    args = c.args()
    leaf = args["norm_q"] = args["norm_q"].detach().clone().requires_grad_()

    def step():
        y, z = rotary_embed(c.q, c.k, c.inv, **args, grad_slab=slab)
        (g,) = torch.autograd.grad((y, z), leaf, (c.dyq, c.dyk))
        return y, g

    eager = rotary_embed(c.q, c.k, c.inv, **args, grad_slab=slab)  # an eager graph that lives
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="is alive"), torch.cuda.graph(graph):
        rotary_embed(c.q, c.k, c.inv, **args, grad_slab=slab)
    del eager, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        c.pos += 11
        c.q.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


# ── CPU ──────────────────────────────────────────────────────────────────────

def _args(**over):
    a = _capi.RotaryArgs()
    r = a.r
    r.dtype, r.total_tokens, r.heads_q, r.heads_k, r.head_dim, r.nseq, r.sign = 1, 10, 4, 2, 64, 0, 1
    r.inv_freq = FAKE
    r.q = _capi.Tensor(FAKE, 0, 256, 64)
    r.k = _capi.Tensor(2 * FAKE, 0, 128, 64)
    r.q_out = _capi.Tensor(3 * FAKE, 0, 256, 64)
    r.k_out = _capi.Tensor(4 * FAKE, 0, 128, 64)
    a.positions, a.rotary_dim, a.interleaved, a.scale = FAKE, 32, 0, 1.0
    for k, v in over.items():
        setattr(r if hasattr(r, k) and not hasattr(_capi.RotaryArgs, k) else a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(), "FNA2_OK"),
    (dict(positions=None), "FNA2_E_SEQLENS"),
    (dict(positions=None, cu_seqlens=FAKE), "FNA2_OK"),
    (dict(cu_seqlens=FAKE), "FNA2_E_SEQLENS"),
    (dict(rotary_dim=0), "FNA2_E_HEAD_DIM"),
    (dict(rotary_dim=7), "FNA2_E_HEAD_DIM"),
    (dict(rotary_dim=66), "FNA2_E_HEAD_DIM"),
    (dict(rotary_dim=64), "FNA2_OK"),
    (dict(rotary_dim=2), "FNA2_OK"),
    (dict(interleaved=2), "FNA2_E_SHAPE"),
    (dict(scale=float("inf")), "FNA2_E_SCALE"),
    (dict(head_dim=96), "FNA2_E_HEAD_DIM"),
    (dict(dtype=9), "FNA2_E_DTYPE"),
    (dict(inv_freq=None), "FNA2_E_NULL"),
    (dict(sign=2), "FNA2_E_SHAPE"),
    (dict(q_out=_capi.Tensor(FAKE + 64, 0, 256, 64)), "FNA2_E_ALIAS"),
    (dict(q_out=_capi.Tensor(FAKE, 0, 256, 64)), "FNA2_OK"),  # in place
    (dict(q=_capi.Tensor(FAKE + 2, 0, 256, 64)), "FNA2_E_STRIDE"),
    (dict(total_tokens=0, q=_capi.empty_tensor()), "FNA2_OK"),
    (dict(norm_q=FAKE), "FNA2_E_DTYPE"),
    (dict(norm_q=FAKE, norm_dtype=2), "FNA2_OK"),
])
def test_check(over, code):
    lib = _capi.lib()
    a = _args(**over)
    assert _capi.STATUS[lib.fna2_check_rotary(ctypes.byref(a))] == code
    if code != "FNA2_OK":
        assert _capi.STATUS[lib.fna2_rotary(ctypes.byref(a), None)] == code


def test_check_backward():
    lib = _capi.lib()
    b = _capi.RotaryBwdArgs()
    b.fwd = _args(norm_q=FAKE, norm_dtype=3)
    b.dq_out, b.dk_out, b.dq, b.dk = b.fwd.r.q, b.fwd.r.k, b.fwd.r.q_out, b.fwd.r.k_out
    st = lambda: _capi.STATUS[lib.fna2_check_rotary_bwd(ctypes.byref(b))]
    assert st() == "FNA2_E_NULL"
    b.dnorm_q = FAKE
    assert st() == "FNA2_E_WORKSPACE"
    need = lib.fna2_rotary_bwd_workspace_bytes(ctypes.byref(b.fwd))
    assert need > 0
    b.workspace, b.workspace_bytes = FAKE, need
    assert st() == "FNA2_OK"
    b.fwd.r.norm_q = None
    b.workspace_bytes = 0
    assert lib.fna2_rotary_bwd_workspace_bytes(ctypes.byref(b.fwd)) == 0 and st() == "FNA2_OK"


def test_struct_layout_matches_header(tmp_path):
    pairs = (("fna2_rotary_args", _capi.RotaryArgs), ("fna2_rotary_bwd_args", _capi.RotaryBwdArgs))
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


@pytest.mark.parametrize("change", [
    dict(positions=None), dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)),
    dict(positions=torch.zeros(3, dtype=torch.int32)), dict(inv_freq=torch.ones(33)),
    dict(inv_freq=torch.ones(0)), dict(q=torch.zeros(5, 64)), dict(k=torch.zeros(4, 2, 64)),
    dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), dict(norm_q=torch.ones(32)),
])
def test_refusals(change):
    a = dict(q=torch.zeros(5, 4, 64), k=torch.zeros(5, 2, 64), inv_freq=torch.ones(32),
             positions=torch.zeros(5, dtype=torch.int32))
    a.update(change)
    # (shapes before the device for all but the norm's, which the GPU check precedes)
    with pytest.raises((AssertionError, RuntimeError)):
        rotary_embed(**a)


def test_needs_the_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_embed(torch.zeros(5, 4, 64), torch.zeros(5, 2, 64), torch.ones(16),
                     positions=torch.zeros(5, dtype=torch.int32))


def test_frequencies():
    inv, s = rotary_frequencies(64)
    ref = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    assert s == 1.0 and np.allclose(inv.double(), ref, rtol=1e-7, atol=0)
    lin, s = rotary_frequencies(64, scaling="linear", factor=4.0)
    assert s == 1.0 and np.allclose(lin.double(), ref / 4, rtol=1e-7, atol=0)
    ntk, s = rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert s == 1.0 and ntk[0] == 1 and np.isclose(float(ntk[-1]), ref[-1] / 4, rtol=1e-6)
    assert (ntk <= inv).all() and (ntk >= lin).all()
    yarn, s = rotary_frequencies(64, scaling="yarn", factor=4.0, original_max_len=2048)
    turns = 2048 * ref / (2 * np.pi)
    y = yarn.double().numpy()
    assert np.isclose(s, 0.1 * np.log(4) + 1)
    assert np.allclose(y[turns > 40], ref[turns > 40], rtol=1e-6)
    assert np.allclose(y[turns < 0.7], ref[turns < 0.7] / 4, rtol=1e-6)
    assert (y <= ref * (1 + 1e-6)).all() and (y >= ref / 4 * (1 - 1e-6)).all()
    one, s = rotary_frequencies(2, scaling="ntk", factor=2.0)
    assert one.tolist() == [0.5]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="linear", factor=0.5)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


@gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("what", ["q", "k", "norm_q", "norm_k", "inv_freq"])
def test_tangents_are_refused(what, native, monkeypatch):
    """Forward-mode differentiation raises, as rope_varlen's does: no output without its tangent."""
    import torch.autograd.forward_ad as fw
    c = Case(9, 2, 1, 64, 32, True, torch.float32)
    args = dict(c.args(), q=c.q.contiguous(), k=c.k.contiguous(), inv_freq=c.inv)
    if not native:
        monkeypatch.setattr(_capi, "native_or_none", lambda: None)
    with fw.dual_level():
        args[what] = fw.make_dual(args[what], torch.ones_like(args[what]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError)):
                rotary_embed(**args)
        with pytest.raises((RuntimeError, NotImplementedError)):
            rotary_embed(**args, grad_slab=_Slab())
