"""The operators of the paged cache, as cases that can be measured.

A paged cache keeps its rows in pages of ``ps`` rows, ``[pages, heads, ps,
features]``, that a block table strings together per sequence.  The operators:

* ``attend``: attention of packed chunks of new tokens (one token, a few
  drafted ones, a piece of a prompt) over the cache, with the low-rank bias
  from cached ``R_k`` pages (``flash_naylis_paged``);
* ``weights``: the same, adding up each cached row's attention weight;
* ``append``: RMSNorm and rotation of the chunks' q and k, and the write of k,
  v and R_k into their pages (``paged_append``);
* ``evict``: the rows of largest accumulated weight kept, the others dropped
  and the cache compacted (``paged_evict``).

``own`` picks the package's kernels; the plain forms are elementary torch
operations in 32 bits (64 for rotation angles).  ``exact()`` restates each
operator in 64 bits, sequence by sequence.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6


def listed():
    return [
        # Serving a small model, one token for each of two short sequences:
        # latency.
        dict(name="decode_few", kind="attend", B=2, chunks=0, M=1, L=500, ragged=False, H=8,
             HKV=4, HG=4, D=64, R=32, ps=16, dtype="bf16"),
        # Serving, one token for each of 64 long sequences, bias from R_k
        # pages, no grouped heads: the cache is read once.
        dict(name="decode_batch", kind="attend", B=64, chunks=0, M=1, L=4096, ragged=False, H=16,
             HKV=16, HG=16, D=128, R=32, ps=64, dtype="bf16"),
        # Five drafted tokens a sequence verified at once, ragged, vanilla
        # heads beside graph heads, an odd page size.
        dict(name="verify_fp16", kind="attend", B=16, chunks=16, M=5, L=2500, ragged=True, H=16,
             HKV=4, HG=12, D=128, R=24, ps=48, dtype="fp16"),
        # One step of a server that mixes a piece of a prompt with 32
        # decoding sequences.
        dict(name="mixed_step", kind="attend", B=33, chunks=1, M=256, L=4096, ragged=True, H=32,
             HKV=8, HG=32, D=128, R=32, ps=64, dtype="bf16"),
        # A piece of a long prompt: bound by the matrix cores.
        dict(name="prompt_chunk", kind="attend", B=1, chunks=1, M=1024, L=16384, ragged=False,
             H=32, HKV=8, HG=32, D=128, R=64, ps=128, dtype="bf16"),
        # One token a sequence with the weights that eviction goes by.
        dict(name="weigh_decode", kind="weights", B=16, chunks=0, M=1, L=8192, ragged=True, H=32,
             HKV=8, HG=0, D=128, R=0, ps=64, dtype="bf16"),
        # Two prompts' last pieces, odd lengths, every row weighed.
        dict(name="weigh_prompt", kind="weights", B=2, chunks=2, M=509, L=7001, ragged=True, H=16,
             HKV=16, HG=16, D=64, R=16, ps=32, dtype="bf16"),
        # The new rows of 64 decoding sequences: a launch.
        dict(name="append_decode", kind="append", B=64, chunks=0, M=1, L=4096, ragged=True, H=16,
             HKV=16, HG=16, D=128, R=32, ps=64, dtype="bf16"),
        # The rows of four long prompts, grouped heads: bandwidth.
        dict(name="append_prompt", kind="append", B=4, chunks=4, M=2048, L=6000, ragged=True, H=32,
             HKV=8, HG=32, D=128, R=32, ps=64, dtype="bf16"),
        # A small cache a little over its budget.
        dict(name="evict_few", kind="evict", B=2, L=1201, ragged=False, budget=1000, recent=100,
             first=4, H=8, HKV=4, HG=4, D=64, R=32, ps=16, dtype="bf16"),
        # 32 long sequences brought back to half their length.
        dict(name="evict_batch", kind="evict", B=32, L=8192, ragged=True, budget=4096, recent=512,
             first=4, H=32, HKV=8, HG=32, D=128, R=32, ps=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    h, kv = rng.choice([(8, 4), (8, 8), (12, 4), (16, 16), (16, 2), (32, 8), (32, 32), (6, 2)])
    hg = rng.choice([h, h, h // 2, 0])
    c = dict(kind=rng.choice(["attend", "attend", "attend", "weights", "append", "evict"]),
             B=_log(rng, 1, 64), L=_log(rng, 64, 16384), ragged=rng.random() < 0.6, H=h, HKV=kv,
             HG=hg, D=rng.choice([64, 128]), R=rng.choice([8, 16, 24, 32, 32, 64]) if hg else 0,
             ps=rng.choice([16, 32, 48, 64, 128, 256]),
             dtype=rng.choice(["bf16", "bf16", "bf16", "fp16"]))
    row = 2 * (2 * kv * c["D"] + hg * c["R"])  # bytes of a cached row
    c["B"] = max(1, min(c["B"], int(2e9) // (row * c["L"])))
    if c["kind"] == "evict":
        c["budget"] = max(8, int(c["L"] * rng.uniform(0.25, 1.1)))
        c["recent"] = int(c["budget"] * rng.uniform(0, 0.4))
        c["first"] = rng.choice([0, 0, 4])
        return c
    mode = rng.choice(["decode", "verify", "prompt", "mixed"])
    c["M"] = {"decode": 1, "verify": rng.randint(2, 9)}.get(mode) or _log(rng, 10, 1024)
    c["M"] = min(c["M"], c["L"])
    c["chunks"] = {"decode": 0, "mixed": min(c["B"], 2)}.get(mode, c["B"])
    # at most the largest listed case's products, and the plain form's padded
    # score matrix within 2^30 values
    while c["B"] > 1 and (work(c)["flops"] > 3.4e11 or c["B"] * h * c["M"] * c["L"] > 1 << 30):
        c["B"] -= 1
        c["chunks"] = min(c["chunks"], c["B"])
    return c


# -- the sizes of a case ------------------------------------------------------

def _rows(case):
    """Rows of each sequence's cache (a chunk's included)."""
    L, B = case["L"], case["B"]
    if not case["ragged"]:
        return [L] * B
    lo = max(L // 3, 1)
    lens = [L - (i * 7919) % (L - lo + 1) for i in range(B)]
    return [max(n, m) for n, m in zip(lens, _chunks(case))]


def _chunks(case):
    """New tokens of each sequence."""
    if case["kind"] == "evict":
        return [0] * case["B"]
    M, n = case["M"], case["chunks"]
    cut = lambda i: (i * 331) % (M // 3 + 1) if case["ragged"] else 0
    return [M - cut(i) if i < n else 1 for i in range(case["B"])]


def _pairs(case):
    return sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(_chunks(case), _rows(case)))


def _kept(case):
    return [min(n, case["budget"]) for n in _rows(case)]


def work(case):
    H, HKV, HG, D, R = (case[x] for x in ("H", "HKV", "HG", "D", "R"))
    T, rows = sum(_chunks(case)), sum(_rows(case))
    k = case["kind"]
    if k == "append":  # every row read once and written once
        n = T * ((H + 2 * HKV) * D + HG * R)
        return dict(bytes=4 * n, flops=10 * T * (H + HKV) * D)
    if k == "evict":
        # the weights read, the kept rows' indexes and weights written, and
        # the rows that move: past the first that is dropped, about all
        kept = sum(_kept(case))
        moved = sum(m for m, n in zip(_kept(case), _rows(case)) if n > m)
        return dict(bytes=HKV * (4 * rows + 8 * kept) + 4 * moved * (2 * HKV * D + HG * R),
                    flops=HKV * rows)
    b = rows * (2 * HKV * D + HG * R) * 2 + T * (2 * H * D + HG * R) * 2
    f = _pairs(case) * (H * 4 * D + HG * 2 * R)
    if k == "weights":
        return dict(bytes=b + 8 * HKV * rows, flops=f + _pairs(case) * H)
    return dict(bytes=b, flops=f)


# -- inputs -------------------------------------------------------------------

def _pool(g, case, heads, feat, dtype, pages):
    return torch.randn(pages, heads, case["ps"], feat, generator=g, device=g.device,
                       dtype=torch.float32).to(dtype) if heads else None


def prepare(case, seed):
    """A cache in use: pools, a block table whose pages lie in no order, the
    lengths, and the chunk's rows as a projection (append) or an append
    (attend) leaves them."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt, ps, B = _DT[case["dtype"]], case["ps"], case["B"]
    H, HKV, HG, D, R = (case[x] for x in ("H", "HKV", "HG", "D", "R"))
    rows, lq = _rows(case), _chunks(case)
    used = [-(-n // ps) for n in rows]
    width, pages = max(used) + 1, sum(used) + 5
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    first = torch.tensor([sum(used[:b]) for b in range(B)], device=dev)[:, None]
    j = torch.arange(width, device=dev)[None]
    inside = j < torch.tensor(used, device=dev)[:, None]
    table = torch.where(inside, perm[(first + j).clamp(max=pages - 1)], -1).to(torch.int32)
    cu = [0]
    for n in lq:
        cu.append(cu[-1] + n)
    T = cu[-1]
    s = dict(case=case, table=table.contiguous(), max_q=max(lq),
             lens=torch.tensor(rows, dtype=torch.int32, device=dev),
             cu=torch.tensor(cu, dtype=torch.int32, device=dev),
             k=_pool(g, case, HKV, D, dt, pages), v=_pool(g, case, HKV, D, dt, pages),
             rk=_pool(g, case, HG, R, torch.bfloat16, pages), rk_new=None, rq=None, gs=None)
    randn = lambda *n: torch.randn(*n, generator=g, device=dev, dtype=torch.float32)
    if HG:
        s["rk"].mul_(R ** -0.5)
        s["gs"] = 1 + 0.25 * randn(HG)
    cap = width * ps
    if case["kind"] == "evict":
        # sums of softmax weights: a few heavy rows, many light ones, some
        # never looked at
        w = torch.exp(2 * randn(B, HKV, cap)) * (randn(B, HKV, cap) > -1.5)
        s["w"] = torch.where(torch.arange(cap, device=dev) < s["lens"][:, None, None], w, 0.0)
        return s
    if case["kind"] == "append":
        # one projection's output [T, q | k | v | R_q | R_k], read in place
        y = randn(T, (H + 2 * HKV) * D + 2 * HG * R).to(dt)
        cut = lambda a, h, f: y[:, a:a + h * f].view(T, h, f)
        s.update(q=cut(0, H, D), k_new=cut(H * D, HKV, D), v_new=cut((H + HKV) * D, HKV, D),
                 wq=1 + 0.1 * randn(D), wk=1 + 0.1 * randn(D),
                 inv=10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float32) / D))
        if HG:
            r = y[:, (H + 2 * HKV) * D + HG * R:].view(T, HG, R)
            s["rk_new"] = r if dt == torch.bfloat16 else r.to(torch.bfloat16)
        return s
    s["q"] = randn(T, H, D).to(dt)
    if HG:  # R_q is a column block of the projection's output
        y = (randn(T, 2 * HG * R) * R ** -0.5).to(torch.bfloat16)
        s["rq"] = y[:, :HG * R].view(T, HG, R)
    if case["kind"] == "weights":
        s["w"] = torch.rand(B, HKV, cap, generator=g, device=dev)
    return s


# -- the operators ------------------------------------------------------------

def _cached(pages, table):
    """Pages [P, h, ps, f] as padded rows [N, h, table width * ps, f], fp32."""
    x = pages[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _attend(s):
    c = s["case"]
    B, H, HKV, HG, D = (c[x] for x in ("B", "H", "HKV", "HG", "D"))
    M, T, dev = s["max_q"], s["q"].shape[0], s["q"].device
    cu, lk = s["cu"].long(), s["lens"].long()
    lq = cu[1:] - cu[:-1]
    i = torch.arange(M, device=dev)
    live = i < lq[:, None]                                     # [B, M]
    tok = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[tok].transpose(1, 2)                    # [B, H, M, D]
    k, v = _cached(s["k"], s["table"]), _cached(s["v"], s["table"])
    L = k.shape[2]
    j = torch.arange(L, device=dev)
    v = torch.where((j < lk[:, None])[:, None, :, None], v, 0.0)
    sc = torch.matmul(q.reshape(B, HKV, -1, D), k.transpose(2, 3)).view(B, H, M, L) * D ** -0.5
    if HG:
        rk = _cached(s["rk"], s["table"])
        rq = s["rq"].float()[tok].transpose(1, 2)
        sc[:, :HG] += torch.matmul(rq, rk.transpose(2, 3)) * s["gs"][:, None, None]
    see = (j <= (lk - lq)[:, None, None] + i[:, None]) & (j < lk[:, None, None]) & live[:, :, None]
    sc = sc.masked_fill_(~see[:, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc.sub_(torch.where(m == -math.inf, 0.0, m)))
    p = p / (p.sum(-1, keepdim=True) + 1e-6)
    out = torch.matmul(p.view(B, HKV, -1, L), v).view(B, H, M, D).transpose(1, 2)
    where = torch.repeat_interleave(torch.arange(B, device=dev), lq, output_size=T)
    out = out[where, torch.arange(T, device=dev) - cu[where]].to(s["q"].dtype)
    if c["kind"] == "attend":
        return out
    w = s["w"]
    w += p.view(B, HKV, -1, L).sum(2)[:, :, :w.shape[2]]
    return out, w


def _slots(s):
    """Page and row within it of every new token, and its position."""
    cu, T = s["cu"].long(), s["q"].shape[0]
    lq = cu[1:] - cu[:-1]
    b = torch.repeat_interleave(torch.arange(len(lq), device=cu.device), lq, output_size=T)
    row = torch.arange(T, device=cu.device) - cu[b] + (s["lens"].long() - lq)[b]
    ps = s["case"]["ps"]
    return s["table"][b, row // ps].long(), row % ps, row


def _norm_rope(x, w, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _append(s):
    page, off, pos = _slots(s)
    ang = pos.double()[:, None, None] * s["inv"].double()
    cos, sin = ang.cos().float(), ang.sin().float()
    dt = s["q"].dtype
    s["k"][page, :, off] = _norm_rope(s["k_new"], s["wk"], cos, sin).to(dt)
    s["v"][page, :, off] = s["v_new"]
    if s["rk"] is not None:
        s["rk"][page, :, off] = s["rk_new"]
    return _norm_rope(s["q"], s["wq"], cos, sin).to(dt), s["k"], s["v"], s["rk"]


def _compact(pages, table, rows, kept, ok):
    """rows[b, h, r] = kept[b, h, r] of each head's rows, where ok."""
    ps = pages.shape[2]
    b, h, r = torch.nonzero(ok, as_tuple=True)
    src = kept[b, h, r]
    x = pages[table[b, src // ps].long(), h, src % ps]
    pages[table[b, r // ps].long(), h, r % ps] = x


def _evict(s):
    c = s["case"]
    n, top = s["lens"].long(), c["budget"]
    w, B, HKV = s["w"], c["B"], c["HKV"]
    cap = w.shape[2]
    j = torch.arange(cap, device=w.device)
    ln = n[:, None, None]
    prio = torch.where((j < c["first"]) | (j >= ln - c["recent"]), math.inf, w)
    prio = torch.where(j < ln, prio, -math.inf)
    order = torch.sort(prio, dim=-1, descending=True, stable=True).indices[..., :top]
    new = torch.minimum(n, torch.full_like(n, top))
    r = torch.arange(order.shape[2], device=w.device)
    ok = (r < new[:, None, None]).expand(B, HKV, -1)
    kept = torch.sort(torch.where(ok, order, cap), dim=-1).values
    got = torch.where(ok, w.gather(2, kept.clamp(max=cap - 1)), 0.0)
    out_w = torch.zeros_like(w)
    out_w[..., :got.shape[2]] = got
    _compact(s["k"], s["table"], c, kept, ok)
    _compact(s["v"], s["table"], c, kept, ok)
    if s["rk"] is not None:
        g = c["H"] // HKV
        heads = torch.arange(c["HG"], device=w.device) // g
        _compact(s["rk"], s["table"], c, kept[:, heads], ok[:, heads])
    idx = torch.full((B, HKV, top), -1, dtype=torch.int32, device=w.device)
    idx[..., :kept.shape[2]] = torch.where(ok, kept, -1).to(torch.int32)
    return idx, new.to(torch.int32), out_w, s["k"], s["v"], s["rk"]


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _append, "evict": _evict}.get(kind, _attend)(s)
    from fna2_amd import paged
    if kind == "append":
        q = paged.paged_append(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["table"],
                               s["lens"], s["cu"], r_k=s["rk_new"], rk_pages=s["rk"],
                               inv_freq=s["inv"], norm_q=s["wq"], norm_k=s["wk"], eps=_EPS)
        return q, s["k"], s["v"], s["rk"]
    if kind == "evict":
        c = s["case"]
        kept, lens, w = paged.paged_evict(s["k"], s["v"], s["table"], s["lens"], s["w"],
                                          c["budget"], recent=c["recent"], first=c["first"],
                                          rk_pages=s["rk"], heads=c["H"])
        return kept, lens, w, s["k"], s["v"], s["rk"]
    out = paged.flash_naylis_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                                   s["max_q"], r_q=s["rq"], rk_pages=s["rk"],
                                   graph_scale=s["gs"], key_weights=s.get("w"))
    return (out, s["w"]) if kind == "weights" else out


# -- the same in 64 bits ------------------------------------------------------

def _exact_attend(s, case):
    H, HKV, HG, D = (case[x] for x in ("H", "HKV", "HG", "D"))
    g, ps = H // HKV, case["ps"]
    outs, w = [], s["w"].double() if case["kind"] == "weights" else None
    t = 0
    for b, (m, n) in enumerate(zip(_chunks(case), _rows(case))):
        ids = s["table"][b, :-(-n // ps)].long()
        rows = lambda p, h: p[ids, h].reshape(-1, p.shape[3])[:n].double()
        hidden = (torch.arange(n, device=ids.device)[None] >
                  n - m + torch.arange(m, device=ids.device)[:, None])
        out = torch.empty(m, H, D, dtype=torch.float64, device=ids.device)
        for h in range(H):
            x = s["q"][t:t + m, h].double() @ rows(s["k"], h // g).t() / math.sqrt(D)
            if h < HG:
                x += s["gs"][h].double() * (s["rq"][t:t + m, h].double() @ rows(s["rk"], h).t())
            x[hidden] = -math.inf
            lse = torch.logsumexp(x, -1, keepdim=True)
            top = x.amax(-1, keepdim=True)  # l + 1e-6 under the maximum, as the operator has it
            p = torch.exp(x - top) / (torch.exp(lse - top) + 1e-6)
            out[:, h] = p @ rows(s["v"], h // g)
            if w is not None:
                w[b, h // g, :n] += p.sum(0)
        outs.append(out)
        t += m
    out = torch.cat(outs)
    return out if w is None else (out, w)


def _exact_append(s, case):
    ps, half = case["ps"], case["D"] // 2
    k, v = s["k"].double(), s["v"].double()
    rk = None if s["rk"] is None else s["rk"].double()

    def turn(x, w, pos):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.double()
        z = torch.complex(x[..., :half], x[..., half:])
        ang = pos.double()[:, None] * s["inv"].double()[None]
        z = z * torch.polar(torch.ones_like(ang), ang)[:, None]
        return torch.cat((z.real, z.imag), -1)

    q, t = [], 0
    for b, (m, n) in enumerate(zip(_chunks(case), _rows(case))):
        pos = torch.arange(n - m, n, device=k.device)
        page, off = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")], pos % ps
        cut = slice(t, t + m)
        q.append(turn(s["q"][cut], s["wq"], pos))
        k[page, :, off] = turn(s["k_new"][cut], s["wk"], pos)
        v[page, :, off] = s["v_new"][cut].double()
        if rk is not None:
            rk[page, :, off] = s["rk_new"][cut].double()
        t += m
    return torch.cat(q), k, v, rk


def exact(case, seed):
    if case["kind"] == "evict":  # whole numbers and copies: nothing is computed
        return None
    H, D = case["H"], case["D"]
    if case["B"] * H > 2100 or (case["kind"] != "append" and work(case)["flops"] > 4e11):
        return None
    s = prepare(case, seed)
    return (_exact_append if case["kind"] == "append" else _exact_attend)(s, case)
