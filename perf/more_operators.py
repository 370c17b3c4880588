"""Operators around the paged cache and the rotary embedding, as cases that
can be measured.

* ``shared``: attention of packed chunks of new tokens over a paged cache in
  which groups of sequences share their first pages (one system prompt, one
  document, many questions), with the low-rank bias from cached ``R_k`` pages
  (``flash_naylis_shared``);
* ``extend``: the books of such a cache kept on the GPU: from lengths and
  counts the pages of the new tokens, the block table, and every token's slot,
  sequence and position (``paged_extend``);
* ``groups``: which neighbouring sequences share how many rows, from the block
  table (``paged_groups``);
* ``rotary``: rotary positions of q and k in two layouts, over part of the
  head, scaled, at given positions, with the QK norm before it
  (``rotary_embed``);
* ``rotary_train``: the same over packed sequences, with its gradients.

``own`` picks the package's kernels; the plain forms are elementary torch
operations in 32 bits (64 for rotation angles and long sums).  ``exact()``
restates what is computed in 64 bits, sequence by sequence.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6


def listed():
    return [
        # Serving a small model: four sequences that share a short document,
        # one token each: latency.
        dict(name="shared_few", kind="shared", G=1, per=4, P=2000, S=100, M=1, ragged=False, H=8,
             HKV=4, HG=4, D=64, R=32, ps=16, dtype="bf16"),
        # 64 users behind one long system prompt, one token each: the prompt
        # is the matrix cores' work, the users' own rows are memory's.
        dict(name="shared_batch", kind="shared", G=1, per=64, P=16384, S=1000, M=1, ragged=True,
             H=32, HKV=8, HG=32, D=128, R=32, ps=64, dtype="bf16"),
        # Four prompts, five drafted tokens a sequence verified at once, vanilla
        # heads beside graph heads, an odd page size.
        dict(name="shared_verify", kind="shared", G=4, per=8, P=3001, S=333, M=5, ragged=True,
             H=16, HKV=4, HG=12, D=128, R=24, ps=48, dtype="fp16"),
        # No grouped heads: 32 sequences behind two long documents.
        dict(name="shared_heads", kind="shared", G=2, per=16, P=8192, S=512, M=1, ragged=False,
             H=16, HKV=16, HG=16, D=128, R=32, ps=128, dtype="bf16"),
        # 16 questions of some 128 tokens to one document, prefilled together:
        # bound by the matrix cores.
        dict(name="shared_prompt", kind="shared", G=1, per=16, P=8192, S=0, M=128, ragged=True,
             H=32, HKV=8, HG=32, D=128, R=64, ps=64, dtype="bf16"),
        # The step of 256 decoding sequences: one token each, now and then a page.
        dict(name="extend_decode", kind="extend", N=256, L=8192, M=1, ps=64),
        # 64 fresh prompts taken in at once.
        dict(name="extend_prompts", kind="extend", N=64, L=0, M=2048, ps=16),
        # Who shares a prefix among 512 sequences, after requests came and went.
        dict(name="groups_batch", kind="groups", N=512, per=24, pages=256, own_pages=16, ps=64),
        # A decode step of 64 sequences, far positions, a quarter of the head,
        # neighbouring features paired.
        dict(name="rotary_decode", kind="rotary", T=64, far=1000000, H=32, HKV=8, D=128, rd=32,
             inter=True, norm=True, scale=1.0, dtype="bf16"),
        # A long prompt of a model scaled for long contexts, the whole head.
        dict(name="rotary_prompt", kind="rotary", T=16384, far=131072, H=32, HKV=8, D=128, rd=128,
             inter=False, norm=False, scale=1.2, dtype="bf16"),
        # A training pack: norm and interleaved rotation, forward and backward.
        dict(name="rotary_train", kind="rotary_train", T=16384, n=64, H=16, HKV=16, D=128, rd=128,
             inter=True, norm=True, scale=1.0, dtype="bf16"),
        # A smaller one in 32 bits, odd lengths, part of a small head.
        dict(name="rotary_train_fp32", kind="rotary_train", T=5003, n=7, H=8, HKV=4, D=64, rd=24,
             inter=False, norm=True, scale=1.1, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared"] * 5 + ["rotary", "rotary_train", "rotary_train", "extend",
                                        "groups"])
    if kind == "extend":
        c = dict(kind=kind, N=_log(rng, 1, 4096), L=rng.choice([0, _log(rng, 16, 16384)]),
                 M=rng.choice([1, rng.randint(2, 9), _log(rng, 10, 4096)]),
                 ps=rng.choice([16, 32, 48, 64, 128, 256]))
        while c["N"] * c["M"] > 200000:
            c["N"] = max(1, c["N"] // 2)
        return c
    if kind == "groups":
        return dict(kind=kind, N=_log(rng, 32, 2048), per=_log(rng, 4, 64),
                    pages=_log(rng, 8, 256), own_pages=_log(rng, 1, 64),
                    ps=rng.choice([16, 48, 64, 128]))
    h, kv = rng.choice([(8, 4), (8, 8), (12, 4), (16, 16), (16, 2), (32, 8), (32, 32), (6, 2)])
    if kind != "shared":
        D = rng.choice([64, 128])
        dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        T = _log(rng, 1, 16384 if dt != "fp32" else 8192)
        if h * D > 2048:
            T = max(1, T // 2)
        c = dict(kind=kind, T=T, H=h, HKV=kv, D=D,
                 rd=rng.choice([D, D, D // 2, D // 4, 24, 2 * rng.randint(1, D // 2)]),
                 inter=rng.random() < 0.5, norm=rng.random() < 0.6,
                 scale=rng.choice([1.0, round(rng.uniform(0.8, 1.5), 3)]), dtype=dt)
        if kind == "rotary":
            c["far"] = _log(rng, T + 1, 2000000)
        else:
            c["n"] = rng.randint(1, min(T, 100))
        return c
    hg = rng.choice([h, h, h // 2, 0])
    c = dict(kind=kind, G=_log(rng, 1, 8), per=_log(rng, 1, 64), P=_log(rng, 64, 16384),
             S=_log(rng, 1, 2000), M=rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 256)]),
             ragged=rng.random() < 0.6, H=h, HKV=kv, HG=hg, D=rng.choice([64, 128]),
             R=rng.choice([8, 16, 24, 32, 32, 64]) if hg else 0,
             ps=rng.choice([16, 32, 48, 64, 128, 256]),
             dtype=rng.choice(["bf16", "bf16", "bf16", "fp16"]))
    # at most the largest listed case's products, and the plain form's padded
    # rows and scores of a group within some gigabytes
    while c["per"] > 1 and (work(c)["flops"] > 1.6e11 or work(c)["bytes"] > 6e8 or
                            c["per"] * c["G"] > 128 or
                            c["per"] * (c["P"] + c["S"] + c["M"]) * max(kv * c["D"], h * c["M"])
                            > 1 << 30):
        c["per"] -= 1
    while c["G"] > 1 and (work(c)["flops"] > 1.6e11 or work(c)["bytes"] > 6e8):
        c["G"] -= 1
    return c


# -- the sizes of a case ------------------------------------------------------

def _members(case):
    """Sequences of each group."""
    n = case["per"]
    return [n - (g * 3) % (n // 2 + 1) if case["ragged"] else n for g in range(case["G"])]


def _prefix(case):
    """Shared rows of each group, whole pages."""
    P, ps = case["P"], case["ps"]
    rows = [P - (g * 613) % (P // 2 + 1) if case["ragged"] else P for g in range(case["G"])]
    return [n // ps * ps for n in rows]


def _own(case):
    """(rows of its own before the chunk, chunk) of each sequence."""
    S, M = case["S"], case["M"]
    out = []
    for i in range(sum(_members(case))):
        cut = (i * 7919) % (S // 2 + 1) if case["ragged"] else 0
        out.append((S - cut, M - (i * 331) % (M // 3 + 1) if case["ragged"] else M))
    return out


def _seqs(case):
    """(group, shared rows, own rows before the chunk, chunk) of each sequence."""
    out, own_rows = [], iter(_own(case))
    for g, (n, p) in enumerate(zip(_members(case), _prefix(case))):
        out += [(g, p, *next(own_rows)) for _ in range(n)]
    return out


def _lens(case):
    """Lengths before the step, and the step's tokens, of ``extend``."""
    L, M = case["L"], case["M"]
    n = range(case["N"])
    return ([L - (i * 7919) % (L // 2 + 1) for i in n], [M - (i * 331) % (M // 3 + 1) for i in n])


def _runs(case):
    """Sequences of the runs of ``groups``, in some order."""
    out, left, i = [], case["N"], 0
    while left > 0:
        out.append(min(1 + (i * 37 + case["per"] - 1) % case["per"], left))
        left -= out[-1]
        i += 1
    return out


def work(case):
    k = case["kind"]
    if k == "extend":
        lens, counts = _lens(case)
        ps, T = case["ps"], sum(counts)
        new = sum(-(-(a + c) // ps) - -(-a // ps) for a, c in zip(lens, counts))
        return dict(bytes=4 * 4 * case["N"] + 8 * new + 16 * T, flops=case["N"] + T)
    if k == "groups":
        # (a run's shared pages are any number up to case["pages"])
        seen = sum(n * (1 + (case["pages"] + 1) // 2 * (n > 1)) for n in _runs(case))
        return dict(bytes=4 * seen + 8 * case["N"], flops=seen)
    H, HKV, D = case["H"], case["HKV"], case["D"]
    if k != "shared":
        es = 4 if case["dtype"] == "fp32" else 2
        n = case["T"] * (H + HKV) * D
        if k == "rotary":
            return dict(bytes=2 * es * n + 4 * case["T"], flops=8 * n)
        # forward: read and written once; backward: the gradient (and the
        # input, with a norm) read, the input's gradient written
        return dict(bytes=(5 if case["norm"] else 4) * es * n, flops=(24 if case["norm"] else 12) * n)
    HG, R = case["HG"], case["R"]
    T = pairs = rows = 0
    for g, p, s, m in _seqs(case):
        T += m
        rows += s + m
        pairs += m * (p + s) + m * (m + 1) // 2
    rows += sum(_prefix(case))
    return dict(bytes=rows * (2 * HKV * D + HG * R) * 2 + T * (2 * H * D + HG * R) * 2,
                flops=pairs * (H * 4 * D + HG * 2 * R))


# -- inputs -------------------------------------------------------------------

def _prepare_shared(case, g, dev):
    dt, ps = _DT[case["dtype"]], case["ps"]
    H, HKV, HG, D, R = (case[x] for x in ("H", "HKV", "HG", "D", "R"))
    seqs, members, prefix = _seqs(case), _members(case), _prefix(case)
    lens = [p + s + m for _, p, s, m in seqs]
    width = max(-(-n // ps) for n in lens) + 1
    total = sum(p // ps for p in prefix) + sum(-(-n // ps) - p // ps
                                               for n, (_, p, _, _) in zip(lens, seqs))
    pages = total + 5
    # pages in no order; a group's sequences begin with the same ones
    free = iter(torch.randperm(pages, generator=g, device=dev).tolist())
    first = [[next(free) for _ in range(p // ps)] for p in prefix]
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    for b, (n, (gr, p, _, _)) in enumerate(zip(lens, seqs)):
        row = first[gr] + [next(free) for _ in range(-(-n // ps) - p // ps)]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    cu, cg = [0], [0]
    for _, _, _, m in seqs:
        cu.append(cu[-1] + m)
    for n in members:
        cg.append(cg[-1] + n)
    T = cu[-1]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    randn = lambda *n: torch.randn(*n, generator=g, device=dev, dtype=torch.float32)
    pool = lambda h, f, t: randn(pages, h, ps, f).to(t)
    s = dict(case=case, table=table.to(dev), lens=ints(lens), cu=ints(cu), cg=ints(cg),
             shared=ints(prefix), max_q=max(m for *_, m in seqs), k=pool(HKV, D, dt),
             v=pool(HKV, D, dt), q=randn(T, H, D).to(dt), rk=None, rq=None, gs=None)
    if HG:
        s["rk"] = pool(HG, R, torch.bfloat16).mul_(R ** -0.5)
        # R_q is a column block of the projection's output
        y = (randn(T, 2 * HG * R) * R ** -0.5).to(torch.bfloat16)
        s["rq"] = y[:, :HG * R].view(T, HG, R)
        s["gs"] = 1 + 0.25 * randn(HG)
    return s


def _prepare_extend(case, g, dev):
    lens, counts = _lens(case)
    ps, N = case["ps"], case["N"]
    have = [-(-n // ps) for n in lens]
    new = sum(-(-(n + c) // ps) - h for n, c, h in zip(lens, counts, have))
    width = max(-(-(n + c) // ps) for n, c in zip(lens, counts)) + 1
    pages = sum(have) + new + 7
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    j = torch.arange(width, device=dev)
    h = torch.tensor(have, device=dev)
    first = (h.cumsum(0) - h)[:, None]
    table = torch.where(j < h[:, None], perm[(first + j).clamp(max=pages - 1)], -1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
    free[:new + 7] = perm[sum(have):]
    return dict(case=case, table=table.to(torch.int32).contiguous(), lens=ints(lens),
                counts=ints(counts), free=free, nfree=ints([new + 7]), T=sum(counts),
                shift=torch.randint(0, 1000, (N,), generator=g, device=dev, dtype=torch.int32))


def _prepare_groups(case, g, dev):
    sizes, N, own_pages = _runs(case), case["N"], case["own_pages"]
    order = torch.randperm(len(sizes), generator=g, device=dev).tolist()
    most = torch.randint(1, case["pages"] + 1, (len(sizes),), generator=g, device=dev).tolist()
    runs = [(sizes[i], m if sizes[i] > 1 else 0) for i, m in zip(order, most)]
    width = case["pages"] + own_pages + 1
    pages = sum(p for _, p in runs) + N * own_pages + 1
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    table, at, b = torch.full((N, width), -1, dtype=torch.int32), 0, 0
    for n, p in runs:
        table[b:b + n, :p] = perm[at:at + p]
        at += p
        for _ in range(n):
            table[b, p:p + own_pages] = perm[at:at + own_pages]
            at += own_pages
            b += 1
    return dict(case=case, table=table.to(dev))


def _prepare_rotary(case, g, dev):
    dt, T = _DT[case["dtype"]], case["T"]
    H, HKV, D, rd = (case[x] for x in ("H", "HKV", "D", "rd"))
    randn = lambda *n: torch.randn(*n, generator=g, device=dev, dtype=torch.float32)
    # q and k as a projection leaves them: column blocks of one output
    y = randn(T, (H + 2 * HKV) * D).to(dt)
    s = dict(case=case, q=y[:, :H * D].view(T, H, D),
             k=y[:, H * D:(H + HKV) * D].view(T, HKV, D), wq=None, wk=None, pos=None, cu=None,
             inv=(10000.0 ** (-torch.arange(0, rd, 2, device=dev, dtype=torch.float64) / rd)
                  / (4.0 if case["scale"] != 1.0 else 1.0)).float())
    if case["norm"]:
        s["wq"], s["wk"] = ((1 + 0.1 * randn(D)).to(dt) for _ in range(2))
    if case["kind"] == "rotary":
        if T <= 256:  # one token a sequence
            s["pos"] = torch.randint(0, case["far"], (T,), generator=g, device=dev,
                                     dtype=torch.int32)
        else:  # a piece of a prompt
            s["pos"] = torch.arange(case["far"] - T, case["far"], device=dev, dtype=torch.int32)
        return s
    cuts = torch.randperm(T - 1, generator=g, device=dev)[:case["n"] - 1] + 1
    ends = torch.tensor([0, T], device=dev)
    s["cu"] = torch.cat((cuts, ends)).sort().values.to(torch.int32)
    s["dyq"], s["dyk"] = randn(T, H, D).to(dt), randn(T, HKV, D).to(dt)
    for n in ("q", "k", "wq", "wk"):
        if s[n] is not None:
            s[n] = s[n].detach().requires_grad_()
    return s


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return {"shared": _prepare_shared, "extend": _prepare_extend, "groups": _prepare_groups}.get(
        case["kind"], _prepare_rotary)(case, g, dev)


# -- the operators ------------------------------------------------------------

def _cached(pages, table):
    """Pages [P, h, ps, f] as padded rows [N, h, table width * ps, f], fp32."""
    x = pages[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _shared(s):
    """A group's sequences at a time, their rows padded to one length."""
    c = s["case"]
    H, HKV, HG, D = (c[x] for x in ("H", "HKV", "HG", "D"))
    M, T, dev = s["max_q"], s["q"].shape[0], s["q"].device
    out = torch.empty_like(s["q"])
    b0 = 0
    for n in _members(c):
        b1 = b0 + n
        cu, lk, table = s["cu"][b0:b1 + 1].long(), s["lens"][b0:b1].long(), s["table"][b0:b1]
        lq = cu[1:] - cu[:-1]
        i = torch.arange(M, device=dev)
        tok = (cu[:-1, None] + i).clamp(max=T - 1)
        q = s["q"].float()[tok].transpose(1, 2)                    # [n, H, M, D]
        k, v = _cached(s["k"], table), _cached(s["v"], table)
        L = k.shape[2]
        j = torch.arange(L, device=dev)
        sc = torch.matmul(q.reshape(n, HKV, -1, D), k.transpose(2, 3)).view(n, H, M, L) * D ** -0.5
        if HG:
            rk = _cached(s["rk"], table)
            rq = s["rq"].float()[tok].transpose(1, 2)
            sc[:, :HG] += torch.matmul(rq, rk.transpose(2, 3)) * s["gs"][:, None, None]
        see = (j <= (lk - lq)[:, None, None] + i[:, None]) & (j < lk[:, None, None])
        sc = sc.masked_fill_(~see[:, None], -math.inf)
        p = torch.exp(sc.sub_(sc.amax(-1, keepdim=True)))
        p /= p.sum(-1, keepdim=True) + 1e-6
        o = torch.matmul(p.view(n, HKV, -1, L), v).view(n, H, M, D).transpose(1, 2)
        out[tok[i < lq[:, None]]] = o[i < lq[:, None]].to(out.dtype)
        b0 = b1
    return out


def _extend(s):
    ps, T, table = s["case"]["ps"], s["T"], s["table"]
    lens, c, dev = s["lens"].long(), s["counts"].long(), table.device
    have, need = (lens + ps - 1) // ps, (lens + c + ps - 1) // ps
    more = need - have
    base = more.cumsum(0) - more
    F = s["nfree"].long()
    j = torch.arange(table.shape[1], device=dev)
    new = (j >= have[:, None]) & (j < need[:, None])
    k = base[:, None] + j - have[:, None]
    table.copy_(torch.where(new, s["free"][(F - 1 - k).clamp(0, len(s["free"]) - 1)], table))
    cu = torch.cat((c.new_zeros(1), c.cumsum(0)))
    b = torch.repeat_interleave(torch.arange(len(c), device=dev), c, output_size=T)
    row = lens[b] + torch.arange(T, device=dev) - cu[b]
    slots = table[b, row // ps].long() * ps + row % ps
    i32 = torch.int32
    return (table, cu.to(i32), (lens + c).to(i32), (F - more.sum()).to(i32), slots, b.to(i32),
            (row + s["shift"][b]).to(i32))


def _groups(s):
    t, ps = s["table"], s["case"]["ps"]
    N, dev = t.shape[0], t.device
    same = ((t[1:] == t[:-1]) & (t[1:] >= 0)).long()
    common = torch.cat((same.new_zeros(1), same.cumprod(1).sum(1)))   # with the one before
    start = common == 0
    g = start.long().cumsum(0) - 1
    cu = torch.full((N + 1,), N, dtype=torch.long, device=dev)
    cu[:N].scatter_reduce_(0, g, torch.arange(N, device=dev), "amin")
    rows = torch.full((N,), 1 << 30, dtype=torch.long, device=dev)
    rows.scatter_reduce_(0, g, torch.where(start, 1 << 30, common), "amin")
    rows = torch.where(rows == 1 << 30, 0, rows) * ps
    return cu.to(torch.int32), rows.to(torch.int32)


def _halves(x, inter):
    return (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, -1)


def _join(a, b, inter):
    return torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)


def _turn(x, c, cos, sin):
    a, b = _halves(x[..., :c["rd"]], c["inter"])
    return torch.cat((_join(a * cos - b * sin, b * cos + a * sin, c["inter"]), x[..., c["rd"]:]), -1)


def _angles(s):
    pos = s["pos"]
    if pos is None:
        t = torch.arange(s["case"]["T"], device=s["cu"].device)
        pos = t - s["cu"].long()[torch.searchsorted(s["cu"].long(), t, right=True) - 1]
    ang = pos.double()[:, None, None] * s["inv"].double()
    f = s["case"]["scale"]
    return (ang.cos() * f).float(), (ang.sin() * f).float()


def _rotary_one(x, w, c, cos, sin):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * w.float()
    return _turn(y, c, cos, sin).to(x.dtype)


def _rotary_grad(x, w, dy, c, cos, sin):
    d = _turn(dy.float(), c, cos, -sin)
    if w is None:
        return d.to(x.dtype), None
    x, w32 = x.float(), w.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    dw = (d * x * r).sum((0, 1), dtype=torch.float64).to(w.dtype)
    d = d * w32
    return (r * (d - x * (r * r * (x * d).mean(-1, keepdim=True)))).to(dy.dtype), dw


def _rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    with torch.no_grad():
        yq, yk = (_rotary_one(s[a], s[w], c, cos, sin) for a, w in (("q", "wq"), ("k", "wk")))
        if c["kind"] == "rotary":
            return yq, yk
        dq, dwq = _rotary_grad(s["q"], s["wq"], s["dyq"], c, cos, sin)
        dk, dwk = _rotary_grad(s["k"], s["wk"], s["dyk"], c, cos, sin)
    return yq, yk, dq, dk, dwq, dwk


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"shared": _shared, "extend": _extend, "groups": _groups}.get(kind, _rotary)(s)
    from fna2_amd import paged, rope
    if kind == "shared":
        return paged.flash_naylis_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                                         s["max_q"], s["cg"], s["shared"], r_q=s["rq"],
                                         rk_pages=s["rk"], graph_scale=s["gs"])
    if kind == "extend":
        x = paged.paged_extend(s["table"], s["lens"], s["counts"], s["free"], s["nfree"], c["ps"],
                               s["T"], position_shift=s["shift"])
        return (s["table"], x.cu_seqlens_q, x.seqlens, x.free_count, x.slots, x.sequences,
                x.positions)
    if kind == "groups":
        return paged.paged_groups(s["table"], c["ps"])
    y = rope.rotary_embed(s["q"], s["k"], s["inv"], positions=s["pos"], cu_seqlens=s["cu"],
                          interleaved=c["inter"], scale=c["scale"], norm_q=s["wq"],
                          norm_k=s["wk"], eps=_EPS)
    if kind == "rotary":
        return y
    leaves = [s[n] for n in ("q", "k", "wq", "wk") if s[n] is not None]
    grads = torch.autograd.grad(y, leaves, (s["dyq"], s["dyk"]))
    return (*(t.detach() for t in y), *grads, *([None] * (4 - len(grads))))


# -- the same in 64 bits ------------------------------------------------------

def _exact_shared(s, case):
    H, HKV, HG, D, ps = (case[x] for x in ("H", "HKV", "HG", "D", "ps"))
    outs, t = [], 0
    for b, (_, p, own_rows, m) in enumerate(_seqs(case)):
        n = p + own_rows + m
        ids = s["table"][b, :-(-n // ps)].long()
        rows = lambda x: x[ids].transpose(0, 1).flatten(1, 2)[:, :n].double()   # [h, n, f]
        spread = lambda x: x.repeat_interleave(H // HKV, 0)
        x = torch.bmm(s["q"][t:t + m].double().transpose(0, 1),
                      spread(rows(s["k"])).transpose(1, 2).contiguous()) / math.sqrt(D)
        if HG:
            x[:HG] += s["gs"].double()[:, None, None] * torch.bmm(
                s["rq"][t:t + m].double().transpose(0, 1),
                rows(s["rk"]).transpose(1, 2).contiguous())
        dev = ids.device
        hidden = torch.arange(n, device=dev) > n - m + torch.arange(m, device=dev)[:, None]
        x.masked_fill_(hidden, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.bmm(e, spread(rows(s["v"]))) / (e.sum(-1, keepdim=True) + 1e-6)
        outs.append(o.transpose(0, 1))
        t += m
    return torch.cat(outs)


def _exact_rotary(s, case):
    rd, inter = case["rd"], case["inter"]
    if s["pos"] is not None:
        pos = s["pos"].double()
    else:
        cu = s["cu"].tolist()
        pos = torch.cat([torch.arange(b - a, device=s["cu"].device) for a, b in zip(cu, cu[1:])])
        pos = pos.double()
    ang = pos[:, None] * s["inv"].double()
    z = torch.polar(torch.full_like(ang, case["scale"]), ang)[:, None]

    def one(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
        r, rest = x[..., :rd], x[..., rd:]
        pair = r.unflatten(-1, (-1, 2)) if inter else r.unflatten(-1, (2, -1)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
        y = y.flatten(-2) if inter else y.transpose(-1, -2).flatten(-2)
        return torch.cat((y, rest), -1)

    train = case["kind"] == "rotary_train"
    leaf = lambda x: None if x is None else x.detach().double().requires_grad_(train)
    q, k, wq, wk = (leaf(s[n]) for n in ("q", "k", "wq", "wk"))
    y = one(q, wq), one(k, wk)
    if not train:
        return y
    leaves = [x for x in (q, k, wq, wk) if x is not None]
    grads = torch.autograd.grad(y, leaves, (s["dyq"].double(), s["dyk"].double()))
    return (*(t.detach() for t in y), *grads, *([None] * (4 - len(grads))))


def exact(case, seed):
    if case["kind"] in ("extend", "groups"):  # whole numbers: nothing is computed
        return None
    s = prepare(case, seed)
    return (_exact_shared if case["kind"] == "shared" else _exact_rotary)(s, case)
