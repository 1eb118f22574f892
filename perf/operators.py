"""Performance cases of the token-routed expert operators and of the products on 4-bit weights.

    route     ``F.expert_route``: the top-k experts of every token with their softmax weights; training adds the
              gradient of the scores
    exchange  ``F.expert_plan`` -> ``F.expert_dispatch`` -> ``F.expert_combine``: tokens into expert order and back, around
              experts whose outputs are given; training adds the gradients of tokens, expert outputs and weights
    experts   ``F.expert_linear``: rows in expert order times their expert's matrix; training adds both gradients
    codes     ``F.linear_4bit``: a few rows times a weight stored in 4 bits, dense or one weight per expert; training adds the
              gradient of the rows

``own`` false: the plain form, elementary torch operations in 32 bits, rounded once at the end. ``own`` true: the calls
of the framework.

Widths: 640 to 2560 are the hidden sizes of ``models/``, 5120 x 13824 is the feed-forward of the Wan 2.2 blocks; numbers of
experts and of experts per token are generic.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
BF16 = torch.bfloat16
NF4 = [-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635, -0.18477343022823334,
       -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
       0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0]


def listed():
    return [
        # One token of a sampler that runs at batch 1: a single row of scores, latency is all that counts.
        dict(name="route 1 token", op="route", tokens=1, experts=64, k=4, dtype="fp32", normalize=True, train=False),
        # The router of a training step: 16384 tokens, 64 experts, both directions.
        dict(name="route train", op="route", tokens=16384, experts=64, k=6, dtype="fp32", normalize=True, train=True),
        # Scores of an odd number of tokens and experts straight from a bf16 linear, weights not renormalised.
        dict(name="route bf16 odd", op="route", tokens=4099, experts=157, k=8, dtype="bf16", normalize=False, train=True),
        # Serving: a handful of tokens into expert order and back.
        dict(name="exchange 7 tokens", op="exchange", tokens=7, experts=32, k=2, dim=2560, padded=False, train=False),
        # A training step's tokens; every token is copied to six experts.
        dict(name="exchange train", op="exchange", tokens=8192, experts=64, k=6, dim=2560, padded=False, train=True),
        # One row for each of a few tokens: bound by reading the experts' weights once.
        dict(name="experts 16 rows", op="experts", rows=16, experts=16, n=5120, k=2560, empty=0, train=False),
        # A prompt's tokens through an up-projection, forward only.
        dict(name="experts prompt", op="experts", rows=8192, experts=16, n=4096, k=2048, empty=0, train=False),
        # A training step: output and both gradients; a third of the experts gets no row.
        dict(name="experts ragged train", op="experts", rows=999, experts=24, n=1336, k=712, empty=8, train=True),
        # The largest training step: many rows per expert, both gradients.
        dict(name="experts train", op="experts", rows=16384, experts=8, n=5120, k=2560, empty=0, train=True),
        # The modulation linear of a quantised model for one image: one row, NF4 codes.
        dict(name="nf4 modulation row", op="codes", rows=1, experts=0, n=15360, k=2560, kind="nf4", block=64, train=False),
        # A wide feed-forward weight in int4 for eight rows, with the gradient of the rows (a frozen base under adapters).
        dict(name="int4 8 rows train", op="codes", rows=8, experts=0, n=13824, k=5120, kind="int4", block=64, train=True),
        # A quantised expert bank that serves twelve routed rows.
        dict(name="nf4 experts 12 rows", op="codes", rows=12, experts=16, n=5120, k=2560, kind="nf4", block=64, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _step(rng, lo, hi, step):
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["route", "exchange", "experts", "experts", "codes", "codes"])
    if op == "route":
        e = _log(rng, 3, 400)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=e, k=rng.randint(1, min(8, e)), dtype=rng.choice(["fp32", "bf16"]),
                    normalize=rng.random() < 0.6, train=rng.random() < 0.6)
    if op == "exchange":
        e = _log(rng, 4, 256)
        k = rng.randint(1, min(8, e))
        d = _step(rng, 64, 4096, 8)
        most = 8192 * 6 * 2560 // (k * d)
        return dict(op=op, tokens=_log(rng, 1, max(2, min(16384, most))), experts=e, k=k, dim=d, padded=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    if op == "experts":
        e = _log(rng, 1, 64)
        n, k = _step(rng, 64, 5120, 8), _step(rng, 64, 5120, 8)
        while e * n * k > 16 * 5120 * 2560:
            e = max(1, e // 2)
        most = max(2, min(16384, 16384 * 5120 * 2560 // (n * k)))
        return dict(op=op, rows=_log(rng, 1, most), experts=e, n=n, k=k, empty=rng.randint(0, e // 2), train=rng.random() < 0.6)
    block = rng.choice([32, 64, 64, 128])
    e = rng.choice([0, 0, _log(rng, 2, 16)])
    n, k = _log(rng, 64, 13824) // 2 * 2, _step(rng, 256, 5120, block)
    while max(1, e) * n * k > 16 * 5120 * 2560:
        e //= 2
    return dict(op=op, rows=rng.randint(1, 16 if e else 8), experts=e, n=n, k=k, kind=rng.choice(["nf4", "int4"]), block=block,
                train=rng.random() < 0.4)


def work(case):
    c = case
    if c["op"] == "route":
        s = 4 if c["dtype"] == "fp32" else 2
        te, tk = c["tokens"] * c["experts"], c["tokens"] * c["k"]
        return {"bytes": te * s + tk * 12 + (te * s + tk * 4 if c["train"] else 0), "flops": te * (4 if c["train"] else 2)}
    if c["op"] == "exchange":
        td, tkd = c["tokens"] * c["dim"], c["tokens"] * c["k"] * c["dim"]
        b = 2 * (td + tkd) + 2 * (tkd + td)                       # x -> rows, rows -> out
        if c["train"]:
            b += 2 * (tkd + td) + 2 * (td + tkd)                  # gradient rows -> dx, dout -> gradient of the expert outputs
        return {"bytes": b + 20 * c["tokens"] * c["k"], "flops": (2 + (5 if c["train"] else 0)) * tkd}
    if c["op"] == "experts":
        rk, rn, w = c["rows"] * c["k"], c["rows"] * c["n"], (c["experts"] - c["empty"]) * c["n"] * c["k"]
        b = 2 * (rk + rn + w)
        if c["train"]:
            b += 2 * (rn + rk + w) + 2 * (c["empty"] * c["n"] * c["k"])        # dy in, dx and dw out
        return {"bytes": b, "flops": 2 * c["rows"] * c["n"] * c["k"] * (3 if c["train"] else 1)}
    e = max(1, min(c["experts"], c["rows"]))
    nk = c["n"] * c["k"]
    b = e * (nk // 2 + 4 * nk // c["block"]) + 2 * c["rows"] * (c["n"] + c["k"])
    return {"bytes": b + (2 * c["rows"] * (c["n"] + c["k"]) if c["train"] else 0),
            "flops": 2 * c["rows"] * nk * (2 if c["train"] else 1)}


# --------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _counts(case, gen, host):
    """Rows of each expert: shares that differ by small factors, as a router's do, some experts without a row."""
    e = case["experts"]
    p = torch.rand(e, generator=host) + 0.25
    p[torch.randperm(e, generator=host)[:case.get("empty", 0)]] = 0
    pick = torch.multinomial(p, case["rows"], replacement=True, generator=host)
    return torch.bincount(pick, minlength=e)


def _codes(case, gen):
    """Codes and scales of a normal weight: blocks of ``block`` values along k, each divided by its largest magnitude, two codes to
    a byte, the even element in the low half."""
    e, n, k, block = max(1, case["experts"]), case["n"], case["k"], case["block"]
    packed = torch.empty(e, n * k // block, block // 2, dtype=torch.uint8, device=DEV)
    scale = torch.empty(e, n * k // block, device=DEV)
    lv = torch.tensor(NF4, device=DEV)
    mid = (lv[1:] + lv[:-1]) / 2
    for i in range(e):
        w = torch.randn(n * k // block, block, generator=gen, device=DEV) / math.sqrt(k)
        s = w.abs().amax(1, keepdim=True)
        if case["kind"] == "nf4":
            q = torch.bucketize(w / s, mid).to(torch.uint8)
        else:
            q = (torch.round(w / s * 7.0) + 8).to(torch.uint8)
        packed[i] = q[:, 0::2] | (q[:, 1::2] << 4)
        scale[i] = s[:, 0]
    return packed.view(-1, block // 2), scale.view(-1)


def _offsets(counts):
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)


def prepare(case, seed):
    gen, host = _gen(seed), torch.Generator().manual_seed(seed)
    c = dict(case)
    st = {"case": c}

    def normal(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    if c["op"] == "route":
        st["scores"] = normal(c["tokens"], c["experts"], std=1.5, dtype=torch.float32 if c["dtype"] == "fp32" else BF16)
        st["dw"] = normal(c["tokens"], c["k"], dtype=torch.float32)
        if c["train"]:
            st["scores"].requires_grad_()
    elif c["op"] == "exchange":
        t, k = c["tokens"], c["k"]
        scores = torch.randn(t, c["experts"], generator=gen, device=DEV) + torch.randn(c["experts"], generator=gen, device=DEV)
        w, idx = torch.topk(scores.softmax(-1), k, dim=-1)
        if c["padded"]:                                          # the last tokens of a padded batch go to no expert
            idx[t - t // 5:] = -1
        st["idx"], st["w"] = idx.contiguous(), (w / w.sum(-1, keepdim=True)).contiguous()
        st["x"], st["y"] = normal(t, c["dim"]), normal(t * k, c["dim"])
        st["dxs"], st["dout"] = normal(t * k, c["dim"]), normal(t, c["dim"])
        if c["train"]:
            for name in ("x", "y", "w"):
                st[name].requires_grad_()
    elif c["op"] == "experts":
        counts = _counts(c, gen, host)
        st["counts"], st["offsets"] = counts.tolist(), _offsets(counts).to(DEV)
        st["x"], st["w"] = normal(c["rows"], c["k"]), normal(c["experts"], c["n"], c["k"], std=c["k"] ** -0.5)
        st["dy"] = normal(c["rows"], c["n"])
        if c["train"]:
            st["x"].requires_grad_()
            st["w"].requires_grad_()
    else:
        st["codes"], st["scale"] = _codes(c, gen)
        st["x"], st["dy"] = normal(c["rows"], c["k"]), normal(c["rows"], c["n"])
        if c["experts"]:
            counts = _counts(c, gen, host)
            st["counts"], st["offsets"] = counts.tolist(), _offsets(counts).to(DEV)
        if c["train"]:
            st["x"].requires_grad_()
        if own:
            from eridiffusion_b200.memory import QuantizedTensor
            shape = (c["experts"], c["n"], c["k"]) if c["experts"] else (c["n"], c["k"])
            st["q"] = QuantizedTensor(c["kind"], st["codes"], st["scale"], shape, c["block"])
    return st


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(st):
    from eridiffusion_b200.ops import functional as F
    c = st["case"]
    grad = torch.autograd.grad
    with torch.set_grad_enabled(c["train"]):
        if c["op"] == "route":
            idx, w = F.expert_route(st["scores"], c["k"], normalize=c["normalize"])
            return (idx, w, *grad(w, st["scores"], st["dw"])) if c["train"] else (idx, w)
        if c["op"] == "exchange":
            plan = F.expert_plan(st["idx"], c["experts"])
            xs = F.expert_dispatch(st["x"], plan)
            out = F.expert_combine(st["y"], st["w"], plan)
            res = (plan.offsets, plan.rows, xs, out)
            if c["train"]:
                res += grad((xs, out), (st["x"], st["y"], st["w"]), (st["dxs"], st["dout"]))
            return res
        if c["op"] == "experts":
            y = F.expert_linear(st["x"], st["w"], st["offsets"])
            return (y, *grad(y, (st["x"], st["w"]), st["dy"])) if c["train"] else y
        y = F.linear_4bit(st["x"], st["q"], st.get("offsets"))
        return (y, *grad(y, st["x"], st["dy"])) if c["train"] else y


def _plain(st):
    c = st["case"]
    with torch.no_grad():
        return {"route": _plain_route, "exchange": _plain_exchange, "experts": _plain_experts, "codes": _plain_codes}[c["op"]](st, c)


def _plain_route(st, c):
    s = st["scores"].float()
    top, idx = torch.sort(s, dim=-1, descending=True, stable=True)
    top, idx = top[:, :c["k"]], idx[:, :c["k"]]
    if c["normalize"]:
        z = torch.exp(top - top[:, :1])
        w = z / z.sum(-1, keepdim=True)
    else:
        z = torch.exp(s - top[:, :1])
        p = z / z.sum(-1, keepdim=True)
        w = p.gather(1, idx)
    if not c["train"]:
        return idx.contiguous(), w
    dot = (w * st["dw"]).sum(-1, keepdim=True)
    if c["normalize"]:
        ds = torch.zeros_like(s).scatter_(1, idx, w * (st["dw"] - dot))
    else:
        ds = p * (torch.zeros_like(s).scatter_(1, idx, st["dw"]) - dot)
    return idx.contiguous(), w, ds.to(st["scores"].dtype)


def _plain_exchange(st, c):
    t, k, e = c["tokens"], c["k"], c["experts"]
    flat = st["idx"].reshape(-1)
    order = torch.sort(torch.where(flat < 0, e, flat), stable=True).indices
    counts = (flat[:, None] == torch.arange(e, device=DEV)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(t * k, device=DEV)
    rows = torch.where(flat < 0, -1, rows).to(torch.int32).view(t, k)
    live = (torch.arange(t * k, device=DEV) < offsets[-1])[:, None]
    here = (rows >= 0)[..., None]
    at = rows.clamp_min(0).long()
    xs = torch.where(live, st["x"][order // k], 0)
    yt = torch.where(here, st["y"][at].float(), 0.0)                                      # [t, k, d]
    out = (st["w"][..., None] * yt).sum(1).to(BF16)
    if not c["train"]:
        return offsets, rows, xs, out
    dx = torch.where(here, st["dxs"][at].float(), 0.0).sum(1).to(BF16)
    do = st["dout"].float()
    dw = (yt * do[:, None]).sum(-1)
    dy = torch.where(live, (st["w"].reshape(-1)[order][:, None] * do[order // k]), 0.0).to(BF16)
    return offsets, rows, xs, out, dx, dy, dw


def _plain_experts(st, c):
    x, w, dy = st["x"].float(), st["w"], st["dy"].float()
    y = torch.empty(c["rows"], c["n"], dtype=BF16, device=DEV)
    dx, dw = torch.empty_like(st["x"]), (torch.empty_like(w) if c["train"] else None)
    lo = 0
    for e, n in enumerate(st["counts"]):
        hi = lo + n
        we = w[e].float()
        y[lo:hi] = x[lo:hi] @ we.t()
        if c["train"]:
            dx[lo:hi] = dy[lo:hi] @ we
            dw[e] = dy[lo:hi].t() @ x[lo:hi]
        lo = hi
    return (y, dx, dw) if c["train"] else y


def _plain_codes(st, c):
    low, high = (st["codes"] & 15).int(), (st["codes"] >> 4).int()
    q = torch.stack([low, high], dim=-1).flatten(1)
    v = torch.tensor(NF4, device=DEV)[q] if c["kind"] == "nf4" else (q.float() - 8.0) / 7.0
    w = (v * st["scale"][:, None]).view(max(1, c["experts"]), c["n"], c["k"])
    x, dy = st["x"].float(), st["dy"].float()
    y, dx = torch.empty_like(dy), torch.empty_like(x)
    lo = 0
    for e, n in enumerate(st.get("counts", [c["rows"]])):
        hi = lo + n
        if n:
            y[lo:hi] = x[lo:hi] @ w[e].t()
            dx[lo:hi] = dy[lo:hi] @ w[e]
        lo = hi
    return (y.to(BF16), dx.to(BF16)) if c["train"] else y.to(BF16)


# ------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    c, st = case, prepare(case, seed)
    with torch.no_grad():
        if c["op"] == "route":
            return _exact_route(st, c)
        if c["op"] == "exchange":
            return _exact_exchange(st, c)
        rows, e = c["rows"], max(1, c["experts"])
        if "counts" in st:
            of = torch.repeat_interleave(torch.arange(e), torch.tensor(st["counts"])).to(DEV)
        else:
            of = torch.zeros(rows, dtype=torch.int64, device=DEV)
        x, dy = st["x"].double(), st["dy"].double()
        y, dx = torch.zeros(rows, c["n"], dtype=torch.float64, device=DEV), torch.zeros_like(x)
        dw = []
        for i in range(e):
            if c["op"] == "experts":
                w = st["w"][i].double()
            else:
                per = c["n"] * c["k"] // c["block"]
                b = st["codes"][i * per:(i + 1) * per].long()
                q = torch.empty(per, c["block"], dtype=torch.int64, device=DEV)
                q[:, 0::2], q[:, 1::2] = b % 16, b // 16
                if c["kind"] == "nf4":
                    v = torch.tensor(NF4, dtype=torch.float32, device=DEV).double()[q]
                else:
                    v = (q - 8).double() / 7
                w = (v * st["scale"][i * per:(i + 1) * per, None].double()).view(c["n"], c["k"])
            mine = (of == i).nonzero()[:, 0]
            y[mine] = torch.einsum("rk,nk->rn", x[mine], w)
            if c["train"]:
                dx[mine] = torch.einsum("rn,nk->rk", dy[mine], w)
                if c["op"] == "experts":
                    dw.append(torch.einsum("rn,rk->nk", dy[mine], x[mine]))
        if not c["train"]:
            return y
        return (y, dx, torch.stack(dw)) if c["op"] == "experts" else (y, dx)


def _exact_route(st, c):
    s = st["scores"].double()
    e = c["experts"]
    left, picks = s.clone(), []
    for _ in range(c["k"]):                                         # the largest that is left, the first of equals
        best = left.amax(1, keepdim=True)
        i = torch.where(left == best, torch.arange(e, device=DEV), e).amin(1)
        picks.append(i)
        left[torch.arange(len(s), device=DEV), i] = -math.inf
    idx = torch.stack(picks, 1)
    chosen = torch.zeros_like(s, dtype=torch.bool).scatter_(1, idx, True)
    base = torch.logsumexp(torch.where(chosen, s, -math.inf) if c["normalize"] else s, 1, keepdim=True)
    p = torch.exp(s - base)
    w = p.gather(1, idx)
    if not c["train"]:
        return idx, w
    g = torch.zeros_like(s).scatter_(1, idx, st["dw"].double())
    dot = (p * g).sum(1, keepdim=True)
    ds = p * (g - dot)
    return idx, w, torch.where(chosen, ds, 0.0) if c["normalize"] else ds


def _exact_exchange(st, c):
    t, k, e = c["tokens"], c["k"], c["experts"]
    flat = st["idx"].reshape(-1).cpu()
    lists = [(flat == i).nonzero()[:, 0] for i in range(e)]
    order = torch.cat(lists)
    offsets = torch.tensor([0] + [len(v) for v in lists]).cumsum(0).to(torch.int32)
    rows = torch.full((t * k,), -1, dtype=torch.int32)
    rows[order] = torch.arange(len(order), dtype=torch.int32)
    order, n = order.to(DEV), len(order)
    token = order // k
    d = c["dim"]
    xs = torch.zeros(t * k, d, dtype=torch.float64, device=DEV)
    xs[:n] = st["x"].double()[token]
    w = st["w"].double().reshape(-1)[order][:, None]
    y = st["y"].double()[:n]
    out = torch.zeros(t, d, dtype=torch.float64, device=DEV).index_add_(0, token, w * y)
    res = (offsets.to(DEV), rows.view(t, k).to(DEV), xs, out)
    if not c["train"]:
        return res
    do = st["dout"].double()[token]
    dx = torch.zeros(t, d, dtype=torch.float64, device=DEV).index_add_(0, token, st["dxs"].double()[:n])
    dy = torch.zeros(t * k, d, dtype=torch.float64, device=DEV)
    dy[:n] = w * do
    dw = torch.zeros(t * k, dtype=torch.float64, device=DEV)
    dw[order] = (y * do).sum(1)
    return res + (dx, dy, dw.view(t, k))
