"""Gradients of gradients through the expert operators and the products on codes, against the PyTorch statements."""
import pytest
import torch

from eridiffusion_b200.memory import quantize
from eridiffusion_b200.models.moe import ExpertBank, moe_linear
from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _apart(g, T, E):
    return torch.stack([torch.randperm(E, device="cuda", generator=g) for _ in range(T)]).float() * 0.3


def _second(fn, leaves, dy, vs):
    """First gradients, and the gradients of their sum weighted by ``vs``, with respect to the leaves and dy."""
    first = torch.autograd.grad(fn(*leaves), leaves, dy, create_graph=True)
    z = sum((f.float() * v.float()).sum() for f, v in zip(first, vs))
    second = torch.autograd.grad(z, (*leaves, dy), allow_unused=True)
    return [f.detach() for f in first], second


def _compare(fn, ref, leaves, dy, g, tol):
    """``tol``: roundings to bf16 between the ends, 2^-8 each, as a share of the norm."""
    vs = [torch.randn(t.shape, device="cuda", generator=g).to(t.dtype) for t in leaves]
    ours = _second(fn, [t.detach().clone().requires_grad_() for t in leaves], dy.detach().clone().requires_grad_(), vs)
    wide = _second(ref, [t.detach().double().requires_grad_() for t in leaves], dy.detach().double().requires_grad_(), vs)
    for a, b in zip((*ours[0], *ours[1]), (*wide[0], *wide[1])):
        if b is None or b.count_nonzero() == 0:
            assert a is None or a.count_nonzero() == 0
        else:
            assert a.shape == b.shape and ((a.double() - b).norm() / b.norm()).item() < tol
    plain = [t.detach().clone().requires_grad_() for t in leaves]              # what the kernels give when nothing is recorded
    for a, b in zip(torch.autograd.grad(fn(*plain), plain, dy), ours[0]):
        assert ((a.double() - b.double()).norm() <= tol * b.double().norm() + 1e-30).item()


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_route(normalize, masked):
    g = torch.Generator(device="cuda").manual_seed(1)
    T, E, k = 9, 12, 3
    allowed = torch.rand(E, device="cuda", generator=g) < 0.7 if masked else None

    def ref(s):
        f = s if allowed is None else s.masked_fill(~allowed, float("-inf"))
        idx = torch.sort(f.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
        top = f.gather(1, idx)
        return torch.softmax(top, -1) if normalize else torch.softmax(f, -1).gather(1, idx)
    _compare(lambda s: F.expert_route(s, k, allowed, normalize)[1], ref, [_apart(g, T, E)], torch.randn(T, k, device="cuda", generator=g), g, 1e-5)


def test_route_of_rows_that_may_choose_nothing():
    s = torch.tensor([[0.0, 1.0, 2.0], [float("-inf")] * 3], device="cuda", requires_grad=True)
    for normalize in (True, False):
        w = F.expert_route(s, 2, normalize=normalize)[1]
        (ds,) = torch.autograd.grad(w, s, torch.tensor([[1.0, 2.0], [3.0, 4.0]], device="cuda"), create_graph=True)
        (dds,) = torch.autograd.grad(ds.square().sum(), s)
        assert ds.isfinite().all() and dds.isfinite().all() and ds[1].count_nonzero() == 0 and dds[1].count_nonzero() == 0


def _plan(g, T, k, E):
    idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(T)])
    idx[1, 0] = -1                                   # a choice of nobody
    return F.expert_plan(idx, E)


def test_dispatch_and_combine():
    g = torch.Generator(device="cuda").manual_seed(2)
    T, k, E, D = 11, 3, 5, 72
    plan = _plan(g, T, k, E)
    _compare(lambda x: F.expert_dispatch(x, plan).square(), lambda x: _dispatch64(x, plan.rows).square(), [_mk(g, T, D)], _mk(g, T * k, D), g, 4 * 2 ** -8)
    _compare(lambda y, w: F.expert_combine(y, w, plan), lambda y, w: _combine64(y, w, plan.rows),
             [_mk(g, T * k, D), torch.rand(T, k, device="cuda", generator=g)], _mk(g, T, D), g, 4 * 2 ** -8)


def _dispatch64(x, rows):
    here = (rows >= 0).flatten()
    token = torch.arange(rows.shape[0], device=x.device).repeat_interleave(rows.shape[1])[here]
    return torch.zeros(rows.numel(), x.shape[1], dtype=x.dtype, device=x.device).index_copy(0, rows.flatten()[here].long(), x[token])


def _combine64(y, w, rows):
    return (w[..., None] * torch.where((rows >= 0)[..., None], y[rows.clamp_min(0).long()], 0.0)).sum(1)


def _linear64(x, w, off):
    b = off.tolist()
    parts = [x[b[e]:b[e + 1]] @ w[e].t() for e in range(w.shape[0])]
    return torch.cat([x.new_zeros(b[0], w.shape[1]), *parts, x.new_zeros(x.shape[0] - b[-1], w.shape[1])])


@pytest.mark.parametrize("counts,N,K", [([3, 0, 5, 1], 40, 72), ([130, 1, 0, 70], 136, 264)])
def test_linear(counts, N, K):
    g = torch.Generator(device="cuda").manual_seed(N)
    R_ = sum(counts) + 2
    off = torch.tensor([1, *(1 + torch.tensor(counts).cumsum(0)).tolist()], dtype=torch.int32, device="cuda")
    _compare(lambda x, w: F.expert_linear(x, w, off), lambda x, w: _linear64(x, w, off),
             [_mk(g, R_, K), _mk(g, len(counts), N, K, std=K ** -0.5)], _mk(g, R_, N), g, 3 * 2 ** -8)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
@pytest.mark.parametrize("experts", [False, True])
def test_codes(kind, experts):
    g = torch.Generator(device="cuda").manual_seed(5)
    q = quantize(_mk(g, 3, 72, 128) if experts else _mk(g, 72, 128), kind)
    off = torch.tensor([0, 2, 2, 7], dtype=torch.int32, device="cuda") if experts else None
    w = q.dequantize(torch.float32).double()
    ref = (lambda x: _linear64(x, w, off).square()) if experts else (lambda x: (x @ w.t()).square())
    _compare(lambda x: F.linear_4bit(x, q, off).square(), ref, [_mk(g, 8, 128)], _mk(g, 8, 72), g, 8 * 2 ** -8)


def test_bias_of_codes():
    g = torch.Generator(device="cuda").manual_seed(6)
    q = quantize(_mk(g, 72, 128), "nf4")
    w = q.dequantize(torch.float32).double()
    _compare(lambda x, b: F.linear_4bit(x, q, bias=b).square(), lambda x, b: (x @ w.t() + b).square(), [_mk(g, 5, 128), _mk(g, 72)], _mk(g, 5, 72), g, 8 * 2 ** -8)


@pytest.mark.parametrize("kind", ["none", "q8", "nf4"])
@pytest.mark.parametrize("T", [5, 200])
def test_moe_linear(kind, T):
    g = torch.Generator(device="cuda").manual_seed(T)
    E, N, K, k = 6, 136, 192, 2
    bank = ExpertBank(kind)
    for e in range(E):
        bank.insert(e, _mk(g, N, K, std=0.07))
    ws = torch.stack([(bank.experts[e] if kind == "none" else bank.experts[e].dequantize(torch.float32)).double() for e in range(E)])
    scores = _apart(g, T, E)

    def ref(x, s):
        idx = torch.sort(s.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
        w = torch.softmax(s.gather(1, idx), -1)
        return (w[..., None] * torch.einsum("tjnk,tk->tjn", ws[idx], x)).sum(1)
    _compare(lambda x, s: moe_linear(x, s, bank, k), ref, [_mk(g, T, K), scores], _mk(g, T, N), g, 8 * 2 ** -8)


@pytest.mark.parametrize("trained", ["x", "w", "both"])
def test_only_what_a_gradient_needs_is_kept(trained):
    """A frozen weight keeps no tokens, a weight without gradient no expert outputs; the gradients are those of the full pass."""
    g = torch.Generator(device="cuda").manual_seed(8)
    T, k, E, D = 20, 2, 4, 64
    plan = _plan(g, T, k, E)
    x, w = _mk(g, T * k, D), _mk(g, E, 72, D, std=0.1)
    y, f = _mk(g, T * k, D), torch.rand(T, k, device="cuda", generator=g)
    dx, dout = _mk(g, T * k, 72), _mk(g, T, D)
    full = [t.clone().requires_grad_() for t in (x, w, y, f)]
    want = [*torch.autograd.grad(F.expert_linear(full[0], full[1], plan.offsets), full[:2], dx),
            *torch.autograd.grad(F.expert_combine(full[2], full[3], plan), full[2:], dout)]
    pick = {"x": (0,), "w": (1,), "both": (0, 1)}[trained]
    for i in pick:
        (x, w)[i].requires_grad_()
        (y, f)[i].requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t.data_ptr()), t)[1], lambda t: t):
        a, b = F.expert_linear(x, w, plan.offsets), F.expert_combine(y, f, plan)
    assert (x.data_ptr() in kept) == (1 in pick) and (y.data_ptr() in kept) == (1 in pick)
    got = [*torch.autograd.grad(a, [(x, w)[i] for i in pick], dx), *torch.autograd.grad(b, [(y, f)[i] for i in pick], dout)]
    assert all(torch.equal(p, q) for p, q in zip(got, [want[i] for i in pick] + [want[2 + i] for i in pick]))


def test_rows_outside_a_plan_are_nobodys():
    """The kernels and the recorded backward pass leave them out alike."""
    g = torch.Generator(device="cuda").manual_seed(9)
    plan = F.expert_plan(torch.tensor([[0, 1], [1, 0], [2, 2]], device="cuda"), 3)
    bad = plan._replace(rows=plan.rows.clone())
    bad.rows[0, 1], bad.rows[1, 0], bad.rows[2, 1] = 6, 2 ** 31 - 1, -7
    good = plan._replace(rows=torch.where(bad.rows < 6, bad.rows, -1).clamp_min(-1))
    y, w, x = _mk(g, 6, 64), torch.rand(3, 2, device="cuda", generator=g), _mk(g, 3, 64)
    dy, dx = _mk(g, 3, 64), _mk(g, 6, 64)
    for create in (False, True):
        got = []
        for p in (bad, good):
            ys, ws, xs = (t.clone().requires_grad_() for t in (y, w, x))
            out, rows = F.expert_combine(ys, ws, p), F.expert_dispatch(xs, p)
            here = (p.rows >= 0) & (p.rows < 6)
            a = torch.autograd.grad(out, (ys, ws), dy, create_graph=create)
            # a row of nobody is not written: compare the others
            used = torch.zeros(6, dtype=torch.bool, device="cuda").index_fill(0, p.rows[here].long(), True)
            got.append((out.detach(), a[0].detach()[used], a[1].detach(), rows.detach()[used], torch.autograd.grad(rows, xs, dx, create_graph=create)[0].detach()))
        assert all(torch.equal(p, q) for p, q in zip(*got))
