"""Token-routed feed-forward on the GPU: the expert bank's path against the product expert by expert, the run of the operators together
with gradients, two streams at once, capture."""
import pytest
import torch

from eridiffusion_b200.memory import QuantizedLinear, quantize
from eridiffusion_b200.models.layers import Linear
from eridiffusion_b200.models.moe import ExpertBank, moe_linear, route_tokens, select_topk_global
from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _moe64(x, scores, weights, k, allowed=None):
    s = scores.double()
    if allowed is not None:
        mask = torch.full_like(s, float("-inf"))
        mask[:, list(allowed)] = 0
        s = s + mask
    top, idx = torch.sort(s, dim=-1, descending=True, stable=True)
    w = torch.softmax(top[:, :k], -1)
    out, mag = 0, 0
    for j in range(k):
        for e, we in weights.items():
            hit = (idx[:, j] == e).double()[:, None] * w[:, j:j + 1]
            y = x.double() @ we.double().t()
            out, mag = out + hit * y, mag + hit * (y.abs() + x.double().abs() @ we.double().abs().t() * x.shape[1] * 2.0 ** -23)
    return out, mag


@pytest.mark.parametrize("kind", ["none", "q8", "nf4"])
@pytest.mark.parametrize("T,E,N,K,k", [(1, 8, 256, 512, 2), (7, 5, 136, 192, 2), (333, 8, 264, 256, 3)])
@pytest.mark.parametrize("resident,missing", [(None, ()), (3, ()), (None, (1, 4))])
def test_bank(T, E, N, K, k, resident, missing, kind):
    g = torch.Generator(device="cuda").manual_seed(T + N)
    bank, weights = ExpertBank(kind), {}
    for e in range(E):
        if e not in missing:
            bank.insert(e, _mk(g, N, K, std=0.05))
            weights[e] = bank.experts[e].dequantize(torch.float32) if kind != "none" else bank.experts[e]
    x, scores = _mk(g, T, K), torch.randn(T, E, device="cuda", generator=g)
    allowed = select_topk_global(scores, resident) if resident else None
    ref, mag = _moe64(x, scores, weights, k, allowed)
    # expert outputs and the sum are rounded to bf16 (2^-8 each); expanded weights, too; the levels of few rows to 2^-11
    for _ in range(2):                                   # the second call finds the bank stacked
        y = moe_linear(x, scores, bank, k=k, resident=resident)
        spread = sum((x.double().abs() @ w.double().abs().t()) for w in weights.values()) * (2.0 ** -8 if kind != "none" else 0.0)
        assert y.dtype == BF and ((y.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * 2 ** -8 * 1.01 + spread + 1e-30).all()
    assert len(bank) == E - len(missing) and {i for i, _ in bank.fetch_topk_bf16(range(E))} == set(weights)


@pytest.mark.parametrize("kind", ["q8", "nf4"])
def test_expanded_a_few_at_a_time(kind, monkeypatch):
    from eridiffusion_b200.models import moe
    g = torch.Generator(device="cuda").manual_seed(3)
    bank = ExpertBank(kind)
    for e in range(7):
        bank.insert(e, _mk(g, 128, 256, std=0.05))
    x, scores = _mk(g, 200, 256), torch.randn(200, 7, device="cuda", generator=g)
    whole = moe_linear(x, scores, bank, k=2)
    monkeypatch.setattr(moe, "_EXPANDED_BYTES", 3 * 2 * 128 * 256)
    assert torch.equal(moe_linear(x, scores, bank, k=2), whole)          # three at a time: the same sums
    monkeypatch.undo()
    assert all(b.data.untyped_storage().nbytes() == b.data.numel() for b in bank.experts.values() if kind == "nf4")     # nothing was stacked


def test_bank_with_changing_residents_is_stacked_once():
    g = torch.Generator(device="cuda").manual_seed(5)
    bank = ExpertBank("none")
    for e in range(6):
        bank.insert(e, _mk(g, 64, 128))
    x = _mk(g, 30, 128)
    moe_linear(x, torch.randn(30, 6, device="cuda", generator=g), bank, k=2, resident=2)
    held = bank._stack[2]
    for _ in range(3):
        moe_linear(x, torch.randn(30, 6, device="cuda", generator=g), bank, k=2, resident=3)
        assert bank._stack[2] is held and all(e.untyped_storage().data_ptr() == held.untyped_storage().data_ptr() for e in bank.experts.values())


def test_bank_follows_a_replaced_expert():
    g = torch.Generator(device="cuda").manual_seed(1)
    bank = ExpertBank("none")
    for e in range(3):
        bank.insert(e, _mk(g, 64, 128))
    x, scores = _mk(g, 20, 128), torch.tensor([[0.0, 5.0, 0.0]], device="cuda").expand(20, 3)
    moe_linear(x, scores, bank, k=1)
    new = _mk(g, 64, 128)
    bank.insert(1, new)
    y = moe_linear(x, scores, bank, k=1)
    ref = x.double() @ new.double().t()
    assert ((y.double() - ref).abs() <= ref.abs() * 2 ** -7 + 1e-3).all()


def test_routes_agree_with_the_cpu_path():
    g = torch.Generator(device="cuda").manual_seed(2)
    s = torch.randn(50, 9, device="cuda", generator=g)
    for allowed in (None, [1, 2, 7]):
        i, w = route_tokens(s, 3, allowed)
        ic, wc = route_tokens(s.cpu(), 3, allowed)
        assert torch.equal(i.cpu(), ic) and torch.allclose(w.cpu(), wc, atol=1e-6) and i.dtype == ic.dtype


def _feed_forward(x, scores, w1, w2, k):
    idx, w = F.expert_route(scores, k)
    plan = F.expert_plan(idx, w1.shape[0])
    h = F.glu(F.expert_linear(F.expert_dispatch(x, plan), w1, plan.offsets), "silu", act_first=True)
    return F.expert_combine(F.expert_linear(h, w2, plan.offsets), w, plan)


def _feed_forward_ref(x, scores, w1, w2, k):
    """The same with PyTorch statements on the given types."""
    idx, w = F.R.expert_route(scores, k)
    off, rows = F.R.expert_plan(idx, w1.shape[0])
    h = F.R.glu(F.R.expert_linear(F.R.expert_dispatch(x, rows), w1, off), "silu", act_first=True)
    return F.R.expert_combine(F.R.expert_linear(h, w2, off), w, rows)


@pytest.mark.parametrize("T,E,D,H,k", [(5, 4, 128, 192, 2), (400, 8, 256, 384, 3)])
def test_feed_forward_and_gradients(T, E, D, H, k):
    g = torch.Generator(device="cuda").manual_seed(T)
    x, scores = _mk(g, T, D).requires_grad_(), torch.randn(T, E, device="cuda", generator=g).requires_grad_()
    w1, w2 = _mk(g, E, 2 * H, D, std=D ** -0.5).requires_grad_(), _mk(g, E, D, H, std=H ** -0.5).requires_grad_()
    dy = _mk(g, T, D)
    out = _feed_forward(x, scores, w1, w2, k)
    grads = torch.autograd.grad(out, (x, scores, w1, w2), dy)
    wide = [t.detach().float().requires_grad_() for t in (x, scores, w1, w2)]
    ref = _feed_forward_ref(*wide, k)
    rgrads = torch.autograd.grad(ref, wide, dy.float())
    # bf16 roundings of 2^-9 rms each lie in a row: rows into the gate (1), gate (2), second product (3), sum (4); backwards as many again
    for a, b, steps in ((out, ref, 4), *((p, q, 8) for p, q in zip(grads, rgrads))):
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() < steps * 2 ** -8
    assert F.kernel_error_check() == {}


def test_feed_forward_in_a_graph_next_to_an_eager_one():
    """The captured run owns its leaves; an eager run of other leaves lives while it is captured and replayed."""
    g = torch.Generator(device="cuda").manual_seed(7)
    T, E, D, H, k = 96, 6, 128, 128, 2
    x, w1, w2, dy = _mk(g, T, D), _mk(g, E, 2 * H, D, std=0.08), _mk(g, E, D, H, std=0.08), _mk(g, T, D)
    scores = torch.randn(T, E, device="cuda", generator=g)
    eager_leaves = [t.clone().requires_grad_() for t in (x, scores, w1, w2)]
    eager = _feed_forward(*eager_leaves, k)
    leaves = [t.clone().requires_grad_() for t in (x, scores, w1, w2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_feed_forward(*leaves, k), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _feed_forward(*leaves, k)
        grads = torch.autograd.grad(out, leaves, dy)
    for seed in range(3):
        gg = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            leaves[1].copy_(torch.randn(T, E, device="cuda", generator=gg))
            eager_leaves[1].copy_(leaves[1])
        graph.replay()
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        o = _feed_forward(*fresh, k)
        assert torch.equal(out, o) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(o, fresh, dy)))
    del eager


def test_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(9)
    sets = []
    for i in range(2):
        sets.append((_mk(g, 300 + i, 256), torch.randn(300 + i, 8, device="cuda", generator=g), _mk(g, 8, 512, 256, std=0.06),
                     _mk(g, 8, 256, 256, std=0.06)))
    ref = [_feed_forward(*s, 2) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [[] for _ in sets]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(_feed_forward(*sets[i], 2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for os, r in zip(outs, ref) for o in os)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
@pytest.mark.parametrize("act,extra", [(None, False), ("gelu", False), ("silu", True)])
def test_quantised_layer_on_few_rows(kind, act, extra):
    g = torch.Generator(device="cuda").manual_seed(4)
    lin = Linear(256, 320, dtype=BF, device="cuda")
    with torch.no_grad():
        lin.weight.copy_(_mk(g, 320, 256, std=0.06))
        lin.bias.copy_(_mk(g, 320))
    q = QuantizedLinear(lin, kind)
    x = _mk(g, 2, 3, 256)
    res, gate = (_mk(g, 2, 3, 320), _mk(g, 2, 320)) if extra else (None, None)
    assert F.on_codes(x, q.q) and not F.on_codes(_mk(g, 9, 256), q.q)
    y = q(x, act=act, residual=res, gate=gate)
    lv = x.double() @ q.q.dequantize(torch.float32).double().t() + lin.bias.detach().double()
    err = lv.abs() * 2 ** -8 + (x.double().abs() @ q.q.dequantize(torch.float32).double().abs().t()) * 2 ** -10
    r, slope = lv, 1.0
    if act is not None:
        r = torch.nn.functional.gelu(lv, approximate="tanh") if act == "gelu" else torch.nn.functional.silu(lv)
        slope = 1.13                                    # largest slope of both
    err = err * slope + r.abs() * 2 ** -8
    if extra:
        err = err * gate.double().abs()[:, None]
        r = res.double() + gate.double()[:, None] * r
        err = err + r.abs() * 2 ** -8
    assert y.shape == r.shape and ((y.double() - r).abs() <= err * 1.01 + 1e-6).all()
