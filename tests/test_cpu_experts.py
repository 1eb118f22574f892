"""Token-routed experts and 4-bit products on the CPU path, and what they refuse."""
import pytest
import torch

from eridiffusion_b200.memory import quantize
from eridiffusion_b200.ops import functional as F


def _moe(x, scores, w1, w2, k):
    """Each token through its experts, one at a time."""
    p = torch.softmax(scores.double(), -1)
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64)
    for t in range(x.shape[0]):
        top = sorted(range(p.shape[1]), key=lambda e: (-p[t, e].item(), e))[:k]
        total = sum(p[t, e] for e in top)
        for e in top:
            out[t] += p[t, e] / total * (w2[e].double() @ torch.relu(w1[e].double() @ x[t].double()))
    return out


def test_a_routed_feed_forward():
    g = torch.Generator().manual_seed(0)
    x, scores = torch.randn(13, 24, generator=g), torch.randn(13, 6, generator=g)
    w1, w2 = torch.randn(6, 16, 24, generator=g) * 0.2, torch.randn(6, 24, 16, generator=g) * 0.2
    idx, w = F.expert_route(scores, 2)
    plan = F.expert_plan(idx, 6)
    h = torch.relu(F.expert_linear(F.expert_dispatch(x, plan), w1, plan.offsets))
    out = F.expert_combine(F.expert_linear(h, w2, plan.offsets), w, plan)
    assert torch.allclose(out.double(), _moe(x, scores, w1, w2, 2), atol=1e-5)


def test_plan_order_and_choices_outside_the_experts():
    plan = F.expert_plan(torch.tensor([[2, 0], [-1, 2], [0, 7], [1, 2]]), 3)
    assert plan.offsets.tolist() == [0, 2, 3, 6]
    assert plan.rows.tolist() == [[3, 0], [-1, 4], [1, -1], [2, 5]]
    x = torch.arange(4.0)[:, None].expand(4, 8)
    assert F.expert_dispatch(x, plan)[:, 0].tolist() == [0, 2, 3, 0, 1, 3, 0, 0]


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    idx = torch.tensor([[1, 0], [2, -1], [1, 2]])
    plan = F.expert_plan(idx, 3)
    x, y, w = (torch.randn(*s, generator=g, requires_grad=True) for s in ((3, 8), (6, 8), (3, 2)))
    bank = torch.randn(3, 5, 8, generator=g, requires_grad=True)
    scores = torch.randn(3, 4, generator=g, requires_grad=True)
    funcs = [(lambda a: F.expert_dispatch(a, plan), (x,)), (lambda a, b: F.expert_combine(a, b, plan), (y, w)),
             (lambda a, b: F.expert_linear(a, b, plan.offsets), (y, bank)), (lambda a: F.expert_route(a, 2)[1], (scores,)),
             (lambda a: F.expert_route(a, 2, normalize=False)[1], (scores,))]
    for f, args in funcs:
        out = f(*args)
        d = torch.randn(out.shape, generator=g)
        for i, (a, da) in enumerate(zip(args, torch.autograd.grad(out, args, d))):
            h = torch.randn(a.shape, generator=g) * 1e-2
            hi, lo = (f(*(b + s * h if j == i else b for j, b in enumerate(args))) for s in (1, -1))
            lhs, rhs = (d * (hi - lo)).sum().item() / 2, (da * h).sum().item()
            assert abs(lhs - rhs) < 2e-4 + 1e-2 * abs(rhs)


def test_rows_of_no_expert_are_zero_and_bounds_stay_inside():
    x, w = torch.ones(6, 8), torch.ones(2, 4, 8)
    y = F.expert_linear(x, w, torch.tensor([1, 3, 4]))
    assert y[:, 0].tolist() == [0, 8, 8, 8, 0, 0]
    # offsets that do not ascend or leave the rows: no row is taken twice, none outside
    assert F.expert_linear(x, w, torch.tensor([-5, 99, 2]))[:, 0].tolist() == [8] * 6


def test_codes_on_the_cpu():
    g = torch.Generator().manual_seed(2)
    w = torch.randn(3, 16, 64, generator=g)
    for kind in ("int4", "nf4"):
        q = quantize(w, kind)
        x = torch.randn(5, 64, generator=g)
        y = F.linear_4bit(x, q, torch.tensor([0, 2, 2, 5]))
        full = q.dequantize(torch.float32)
        assert torch.allclose(y[:2], x[:2] @ full[0].t(), atol=1e-5) and torch.allclose(y[2:], x[2:] @ full[2].t(), atol=1e-5)
        d = quantize(w[0], kind)
        assert torch.allclose(F.linear_4bit(x[None], d, bias=torch.ones(16)), (x @ d.dequantize(torch.float32).t() + 1)[None], atol=1e-5)


@pytest.mark.parametrize("call", [
    lambda: F.expert_route(torch.zeros(4), 1), lambda: F.expert_route(torch.zeros(2, 4), 0), lambda: F.expert_route(torch.zeros(2, 4), 5),
    lambda: F.expert_route(torch.zeros(2, 4, dtype=torch.int32), 1), lambda: F.expert_route(torch.zeros(2, 4), 1, allowed=torch.ones(4)),
    lambda: F.expert_route(torch.zeros(2, 4), 1, allowed=torch.ones(3, dtype=torch.bool)),
    lambda: F.expert_plan(torch.zeros(4, dtype=torch.int64), 2), lambda: F.expert_plan(torch.zeros(4, 1), 2),
    lambda: F.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 0), lambda: F.expert_plan(torch.zeros(4, 0, dtype=torch.int64), 3),
    lambda: F.expert_dispatch(torch.zeros(3, 8), F.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 2)),
    lambda: F.expert_combine(torch.zeros(4, 8), torch.zeros(4, 2), F.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 2)),
    lambda: F.expert_combine(torch.zeros(5, 8), torch.zeros(4, 1), F.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 2)),
    lambda: F.expert_linear(torch.zeros(4, 8), torch.zeros(2, 4, 9), torch.zeros(3, dtype=torch.int32)),
    lambda: F.expert_linear(torch.zeros(4, 8), torch.zeros(2, 4, 8), torch.zeros(2, dtype=torch.int32)),
    lambda: F.expert_linear(torch.zeros(4, 8), torch.zeros(2, 4, 8), torch.zeros(3)),
    lambda: F.expert_linear(torch.zeros(4, 8), torch.zeros(2, 4, 8, dtype=torch.float64), torch.zeros(3, dtype=torch.int32)),
    lambda: F.linear_4bit(torch.zeros(4, 64), quantize(torch.ones(8, 64), "int8")),
    lambda: F.linear_4bit(torch.zeros(4, 64), quantize(torch.ones(2, 8, 64), "int4")),
    lambda: F.linear_4bit(torch.zeros(4, 64), quantize(torch.ones(8, 64), "int4"), torch.zeros(2, dtype=torch.int32)),
    lambda: F.linear_4bit(torch.zeros(4, 32), quantize(torch.ones(8, 64), "int4")),
    lambda: F.linear_4bit(torch.zeros(4, 64), quantize(torch.ones(8, 64), "int4"), bias=torch.zeros(4)),
    lambda: F.linear_4bit(torch.zeros(4, 64), quantize(torch.ones(2, 8, 64), "int4"), torch.zeros(3, dtype=torch.int32), torch.zeros(8)),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()
