"""A plan's rows outside [0, T * k) are nobody's: neither copied nor added, in either direction."""
import torch

from eridiffusion_b200.ops import functional as F


def test_rows_outside_are_nobodys():
    idx = torch.tensor([[0, 1], [1, 0], [2, 2]])
    plan = F.expert_plan(idx, 3)
    bad = plan._replace(rows=plan.rows.clone())
    bad.rows[0, 1], bad.rows[1, 0], bad.rows[2, 1] = 6, 2 ** 31 - 1, -7
    good = plan._replace(rows=torch.where(bad.rows < 6, bad.rows, -1).clamp_min(-1))
    x, y, w = (torch.randn(*s, dtype=torch.float64).float() for s in ((3, 8), (6, 8), (3, 2)))
    for p in (bad, good):
        x.requires_grad_(), y.requires_grad_(), w.requires_grad_()
    a, b = [(F.expert_dispatch(x, p), F.expert_combine(y, w, p)) for p in (bad, good)]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for i, leaves in ((0, (x,)), (1, (y, w))):
        for p, q in zip(torch.autograd.grad(a[i].square().sum(), leaves), torch.autograd.grad(b[i].square().sum(), leaves)):
            assert torch.equal(p, q)
