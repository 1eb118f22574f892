"""Offsets that do not ascend or leave the rows: every operator gives a row to the same expert, that of their running maximum inside
[0, rows], in both directions."""
import pytest
import torch

from eridiffusion_b200.memory import quantize
from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
CASES = {"falls": ([0, 12, 4, 16], 16), "starts late": ([3, 1, 9, 2], 16), "behind the rows": ([0, 40, 5, 50], 16), "below zero": ([-7, -1, 6, 5], 16),
         "all fall": ([16, 8, 4, 0], 16), "past a warp": ([0] * 30 + [9, 3, 5, 11, 2, 14, 0, 64, 1], 16), "one row": ([5, -5, 1, 0], 1)}


def _owners(off, rows):
    out, top = [-1] * rows, 0
    bounds = []
    for o in off:
        top = max(top, min(max(o, 0), rows))
        bounds.append(top)
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        out[a:b] = [e] * (b - a)
    return out


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _check(got, ref, mag, terms, share=0.0):
    """bf16 output (2^-8 of itself), sums in 32 bits, ``share``: what the operands were rounded by."""
    assert ((got.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * (terms * 2 ** -23 + share) + 1e-30).all()


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_same_rows_in_both_directions(name, dtype):
    off, rows = CASES[name]
    E, N, K = len(off) - 1, 88, 128
    own = _owners(off, rows)
    g = torch.Generator(device="cuda").manual_seed(rows + E)
    o = torch.tensor(off, dtype=dtype, device="cuda")
    x, dy, w = _mk(g, rows, K), _mk(g, rows, N), _mk(g, E, N, K, std=0.1)
    pick = torch.zeros(rows, E, dtype=torch.float64, device="cuda")
    for r, e in enumerate(own):
        if e >= 0:
            pick[r, e] = 1
    for kind in (None, "int4", "nf4"):
        q = None if kind is None else quantize(w, kind)
        wd = w.double() if q is None else q.dequantize(torch.float32).double()
        share = 0.0 if q is None else 2.0 ** -10          # levels and dy * scale in 11 bits each
        leaves = [x.clone().requires_grad_()] + ([w.clone().requires_grad_()] if q is None else [])
        y = F.expert_linear(*leaves, o) if q is None else F.linear_4bit(leaves[0], q, o)
        grads = torch.autograd.grad(y, leaves, dy)
        xd, dd = x.double(), dy.double()
        rows_w, rows_wa = torch.einsum("re,enk->rnk", pick, wd), torch.einsum("re,enk->rnk", pick, wd.abs())
        _check(y.detach(), torch.einsum("rnk,rk->rn", rows_w, xd), torch.einsum("rnk,rk->rn", rows_wa, xd.abs()), K, share)
        _check(grads[0], torch.einsum("rnk,rn->rk", rows_w, dd), torch.einsum("rnk,rn->rk", rows_wa, dd.abs()), N, share)
        if q is None:
            _check(grads[1], torch.einsum("re,rn,rk->enk", pick, dd, xd), torch.einsum("re,rn,rk->enk", pick, dd.abs(), xd.abs()), rows)
    assert F.kernel_error_check() == {}


def test_offsets_wider_than_32_bits():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = _mk(g, 10, 128), _mk(g, 2, 88, 128)
    q = quantize(w, "nf4")
    wide = torch.tensor([0, 4, 2 ** 32 + 1], device="cuda")              # the low 32 bits are 1
    near = torch.tensor([-2 ** 32 + 9, 4, 10], device="cuda")
    want = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    for off in (wide, near):
        assert torch.equal(F.expert_linear(x, w, off), F.expert_linear(x, w, want))
        assert torch.equal(F.linear_4bit(x, q, off), F.linear_4bit(x, q, want))
    assert torch.equal(F.R.expert_linear(x, w, wide), F.R.expert_linear(x, w, want))
