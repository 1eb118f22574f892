"""A 4-bit layer on few rows takes and gives what the same layer takes and gives on many."""
import pytest
import torch

from eridiffusion_b200.memory import QuantizedLinear
from eridiffusion_b200.models.layers import Linear
from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _layer(g, n, k, kind, dtype=BF):
    lin = Linear(k, n, dtype=dtype, device="cuda")
    with torch.no_grad():
        lin.weight.copy_(_mk(g, n, k, std=0.06))
        lin.bias.copy_(_mk(g, n))
    return QuantizedLinear(lin, kind)


@pytest.mark.parametrize("n", [320, 84])
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("gated,summed", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("lead", [(6,), (1,), (), (2, 3), (2, 1), (2, 1, 3), (2, 2, 2)])
def test_gate_and_residual_of_any_rank(lead, gated, summed, act, n):
    g = torch.Generator(device="cuda").manual_seed(n + len(lead))
    q = _layer(g, n, 256, "nf4")
    x = _mk(g, *lead, 256)
    tokens = lead[-1] if lead else 1
    batch = max(1, x.numel() // 256 // tokens)
    res, gate = _mk(g, *lead, n) if summed else None, _mk(g, batch, n) if gated else None
    assert F.on_codes(x, q.q)
    y = q(x, act=act, residual=res, gate=gate)
    w, xd = q.q.dequantize(torch.float32).double(), x.double()
    ref = xd @ w.t() + q.bias.detach().double()
    # output and activation are rounded to bf16 (2^-8 each), levels to 2^-11; 1.13: the activations' largest slope
    err = ref.abs() * 2 ** -8 + (xd.abs() @ w.abs().t()) * 2 ** -10
    if act is not None:
        ref = torch.nn.functional.gelu(ref, approximate="tanh") if act == "gelu" else torch.nn.functional.silu(ref)
        err = err * 1.13 + ref.abs() * 2 ** -8
    ref, err = ref.reshape(batch, tokens, n), err.reshape(batch, tokens, n)
    if gated:
        ref, err = ref * gate.double()[:, None], err * gate.double().abs()[:, None]
    if summed:
        ref = ref + res.double().reshape(ref.shape)
    err = err + ref.abs() * 2 ** -8
    assert y.shape == (*lead, n) and y.dtype == BF and ((y.double().reshape(ref.shape) - ref).abs() <= err * 1.01 + 1e-6).all()


def test_gradients_of_gate_and_residual():
    g = torch.Generator(device="cuda").manual_seed(3)
    q = _layer(g, 320, 256, "int4")
    leaves = [t.requires_grad_() for t in (_mk(g, 6, 256), _mk(g, 6, 320), _mk(g, 1, 320))]
    x, res, gate = leaves
    dy = _mk(g, 6, 320)
    grads = torch.autograd.grad(q(x, residual=res, gate=gate), leaves, dy)
    w = q.q.dequantize(torch.float32).double()
    y = x.detach().double() @ w.t() + q.bias.detach().double()
    refs = ((dy.double() * gate.detach().double()) @ w, dy.double(), (dy.double() * y).sum(0, keepdim=True))
    for a, r in zip(grads, refs):                # a handful of bf16 roundings between the ends
        assert a.shape == r.shape and ((a.double() - r).norm() / r.norm()).item() < 4 * 2 ** -8


def test_what_the_codes_do_not_take_goes_the_usual_way():
    g = torch.Generator(device="cuda").manual_seed(5)
    q = _layer(g, 320, 256, "nf4")
    x = _mk(g, 1, 3, 256)
    with pytest.raises(KeyError):
        q(x, act="tanh")
    wide = torch.randn(1, 1, 320, device="cuda", generator=g).to(BF)      # a residual that broadcasts, as on the expanded weight
    want = F.linear(x, q.weight, q.bias, residual=wide)
    y = q(x, residual=wide)
    assert y.shape == want.shape and torch.equal(y, want)
    double = _layer(g, 320, 256, "nf4", dtype=torch.float32)
    with pytest.raises(RuntimeError):
        double(x)                                # types that do not go together, as before
    assert q(x[:, :0]).shape == (1, 0, 320)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
def test_trained_after_quantising_in_inference_mode(kind):
    g = torch.Generator(device="cuda").manual_seed(7)
    with torch.inference_mode():
        q = _layer(g, 320, 256, kind)
    q.bias = None
    x, dy = _mk(g, 3, 256).requires_grad_(), _mk(g, 3, 320)
    (dx,) = torch.autograd.grad(q(x), x, dy)
    w = q.q.dequantize(torch.float32).double()
    assert ((dx.double() - dy.double() @ w).norm() / (dy.double() @ w).norm()).item() < 2 ** -7
