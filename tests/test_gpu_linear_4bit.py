"""Products with int4 / NF4 codes against their definition in 64 bits (weight = level * scale): dense and per expert, rows of no
expert, gradient of the rows. A rounding to bf16 is off by 2^-8 of the value at most, a sum of n fp32 products by n 2^-23 of the
sum of their magnitudes, the level of a code by 2^-11 of itself (it is multiplied as fp16)."""
import pytest
import torch

from eridiffusion_b200.memory import NF4_LEVELS, QuantizedTensor, quantize
from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _weight64(q):
    lo, hi = (q.data & 15).long(), (q.data >> 4).long()
    c = torch.stack([lo, hi], -1).flatten(1)
    v = (c - 8).double() / 7 if q.kind == "int4" else NF4_LEVELS.cuda().double()[c]
    return (v * q.scale.double()[:, None]).view(q.shape)


def _near(a, ref, mag, terms, expanded=False):
    # sums, a level's 2^-11 and the scale of a row's block as a power of two; the rounding to bf16. More rows than are multiplied with
    # the codes meet the weight expanded to bf16: every weight, and with it every product, is off by up to 2^-8 of itself
    bad = ~((a.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * (terms * 2 ** -23 + (2 ** -8 if expanded else 2 ** -11)))
    assert a.shape == ref.shape and not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), a[bad][:4].tolist(), ref[bad][:4].tolist())


def _random(g, kind, shape, block):
    n = 1
    for s in shape:
        n *= s
    codes = torch.randint(0, 256, (n // block, block // 2), device="cuda", generator=g, dtype=torch.uint8)
    scale = torch.rand(n // block, device="cuda", generator=g) * 0.1 + 1e-4
    return QuantizedTensor(kind, codes, scale, shape, block)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
@pytest.mark.parametrize("M,N,K,block", [(1, 1, 32, 32), (1, 64, 256, 64), (2, 33, 192, 64), (3, 100, 96, 32), (5, 257, 640, 128), (8, 1000, 1280, 64),
                                         (7, 520, 2560, 256), (4, 130, 1088, 64)])
def test_dense(M, N, K, block, kind):
    g = _gen(M * N + K)
    q = _random(g, kind, (N, K), block)
    x = _mk(g, M, K + 8)[:, :K].requires_grad_()
    bias = _mk(g, N).requires_grad_()
    dy = _mk(g, M, N)
    y = F.linear_4bit(x, q, bias=bias)
    dx, db = torch.autograd.grad(y, (x, bias), dy)
    w = _weight64(q)
    _near(y.detach(), x.detach().double() @ w.t() + bias.detach().double(), x.detach().double().abs() @ w.abs().t() + bias.detach().double().abs(), K)
    _near(dx, dy.double() @ w, dy.double().abs() @ w.abs(), N)
    _near(db, dy.double().sum(0), dy.double().abs().sum(0), M)
    plain = F.linear_4bit(x.detach(), q)
    _near(plain, x.detach().double() @ w.t(), x.detach().double().abs() @ w.abs().t(), K)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
@pytest.mark.parametrize("counts,first,rest", [([1], 0, 0), ([0, 3, 0, 1], 0, 0), ([9, 0, 17, 8], 0, 0), ([2, 2], 3, 5), ([0, 0, 0], 0, 4), ([1] * 12, 0, 0)])
def test_experts(counts, first, rest, kind):
    E, N, K, block = len(counts), 72, 320, 64
    g = _gen(sum(counts) + E)
    q = _random(g, kind, (E, N, K), block)
    off = torch.tensor([0, *counts]).cumsum(0).add(first).to(torch.int32).cuda()
    R = sum(counts) + first + rest
    x, dy = _mk(g, R, K), _mk(g, R, N)
    own = torch.zeros(R, dtype=torch.bool, device="cuda")
    own[first:first + sum(counts)] = True
    x[~own], dy[~own] = float("nan"), float("nan")
    x.requires_grad_()
    y = F.linear_4bit(x, q, off)
    (dx,) = torch.autograd.grad(y, x, dy)
    w = _weight64(q)
    of = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).cuda()
    we = w[of]
    xs, ds = x.detach()[own].double(), dy[own].double()
    _near(y.detach()[own], torch.einsum("rk,rnk->rn", xs, we), torch.einsum("rk,rnk->rn", xs.abs(), we.abs()), K)
    _near(dx[own], torch.einsum("rn,rnk->rk", ds, we), torch.einsum("rn,rnk->rk", ds.abs(), we.abs()), N)
    assert (y.detach()[~own] == 0).all() and (dx[~own] == 0).all()


@pytest.mark.parametrize("kind", ["int4", "nf4"])
def test_values_of_wide_range_and_special_ones(kind):
    """Rows whose magnitudes span the whole range of bf16 next to each other keep their 2^-8; infinities and NaN stay in their row."""
    g = _gen(4)
    q = _random(g, kind, (64, 256), 64)
    w = _weight64(q)
    x = _mk(g, 6, 256)
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -100
    x[2, ::2] *= 2.0 ** 60
    x[3] = 0
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    y = F.linear_4bit(x, q)
    for r in range(4):
        _near(y[r], w @ x[r].double(), w.abs() @ x[r].double().abs(), 256)
    codes = torch.stack([q.data & 15, q.data >> 4], -1).flatten(1).view(64, 256)
    zero = codes[:, 7] == (8 if kind == "int4" else 7)
    assert y[4][zero].isnan().all() and y[4][~zero].isinf().all() and (y[4][~zero] > 0).eq(w[~zero, 7] > 0).all()
    assert y[5].isnan().all()


def test_more_rows_and_other_shapes_expand_the_weight():
    g = _gen(6)
    w = torch.randn(256, 512, device="cuda", generator=g) * 0.05
    for kind in ("int4", "nf4"):
        q = quantize(w, kind)
        for shape in ((40, 512), (3, 100, 512)):
            x = _mk(g, *shape)
            y = F.linear_4bit(x, q)
            ref = x.double() @ _weight64(q).t()
            mag = x.double().abs() @ _weight64(q).abs().t()
            assert y.shape == ref.shape
            assert ((y.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * (2 ** -8 + 512 * 2 ** -23)).all()
        lead = F.linear_4bit(_mk(g, 2, 1, 512), q)
        assert lead.shape == (2, 1, 256)


def test_gradient_against_differences():
    """Linear in x: <dy, y(x + h) - y(x)> = <dx, h> but for roundings."""
    g = _gen(8)
    q = _random(g, "nf4", (200, 256), 64)
    x, dy = _mk(g, 4, 256).requires_grad_(), _mk(g, 4, 200)
    y = F.linear_4bit(x, q)
    (dx,) = torch.autograd.grad(y, x, dy)
    moved = x.detach() + _mk(g, 4, 256)
    h = moved.double() - x.detach().double()
    y1 = F.linear_4bit(moved, q)
    lhs, rhs = (dy.double() * (y1.double() - y.detach().double())).sum(), (dx.double() * h).sum()
    err = (dy.double() * y1.double() * 2 ** -8).norm() + (dy.double() * y.detach().double() * 2 ** -8).norm() + (dx.double() * h * 2 ** -8).norm()
    assert (lhs - rhs).abs() <= 6 * err


def test_in_a_graph():
    g = _gen(9)
    q = _random(g, "int4", (4, 136, 320), 64)
    x, dy = _mk(g, 12, 320).requires_grad_(), _mk(g, 12, 136)
    off = torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(F.linear_4bit(x, q, off), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.linear_4bit(x, q, off)
        (dx,) = torch.autograd.grad(y, x, dy)
    for counts in ([3, 3, 3, 3], [12, 0, 0, 0], [0, 1, 10, 1]):
        off.copy_(torch.tensor([0, *counts]).cumsum(0))
        graph.replay()
        fresh = F.linear_4bit(x, q, off)
        assert torch.equal(y, fresh) and torch.equal(dx, torch.autograd.grad(fresh, x, dy)[0])


@pytest.mark.parametrize("kind", ["int4", "nf4"])
@pytest.mark.parametrize("E,N,K,block", [(64, 2000, 320, 64), (48, 2000, 320, 64), (40, 1208, 1024, 64), (24, 3000, 160, 32)])
def test_many_experts_per_cta(E, N, K, block, kind):
    """More tiles than CTAs, so that a CTA goes on from one expert's rows to the next one's."""
    g = _gen(E + N)
    q = _random(g, kind, (E, N, K), block)
    counts = [1 + (i % 3 == 0) - (i % 7 == 3) for i in range(E)]
    off = torch.tensor([0, *counts]).cumsum(0).to(torch.int32).cuda()
    R = sum(counts)
    x, dy = _mk(g, R, K).requires_grad_(), _mk(g, R, N)
    y = F.linear_4bit(x, q, off)
    (dx,) = torch.autograd.grad(y, x, dy)
    we = _weight64(q)[torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).cuda()]
    xd, dd, expanded = x.detach().double(), dy.double(), R > F.CODES_EXPERT_ROWS       # (the first case: 77 rows)
    _near(y.detach(), torch.einsum("rk,rnk->rn", xd, we), torch.einsum("rk,rnk->rn", xd.abs(), we.abs()), K, expanded)
    _near(dx, torch.einsum("rn,rnk->rk", dd, we), torch.einsum("rn,rnk->rk", dd.abs(), we.abs()), N, expanded)


@pytest.mark.parametrize("kind", ["int4", "nf4"])
def test_long_rows_take_several_passes(kind):
    """x of eight rows does not fit next to the rings: the codes are read once per few rows."""
    g = _gen(17)
    q = _random(g, kind, (50, 16384), 64)
    x, dy = _mk(g, 8, 16384).requires_grad_(), _mk(g, 8, 50)
    y = F.linear_4bit(x, q)
    (dx,) = torch.autograd.grad(y, x, dy)
    w = _weight64(q)
    _near(y.detach(), x.detach().double() @ w.t(), x.detach().double().abs() @ w.abs().t(), 16384)
    _near(dx, dy.double() @ w, dy.double().abs() @ w.abs(), 50)


def test_codes_of_another_size_are_refused():
    g = _gen(19)
    q = _random(g, "int4", (64, 128), 64)
    x = _mk(g, 2, 128)
    for data, scale in ((q.data[:-1], q.scale), (q.data, q.scale[:-1])):
        with pytest.raises(ValueError):
            F.linear_4bit(x, QuantizedTensor("int4", data, scale, (64, 128), 64))
    with pytest.raises(ValueError):
        F.linear_4bit(x, QuantizedTensor("int4", q.data.cpu(), q.scale, (64, 128), 64))
