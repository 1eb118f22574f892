"""Token-routed experts against their definitions in 64 bits: router, plan, dispatch and combine, grouped product, and the run of
them together. A rounding to bf16 is off by 2^-8 of the value at most, a sum of n fp32 products by n 2^-23 of the sum of their
magnitudes (the tensor cores cut the aligned products off instead of rounding them)."""
import math

import pytest
import torch

from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _offsets(counts, first=0):
    return torch.tensor([0, *counts], dtype=torch.int32).cumsum(0).add(first).to(torch.int32).cuda()


# ------------------------------------------------------------------------------------------- router
def _route64(scores, k, allowed, normalize, dw):
    s = scores.double().cpu()
    if allowed is not None:
        s = torch.where(allowed.cpu(), s, -math.inf)
    idx = torch.tensor([sorted(range(s.shape[1]), key=lambda e: (-r[e].item(), e))[:k] for r in s])
    s.requires_grad_()
    top = s.gather(1, idx)
    if normalize:
        w = torch.softmax(top, -1)
    else:
        w = torch.softmax(s, -1).gather(1, idx)
    (ds,) = torch.autograd.grad(w, s, dw.double().cpu())
    return idx, w.detach(), ds


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 4), (9, 3, 3), (33, 32, 32), (257, 33, 8), (40, 129, 2), (17, 300, 6), (5, 1000, 32),
                                   (3, 1024, 7)])
def test_route(T, E, k, dtype, normalize):
    g = _gen(T * E + k)
    wide = torch.randn(T, E + 3, device="cuda", generator=g).mul(3).to(dtype)
    scores = wide[:, :E].detach().requires_grad_()                  # rows of another stride
    allowed = torch.rand(E, device="cuda", generator=g) < 0.7
    allowed[torch.randperm(E, generator=g, device="cuda")[:k]] = True
    dw = torch.randn(T, k, device="cuda", generator=g)
    for al in (None, allowed):
        idx, w = F.expert_route(scores, k, allowed=al, normalize=normalize)
        ri, rw, rds = _route64(scores.detach(), k, al, normalize, dw)
        assert idx.dtype == torch.int64 and w.dtype == torch.float32
        assert torch.equal(idx.cpu(), ri)
        # exponentials and quotient at 2^-22, the sum of E terms at E 2^-24
        assert ((w.cpu().double() - rw).abs() <= rw * (2 ** -20 + E * 2 ** -24) + 1e-37).all()
        (ds,) = torch.autograd.grad(w, scores, dw)
        assert ds.dtype == dtype and ds.shape == scores.shape
        p = torch.softmax(scores.detach().double().cpu() if al is None else torch.where(al.cpu(), scores.detach().double().cpu(), -math.inf), -1)
        p = torch.maximum(p, torch.zeros_like(p).scatter_(1, ri, rw))
        bound = p * (dw.abs().max().item() * (E + 64) * 2 ** -22) + rds.abs() * (torch.finfo(dtype).eps / 2) + 1e-37
        assert ((ds.cpu().double() - rds).abs() <= bound).all()
        if normalize:
            assert (ds.cpu().scatter(1, ri, 0) == 0).all()


def test_route_equal_scores_go_to_the_lowest_index():
    s = torch.tensor([[0.0, -0.0, 0.0, 1.0, 1.0], [2.0, 2.0, 2.0, 2.0, 2.0]], device="cuda")
    idx, w = F.expert_route(s, 4)
    assert idx.tolist() == [[3, 4, 0, 1], [0, 1, 2, 3]]
    assert torch.allclose(w[1], torch.full((4,), 0.25, device="cuda"), atol=2 ** -22)
    many = torch.zeros(3, 200, device="cuda", dtype=BF)
    assert F.expert_route(many, 8)[0].tolist() == [list(range(8))] * 3


def test_route_rows_without_an_expert_and_special_values():
    inf, nan = math.inf, math.nan
    s = torch.tensor([[-inf] * 4, [1.0, -inf, -inf, -inf], [1.0, nan, 2.0, 0.0], [inf, 0.0, 1.0, 2.0], [-3.4e38, -inf, -3.4e38, -inf]],
                     device="cuda").requires_grad_()
    for normalize in (True, False):
        idx, w = F.expert_route(s, 2, normalize=normalize)
        assert idx.tolist() == [[0, 1], [0, 1], [1, 2], [0, 3], [0, 2]]
        assert w[0].tolist() == [0, 0] and w[1].tolist() == [1, 0] and w[2].isnan().all() and w[3].isnan().all()
        assert torch.allclose(w[4], torch.full((2,), 0.5, device="cuda"), atol=2 ** -22)
        (ds,) = torch.autograd.grad(w[[0, 1, 4]].sum() + w[4, 0], s, retain_graph=True)
        assert (ds[0] == 0).all() and (ds[1] == 0).all() and torch.isfinite(ds[4]).all() and ds[4, 0] > 0
        r = F.R.expert_route(s.detach().cpu(), 2, None, normalize)
        assert torch.equal(r[0], idx.cpu()) and torch.allclose(r[1], w.detach().cpu(), atol=2 ** -20, equal_nan=True)


def test_route_without_tokens():
    idx, w = F.expert_route(torch.empty(0, 8, device="cuda"), 2)
    assert idx.shape == w.shape == (0, 2)


# ------------------------------------------------------------------------------------------- plan, dispatch, combine
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (7, 2, 32), (129, 3, 5), (1024, 4, 64), (1366, 3, 7), (2731, 6, 256), (5000, 5, 1024),
                                   (30001, 8, 33)])
def test_plan(T, k, E, dtype):
    g = _gen(T + k + E)
    idx = torch.randint(-1, E + (1 if T % 2 else 0), (T, k), device="cuda", generator=g).to(dtype)     # some outside [0, E)
    plan = F.expert_plan(idx, E)
    offsets, rows = (t.cpu() for t in plan)
    ro, rr = F.R.expert_plan(idx.cpu(), E)
    assert torch.equal(offsets, ro) and torch.equal(rows, rr)
    again = F.expert_plan(idx, E)
    assert all(torch.equal(a, b) for a, b in zip(plan, again))


def test_plan_of_one_expert_only():
    for n in (1, 4097, 20000):
        plan = F.expert_plan(torch.full((n, 1), 3, device="cuda"), 5)
        assert plan.offsets.tolist() == [0, 0, 0, 0, n, n] and torch.equal(plan.rows[:, 0].cpu(), torch.arange(n, dtype=torch.int32))
        none = F.expert_plan(torch.full((n, 1), 9, device="cuda"), 5)
        assert none.offsets.tolist() == [0] * 6 and (none.rows == -1).all()


@pytest.mark.parametrize("T,k,E,D", [(1, 1, 1, 8), (7, 2, 32, 640), (65, 9, 12, 136), (300, 17, 40, 1288), (1000, 4, 8, 72), (5000, 1, 9, 264), (4000, 3, 9, 72),
                                     (1500, 8, 64, 2312), (700, 9, 16, 4104)])       # with more tokens than the kernels hold at a time
@pytest.mark.parametrize("padded", [False, True])
def test_dispatch_and_combine(T, k, E, D, padded):
    g = _gen(T + k + D)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g)           # the same expert twice for a token, too
    if padded:
        idx[T // 2:] = -1
    plan = F.expert_plan(idx, E)
    live = int(plan.offsets[-1])
    x = _mk(g, T, D + 8)[:, :D].requires_grad_()
    y = _mk(g, T * k, D + 8)[:, :D]
    y[live:] = float("nan")                                                 # rows of nobody
    y.requires_grad_()
    w = torch.rand(T, k, device="cuda", generator=g).requires_grad_()
    xs, out = F.expert_dispatch(x, plan), F.expert_combine(y, w, plan)
    rows, here = plan.rows.long().clamp_min(0), (plan.rows >= 0)
    flat = plan.rows.reshape(-1).long()
    choice = torch.empty(live, dtype=torch.int64, device="cuda")          # of every row
    choice[flat[flat >= 0]] = torch.arange(T * k, device="cuda")[flat >= 0]
    token = choice // k
    assert torch.equal(xs[:live], x.detach()[token]) and (xs[live:] == 0).all()
    yt = torch.where(here[..., None], y.detach().double()[rows], 0.0)
    ref = (w.detach().double()[..., None] * yt).sum(1)
    mag = (w.detach().double()[..., None] * yt.abs()).sum(1)
    assert ((out.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * k * 2 ** -23).all()
    dxs, dout = _mk(g, T * k, D), _mk(g, T, D)
    dxs[live:] = float("nan")
    dx, dy, dw = torch.autograd.grad((xs, out), (x, y, w), (dxs, dout))
    dt = torch.where(here[..., None], dxs.double()[rows], 0.0)
    assert ((dx.double() - dt.sum(1)).abs() <= dt.sum(1).abs() * 2 ** -8 + dt.abs().sum(1) * k * 2 ** -23).all()
    rdy = w.detach().double().reshape(-1)[choice][:, None] * dout.double()[token]
    assert ((dy[:live].double() - rdy).abs() <= rdy.abs() * (2 ** -8 + 2 ** -23)).all() and (dy[live:] == 0).all()
    prod = yt * dout.double()[:, None]
    assert ((dw.double() - prod.sum(-1)).abs() <= prod.abs().sum(-1) * D * 2 ** -23).all() and (dw[~here] == 0).all()


def test_combine_gradients_on_demand_and_weights_of_another_type():
    g = _gen(3)
    plan = F.expert_plan(torch.randint(0, 4, (20, 2), device="cuda", generator=g), 4)
    y, w = _mk(g, 40, 64), torch.rand(20, 2, device="cuda", generator=g)
    d = _mk(g, 20, 64)
    full = torch.autograd.grad(F.expert_combine(y.requires_grad_(), w.requires_grad_(), plan), (y, w), d)
    only_y = torch.autograd.grad(F.expert_combine(y, w.detach(), plan), y, d)
    only_w = torch.autograd.grad(F.expert_combine(y.detach(), w, plan), w, d)
    assert torch.equal(full[0], only_y[0]) and torch.equal(full[1], only_w[0])
    half = w.detach().to(BF).requires_grad_()
    (dh,) = torch.autograd.grad(F.expert_combine(y, half, plan), half, d)
    assert dh.dtype == BF


# ------------------------------------------------------------------------------------------- grouped product
def _linear64(x, w, offsets, dy):
    b = offsets.tolist()
    x, w, dy = x.double(), w.double(), dy.double()
    y, dx, dw = x.new_zeros(x.shape[0], w.shape[1]), torch.zeros_like(x), torch.zeros_like(w)
    my, mx, mw = torch.zeros_like(y), torch.zeros_like(dx), torch.zeros_like(dw)       # sums of magnitudes
    for e in range(w.shape[0]):
        s = slice(b[e], b[e + 1])
        y[s], my[s] = x[s] @ w[e].t(), x[s].abs() @ w[e].abs().t()
        dx[s], mx[s] = dy[s] @ w[e], dy[s].abs() @ w[e].abs()
        dw[e], mw[e] = dy[s].t() @ x[s], dy[s].abs().t() @ x[s].abs()
    return (y, my), (dx, mx), (dw, mw)


def _near(a, ref, mag, terms):
    assert a.shape == ref.shape
    bad = ~((a.double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * terms * 2 ** -23)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), a[bad][:4].tolist(), ref[bad][:4].tolist())


COUNTS = [[1], [0, 5, 0], [33, 0, 1, 64, 65, 2, 0, 31], [0, 0, 0, 7], [130, 1, 200, 64], [300, 257, 0, 1, 511], [1000, 2, 255, 256],
          [3] * 40, [64, 128, 192, 0, 256]]


@pytest.mark.parametrize("N,K", [(8, 8), (136, 72), (264, 520), (1000, 264), (512, 64)])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
def test_linear(counts, N, K):
    g = _gen(sum(counts) + N + K)
    R, E = sum(counts), len(counts)
    off = _offsets(counts)
    x = _mk(g, R, K + 8)[:, :K].requires_grad_()                     # rows of another stride
    w = _mk(g, E, N, K, std=K ** -0.5).requires_grad_()
    dy = _mk(g, R, N + 16)[:, 8:N + 8]
    y = F.expert_linear(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    (ry, my), (rx, mx), (rw, mw) = _linear64(x.detach(), w.detach(), off, dy)
    _near(y.detach(), ry, my, K)
    _near(dx, rx, mx, N)
    _near(dw, rw, mw, max(counts))
    assert F.kernel_error_check() == {}


@pytest.mark.parametrize("columns", [32, 64, 128, 256])
def test_linear_every_tile_height(columns):
    counts = [columns - 1, 0, columns + 1, 1, 2 * columns, 70]
    g = _gen(columns)
    R, E, N, K = sum(counts), len(counts), 328, 200
    x, w, off = _mk(g, R, K), _mk(g, E, N, K, std=K ** -0.5), _offsets(counts)
    dy = _mk(g, R, N)
    x.requires_grad_()
    y = F.N.ops().expert_linear(x, w, off, columns, False)
    (dx,) = torch.autograd.grad(y, x, dy)
    (ry, my), (rx, mx), _ = _linear64(x.detach(), w, off, dy)
    _near(y.detach(), ry, my, K)
    _near(dx, rx, mx, N)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_linear_rows_of_nobody_and_other_experts_stay_out(bad):
    """Rows outside the offsets and rows of a neighbouring expert hold NaN or infinities: nothing of theirs shows elsewhere."""
    g = _gen(5)
    counts, N, K = [70, 3, 0, 100], 136, 264
    off = _offsets(counts, first=9)
    R = sum(counts) + 9 + 50
    x, w, dy = _mk(g, R, K), _mk(g, 4, N, K, std=0.06), _mk(g, R, N)
    x[:9], dy[:9], x[-50:], dy[-50:] = bad, bad, bad, bad
    x[9 + 70:9 + 73], dy[9 + 70:9 + 73] = bad, bad                   # the second expert's three rows
    w[1] = bad
    w[2] = bad                                                       # an expert without rows
    x.requires_grad_(), w.requires_grad_()
    y = F.expert_linear(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    keep = torch.ones(R, dtype=torch.bool)
    keep[:9] = keep[-50:] = keep[79:82] = False
    (ry, my), (rx, mx), (rw, mw) = _linear64(x.detach(), w.detach(), off, dy)
    _near(y.detach()[keep], ry[keep], my[keep], K)
    _near(dx[keep], rx[keep], mx[keep], N)
    for t in (y.detach(), dx):
        assert (t[:9] == 0).all() and (t[-50:] == 0).all() and not torch.isfinite(t[79:82]).any()
    for e in (0, 3):
        _near(dw[e], rw[e], mw[e], 100)
    assert (dw[2] == 0).all() and not torch.isfinite(dw[1]).any()


def test_linear_without_rows_and_without_owned_rows():
    w = torch.randn(3, 16, 24, device="cuda").to(BF).requires_grad_()
    x = torch.empty(0, 24, device="cuda", dtype=BF).requires_grad_()
    y = F.expert_linear(x, w, torch.zeros(4, dtype=torch.int32, device="cuda"))
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 16, device="cuda", dtype=BF))
    assert y.shape == (0, 16) and dx.shape == (0, 24) and (dw == 0).all()
    x = torch.randn(100, 24, device="cuda").to(BF).requires_grad_()
    y = F.expert_linear(x, w, torch.zeros(4, dtype=torch.int64, device="cuda"))
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert (y == 0).all() and (dx == 0).all() and (dw == 0).all()


def test_linear_gradient_against_differences():
    """The product is linear in each argument, so a difference of any size is exact but for roundings: <dy, y(x + h) - y(x)> = <dx, h>."""
    g = _gen(11)
    counts, N, K = [40, 0, 90, 5], 264, 136
    off = _offsets(counts)
    R, E = sum(counts), len(counts)
    x, w, dy = _mk(g, R, K).requires_grad_(), _mk(g, E, N, K, std=0.1).requires_grad_(), _mk(g, R, N)
    y = F.expert_linear(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for t, d, shape in ((x, dx, (R, K)), (w, dw, (E, N, K))):
        h = (t.detach() + _mk(g, *shape)) - t.detach()               # representable
        moved = (t.detach() + h)
        h = moved.double() - t.detach().double()
        args = (moved, w.detach()) if t is x else (x.detach(), moved)
        diff = F.expert_linear(*args, off).double() - y.detach().double()
        lhs, rhs = (dy.double() * diff).sum(), (d.double() * h).sum()
        # every y is off by 2^-8 of itself and every gradient element by 2^-8 of itself; independent roundings add up as squares
        err = (dy.double() * y.detach().double() * 2 ** -8).norm() * 2 + (d.double() * h * 2 ** -8).norm()
        assert (lhs - rhs).abs() <= 6 * err


def test_linear_adds_into_a_gradient_buffer():
    g = _gen(12)
    counts, N, K = [40, 0, 90], 72, 136
    off = _offsets(counts)
    x, dy = _mk(g, 130, K), _mk(g, 130, N)
    w = torch.nn.Parameter(_mk(g, 3, N, K))
    first = _mk(g, 3, N, K)
    w.grad = first.clone()
    held = w.grad
    F.expert_linear(x, w, off).backward(dy)
    _, _, (rw, mw) = _linear64(x, w.detach(), off, dy)
    ref = rw + first.double()
    assert w.grad.data_ptr() == held.data_ptr()
    _near(w.grad, ref, mw + first.double().abs(), 100)
    assert torch.equal(w.grad[1], first[1])


def test_linear_in_a_graph_follows_the_offsets():
    g = _gen(13)
    N, K, R, E = 264, 200, 300, 5
    x, w, dy = _mk(g, R, K).requires_grad_(), _mk(g, E, N, K, std=0.1).requires_grad_(), _mk(g, R, N)
    off = _offsets([60] * 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(F.expert_linear(x, w, off), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.expert_linear(x, w, off)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    for counts in ([60] * 5, [0, 299, 0, 1, 0], [300, 0, 0, 0, 0], [7, 100, 64, 65, 20]):
        off.copy_(_offsets(counts))
        graph.replay()
        (ry, my), (rx, mx), (rw, mw) = _linear64(x.detach(), w.detach(), off, dy)
        _near(y.detach(), ry, my, K)
        _near(dx, rx, mx, N)
        _near(dw, rw, mw, R)


def test_on_another_stream():
    g = _gen(14)
    x, w, off = _mk(g, 500, 512), _mk(g, 4, 512, 512, std=0.05), _offsets([100, 150, 0, 250])
    ref = F.expert_linear(x, w, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = x * 1                                    # made on the side stream: a launch elsewhere would not wait for it
        y = F.expert_linear(late, w, off)
    side.synchronize()
    assert torch.equal(y, ref)


def test_first_call_of_a_thread():
    """Operand maps are encoded by the driver, which wants a context of the calling thread; a new thread has none yet."""
    import threading
    g = _gen(15)
    x, w, off = _mk(g, 48, 88), _mk(g, 2, 40, 88, std=0.1), _offsets([20, 28])
    ref = F.expert_linear(x, w, off)
    x2, w2 = x.clone(), w.clone()               # other addresses: nothing of theirs is encoded yet
    torch.cuda.synchronize()
    got = []

    def call():
        try:
            got.append(F.expert_linear(x2, w2, off))
        except RuntimeError as e:
            got.append(e)
    t = threading.Thread(target=call)
    t.start(), t.join()
    torch.cuda.synchronize()
    assert torch.is_tensor(got[0]) and torch.equal(got[0], ref), got[0]
