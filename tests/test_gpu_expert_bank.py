"""``moe_linear`` on an ``ExpertBank`` whose entries change, are held elsewhere, or are first used in unusual places."""
import pytest
import torch

from eridiffusion_b200.memory import QuantizedTensor
from eridiffusion_b200.models.moe import ExpertBank, moe_linear, route_tokens

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
E, N, K = 6, 136, 192


def _mk(g, *s, std=1.0):
    return (torch.randn(*s, device="cuda", generator=g) * std).to(BF)


def _weight64(e):
    return (e.dequantize(torch.float32) if isinstance(e, QuantizedTensor) else e).detach().double()


def _near(y, x, scores, bank, k=2):
    """Against 64 bits: expert outputs and their sum are rounded to bf16 (2^-8 of themselves each); expanded weights 2^-8, levels of
    few rows 2^-11 of themselves; sums over K in 32 bits."""
    top, idx = torch.sort(scores.double(), dim=-1, descending=True, stable=True)
    w = torch.softmax(top[:, :k], -1)
    ref, err = 0, 0
    for j in range(k):
        for e, q in bank.experts.items():
            hit = (idx[:, j] == e).double()[:, None] * w[:, j:j + 1]
            we, xd = _weight64(q), x.detach().double()
            p = xd @ we.t()
            ref = ref + hit * p
            err = err + hit * (p.abs() * 2 ** -8 + (xd.abs() @ we.abs().t()) * (K * 2 ** -23 + (2 ** -8 if isinstance(q, QuantizedTensor) else 0)))
    assert y.dtype == BF and ((y.double() - ref).abs() <= (ref.abs() * 2 ** -8 + err) * 1.01 + 1e-30).all()


def _bank(kind, g, held=None):
    bank = ExpertBank(kind)
    for e in range(E):
        w = _mk(g, N, K, std=0.07)
        if held is not None:
            held.append(w)
        bank.insert(e, w)
    return bank


def _inputs(g, T):
    return _mk(g, T, K), torch.randn(T, E, device="cuda", generator=g)


@pytest.mark.parametrize("T", [1, 5, 300])
def test_changes_of_the_callers_weights_are_followed(T):
    g = torch.Generator(device="cuda").manual_seed(T)
    held = []
    bank = _bank("none", g, held)
    x, scores = _inputs(g, T)
    for _ in range(3):
        _near(moe_linear(x, scores, bank), x, scores, bank)
        assert all(torch.equal(bank.experts[i], w) for i, w in enumerate(held))
        for w in held:
            w.copy_(_mk(g, N, K, std=0.07))


@pytest.mark.parametrize("T", [1, 5, 300])
@pytest.mark.parametrize("kind", ["none", "nf4"])
def test_changes_of_entries_are_followed(kind, T):
    g = torch.Generator(device="cuda").manual_seed(T + 1)
    bank = _bank(kind, g)
    x, scores = _inputs(g, T)
    entries = list(bank.experts.values())
    for _ in range(3):
        _near(moe_linear(x, scores, bank), x, scores, bank)
        for e in entries:
            (e.scale if kind == "nf4" else e).mul_(1.5)
        assert all(bank.experts[i] is e for i, e in enumerate(entries))


def _capture(fn):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.parametrize("called_before", [False, True])
@pytest.mark.parametrize("T", [1, 5, 300])
@pytest.mark.parametrize("kind", ["none", "q8", "nf4"])
def test_captured_call(kind, T, called_before):
    """The first call of a bank may be captured: replays follow the entries, also after eager calls and other allocations."""
    g = torch.Generator(device="cuda").manual_seed(T + 2)
    bank = _bank(kind, g)
    x, scores = _inputs(g, T)
    if called_before:
        moe_linear(x, scores, bank)
    at = [(e.data if isinstance(e, QuantizedTensor) else e).data_ptr() for e in bank.experts.values()]
    graph, y = _capture(lambda: moe_linear(x, scores, bank))
    for i in range(3):
        junk = [torch.full((E * N * K,), float("nan"), device="cuda", dtype=BF) for _ in range(4)]
        x.copy_(_mk(g, T, K))
        scores.copy_(torch.randn(T, E, device="cuda", generator=g))
        for e in bank.experts.values():
            (e.scale if isinstance(e, QuantizedTensor) else e).mul_(1.25)
        graph.replay()
        _near(y, x, scores, bank)
        _near(moe_linear(x, scores, bank), x, scores, bank)
        del junk
    assert [(e.data if isinstance(e, QuantizedTensor) else e).data_ptr() for e in bank.experts.values()] == at


def test_fetched_under_capture_then_called():
    g = torch.Generator(device="cuda").manual_seed(4)
    bank = _bank("none", g)
    x, scores = _inputs(g, 5)
    out = torch.empty(N, K, device="cuda", dtype=BF)
    graph, _ = _capture(lambda: out.copy_(bank.fetch_topk_bf16([2])[0][1] * 2))
    _near(moe_linear(x, scores, bank), x, scores, bank)
    junk = [torch.full((N * K,), float("nan"), device="cuda", dtype=BF) for _ in range(2 * E)]
    graph.replay()
    assert torch.equal(out, bank.experts[2] * 2)
    del junk


def _junk(n=3 * E):
    return [torch.full((N * K,), float("nan"), device="cuda", dtype=BF) for _ in range(n)] + [torch.full((E * N * K,), float("nan"), device="cuda", dtype=BF)]


@pytest.mark.parametrize("kind", ["none", "nf4"])
def test_first_call_on_another_stream(kind):
    """The first call waits on a busy stream: what the bank's own stream allocates and writes meanwhile is not its weights, and a third
    stream finds them without waiting for the first one."""
    g = torch.Generator(device="cuda").manual_seed(6)
    bank = _bank(kind, g)
    want = [_weight64(e).clone() for e in bank.experts.values()]
    x, scores = _inputs(g, 5)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(40_000_000)
        y = moe_linear(x, scores, bank)
    junk = _junk()
    with torch.cuda.stream(other):
        z = moe_linear(x, scores, bank)
    torch.cuda.synchronize()
    assert all(torch.equal(_weight64(e), w) for e, w in zip(bank.experts.values(), want))
    _near(y, x, scores, bank)
    _near(z, x, scores, bank)
    del junk


@pytest.mark.parametrize("kind", ["none", "nf4"])
def test_bank_dropped_while_another_stream_reads_it(kind):
    g = torch.Generator(device="cuda").manual_seed(8)
    bank = _bank(kind, g)
    x, scores = _inputs(g, 5)
    first = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        y = moe_linear(x, scores, bank)
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)
    z = moe_linear(x, scores, bank)
    bank.experts.clear()
    del bank
    with torch.cuda.stream(first):
        junk = _junk()
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    del junk


@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("inserted_inside", [False, True])
@pytest.mark.parametrize("kind", ["none", "nf4"])
def test_training_after_a_call_in_inference_mode(kind, inserted_inside, T):
    g = torch.Generator(device="cuda").manual_seed(10)
    with torch.inference_mode(inserted_inside):
        bank = _bank(kind, g)
    x, scores = _inputs(g, T)
    with torch.inference_mode():
        _near(moe_linear(x, scores, bank), x, scores, bank)
    x.requires_grad_()
    scores.requires_grad_()
    y = moe_linear(x, scores, bank)
    dx, ds = torch.autograd.grad(y, (x, scores), torch.ones_like(y))
    assert dx.isfinite().all() and ds.isfinite().all() and dx.count_nonzero() > 0 and ds.count_nonzero() > 0


def _far_apart(g, T):
    """Scores whose order no small step changes."""
    return torch.stack([torch.randperm(E, device="cuda", generator=g) for _ in range(T)]).float()


@pytest.mark.parametrize("dual", ["x", "scores"])
def test_forward_mode(dual):
    g = torch.Generator(device="cuda").manual_seed(11)
    bank = _bank("none", g)
    x, scores = _mk(g, 7, K), _far_apart(g, 7)
    tangent = torch.randn(7, K if dual == "x" else E, device="cuda", generator=g)
    with torch.autograd.forward_ad.dual_level():
        if dual == "x":
            y = moe_linear(torch.autograd.forward_ad.make_dual(x, tangent.to(BF)), scores, bank)
        else:
            y = moe_linear(x, torch.autograd.forward_ad.make_dual(scores, tangent), bank)
        out = torch.autograd.forward_ad.unpack_dual(y)
    top, idx = torch.sort(scores.double(), dim=-1, descending=True)
    w = torch.softmax(top[:, :2], -1)
    experts = torch.stack([bank.experts[e].double() for e in range(E)])[idx[:, :2]]                # [T, 2, N, K]
    if dual == "x":
        ref = (w[..., None] * torch.einsum("tjnk,tk->tjn", experts, tangent.to(BF).double())).sum(1)
    else:
        dtop = tangent.double().gather(1, idx[:, :2])
        dw = w * (dtop - (w * dtop).sum(-1, keepdim=True))
        ref = (dw[..., None] * torch.einsum("tjnk,tk->tjn", experts, x.double())).sum(1)
    assert out.tangent is not None and ((out.tangent.double() - ref).norm() / ref.norm()).item() < 2 ** -6


def test_router_under_transforms():
    g = torch.Generator(device="cuda").manual_seed(12)
    s = torch.stack([_far_apart(g, 5) for _ in range(3)])
    idx, w = torch.func.vmap(lambda t: route_tokens(t, 2))(s)
    for b in range(3):
        i1, w1 = route_tokens(s[b], 2)
        assert torch.equal(idx[b], i1) and torch.allclose(w[b], w1, atol=1e-6)
    _, dw = torch.func.jvp(lambda t: route_tokens(t, 2)[1], (s[0],), (torch.ones_like(s[0]),))
    assert dw.abs().max().item() < 1e-6           # weights do not change when all scores grow alike


@pytest.mark.parametrize("T", [1, 5, 30, 400])
@pytest.mark.parametrize("kind", ["none", "q8", "nf4"])
def test_against_the_weights_that_are_multiplied(kind, T):
    """Expanded weights are bf16 as they are; codes on few rows are levels in 11 bits times their scale. What is left are the roundings of
    the chosen experts' outputs and of their sum (2^-8 of themselves each) and sums over K in 32 bits."""
    from eridiffusion_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(T + 20)
    bank = _bank(kind, g)
    x, scores = _inputs(g, T)
    on_codes = kind == "nf4" and 2 * T <= F.CODES_EXPERT_ROWS
    ws = torch.stack([_weight64(e) if kind == "none" or on_codes else e.dequantize(BF).double() for e in bank.experts.values()])
    top, idx = torch.sort(scores.double(), dim=-1, descending=True, stable=True)
    w, xd = torch.softmax(top[:, :2], -1), x.double()
    ref = torch.einsum("tjnk,tk->tjn", ws[idx[:, :2]], xd)
    mag = torch.einsum("tjnk,tk->tjn", ws[idx[:, :2]].abs(), xd.abs())
    err = (w[..., None] * (ref.abs() * 2 ** -8 + mag * (K * 2 ** -23 + (2 ** -11 if on_codes else 0)))).sum(1)
    ref = (w[..., None] * ref).sum(1)
    y = moe_linear(x, scores, bank)
    assert ((y.double() - ref).abs() <= (ref.abs() * 2 ** -8 + err) * 1.01 + 1e-30).all()


@pytest.mark.parametrize("what", ["absent", "resident"])
def test_captures_that_need_the_host_are_refused(what):
    g = torch.Generator(device="cuda").manual_seed(30)
    bank = _bank("none", g)
    x, scores = _inputs(g, 5)
    if what == "absent":
        del bank.experts[2]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(graph):
            moe_linear(x, scores, bank, resident=3 if what == "resident" else None)
    torch.cuda.synchronize()
    y = moe_linear(x, scores, bank)
    if what == "resident":
        _near(y, x, scores, bank)
