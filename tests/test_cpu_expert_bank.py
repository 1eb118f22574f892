"""Stacking of an expert bank: which entries may be moved, and that every holder of an entry goes on seeing the bank's values."""
import copy
import gc

import pytest
import torch

from eridiffusion_b200.memory import QuantizedTensor, quantize
from eridiffusion_b200.models.moe import ExpertBank

BF = torch.bfloat16


def _weights(n, shape=(24, 64)):
    g = torch.Generator().manual_seed(n)
    return [torch.randn(*shape, generator=g).to(BF) for _ in range(n)]


def test_changes_of_a_callers_tensor_are_seen():
    ws = _weights(3)
    bank = ExpertBank("none")
    for i, w in enumerate(ws):
        bank.insert(i, w)
    bank.stacked(range(3))
    ws[1].add_(1.0)
    assert all(torch.equal(a, b) for (_, a), b in zip(bank.fetch_topk_bf16(range(3)), ws))
    assert bank.stacked(range(3)) is None


def test_entries_that_nobody_else_holds_are_moved():
    ws = _weights(3)
    bank = ExpertBank("none")
    for i, w in enumerate(ws):
        bank.insert(i, w.clone())
    entries = [bank.experts[i] for i in range(3)]
    whole = bank.stacked(range(3))
    assert whole is bank.stacked(range(3)) and torch.equal(whole, torch.stack(ws))
    assert all(bank.experts[i] is e and e.untyped_storage().data_ptr() == whole.untyped_storage().data_ptr() for i, e in enumerate(entries))
    entries[2].mul_(2.0)                                       # a change of an entry is a change of the stack
    assert torch.equal(bank.stacked(range(3))[2], ws[2] * 2)


def test_codes_of_a_callers_weight_stay_the_callers():
    qs = [quantize(w, "nf4") for w in _weights(3)]
    bank = ExpertBank("nf4")
    for i, q in enumerate(qs):
        bank.insert(i, q)
    want = [q.dequantize(torch.float32) for q in qs]
    whole = bank.stacked(range(3))
    assert torch.equal(whole.dequantize(torch.float32), torch.stack(want))
    qs[0].scale.mul_(2.0)                                      # through the caller's object, after the move
    assert torch.equal(bank.stacked(range(3)).dequantize(torch.float32)[0], want[0] * 2)
    held = qs[1].data.view(-1)                                 # another holder of the memory: no further move
    qs[2].data = qs[2].data.clone()
    assert bank.stacked(range(3)) is None
    held.zero_()
    assert torch.equal(bank.experts[1].dequantize(torch.float32), torch.full((24, 64), -1.0) * qs[1].scale.repeat_interleave(64).view(24, 64))


def test_a_replaced_expert_is_stacked_anew():
    ws = _weights(4)
    bank = ExpertBank("none")
    for i in range(3):
        bank.insert(i, ws[i].clone())
    bank.stacked(range(3))
    bank.insert(1, ws[3].clone())
    assert torch.equal(bank.stacked(range(3)), torch.stack([ws[0], ws[3], ws[2]]))
    bank.experts[0].data = ws[1].clone()
    assert torch.equal(bank.stacked(range(3)), torch.stack([ws[1], ws[3], ws[2]]))


@pytest.mark.parametrize("what", ["twice", "dtype", "shape", "gradient", "strides", "kinds", "int8"])
def test_what_is_not_stacked(what):
    a, b = _weights(2, (64, 64))
    bank = ExpertBank("none")
    bank.insert(0, a.clone())
    bank.insert(1, b.clone())
    if what == "twice":
        bank.experts[1] = bank.experts[0]
    elif what == "dtype":
        bank.experts[1] = b.float()
    elif what == "shape":
        bank.experts[1] = b[:32].clone()
    elif what == "gradient":
        bank.experts[1].requires_grad_()
    elif what == "strides":
        bank.experts[1].t_()
    else:
        bank.experts[1] = quantize(b, "nf4" if what == "kinds" else "int8")
        if what == "int8":
            bank.experts[0] = quantize(a, "int8")
    before = {i: (e.dequantize(torch.float32) if isinstance(e, QuantizedTensor) else e.detach().clone()) for i, e in bank.experts.items()}
    assert bank.stacked((0, 1)) is None
    for i, e in bank.experts.items():
        now = e.dequantize(torch.float32) if isinstance(e, QuantizedTensor) else e
        assert now.dtype == before[i].dtype and torch.equal(now, before[i])


def test_copies_of_a_stacked_bank_are_their_own():
    bank = ExpertBank("none")
    for i, w in enumerate(_weights(2)):
        bank.insert(i, w.clone())
    whole = bank.stacked((0, 1)).clone()
    other = copy.deepcopy(bank)
    other.experts[0].zero_()
    gc.collect()
    assert torch.equal(bank.stacked((0, 1)), whole)
    assert other.stacked((0, 1))[0].count_nonzero() == 0 and torch.equal(other.stacked((0, 1))[1], whole[1])


@pytest.mark.parametrize("first", ["stacked", "fetched"])
def test_nothing_moves_once_a_graph_reads_the_bank(first, monkeypatch):
    from eridiffusion_b200.models import moe
    bank = ExpertBank("none")
    for i, w in enumerate(_weights(3)):
        bank.insert(i, w.clone())
    at = [bank.experts[i].data_ptr() for i in range(3)]
    monkeypatch.setattr(moe, "_capturing", lambda device: True)
    if first == "stacked":
        assert bank.stacked(range(3)) is None
    else:
        bank.fetch_topk_bf16([0])
    monkeypatch.undo()
    assert bank.stacked(range(3)) is None                      # a replay reads the entries where they were
    assert [bank.experts[i].data_ptr() for i in range(3)] == at


def test_a_stack_made_before_a_capture_is_kept_by_it(monkeypatch):
    from eridiffusion_b200.models import moe
    ws = _weights(4)
    bank = ExpertBank("none")
    for i in range(3):
        bank.insert(i, ws[i].clone())
    whole = bank.stacked(range(3))
    at = whole.data_ptr()
    monkeypatch.setattr(moe, "_capturing", lambda device: True)
    bank._fix_if_captured()
    assert bank.stacked(range(3)) is whole
    monkeypatch.undo()
    del whole
    bank.insert(3, ws[3].clone())
    assert bank.stacked(range(4)) is None and [bank.experts[i].data_ptr() for i in range(3)] == [at + i * 24 * 64 * 2 for i in range(3)]


def test_memory_of_another_streams_stack_is_recorded(monkeypatch):
    """A stack is ready for every stream when it is made, and what another stream reads of it is not given to others before."""
    from types import SimpleNamespace
    from eridiffusion_b200.models import moe

    class OnGpu(torch.Tensor):
        is_cuda = True
        log = []

        def record_stream(self, stream):
            self.log.append(stream.cuda_stream)
    bank, device, now = ExpertBank("none"), torch.device("cuda", 0), [7]
    for i, w in enumerate(_weights(2)):
        bank.insert(i, w.clone())
    synced = []
    monkeypatch.setattr(torch, "stack", lambda ts: torch.cat([t[None] for t in ts]).as_subclass(OnGpu))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d: synced.append([bank.experts[i].data_ptr() for i in range(2)]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=now[0]))
    monkeypatch.setattr(moe, "_stream", lambda d: now[0])
    monkeypatch.setattr(moe, "_device", lambda w: device)
    monkeypatch.setattr(moe, "_capturing", lambda d: False)
    before = [bank.experts[i].data_ptr() for i in range(2)]
    whole = bank.stacked((0, 1))
    assert synced == [before] and [bank.experts[i].data_ptr() for i in range(2)] != before       # filled before the old memory goes
    assert OnGpu.log == []
    now[0] = 8
    assert bank.stacked((0, 1)) is whole and OnGpu.log == [8] and len(synced) == 1


def test_a_stack_made_in_inference_mode_is_an_ordinary_tensor():
    bank, made_inside = ExpertBank("none"), ExpertBank("none")
    for i, w in enumerate(_weights(2)):
        bank.insert(i, w.clone())
    with torch.inference_mode():
        whole = bank.stacked((0, 1))
        for i, w in enumerate(_weights(2)):
            made_inside.insert(i, w.clone())
        assert made_inside.stacked((0, 1)) is None             # they cannot be saved for a backward pass, as stack or alone
    assert not whole.is_inference() and not any(e.is_inference() for e in bank.experts.values())
    x = torch.ones(1, 64, dtype=BF, requires_grad=True)
    (x @ bank.stacked((0, 1))[0].t()).sum().backward()
    assert x.grad is not None


def test_a_bank_that_does_not_fit_twice_stays_where_it_is(monkeypatch):
    ws = _weights(2)
    bank = ExpertBank("none")
    for i, w in enumerate(ws):
        bank.insert(i, w.clone())
    tries = []

    def full(tensors):
        tries.append(tensors)
        raise torch.OutOfMemoryError
    monkeypatch.setattr(torch, "stack", full)
    assert bank.stacked((0, 1)) is None and bank.stacked((0, 1)) is None and len(tries) == 1
    assert all(torch.equal(bank.experts[i], w) for i, w in enumerate(ws))
