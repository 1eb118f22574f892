"""Quantised expert bank and expert selection.

Reference: ``QuantKind{None, Q8, NF4}``, ``QWeight``, ``quantize_weight`` / ``dequantize_to_bf16``,
``ExpertBank{insert, fetch_topk_bf16}`` and ``select_topk_global`` (crates/models/wan22/src/
moe_quant.rs:6-48). In the reference the quantiser is a pass-through and the selection returns the
first k ids. Here the bank stores real int8 / NF4 codes (``memory.quantize``; expanded by the
dequantisation kernel on the GPU) and the selection is a top-k over router scores. On the GPU the tokens
are put into expert order (``F.expert_plan`` / ``expert_dispatch``), meet all experts in one grouped product
(``F.expert_linear``, or ``F.linear_4bit`` on the codes of a 4-bit bank and few rows) and are added up again
(``F.expert_combine``). Nothing is read back where the bank's weights can be stacked (``ExpertBank.stacked``) and all experts are
resident; int8 codes, 4-bit codes of many rows and weights that someone else holds are expanded or joined for each call, only
the experts that some token uses, which are read back.

Wan 2.2 itself is not token-routed: its two "experts" are two whole transformers chosen by the
timestep (``models/nextdit.py``: ``WanDualExpert``); the bank serves that case too (two entries,
one resident in bf16 at a time) and token-routed feed-forward experts.
"""
from __future__ import annotations

import collections
import enum
import sys
import threading

import torch
from torch.autograd import forward_ad

from ..memory import QuantizedTensor, dequantize, quantize
from ..ops import _native as N
from ..ops import functional as F


class QuantKind(str, enum.Enum):
    NONE = "none"
    Q8 = "q8"
    NF4 = "nf4"


def quantize_weight(w: torch.Tensor, kind: QuantKind | str):
    kind = QuantKind(kind)
    if kind == QuantKind.NONE:
        return w.detach().to(torch.bfloat16)
    return quantize(w, "int8" if kind == QuantKind.Q8 else "nf4")


def dequantize_to_bf16(qw) -> torch.Tensor:
    return dequantize(qw, torch.bfloat16) if isinstance(qw, QuantizedTensor) else qw.to(torch.bfloat16)


_MOVING = threading.Lock()


class ExpertBank:
    def __init__(self, kind: QuantKind | str = QuantKind.Q8):
        self.kind = QuantKind(kind)
        self.experts: dict[int, object] = {}
        self._stack = None              # (ids, what their entries are slices of, the stacked weight)
        self._streams = set()           # whose memory stacks are
        self._fixed = False             # a captured graph reads the entries where they lie, or they do not fit twice

    def insert(self, expert_id: int, weight):
        """``weight``: a tensor (quantised on insertion) or an already quantised weight."""
        self.experts[expert_id] = weight if isinstance(weight, QuantizedTensor) else quantize_weight(weight, self.kind)

    def __len__(self):
        return len(self.experts)

    def nbytes(self) -> int:
        return sum(q.nbytes() if isinstance(q, QuantizedTensor) else q.numel() * q.element_size()
                   for q in self.experts.values())

    def fetch_topk_bf16(self, ids):
        """[(id, bf16 weight)] for the ids that are present, in the order asked."""
        self._fix_if_captured()
        ids = [int(i) for i in ids if int(i) in self.experts]
        return [(i, dequantize_to_bf16(e)) for i, e in zip(ids, self._here([self.experts[i] for i in ids]))]

    def _fix_if_captured(self) -> bool:
        """Whether the current stream captures; the entries then stay where they lie, for the replays."""
        captured = _capturing(next((_device(e) for e in self.experts.values()), None))
        self._fixed |= captured
        return captured

    def _here(self, weights):
        """``weights``, entries or stacks, for the current stream: memory of another stream's stack may not be given to others
        before this stream has read it."""
        if self._streams and weights and _device(weights[0]).type == "cuda":
            device = _device(weights[0])
            if self._streams != {_stream(device)}:
                for w in weights:
                    for t in (w.data, w.scale) if isinstance(w, QuantizedTensor) else (w,):
                        t.record_stream(torch.cuda.current_stream(device))
        return weights

    def stacked(self, ids):
        """The weights of the present experts ``ids`` as one [len(ids), N, K] tensor or, for 4-bit codes, one ``QuantizedTensor`` of
        that shape. The entries are moved into it (the same tensor objects on other memory), so that nothing is held twice and a
        change of an entry is a change of the stack. None where someone else holds an entry's memory (a caller's tensor, whose
        changes in place the bank has to follow), where an entry records gradients or was made in inference mode, where a captured
        graph reads the entries (a call under capture moves nothing: the copies would only be recorded), where the device has
        no room for a second copy meanwhile, or where the entries are of different shapes, kinds or devices, or not stored as
        bf16, int4 or NF4."""
        with _MOVING:
            weight = self._stacked(tuple(ids))
        return None if weight is None else self._here([weight])[0]

    def _stacked(self, ids):
        entries = [self.experts[i] for i in ids]
        if self._stack is not None and self._stack[0] == ids and _lie_in(self._stack[1], self._stack[2], entries):
            return self._stack[2]
        if self._fix_if_captured() or self._fixed:
            return None
        self._stack = None
        parts = _stackable(entries)
        if parts is None or not _sole_holders([t for part in parts for t in part]):
            return None
        try:
            with torch.inference_mode(False), torch.no_grad():       # it outlives this call and its mode
                joined = [torch.stack(part) for part in parts]
        except torch.OutOfMemoryError:
            self._fixed = True
            return None
        if joined[0].is_cuda:
            # every stream finds the stack filled, and nothing reads the old memory any more when it is given back
            torch.cuda.synchronize(joined[0].device)
            self._streams.add(_stream(joined[0].device))
        for whole, part in zip(joined, parts):
            for t, home in zip(part, whole):
                t.data = home
        first, weight = entries[0], joined[0]
        if isinstance(first, QuantizedTensor):
            weight = QuantizedTensor(first.kind, joined[0].flatten(0, 1), joined[1].flatten(), (len(ids), *first.shape), first.block)
        self._stack = (ids, joined, weight)
        return weight


def _lie_in(joined, weight, entries) -> bool:
    """Whether the entries still are the slices of their stack."""
    if not isinstance(weight, QuantizedTensor):
        return not any(isinstance(e, QuantizedTensor) for e in entries) and N.ops().are_slices(joined[0], entries)
    like = (weight.kind, tuple(weight.shape[1:]), weight.block)
    return all(isinstance(e, QuantizedTensor) and (e.kind, tuple(e.shape), e.block) == like for e in entries) \
        and N.ops().are_slices(joined[0], [e.data for e in entries]) and N.ops().are_slices(joined[1], [e.scale for e in entries])


def _holders(t):
    """Holders of a tensor's memory: tensors (one more for the storage object made here), and references to that object."""
    storage = t.untyped_storage()
    return storage._cdata, torch._C._storage_Use_Count(storage._cdata), sys.getrefcount(storage)


def _sole_holders(tensors) -> bool:
    """Whether nothing but these tensors holds their memory, so that it may be given up when they are moved."""
    here = collections.Counter(t.untyped_storage()._cdata for t in tensors)
    _, alone, refs = _holders(torch.empty(1))
    return all((users, r) == (alone - 1 + here[key], refs) for key, users, r in map(_holders, tensors))


def _stackable(entries):
    """The tensors to stack, entry by entry: [weights] or [codes, scales]; None where they do not go together."""
    first = entries[0]
    if isinstance(first, QuantizedTensor):
        if first.kind not in ("int4", "nf4") or len(first.shape) != 2 \
                or any(not isinstance(e, QuantizedTensor) or (e.kind, tuple(e.shape), e.block) != (first.kind, tuple(first.shape), first.block) for e in entries):
            return None
        parts = [[e.data for e in entries], [e.scale for e in entries]]
    else:
        if any(isinstance(e, QuantizedTensor) or e.dim() != 2 or e.dtype != torch.bfloat16 for e in entries):
            return None
        parts = [list(entries)]
    for part in parts:
        t0 = part[0]
        if len({id(t) for t in part}) != len(part) or any(
                t.shape != t0.shape or t.dtype != t0.dtype or t.device != t0.device or not t.is_contiguous() or t.requires_grad
                or t.is_inference() for t in part):
            return None
    return parts


def select_topk_global(scores_or_total, k: int):
    """With an int: the first ``k`` ids (the reference's behaviour). With router scores
    ``[tokens, experts]``: the ``k`` experts with the largest total probability mass over all
    tokens, i.e. the set worth keeping resident for this batch."""
    if isinstance(scores_or_total, int):
        return list(range(min(k, scores_or_total)))
    s = scores_or_total.float().softmax(-1).sum(0)
    return torch.topk(s, min(k, s.numel())).indices.tolist()


def _plain(*ts) -> bool:
    """Whether the kernels take these tensors: no forward-mode tangents, no transform (vmap, jvp, ..) and no subclass, for
    which only PyTorch's own operations have rules."""
    if torch._C._are_functorch_transforms_active() or any(type(t) not in (torch.Tensor, torch.nn.Parameter) for t in ts):
        return False
    return forward_ad._current_level < 0 or all(forward_ad.unpack_dual(t).tangent is None for t in ts)


def route_tokens(scores: torch.Tensor, k: int, allowed=None):
    """Per-token top-k routing: returns (expert ids [tokens, k], normalised weights [tokens, k]).
    ``allowed``: restrict the choice to these expert ids (the resident set)."""
    if scores.is_cuda and scores.dim() == 2 and F.get_backend() == "fused" and _plain(scores):
        mask = None
        if allowed is not None:
            mask = torch.zeros(scores.shape[1], dtype=torch.bool)
            mask[list(allowed)] = True
            mask = mask.to(scores.device)
        return F.expert_route(scores, k, allowed=mask)
    s = scores.float()
    if allowed is not None:
        mask = torch.full_like(s, float("-inf"))
        mask[:, list(allowed)] = 0
        s = s + mask
    w, idx = torch.topk(s.softmax(-1), k, dim=-1)
    return idx, w / w.sum(-1, keepdim=True).clamp_min(1e-12)


def moe_linear(x: torch.Tensor, scores: torch.Tensor, bank: ExpertBank, k: int = 2, resident: int | None = None):
    """y[t] = sum_j w[t, j] * x[t] @ W[e(t, j)]^T over the top-k experts of each token, expanding only
    the experts some token uses (at most ``resident`` of them, chosen by ``select_topk_global``)."""
    allowed = select_topk_global(scores, resident) if resident else None
    idx, w = route_tokens(scores, k, allowed)
    y = _moe_grouped(x, idx, w, scores.shape[-1], bank, resident)
    if y is not None:
        return y
    out = None
    for e, We in bank.fetch_topk_bf16(sorted(set(idx.flatten().tolist()))):
        hit = idx == e                                              # [T, k]
        rows = hit.any(-1)
        y = x[rows].to(We.dtype) @ We.t()
        if out is None:
            out = torch.zeros(x.shape[0], We.shape[0], dtype=torch.float32, device=x.device)
        out[rows] += y.float() * (w * hit)[rows].sum(-1, keepdim=True)
    return out.to(x.dtype)


def _moe_grouped(x, idx, w, total: int, bank: ExpertBank, resident):
    """``moe_linear`` as one grouped product on the GPU; None where that does not apply."""
    if not (x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.shape[0] > 0 and F.get_backend() == "fused" and _plain(x, w)):
        return None
    ids = [i for i in range(total) if i in bank.experts]
    if not ids:
        return None
    first = bank.experts[ids[0]]
    if tuple(first.shape) != (first.shape[0], x.shape[1]):
        return None
    weight, entries, captured = None, None, bank._fix_if_captured()
    if not isinstance(first, QuantizedTensor) or (first.kind in ("int4", "nf4") and x.shape[0] * idx.shape[1] <= F.CODES_EXPERT_ROWS):
        weight = bank.stacked(ids)           # all that are present, whatever is allowed: stacked once
    if weight is None:
        # codes of many rows, and weights that are not stacked: a few at a time, and only the experts that some token uses
        # (all of them under capture, where nothing can be read back)
        if not captured:
            used = set(idx.flatten().tolist())
            ids = [i for i in ids if i in used]
        entries = bank._here([bank.experts[i] for i in ids])
        if not ids or any(tuple(e.shape) != tuple(first.shape) for e in entries):
            return None
    if any(_device(e) != x.device for e in entries or (weight,)):
        return None
    if len(ids) != total:                    # the experts' places in the bank; an absent expert adds nothing
        if captured:
            raise RuntimeError("moe_linear: a bank with absent experts cannot be captured (their places are copied from the host)")
        place = torch.full((total,), -1, dtype=torch.int64)
        place[ids] = torch.arange(len(ids))
        idx = place.to(x.device)[idx]
    plan = F.expert_plan(idx, len(ids))
    xs = F.expert_dispatch(x, plan)
    if isinstance(weight, QuantizedTensor):
        y = F.linear_4bit(xs, weight, plan.offsets)
    elif weight is not None:
        y = F.expert_linear(xs, weight, plan.offsets)
    else:
        n, k = first.shape
        step = max(1, min(len(ids), resident or len(ids), _EXPANDED_BYTES // (2 * n * k)))
        y = None
        for a in range(0, len(ids), step):
            part = entries[a:a + step]
            rows_y = F.expert_linear(xs, _expanded(part), plan.offsets[a:a + len(part) + 1])        # zeros for the rows of other experts
            y = rows_y if y is None else y + rows_y
    return F.expert_combine(y, w, plan)


def _capturing(device) -> bool:
    if device is None or device.type != "cuda":
        return False
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream if N._raw_stream is None else N._raw_stream(device.index)


def _device(weight):
    return weight.data.device if isinstance(weight, QuantizedTensor) else weight.device


def _expanded(entries):
    """bf16 weights of some experts, [len(entries), N, K]."""
    if not all(isinstance(e, QuantizedTensor) for e in entries):
        return torch.stack([dequantize_to_bf16(e) for e in entries])
    weight = torch.empty(len(entries), *entries[0].shape, dtype=torch.bfloat16, device=entries[0].data.device)
    for out, q in zip(weight, entries):
        w_bf16 = dequantize(q, torch.bfloat16, out=out)
        if w_bf16 is not out:
            out.copy_(w_bf16)
    return weight


_EXPANDED_BYTES = 1 << 30        # most bytes of expanded experts at a time
