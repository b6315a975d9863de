"""AdamW over many tensors at once (``fh_adamw_many``, fithubert_amd/csrc/adamw_many.hip), moments in 32 or in 8 bits.

The student's own optimizer step (``fh_adamw`` / ``fh_adamw_amp``, reference train.py:407-421) works on one flat fp32 buffer.  What is
trained beside the student -- adapters (``fithubert_amd.adapters``), downstream heads, a teacher or upstream that is fine-tuned as an
ordinary ``nn.Module`` -- comes as a list of tensors, hundreds of them often a few thousand elements long: here the whole list is one
launch per 160 tensors.

* ``adamw_many``: the functional form; ``adamw_moments`` makes the moments it updates.
* ``ManyAdamW``: a ``torch.optim.Optimizer`` over it (parameter groups, schedulers, ``state_dict``).

8-bit moments take 2.03 bytes per parameter instead of 8: m and sqrt(v) as e4m3 codes over one fp32 scale per 256 elements, rounded by
chance with draws that are a function of (seed, place) alone.
"""
from __future__ import annotations

from array import array
from itertools import chain
from operator import attrgetter
from typing import List, Sequence, Tuple

import torch

from . import _lib as L

BLOCK = 256   # elements that share one scale; every tensor's moments begin at a multiple of it

_dtype, _device, _contiguous, _numel, _data_ptr = attrgetter("dtype"), torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.numel, torch.Tensor.data_ptr
_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def moment_blocks(sizes: Sequence[int]) -> int:
    """blocks of 256 elements that tensors of these sizes take in the flat moments"""
    return sum([(n + BLOCK - 1) // BLOCK for n in sizes])


def adamw_moments(params: Sequence[torch.Tensor], bits: int = 32) -> List[torch.Tensor]:
    """Zero moments for ``adamw_many`` over ``params``: [m, v] flat fp32, or with ``bits=8`` [m codes, m scales, root codes, root
    scales] (float8_e4m3fn, one fp32 scale per 256 elements).  Tensor i's part begins at the block that ``moment_blocks`` of the tensors in
    front of it gives; what pads its last block stays zero."""
    if bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits, not {bits}")
    if not params:
        raise ValueError("no tensors")
    nb, dev = moment_blocks([p.numel() for p in params]), params[0].device
    if bits == 32:
        return [torch.zeros(nb * BLOCK, device=dev) for _ in range(2)]
    return [t for _ in range(2) for t in (torch.zeros(nb * BLOCK, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(nb, device=dev))]


def adamw_many(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moments: Sequence[torch.Tensor], *, step: int, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, grad_scale: float = 1.0,
               seed: int = 0) -> None:
    """One AdamW step in place: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2 with g = grad * grad_scale, then
    p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps); ``step`` counts from 1.

    ``params``: contiguous CUDA tensors of one type (fp32, bf16 or fp16) on one device, none twice and none overlapping another (a tensor given
    twice is refused; an overlap cannot be seen).  ``grads``: one per parameter, of its size (in the order of its elements) and all of one type, or None: that parameter and its
    moments are left alone.  ``moments``: as ``adamw_moments`` makes them, updated in place.  Arithmetic is fp32 throughout; a 16-bit parameter is rounded
    to nearest once, so a change below half its spacing is lost.  ``seed`` draws the rounding of 8-bit moments: give each step its own
    (the step's number will do).  Their root is right on average, its square up to 5 % too large.  Runs on the current stream of the tensors' device; all scalars are part of the launch, so a captured
    call repeats the same ``step`` and ``seed`` on every replay."""
    call = _checked(params, grads, moments, step, lr, betas, eps, weight_decay, grad_scale, seed)
    if call is not None:
        _launch(*call)


def _checked(params, grads, moments, step, lr, betas, eps, weight_decay, grad_scale, seed):
    """adamw_many up to its launch, every refusal included: what `_launch` takes (the gradients' contiguous copies among it), None where there is nothing to do"""
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} parameters and {len(grads)} gradients")
    if step < 1 or not all(0 <= b < 1 for b in betas):
        raise ValueError(f"step {step} counts from 1, betas {betas} lie in [0, 1)")
    if not params:
        return None
    L.native_call("adamw_many", chain(params, grads))
    with torch.no_grad():
        dev, pdt = params[0].device, params[0].dtype
        if pdt not in _DT or dev.type != "cuda":
            raise ValueError(f"parameters are fp32, bf16 or fp16 tensors on the GPU, got {pdt} on {dev}")
        held = [g for g in grads if g is not None]
        if not held:
            return None
        gdt = held[0].dtype
        if gdt not in _DT:
            raise ValueError(f"gradients are fp32, bf16 or fp16, got {gdt}")
        # (a call's time on the host is these looks at every tensor: each is one pass of a C function over the list)
        if set(map(_dtype, params)) != {pdt} or set(map(_dtype, held)) != {gdt} or set(map(_device, params)) | set(map(_device, held)) != {dev.index}:
            raise ValueError(f"parameters are of one type, gradients are of one type, all on one GPU ({pdt}, {gdt}, {dev})")
        if not all(map(_contiguous, params)):
            raise ValueError("parameters are contiguous")
        if len(held) == len(grads) and all(map(_contiguous, held)):
            held = grads
        else:
            held = [g if g is None or g.is_contiguous() else g.contiguous() for g in grads]
        sizes = list(map(_numel, params))
        if sizes != (list(map(_numel, held)) if held is grads else [n if g is None else g.numel() for n, g in zip(sizes, held)]):
            raise ValueError("a gradient has another size than its parameter")
        at = list(map(_data_ptr, params))
        if len(set(at)) != len(at) and len({a for a, k in zip(at, sizes) if k}) != len([k for k in sizes if k]):
            raise ValueError("a parameter is given twice")
        gat = list(map(_data_ptr, held)) if held is grads else [0 if g is None else g.data_ptr() for g in held]
        bits = {2: 32, 4: 8}.get(len(moments))
        nb = moment_blocks(sizes)
        want = [(torch.float32, nb * BLOCK)] * 2 if bits == 32 else [(torch.float8_e4m3fn, nb * BLOCK), (torch.float32, nb)] * 2
        if bits is None or any(t.dtype != d or t.numel() != k or t.device != dev or not t.is_contiguous() for t, (d, k) in zip(moments, want)):
            raise ValueError(f"moments do not fit the parameters ({nb} blocks on {dev}): make them with adamw_moments")
        mp = [t.data_ptr() for t in moments]
        if nb and (len(set(mp)) != len(mp) or (mp[0] | mp[len(mp) // 2]) & 15):
            raise ValueError("moments are tensors of their own, m and v at multiples of 16 bytes")
        m, ms, v, vs = (mp[0], None, mp[1], None) if bits == 32 else mp
        scalars = lr, betas[0], betas[1], eps, weight_decay, step, grad_scale, seed & 0xFFFFFFFF
        return dev, (_DT[pdt], _DT[gdt]), array("Q", at), array("Q", gat), array("q", sizes), (bits, m, ms, v, vs), scalars, params, held, held is grads


def _launch(dev, types, at, gat, sizes, moments, scalars, params, held, every):
    with torch.cuda.device(dev):
        L.check(L.lib().fh_adamw_many(*types, at.buffer_info()[0], gat.buffer_info()[0], sizes.buffer_info()[0], len(sizes), *moments, *scalars,
                                      torch.cuda.current_stream(dev).cuda_stream), "fh_adamw_many")
    torch.autograd.graph.increment_version(params if every else [p for p, g in zip(params, held) if g is not None])


class ManyAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` in one launch per parameter group (and type), with ``bits`` = 32 or 8 bits per moment.

    The step count is the group's own (a parameter without a gradient is left out of a step and still shares the count).  ``step`` takes a
    ``grad_scale`` (1 / (world * accumulation * loss scale)).  The moments belong to a group's parameters, types and devices as its first step meets them: a later step or
    ``state_dict`` with others is refused.  Sparse gradients and steps inside a graph capture are refused: the step number
    would be the same on every replay."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, bits: int = 32):
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError(f"lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        if bits not in (8, 32):
            raise ValueError(f"moments are held in 8 or 32 bits, not {bits}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, bits=bits, steps=0))
        self._moments = {}   # (group, device, type) -> [tensors, moments]

    def _sets(self, k, group, anew=False):
        sets = {}
        for p in group["params"]:
            sets.setdefault((k, str(p.device), str(p.dtype)), []).append(p)
        for key, ps in sets.items():
            held = self._moments.get(key)
            if held is None or len(held[0]) != len(ps) or any(a is not b for a, b in zip(held[0], ps)):
                if group["steps"] and not anew:   # (zero moments under a running count: its bias corrections would multiply the step)
                    raise RuntimeError("a group's parameters changed after its first step: add new ones as a group of their own; where a type or a device changed, "
                                       "make a new optimizer and load this one's state_dict (taken before the change) into it")
                self._moments[key] = held = [ps, adamw_moments(ps, group["bits"])]
            yield held

    @torch.no_grad()
    def step(self, closure=None, grad_scale: float = 1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ManyAdamW.step inside a graph capture would repeat one step number: call adamw_many with scalars of your own")
        calls, steps = [], []   # (every refusal comes before the first launch: a refused step leaves all parameters, moments and counts)
        for k, group in enumerate(self.param_groups):
            if all(p.grad is None for p in group["params"]):
                continue
            step = group["steps"] + 1
            steps.append((group, step))
            for ps, moments in self._sets(k, group):
                by = {}
                for p in ps:
                    if p.grad is not None:
                        by.setdefault(p.grad.dtype, None)
                for dt in by:   # one launch per gradient type; the others' tensors sit it out
                    calls.append(_checked(ps, [p.grad if p.grad is not None and p.grad.dtype == dt else None for p in ps], moments, step, float(group["lr"]), group["betas"],
                                          group["eps"], group["weight_decay"], grad_scale, step))
        for call in calls:
            if call is not None:
                _launch(*call)
        for group, step in steps:
            group["steps"] = step
        return loss

    def __getstate__(self):   # copies and pickles carry the moments too
        return dict(super().__getstate__(), _moments=self._moments)

    def state_dict(self):
        """torch's form with the flat moments of each group under 'moments' (in the order of its parameters, one set per device and type)"""
        d = super().state_dict()
        d["moments"] = [[[t.clone() for t in held[1]] for held in self._sets(k, g)] if g["steps"] else None for k, g in enumerate(self.param_groups)]
        return d

    def load_state_dict(self, state_dict):
        d = dict(state_dict)
        if "moments" not in d:
            raise ValueError("a state of ManyAdamW's own: this one holds no 'moments'")
        saved = d.pop("moments")
        before = {n: self.__dict__[n] for n in ("state", "param_groups", "_moments")}
        try:
            super().load_state_dict(d)
            self._moments = {}
            for k, (group, sets) in enumerate(zip(self.param_groups, saved)):
                if sets is None:
                    continue
                here = list(self._sets(k, group, anew=True))
                if len(here) != len(sets):
                    raise ValueError(f"group {k}: the state holds {len(sets)} sets of moments, the parameters make {len(here)}")
                for (_, mine), theirs in zip(here, sets):
                    if [(t.shape, t.dtype) for t in mine] != [(t.shape, t.dtype) for t in theirs]:
                        raise ValueError(f"group {k}: the state's moments do not fit the parameters")
                    for a, b in zip(mine, theirs):
                        a.copy_(b)
        except BaseException:   # (what was there goes on: not the new counts over moments of zeros)
            self.__dict__.update(before)
            raise
