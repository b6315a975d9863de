"""Low-rank adapters of many requests beside one frozen projection (``fh_adapter_linear_*``, fithubert_amd/csrc/adapters.hip).

One upstream encoder serves -- or trains -- several downstream tasks: the rows of a batch belong to requests, each request names its
task's adapter, and every Linear of the shared encoder (modules/module.py:498-515) becomes

    y = adapter_linear(x, weight, bias, lora_a, lora_b, scaling, seg_start, seg_adapter)

i.e. y[i] = x[i] weight^T + bias + scaling[a] (x[i] lora_a[a]^T) lora_b[a]^T with the adapter a of the row's request.  Differentiable in x, lora_a and
lora_b; the projection is frozen.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
import torch.nn.functional as F

from . import _lib as L

_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _dense(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _desc(x, a, N, scaling, start, which) -> L.AdapterC:
    (M, K), (n, R, _) = x.shape, a.shape
    return L.AdapterC(M, K, N, R, n, which.shape[0], start.data_ptr(), which.data_ptr(), scaling.data_ptr())


def _scratch(dt, d, backward, dev):
    n = L.lib().fh_adapter_scratch_bytes(dt, C.byref(d), backward)
    if n < 0:
        raise ValueError("fh_adapter_linear: arguments refused")
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


_stream = torch._C._cuda_getCurrentRawStream   # (what torch.cuda.current_stream(..).cuda_stream gives, without an object on the way: a call of a few rows is the host's time)


def _forward(x, weight, bias, a, b, scaling, start, which):
    dt, dev = _DT[x.dtype], x.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _forward(x, weight, bias, a, b, scaling, start, which)
    d = _desc(x, a, weight.shape[0], scaling, start, which)
    h, y = x.new_empty((x.shape[0], a.shape[1])), x.new_empty((x.shape[0], weight.shape[0]))
    scratch = _scratch(dt, d, 0, dev)
    L.check(L.lib().fh_adapter_linear_forward(dt, C.byref(d), x.data_ptr(), weight.data_ptr(), _ptr(bias), a.data_ptr(), b.data_ptr(), h.data_ptr(), y.data_ptr(),
                                              _ptr(scratch), _stream(dev.index)), "fh_adapter_linear_forward")
    return y, h


def _backward(x, weight, a, b, scaling, start, which, h, dy, need):
    L.native_call("adapter_linear", (x, weight, a, b, scaling, dy))
    dt, dev = _DT[x.dtype], x.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _backward(x, weight, a, b, scaling, start, which, h, dy, need)
    d = _desc(x, a, weight.shape[0], scaling, start, which)
    dx, da, db = (t.new_empty(t.shape) if n else None for t, n in zip((x, a, b), need))
    scratch = _scratch(dt, d, 1, dev)
    L.check(L.lib().fh_adapter_linear_backward(dt, C.byref(d), x.data_ptr(), weight.data_ptr(), a.data_ptr(), b.data_ptr(), h.data_ptr(), dy.data_ptr(),
                                               _ptr(dx), _ptr(da), _ptr(db), _ptr(scratch), _stream(dev.index)), "fh_adapter_linear_backward")
    return dx, da, db


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, a, b, scaling, start, which):
        y, h = _forward(x, weight, bias, a, b, scaling, start, which)
        ctx.save_for_backward(x, weight, a, b, scaling, start, which, h)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, a, b, scaling, start, which, h = ctx.saved_tensors
        need = ctx.needs_input_grad
        # (saved-tensor hooks may give back other strides)
        dx, da, db = _backward(_dense(x), _dense(weight), _dense(a), _dense(b), scaling.contiguous(), start.contiguous(), which.contiguous(), _dense(h), _dense(dy),
                               (need[0], need[3], need[4]))
        return dx, None, None, da, db, None, None, None


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: torch.Tensor,
                   seg_start: torch.Tensor, seg_adapter: torch.Tensor) -> torch.Tensor:
    """x [rows][K] (or [..][K], rows counted in order) -> [..][N].

    ``weight`` [N][K], ``lora_a`` [adapters][R][K], ``lora_b`` [adapters][N][R]: x's type (fp32, bf16 or fp16); ``bias`` [N] or None and ``scaling`` [adapters]: fp32.
    Request s is the rows ``seg_start[s]`` .. ``seg_start[s + 1]`` - 1 (int32, ascending, one more than there are requests) and uses adapter ``seg_adapter[s]`` (int32; -1, or
    any number that is no adapter's: none).  Rows in front of the first and behind the last request get the shared projection alone.  Several requests may
    name one adapter; both tensors stay on the device and are not looked at on the host.

    K and N are multiples of 8; a rank that is no multiple of 8 is padded with zeros (copies of the factors in every call: better keep them padded), at
    most 128.  16-bit modes round x lora_a^T * scaling (backward: dy lora_b * scaling) to the element type; where many requests are short (under 16 rows on average in
    a batch that is too large for the kernel of few rows) the adapter's part of y (dx) is rounded once more before it is added.  Sums are fp32 and the gradients of the factors leave them rounded once.  ``weight``, ``bias`` and ``scaling`` take no gradient: one that requires it is refused.
    The call cannot be recorded (torch.jit.trace, make_fx) and has no forward-mode derivative: both are refused."""
    if x.dim() < 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError(f"x [..][K], weight [N][K], lora_a [n][R][K], lora_b [n][N][R]: got {tuple(x.shape)}, {tuple(weight.shape)}, {tuple(lora_a.shape)}, {tuple(lora_b.shape)}")
    (N, K), (n, R) = weight.shape, lora_a.shape[:2]
    if x.shape[-1] != K or lora_a.shape != (n, R, K) or lora_b.shape != (n, N, R) or n < 1:
        raise ValueError(f"x [..][K], weight [N][K], lora_a [n][R][K], lora_b [n][N][R]: got {tuple(x.shape)}, {tuple(weight.shape)}, {tuple(lora_a.shape)}, {tuple(lora_b.shape)}")
    dt = x.dtype
    if dt not in _DT or weight.dtype != dt or lora_a.dtype != dt or lora_b.dtype != dt:
        raise ValueError(f"x, weight and the factors are fp32, bf16 or fp16, all of one type: got {x.dtype}, {weight.dtype}, {lora_a.dtype}, {lora_b.dtype}")
    if K < 8 or N < 8 or K % 8 or N % 8 or not 1 <= R <= 128:
        raise ValueError(f"K {K} and N {N} are multiples of 8, the rank {R} lies in 1 .. 128")
    if scaling.shape != (n,) or scaling.dtype != torch.float32 or (bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32)):
        raise ValueError("scaling [n] and bias [N] are fp32")
    if seg_adapter.dim() != 1 or seg_start.shape != (seg_adapter.shape[0] + 1,) or seg_start.dtype != torch.int32 or seg_adapter.dtype != torch.int32:
        raise ValueError(f"seg_start [requests + 1] and seg_adapter [requests] are int32: got {tuple(seg_start.shape)} {seg_start.dtype}, {tuple(seg_adapter.shape)} {seg_adapter.dtype}")
    gpu = x.get_device()   # (-1: not on one)
    if gpu < 0 or not (weight.get_device() == lora_a.get_device() == lora_b.get_device() == scaling.get_device() == seg_start.get_device() == seg_adapter.get_device() == gpu) \
            or (bias is not None and bias.get_device() != gpu):
        raise ValueError(f"all tensors live on one GPU (x: {x.device})")
    grad = torch.is_grad_enabled()
    if grad and (weight.requires_grad or scaling.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("the shared projection and the scalings are frozen: detach weight, bias and scaling")
    L.native_call("adapter_linear", (x, weight, bias, lora_a, lora_b, scaling))
    if R % 8:
        lora_a, lora_b = F.pad(lora_a, (0, 0, 0, -R % 8)), F.pad(lora_b, (0, -R % 8))
    flat = _dense(x if x.dim() == 2 else x.reshape(-1, K))
    args = (flat, _dense(weight), _dense(bias) if bias is not None else None, _dense(lora_a), _dense(lora_b), scaling.contiguous(), seg_start.contiguous(), seg_adapter.contiguous())
    if grad and (x.requires_grad or lora_a.requires_grad or lora_b.requires_grad):
        y = _AdapterLinear.apply(*args)
    else:
        y = _forward(*args)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)
