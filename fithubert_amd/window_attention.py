"""Attention inside a sliding window with a few first keys that stay visible (``fh_window_attention_*``,
fithubert_amd/csrc/window_attention.hip): what replaces the full self-attention of modules/module.py:558-564 where a recording is too
long for every frame against every frame, and in streaming, where a few new frames meet a cache.

    y = window_attention(q, k, v, left=128, right=16, sinks=4, key_len=lengths)

Differentiable in q, k and v; no T x T tensor exists in either direction.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _lib as L

_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place: channels contiguous, address and strides multiples of 16 bytes, frames and heads at most 2^23 elements
    apart (strides of axes of length 1 do not count); a contiguous copy otherwise"""
    if t.is_contiguous() and t.data_ptr() % 16 == 0 and t.shape[2] * t.shape[3] <= 1 << 23:
        return t
    vec = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % vec == 0 and (s <= 1 << 23 or not i) for i, (s, n) in enumerate(zip(t.stride()[:-1], t.shape[:-1])) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _dense(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _per_entry(x, B: int, dev: torch.device, name: str) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if not torch.is_tensor(x):
        return torch.full((B,), int(x), dtype=torch.int32, device=dev)
    if x.dim() != 1 or x.shape[0] != B or x.dtype.is_floating_point or x.dtype == torch.bool:
        raise ValueError(f"{name}: one integer per entry ({B}), got {tuple(x.shape)} {x.dtype}")
    if x.dtype == torch.int32 and x.device == dev and x.is_contiguous():
        return x
    return x.to(device=dev).clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32).contiguous() if x.dtype == torch.int64 else x.to(device=dev, dtype=torch.int32).contiguous()


def _desc(q, k, v, left, right, sinks, scale, key_len, q_start) -> L.WindowAttentionC:
    (B, Tq, Hq, dh), (_, Tk, Hkv, _) = q.shape, k.shape
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    many = (B > 1, Tq > 1, Hq > 1), (B > 1, Tk > 1, Hkv > 1)   # (an axis of length 1 is never stepped along: its stride may be anything)
    return L.WindowAttentionC(B, Tq, Tk, Hq, Hkv, dh, left, right, sinks, scale, _ptr(key_len), _ptr(q_start), sq[0] * many[0][0], sq[1] * many[0][1],
                              sq[2] * many[0][2], sk[0] * many[1][0], sk[1] * many[1][1], sk[2] * many[1][2], sv[0] * many[1][0], sv[1] * many[1][1], sv[2] * many[1][2])


def _scratch(dt, d, backward, dev):
    n = L.lib().fh_window_attention_scratch_bytes(dt, C.byref(d), backward)
    if n < 0:
        raise ValueError("fh_window_attention: arguments refused")
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


_stream = torch._C._cuda_getCurrentRawStream   # (what torch.cuda.current_stream(..).cuda_stream gives, without an object on the way: a call of a few frames is the host's time)


def _forward(q, k, v, d, want_lse):
    dt, dev = _DT[q.dtype], q.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _forward(q, k, v, d, want_lse)
    out = q.new_empty(q.shape)
    lse = q.new_empty(q.shape[:3], dtype=torch.float32) if want_lse else None
    scratch = _scratch(dt, d, 0, dev)
    L.check(L.lib().fh_window_attention_forward(dt, C.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(scratch), _stream(dev.index)),
            "fh_window_attention_forward")
    return out, lse


def _backward(q, k, v, out, lse, dout, d):
    L.native_call("window_attention", (q, k, v, dout))
    dt, dev = _DT[q.dtype], q.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _backward(q, k, v, out, lse, dout, d)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    scratch = _scratch(dt, d, 1, dev)
    L.check(L.lib().fh_window_attention_backward(dt, C.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(), dq.data_ptr(),
                                                 dk.data_ptr(), dv.data_ptr(), _ptr(scratch), _stream(dev.index)), "fh_window_attention_backward")
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_len, q_start, d):
        out, lse = _forward(q, k, v, d, True)
        ctx.save_for_backward(q, k, v, out, lse, key_len, q_start)
        ctx.d, ctx.strides = d, (q.stride(), k.stride(), v.stride())
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_len, q_start = ctx.saved_tensors
        q, k, v, d = _aligned(q), _aligned(k), _aligned(v), ctx.d
        if ctx.strides == (q.stride(), k.stride(), v.stride()):
            d.key_len, d.q_start = _ptr(key_len), _ptr(q_start)
        else:   # (saved-tensor hooks may give back tensors with addresses and strides of their own)
            d = _desc(q, k, v, d.left, d.right, d.sinks, d.scale, key_len, q_start)
        return _backward(q, k, v, _dense(out), _dense(lse), _dense(dout), d) + (None, None, None)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, left: int = -1, right: int = -1, sinks: int = 0,
                     key_len: Optional[torch.Tensor] = None, q_start: Union[None, int, torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T over the visible keys) v -> [B][Tq][Hq][dh].

    ``q`` [B][Tq][Hq][dh], ``k``, ``v`` [B][Tk][Hkv][dh]: fp32, bf16 or fp16 on one GPU, dh a multiple of 8 up to 128, Hq a multiple of Hkv (query head h
    reads key head h // (Hq // Hkv)), up to 65535 entries.  Any strides with contiguous channels -- slices of a packed q|k|v projection, a cache longer than it is
    filled -- are read in place when addresses and strides are multiples of 16 bytes, copied otherwise.

    Query i of entry b stands at position p = ``q_start[b]`` + i (default 0; required as soon as Tq != Tk) and sees key s when s < ``key_len[b]``
    (default Tk), s <= p + ``right`` and (s >= p - ``left`` or s < ``sinks``); a ``left`` or ``right`` that is negative, or 2^31 - 1 and more, is no limit.  A row that sees no key
    gives zeros and takes part in no gradient.  Keys that no row of the call sees may hold anything; an infinity or NaN in a key that some rows see
    may reach rows near them that do not (0 x inf), one in a row's query or gradient the gradients of keys near those it sees.  ``scale`` > 0, default dh ** -0.5.

    16-bit modes round the probabilities (backward: and dS) to the element type in front of the second products, and the backward pass takes sum(dout out) from the rounded
    output; softmax and sums are fp32.  In fp16 a dS above
    65504 is infinite and one below 2^-25 is 0: scale the loss so that gradients lie between.  Nothing depends on the order of atomics: equal calls give equal bits.
    The call cannot be recorded (torch.jit.trace, make_fx) and has no forward-mode derivative: both are refused."""
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B][Tq][Hq][dh], k and v [B][Tk][Hkv][dh]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v are fp32, bf16 or fp16, all of one type: got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.device.type != "cuda" or k.device != q.device or v.device != q.device:
        raise ValueError(f"q, k, v live on one GPU: got {q.device}, {k.device}, {v.device}")
    B, Tq, Hq, dh = q.shape
    if Hq < 1 or k.shape[2] < 1 or Hq % k.shape[2] or dh % 8 or not 8 <= dh <= 128:
        raise ValueError(f"heads of 8 to 128 channels (a multiple of 8), query heads a multiple of key heads: got {Hq} x {dh} over {k.shape[2]}")
    if q_start is None and Tq != k.shape[1]:
        raise ValueError(f"{Tq} queries and {k.shape[1]} keys: q_start says where the queries stand")
    scale = dh ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError(f"scale {scale}")
    L.native_call("window_attention", (q, k, v))
    far = (1 << 31) - 1
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    key_len, q_start = _per_entry(key_len, B, q.device, "key_len"), _per_entry(q_start, B, q.device, "q_start")
    d = _desc(q, k, v, max(-1, min(int(left), far)), max(-1, min(int(right), far)), max(0, min(int(sinks), far)), scale, key_len, q_start)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, key_len, q_start, d)
    return _forward(q, k, v, d, False)[0]
