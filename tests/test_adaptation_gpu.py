"""GPU: the adaptation operators together, as a layer uses them -- adapters beside the q | k | v projection, window attention over it, adapters beside
the output projection, backward, one optimizer step -- against the same layer in 64 bits; and its streaming form against the whole recording.

The bounds are carried through the layer to first order (u = eps / 2 of the element type, f = 2^-24; |.| elementwise, E(t) the bound of t, n = terms of a sum):
  adapters   h = s x A^T:  E(h) = s E(x)|A|^T + n f s |x||A|^T + u |h|;   y = x W^T + h B^T + bias:  E(y) = E(x)|W|^T + E(h)|B|^T + n f (magnitudes) + u |part| + u |y|
             backward the same with dy, W, B, A;  dA = G^T x:  E = E(G)^T|x| + |G|^T E(x) + n f |G|^T|x| + u |dA|, dB alike
  attention  scores: E(S) = scale (E(q)|k| + |q| E(k)) + (dh + 8) f scale |q||k|; a probability is off by a factor 1 +- r with r = exp(2 max over the row's visible keys of E(S)
             + 2^-20) - 1;   out: E = P E(v) + (u + r + n f) P|v| + u |out|
             dP = dout v^T: E = E(dout)|v| + |dout| E(v) + dh f |dout||v|;   D = sum dout out: E = sum E(dout)|out| + |dout| E(out) + dh f |dout||out|
             dS = scale P (dP - D): E = scale P (E(dP) + E(D)) + (r + u + n f) scale P (|dP| + |D|)
             dq = dS k: E = E(dS)|k| + |dS| E(k) + n f |dS||k| + u |dq|, dk alike;  dv = P^T dout: E = (r + u + n f) P^T|dout| + P^T E(dout) + u |dv|
fp16 would add its smallest spacing; the layer is run in fp32 and bf16.  Products of two bounds are left out above and paid for by 5 %."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fithubert_amd.adapters import adapter_linear  # noqa: E402
from fithubert_amd.optim import ManyAdamW, adamw_many, adamw_moments  # noqa: E402
from fithubert_amd.window_attention import window_attention  # noqa: E402

DEV = "cuda"
F = 2.0 ** -24


def make(seed, dtype, B, T, D, H, n, R):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, f=1.0: (torch.randn(*s, device=DEV, generator=g) * f).to(dtype)  # noqa: E731
    return dict(x=r(B, T, D), w1=r(3 * D, D, f=D ** -0.5), b1=torch.randn(3 * D, device=DEV, generator=g) * 0.1, w2=r(D, D, f=D ** -0.5), b2=torch.randn(D, device=DEV, generator=g) * 0.1,
                a1=r(n, R, D, f=D ** -0.5), u1=r(n, 3 * D, R, f=0.3 * R ** -0.5), a2=r(n, R, D, f=D ** -0.5), u2=r(n, D, R, f=0.3 * R ** -0.5),
                scaling=torch.rand(n, device=DEV, generator=g) + 0.5, dy=r(B, T, D))


LEAVES = ("x", "a1", "u1", "a2", "u2")


def layer(s, H, start, which, **at):
    B, T, D = s["x"].shape
    qkv = adapter_linear(s["x"], s["w1"], s["b1"], s["a1"], s["u1"], s["scaling"], start, which).view(B, T, 3, H, D // H)
    y = window_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], **at)
    return adapter_linear(y.reshape(B, T, D), s["w2"], s["b2"], s["a2"], s["u2"], s["scaling"], start, which)


def step(s, H, start, which, **at):
    leaves = {n: s[n].detach().clone().requires_grad_(True) for n in LEAVES}
    y = layer(dict(s, **leaves), H, start, which, **at)
    return dict(zip(("y",) + LEAVES, (y.detach(),) + torch.autograd.grad(y, list(leaves.values()), s["dy"])))


def lin(x, ex, w, bias, a, b, scaling, rows, u):
    """adapters forward on [M][K]: y, E(y), h, E(h)"""
    K, R = w.shape[1], a.shape[1]
    y, e = x @ w.T + bias, ex @ w.abs().T + (K + 8) * F * (x.abs() @ w.abs().T + bias.abs())
    h, eh = (torch.zeros(x.shape[0], R, device=DEV, dtype=torch.float64) for _ in range(2))
    for i, j, k in rows:
        f = scaling[k]
        h[i:j] = f * x[i:j] @ a[k].T
        eh[i:j] = f * (ex[i:j] @ a[k].abs().T + (K + 8) * F * (x[i:j].abs() @ a[k].abs().T)) + u * h[i:j].abs()
        part = h[i:j] @ b[k].T
        y[i:j] += part
        e[i:j] += (eh[i:j] + (R + 8) * F * h[i:j].abs()) @ b[k].abs().T + u * part.abs()
    return y, e + u * y.abs(), h, eh


def lin_back(dy, ed, x, ex, w, a, b, scaling, rows, h, eh, u):
    M = x.shape[0]
    bt, at = b.transpose(1, 2), a.transpose(1, 2)
    dx, edx, g, eg = lin(dy, ed, w.T, torch.zeros(w.shape[1], device=DEV, dtype=torch.float64), bt, at, scaling, rows, u)
    out = {"x": (dx, edx)}
    da, db, ea, eb = torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(a), torch.zeros_like(b)
    for i, j, k in rows:
        X, EX, Y, EY, g_, eg_, h_, eh_ = (t[i:j] for t in (x, ex, dy, ed, g, eg, h, eh))
        da[k] += g_.T @ X
        ea[k] += eg_.T @ X.abs() + g_.abs().T @ EX + (M + 8) * F * (g_.abs().T @ X.abs())
        db[k] += Y.T @ h_
        eb[k] += EY.T @ h_.abs() + Y.abs().T @ eh_ + (M + 8) * F * (Y.abs().T @ h_.abs())
    out["a"], out["b"] = (da, ea + u * da.abs()), (db, eb + u * db.abs())
    return out


def visible(T, key_len, left, right, sinks):
    p, k = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)[None]
    return ((k <= p + right) & ((k >= p - left) | (k < sinks)))[None] & (k[None] < key_len[:, None, None])


def expected(s, H, start, which, left, right, sinks, key_len):
    """{name: (value, bound)} of a step in 64 bits"""
    u = F if s["x"].dtype == torch.float32 else torch.finfo(s["x"].dtype).eps / 2
    up = 0.0 if s["x"].dtype == torch.float32 else u
    B, T, D = s["x"].shape
    dh, M = D // H, B * T
    rows = [(i, j, k) for i, j, k in zip(start.tolist(), start.tolist()[1:], which.tolist()) if k >= 0 and j > i]
    d = {n: t.double() for n, t in s.items()}
    x, dy = d["x"].view(M, D), d["dy"].view(M, D)
    zero = torch.zeros_like(x)
    qkv, eqkv, h1, eh1 = lin(x, zero, d["w1"], d["b1"], d["a1"], d["u1"], s["scaling"].double(), rows, u)
    heads = lambda t: t.view(B, T, 3, H, dh).permute(2, 0, 3, 1, 4)  # noqa: E731
    (q, k, v), (eq, ek, ev) = heads(qkv), heads(eqkv)
    tr = lambda t: t.transpose(-1, -2)  # noqa: E731
    mask, scale, n = visible(T, key_len, left, right, sinks)[:, None], dh ** -0.5, T + 8
    S = (q @ tr(k) * scale).masked_fill(~mask, -math.inf)
    eS = torch.where(mask, scale * (eq @ tr(k).abs() + q.abs() @ tr(ek) + (dh + 8) * F * (q.abs() @ tr(k).abs())), 0.0)
    P = torch.where(mask, torch.softmax(S, -1), 0.0)
    r = torch.expm1(2 * eS.amax(-1, keepdim=True) + 2.0 ** -20)
    att = P @ v
    eatt = P @ ev + (up + r + n * F) * (P @ v.abs()) + u * att.abs()
    flat = lambda t: t.permute(0, 2, 1, 3).reshape(M, D)  # noqa: E731
    y, ey, h2, eh2 = lin(flat(att), flat(eatt), d["w2"], d["b2"], d["a2"], d["u2"], s["scaling"].double(), rows, u)
    back = lin_back(dy, zero, flat(att), flat(eatt), d["w2"], d["a2"], d["u2"], s["scaling"].double(), rows, h2, eh2, u)
    res = {"y": (y, ey), "a2": back["a"], "u2": back["b"]}
    unflat = lambda t: t.view(B, T, H, dh).permute(0, 2, 1, 3)  # noqa: E731
    do, edo = (unflat(t) for t in back["x"])
    dP, edP = do @ tr(v), edo @ tr(v).abs() + do.abs() @ tr(ev) + (dh + 8) * F * (do.abs() @ tr(v).abs())
    Dl, eD = (do * att).sum(-1, keepdim=True), (edo * att.abs() + do.abs() * (eatt + (dh + 8) * F * att.abs())).sum(-1, keepdim=True)
    dS = scale * P * (dP - Dl)
    edS = scale * P * (edP + eD) + (r + up + n * F) * scale * P * (dP.abs() + Dl.abs())
    rP = (r + up + n * F) * P
    dq, dk, dv = dS @ k, tr(dS) @ q, tr(P) @ do
    edq = edS @ k.abs() + dS.abs() @ ek + n * F * (dS.abs() @ k.abs()) + u * dq.abs()
    edk = tr(edS) @ q.abs() + tr(dS).abs() @ eq + n * F * (tr(dS).abs() @ q.abs()) + u * dk.abs()
    edv = tr(rP) @ do.abs() + tr(P) @ edo + u * dv.abs()
    pack = lambda *t: torch.stack(t).permute(1, 3, 0, 2, 4).reshape(M, 3 * D)  # noqa: E731
    back = lin_back(pack(dq, dk, dv), pack(edq, edk, edv), x, zero, d["w1"], d["a1"], d["u1"], s["scaling"].double(), rows, h1, eh1, u)
    return dict(res, x=back["x"], a1=back["a"], u1=back["b"])


def near(got, want):
    for n, (value, bound) in want.items():
        off = (got[n].double().view_as(value) - value).abs()
        assert torch.isfinite(got[n]).all(), n
        assert (off <= 1.05 * bound + 1e-30).all(), f"{n}: {(off / bound.clamp_min(1e-300)).max().item():.2f} times its bound"


CASES = [(2, 75, 480, 12, 3, 8, 64, 64, 0, [75, 41]), (3, 33, 64, 4, 2, 16, 5, 0, 2, [33, 1, 20]), (1, 700, 128, 2, 4, 24, 100, 20, 4, [700])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,H,n,R,left,right,sinks,lens", CASES)
def test_a_layer_forward_and_backward(dtype, B, T, D, H, n, R, left, right, sinks, lens):
    s = make(T, dtype, B, T, D, H, n, R)
    start = torch.tensor([T * b for b in range(B + 1)], dtype=torch.int32, device=DEV)      # a request per recording
    which = torch.tensor([(2 * b + 1) % n for b in range(B)], dtype=torch.int32, device=DEV)
    lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = step(s, H, start, which, left=left, right=right, sinks=sinks, key_len=lens)
    near(got, expected(s, H, start, which, left, right, sinks, lens))


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_eager_and_captured(bits):
    """Three steps of the layer and its optimizer, once eager and once with forward and backward replayed from a graph (its leaves its own): the same bits."""
    B, T, D, H, n, R = 2, 60, 96, 4, 3, 8
    s = make(5, torch.bfloat16, B, T, D, H, n, R)
    start = torch.tensor([0, T, 2 * T], dtype=torch.int32, device=DEV)
    which = torch.tensor([2, 0], dtype=torch.int32, device=DEV)
    at = dict(left=8, right=2, sinks=1, key_len=torch.tensor([60, 33], dtype=torch.int32, device=DEV))
    names = LEAVES[1:]
    a = {k: torch.nn.Parameter(s[k].float()) for k in names}
    opt = ManyAdamW(a.values(), lr=1e-2, bits=bits)
    low = lambda p: {k: t.detach().to(torch.bfloat16) for k, t in p.items()}  # noqa: E731
    for _ in range(3):
        grads = step(dict(s, **low(a)), H, start, which, **at)
        for k in names:
            a[k].grad = grads[k].float()
        opt.step()

    b = {k: s[k].float() for k in names}
    moments = adamw_moments(list(b.values()), bits)
    leaves = {k: s[k].clone().requires_grad_(True) for k in LEAVES}
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(s, H, start, which, **at)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(dict(s, **leaves), H, start, which, **at)
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"])
    for i in range(3):
        with torch.no_grad():
            for k in names:
                leaves[k].copy_(b[k])
        for t in grads:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        torch.ones(300, 300, device=DEV).cumsum(0).sum().item()
        adamw_many(list(b.values()), list(grads[1:]), moments, step=i + 1, lr=1e-2, weight_decay=1e-2, seed=i + 1)
    assert all(torch.equal(a[k], b[k]) for k in names)
    assert all(not torch.equal(a[k][2], s[k].float()[2]) for k in names)            # (adapters that requests name have moved,
    moved = {k: (a[k][1] / s[k].float()[1] - (1 - 1e-4) ** 3).abs() for k in names}  # the one that none names has only decayed: lr * weight_decay a step)
    assert all((m[s[k][1] != 0] < 8 * 2.0 ** -24).all() for k, m in moved.items())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_live_requests_frame_by_frame(dtype):
    """Three live requests, each with its adapter and its cache, advance a frame per call: the layer of the whole recordings, row by row."""
    B, T, D, H, n, R = 3, 23, 128, 4, 3, 8
    left, sinks, dh = 6, 2, 32
    s = make(6, dtype, B, T, D, H, n, R)
    frame = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    which = torch.tensor([1, 2, 0], dtype=torch.int32, device=DEV)
    cache = torch.full((2, B, 64, H, dh), float("nan"), dtype=dtype, device=DEV)     # (rows behind the last frame hold nothing yet)
    rows = []
    with torch.no_grad():
        for t in range(T):
            qkv = adapter_linear(s["x"][:, t], s["w1"], s["b1"], s["a1"], s["u1"], s["scaling"], frame, which).view(B, 1, 3, H, dh)
            cache[0, :, t], cache[1, :, t] = qkv[:, 0, 1], qkv[:, 0, 2]
            at = torch.full((B,), t, dtype=torch.int32, device=DEV)
            y = window_attention(qkv[:, :, 0], cache[0], cache[1], left=left, right=0, sinks=sinks, key_len=at + 1, q_start=at)
            rows.append(adapter_linear(y.view(B, D), s["w2"], s["b2"], s["a2"], s["u2"], s["scaling"], frame, which))
    start = torch.arange(0, B * T + 1, T, dtype=torch.int32, device=DEV)
    want = expected(s, H, start, which, left, 0, sinks, torch.full((B,), T, device=DEV))
    near({"y": torch.stack(rows, 1)}, {"y": want["y"]})


def _operators():
    """name -> (a differentiable input, the operator as a function of it)"""
    g = torch.Generator(device=DEV).manual_seed(71)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    q, x = r(2, 9, 4, 16), r(10, 16)
    rest = r(24, 16), r(24), r(2, 8, 16), r(2, 24, 8), torch.ones(2, device=DEV), torch.tensor([0, 4, 10], device=DEV, dtype=torch.int32), torch.tensor([1, 0], device=DEV, dtype=torch.int32)
    return {"window_attention": (q, lambda t: window_attention(t, q, q, left=3, right=0)), "adapter_linear": (x, lambda t: adapter_linear(t, *rest))}


@pytest.mark.parametrize("name", ["window_attention", "adapter_linear"])
def test_compiled_programs_call_the_kernels(name):
    x, f = _operators()[name]
    leaf = x.clone().requires_grad_(True)
    g = torch.compile(lambda t: f(t * 2) + 1, backend="eager")
    assert torch.equal(g(x), f(x * 2) + 1) and torch.equal(g(x + 1), f((x + 1) * 2) + 1)
    y = g(leaf)
    assert torch.equal(torch.autograd.grad(y, leaf, torch.ones_like(y))[0], torch.autograd.grad(f(leaf * 2) + 1, leaf, torch.ones_like(y))[0])


@pytest.mark.parametrize("name", ["window_attention", "adapter_linear"])
def test_no_derivative_is_lost_and_no_trace_is_empty(name):
    """Forward-mode derivatives and recorded programs: a native call would drop the one and leave the other with an output that nothing writes, so both are refused."""
    import torch.autograd.forward_ad as fwAD
    from torch.fx.experimental.proxy_tensor import make_fx
    x, f = _operators()[name]
    want = f(x)
    leaf = x.clone().requires_grad_(True)
    dy = torch.ones_like(want)
    grad = torch.autograd.grad(f(leaf), leaf, dy)[0]
    back = lambda t: torch.autograd.grad(f(t), t, dy)[0]  # noqa: E731
    for nograd in (False, True):
        with fwAD.dual_level(), torch.set_grad_enabled(not nograd):
            for t in (x, leaf):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(fwAD.make_dual(t, torch.ones_like(x)))
            assert torch.equal(f(x), want)                       # (no tangent: nothing to lose)
    with fwAD.dual_level():
        y = f(leaf)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fwAD.make_dual(dy, dy))
    for t, fn in ((x, f), (leaf, f), (leaf, back)):
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(fn, (t,), check_trace=False)
        for kw in ({}, dict(pre_dispatch=True)):
            with pytest.raises(RuntimeError, match="recorded"):
                make_fx(fn, **kw)(t)
    assert torch.equal(f(x), want) and torch.equal(back(leaf), grad)
