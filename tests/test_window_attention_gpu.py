"""GPU: window attention (fithubert_amd.window_attention) against its definition in 64 bits, forward and backward.

Tolerances are elementwise and follow from the roundings (u = eps / 2 of the element type, nz = the fp32 part):
  scores            off by at most ds = (dh + 8) 2^-24 max sum |q k| scale (a dot product of dh terms and the scaling), so a probability by a
                    factor 1 +- 2 (ds + 2^-21) (its own score and the log-sum-exp's; v_exp_f32 and the sums: the 2^-21)
  nz                2 (ds + 2^-21) + n 2^-24  (a sum over n keys or rows)
  out               u sum P|v| (P rounded in front of the product) + u |out| + nz sum P|v|
  dS = scale P (dP - D): u |dS| (rounded) + nz scale P (|dout||v| + |D|) + scale P eD, eD = sum |dout| e_out (D reads the rounded out)
  dq, dk            the error of dS times |k|, |q| summed, + u |result| + nz sum |dS||k|;   dv: u sum P|dout| + u |dv| + nz sum P|dout|
fp16 adds half its smallest spacing, 2^-25, per rounded P, dS and stored value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fithubert_amd.window_attention import window_attention  # noqa: E402

DEV = "cuda"


def seen(Tq, Tk, key_len, q_start, left, right, sinks):
    p = (q_start[:, None] + torch.arange(Tq, device=DEV))[:, :, None]
    s = torch.arange(Tk, device=DEV)[None, None]
    m = (s < key_len[:, None, None]).expand(-1, Tq, -1)
    if right >= 0:
        m = m & (s <= p + right)
    return m & ((s >= p - left) | (s < sinks)) if left >= 0 else m


def reference(q, k, v, dout, mask, scale):
    """values and bounds in 64 bits: {name: (value, bound)}"""
    u = torch.finfo(q.dtype).eps / 2 if q.dtype != torch.float32 else 2.0 ** -24
    low = q.dtype != torch.float32
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    B, Tq, Hq, dh = q.shape
    G = Hq // k.shape[2]
    Q, K, V = q.double().permute(0, 2, 1, 3), k.double().permute(0, 2, 1, 3).repeat_interleave(G, 1), v.double().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    hidden = ~mask[:, None]
    K, V = (torch.where(mask.any(1)[:, None, :, None], t, 0.0) for t in (K, V))        # (what nobody sees may be anything)
    x = (Q @ K.transpose(2, 3) * scale).masked_fill(hidden, -math.inf)
    ds_max = (dh + 8) * 2.0 ** -24 * (Q.abs() @ K.abs().transpose(2, 3) * scale).max().item()
    P = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e300))
    P = torch.where(hidden, 0.0, P)
    P = P / P.sum(-1, keepdim=True).clamp_min(1e-300)
    n = max(mask.sum(-1).max().item(), mask.sum(1).max().item() * G) + 8
    nz = 2 * (ds_max + 2.0 ** -21) + n * 2.0 ** -24
    up = u if low else 0.0
    vis = mask[:, None].double()
    out = P @ V
    pv = P @ V.abs()
    e_out = (up + nz) * pv + u * out.abs() + tiny * (vis @ V.abs()) + tiny
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    fold = lambda t: back(t).reshape(B, -1, k.shape[2], G, dh).sum(3)  # noqa: E731
    res = {"out": (back(out), back(e_out))}
    if dout is None:
        return res
    dO = dout.double().permute(0, 2, 1, 3)
    D = (dO * out).sum(-1, keepdim=True)
    eD = (dO.abs() * e_out).sum(-1, keepdim=True) + dh * 2.0 ** -24 * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    dS = scale * P * (dO @ V.transpose(2, 3) - D)
    e_dS = up * dS.abs() + nz * scale * P * (dO.abs() @ V.abs().transpose(2, 3) + D.abs()) + scale * P * eD + tiny * vis
    Pt, St, Et = P.transpose(2, 3), dS.transpose(2, 3), e_dS.transpose(2, 3)
    dq, dk, dv = dS @ K, St @ Q, Pt @ dO
    res["dq"] = (back(dq), back(e_dS @ K.abs() + u * dq.abs() + nz * (dS.abs() @ K.abs()) + tiny))
    dk, dv = fold(dk), fold(dv)
    res["dk"] = (dk, fold(Et @ Q.abs() + nz * (St.abs() @ Q.abs())) + u * dk.abs() + tiny)
    res["dv"] = (dv, fold((up + nz) * (Pt @ dO.abs()) + tiny * (vis.transpose(2, 3) @ dO.abs())) + u * dv.abs() + tiny)
    return res


def near(name, got, value, bound):
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), name
    worst = (off / bound.clamp_min(1e-300)).max().item()
    assert (off <= bound + 1e-30).all(), f"{name}: {worst:.2f} times its bound"


def inputs(seed, dtype, B, Tq, Tk, Hq, Hkv, dh, packed=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if packed:
        x = torch.randn(B, Tk, (Hq + 2 * Hkv) * dh, device=DEV, generator=g).to(dtype)
        q, k, v = x.split([Hq * dh, Hkv * dh, Hkv * dh], -1)
        return q.view(B, Tq, Hq, dh), k.view(B, Tk, Hkv, dh), v.view(B, Tk, Hkv, dh), torch.randn(B, Tq, Hq, dh, device=DEV, generator=g).to(dtype)
    return tuple(torch.randn(*s, device=DEV, generator=g).to(dtype) for s in ((B, Tq, Hq, dh), (B, Tk, Hkv, dh), (B, Tk, Hkv, dh), (B, Tq, Hq, dh)))


def run(q, k, v, dout, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = window_attention(q, k, v, **kw)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + torch.autograd.grad(out, (q, k, v), dout)))


def check(q, k, v, dout, left, right, sinks, key_len=None, q_start=None, scale=None):
    B, Tq = q.shape[:2]
    kl = torch.full((B,), k.shape[1], device=DEV) if key_len is None else torch.tensor(key_len, device=DEV)
    qs = torch.zeros(B, dtype=torch.long, device=DEV) if q_start is None else torch.tensor(q_start, device=DEV)
    ref = reference(q, k, v, dout, seen(Tq, k.shape[1], kl, qs, left, right, sinks), scale or q.shape[3] ** -0.5)
    kw = dict(left=left, right=right, sinks=sinks, scale=scale, key_len=None if key_len is None else kl.int(), q_start=None if q_start is None else qs.int())
    got = run(q, k, v, dout, **kw) if dout is not None else {"out": window_attention(q, k, v, **kw)}
    for n in got:
        near(n, got[n], *ref[n])
    return got


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,Hq,Hkv,dh,left,right,sinks", [
    (1, 1, 1, 8, 0, 0, 0), (2, 3, 1, 40, 0, 0, 1), (63, 4, 4, 64, 10, 0, 0), (64, 2, 1, 128, 5, 5, 2), (65, 12, 12, 40, 64, 64, 0),
    (129, 8, 2, 64, 31, 0, 4), (200, 6, 2, 80, 17, 40, 130), (257, 4, 1, 96, 100, 3, 64), (321, 5, 1, 48, -1, 0, 0), (190, 2, 2, 56, 20, -1, 3),
    (130, 2, 2, 64, -1, -1, 0), (515, 4, 2, 128, 70, 0, 16), (700, 2, 1, 64, 0, 0, 0), (400, 3, 3, 72, 5, 200, 1000)])
def test_self_attention(dtype, T, Hq, Hkv, dh, left, right, sinks):
    q, k, v, dout = inputs(T + dh, dtype, 2, T, T, Hq, Hkv, dh)
    check(q, k, v, dout, left, right, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("left,right,sinks", [(20, 0, 0), (20, 10, 5), (0, 0, 0), (-1, 0, 0), (3, -1, 0)])
def test_ragged_lengths_leave_rows_without_keys(dtype, left, right, sinks):
    T = 150
    q, k, v, dout = inputs(7, dtype, 5, T, T, 4, 2, 40)
    got = check(q, k, v, dout, left, right, sinks, key_len=[T, 0, 1, 64, 97])
    assert (got["out"][1] == 0).all() and all((got[n][1] == 0).all() for n in ("dq", "dk", "dv"))
    if left == 20 and sinks == 0:
        assert (got["out"][2, 22:] == 0).all() and (got["dq"][2, 22:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("left,right,sinks", [(20, 0, 0), (3, 9, 0), (-1, 0, 4)])
def test_rows_without_keys_may_hold_anything(dtype, left, right, sinks):
    T = 150
    q, k, v, dout = inputs(8, dtype, 4, T, T, 4, 2, 48)
    kw = dict(left=left, right=right, sinks=sinks, key_len=torch.tensor([100, 0, 1, 64], device=DEV, dtype=torch.int32), q_start=torch.tensor([0, 3, 0, -20], device=DEV, dtype=torch.int32))
    empty = ~seen(T, T, kw["key_len"], kw["q_start"], left, right, sinks).any(-1)
    assert empty[1].all() and empty.sum() > T
    clean = run(q, k, v, dout, **kw)
    for bad in (math.nan, math.inf):
        q2, d2 = q.clone(), dout.clone()
        q2[empty], d2[empty] = bad, bad
        dirty = run(q2, k, v, d2, **kw)
        assert (dirty["out"][empty] == 0).all() and (dirty["dq"][empty] == 0).all()
        assert all(torch.equal(clean[n], dirty[n]) for n in clean), bad


@pytest.mark.parametrize("dtype", TYPES)
def test_what_no_row_sees_may_be_anything(dtype):
    T = 200
    q, k, v, dout = inputs(3, dtype, 2, T, T, 4, 2, 64)
    clean = run(q, k, v, dout, left=16, right=0, sinks=2, key_len=torch.tensor([120, T], device=DEV))
    for bad in (math.inf, -math.inf, math.nan, torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[0, 120:], v2[0, 120:] = bad, bad
        dirty = run(q, k2, v2, dout, left=16, right=0, sinks=2, key_len=torch.tensor([120, T], device=DEV))
        for n in clean:
            assert torch.equal(clean[n], dirty[n]), (n, bad)
        # a cache that is longer than what it holds, and whose oldest frames have been given back
        new = window_attention(q[:, 90:92], k, v, left=16, right=0, sinks=2, q_start=torch.tensor([90, 90], device=DEV))
        k2, v2 = k.clone(), v.clone()
        k2[:, 92:], v2[:, 92:] = bad, bad
        k2[:, 2:74], v2[:, 2:74] = bad, bad
        assert torch.equal(new, window_attention(q[:, 90:92], k2, v2, left=16, right=0, sinks=2, q_start=torch.tensor([90, 90], device=DEV))), bad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,dh,left,sinks", [(3, 1, 1000, 8, 2, 64, 255, 4), (2, 1, 4097, 4, 4, 40, -1, 0), (1, 1, 9000, 16, 1, 128, 5000, 7), (2, 7, 640, 6, 6, 96, 64, 70),
                                                          (1, 16, 3001, 16, 2, 128, -1, 0), (2, 33, 700, 4, 2, 80, 100, 0), (70, 1, 300, 4, 2, 64, 63, 1), (1, 3, 5, 1, 1, 8, 2, 0)])
def test_a_few_frames_against_a_cache(dtype, B, Tq, Tk, Hq, Hkv, dh, left, sinks):
    q, k, v, dout = inputs(Tk + Tq, dtype, B, Tq, Tk, Hq, Hkv, dh)
    lens = [max(Tq, Tk - 13 * b * b) for b in range(B)]
    check(q, k, v, None, left, 0, sinks, key_len=lens, q_start=[n - Tq for n in lens])
    check(q, k, v, dout, left, 2, sinks, key_len=lens, q_start=[n - Tq - 1 for n in lens])     # (and its gradients)
    check(q, k, v, None, left, 0, sinks, key_len=[0] * B, q_start=[n - Tq for n in lens])        # nothing to see


def test_chunks_of_a_stream_give_the_whole():
    T, n = 230, 23
    q, k, v, _ = inputs(5, torch.float16, 2, T, T, 4, 2, 64)
    whole = window_attention(q, k, v, left=50, right=0, sinks=3)
    for i in range(0, T, n):
        part = window_attention(q[:, i:i + n], k, v, left=50, right=0, sinks=3, q_start=i)
        value, bound = reference(q[:, i:i + n], k, v, None, seen(n, T, torch.full((2,), T, device=DEV), torch.full((2,), i, device=DEV), 50, 0, 3), 0.125)["out"]
        near("chunk", part, value, bound)
        near("whole", whole[:, i:i + n], value, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_projections_and_odd_strides(dtype):
    q, k, v, dout = inputs(11, dtype, 2, 100, 100, 6, 2, 40, packed=True)
    assert not q.is_contiguous()
    a = check(q, k, v, dout, 30, 5, 2)
    b = run(*(t.contiguous() for t in (q, k, v)), dout, left=30, right=5, sinks=2)
    assert all(torch.equal(a[n], b[n]) for n in a)
    # head-major tensors, and slices whose addresses and strides no 16-byte access fits
    hm = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        w = torch.zeros(*t.shape[:3], t.shape[3] + 3, device=DEV, dtype=dtype)
        w[..., 1:-2] = t
        odd.append(w[..., 1:-2])
    for other in (hm, odd):
        c = run(*other, dout.transpose(1, 2).contiguous().transpose(1, 2), left=30, right=5, sinks=2)
        assert all(torch.equal(a[n], c[n]) for n in a)


def test_gradients_against_differences():
    T = 40
    q, k, v, dout = (t.double() for t in inputs(2, torch.float32, 1, T, T, 4, 2, 16))
    f = lambda a, b, c: (window_attention(a.float(), b.float(), c.float(), left=9, right=2, sinks=2).double() * dout).sum().item()  # noqa: E731
    got = run(q.float(), k.float(), v.float(), dout.float(), left=9, right=2, sinks=2)
    g = torch.Generator(device=DEV).manual_seed(1)
    for i, n in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            d = torch.randn(q.shape if i == 0 else k.shape, device=DEV, generator=g, dtype=torch.float64)
            h, a, b = 1e-2, [q, k, v], [q, k, v]
            a[i], b[i] = a[i] + h * d, b[i] - h * d
            diff = (f(*a) - f(*b)) / (2 * h)
            # third-order term of the difference (h^2 times values of order 10) and 2^-24 sqrt(2560) |out| of fp32 noise over 2 h
            assert abs(diff - (got[n].double() * d).sum().item()) < 2e-2 * max(1.0, abs(diff)), n


def test_equal_calls_give_equal_bits_and_scale_is_taken():
    q, k, v, dout = inputs(9, torch.bfloat16, 2, 300, 300, 8, 2, 64)
    a = check(q, k, v, dout, 60, 0, 140, scale=0.3)
    for _ in range(3):
        b = run(q, k, v, dout, left=60, right=0, sinks=140, scale=0.3)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_streams_and_a_captured_call():
    q, k, v, dout = inputs(21, torch.bfloat16, 2, 200, 200, 4, 2, 64)
    want = run(q, k, v, dout, left=40, right=0, sinks=4)
    token = window_attention(q[:, 150:151], k, v, left=150, right=0, q_start=150)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = run(q, k, v, dout, left=40, right=0, sinks=4)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(want[n], got[n]) for n in want)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    g = torch.cuda.CUDAGraph()
    start = torch.tensor([150, 150], dtype=torch.int32, device=DEV)
    with torch.cuda.stream(st):
        for _ in range(2):
            torch.autograd.grad(window_attention(*leaves, left=40, right=0, sinks=4), leaves, dout)
            window_attention(q[:, 150:151], k, v, left=150, right=0, q_start=start)
    torch.cuda.current_stream().wait_stream(st)
    with torch.cuda.graph(g):
        out = window_attention(*leaves, left=40, right=0, sinks=4)
        grads = torch.autograd.grad(out, leaves, dout)
        one = window_attention(q[:, 150:151], k, v, left=150, right=0, q_start=start)
    for i in range(4):
        for t in (out, one) + grads:
            t.detach().zero_()
        g.replay()
        torch.cuda.synchronize()
        for n, t in zip(("out", "dq", "dk", "dv"), (out,) + grads):
            assert torch.equal(want[n], t), (n, i)
        assert torch.equal(one, token)
        torch.ones(1000, 1000, device=DEV).cumsum(0).sum().item()
    with torch.no_grad():                                # new inputs and new positions in the captured buffers
        leaves[0].copy_(q.flip(1))
        start.fill_(100)
    g.replay()
    torch.cuda.synchronize()
    again = run(q.flip(1), k, v, dout, left=40, right=0, sinks=4)
    assert torch.equal(again["dk"], grads[1]) and torch.equal(again["out"], out)
    assert torch.equal(one, window_attention(q[:, 150:151], k, v, left=150, right=0, q_start=100))


def test_a_cache_past_32_bit_offsets():
    """the last entries of a cache of more than 2^31 elements"""
    B, Tk, Hkv, dh = 3, 700_000, 8, 128
    k = torch.empty(B, Tk, Hkv, dh, device=DEV, dtype=torch.float16)
    g = torch.Generator(device=DEV).manual_seed(4)
    k[2, -600:] = torch.randn(600, Hkv, dh, device=DEV, generator=g)
    q = torch.randn(B, 1, 16, dh, device=DEV, generator=g).half()
    got = window_attention(q, k, k, left=511, right=0, q_start=torch.full((B,), Tk - 1, device=DEV), key_len=torch.tensor([0, 0, Tk], device=DEV))
    tail = k[2:, -512:].clone()
    value, bound = reference(q[2:], tail, tail, None, torch.ones(1, 1, 512, dtype=torch.bool, device=DEV), dh ** -0.5)["out"]
    near("out", got[2:], value, bound)
    assert (got[:2] == 0).all()


def test_saved_tensors_that_come_back_elsewhere():
    """Activations parked in host memory between the passes, and hooks that give back other strides."""
    q, k, v, dout = inputs(21, torch.bfloat16, 2, 70, 70, 4, 2, 64, packed=True)
    at = dict(left=9, right=3, sinks=2)
    want = run(q, k, v, dout, key_len=torch.tensor([70, 31], device=DEV), q_start=torch.tensor([0, 2], device=DEV), **at)
    other = lambda t: torch.empty((2,) + t.shape, dtype=t.dtype, device=t.device).permute(*range(1, t.dim() + 1), 0)[..., 0].copy_(t)  # noqa: E731
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), other)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        with hooks:
            out = window_attention(*leaves, key_len=torch.tensor([70, 31], device=DEV), q_start=torch.tensor([0, 2], device=DEV), **at)
        torch.empty(1000, device=DEV, dtype=torch.int32).fill_(-1)
        got = torch.autograd.grad(out, leaves, dout)
        assert all(torch.equal(want[n], t) for n, t in zip(("dq", "dk", "dv"), got))


def test_wide_integers_are_limited_not_wrapped():
    q, k, v, _ = inputs(22, torch.float32, 2, 20, 20, 2, 2, 32)
    a = window_attention(q, k, v, left=5, right=0, key_len=torch.tensor([2 ** 32 + 7, 20], device=DEV), q_start=torch.tensor([0, 2 ** 32], device=DEV))
    assert torch.equal(a[0], window_attention(q, k, v, left=5, right=0)[0]) and (a[1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk", [(0, 7, 7), (2, 0, 9), (2, 70, 0), (2, 3, 0), (0, 0, 0)])
def test_no_frames(dtype, B, Tq, Tk):
    q, k, v, dout = inputs(23, dtype, B, Tq, Tk, 4, 2, 32)
    got = run(q, k, v, dout, left=3, right=0, sinks=2, q_start=0)
    assert [got[n].shape for n in ("out", "dq", "dk", "dv")] == [q.shape, q.shape, k.shape, v.shape]
    assert all((got[n] == 0).all() for n in got)


def test_refusals_on_the_gpu():
    q, k, v, _ = inputs(24, torch.bfloat16, 2, 9, 9, 4, 2, 32)
    for kw in (dict(key_len=torch.tensor([1], device=DEV)), dict(key_len=torch.tensor([1.0, 2.0], device=DEV)), dict(q_start=torch.tensor([[1, 2]], device=DEV))):
        with pytest.raises(ValueError):
            window_attention(q, k, v, **kw)
    with pytest.raises(ValueError):
        window_attention(q[:, :3], k, v)                     # where do three queries stand among nine keys?
    with pytest.raises(ValueError):
        window_attention(q, k.cpu(), v)
    y = window_attention(q.requires_grad_(True), k, v)
    g = torch.autograd.grad(y, q, torch.ones_like(y), create_graph=True)[0]
    with pytest.raises(RuntimeError):                        # no second derivatives
        torch.autograd.grad(g.sum(), q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,dh,left,right,sinks", [(2, 40, 300, 4, 2, 64, 30, 0, 0), (2, 40, 300, 4, 2, 40, 30, 7, 3), (2, 3, 200, 6, 2, 128, 5, 2, 1), (3, 70, 500, 2, 2, 96, 0, 0, 70),
                                                                (8, 40, 1024, 8, 8, 64, 100, 3, 2)])
def test_keys_that_no_row_sees_take_no_gradient(dtype, B, Tq, Tk, Hq, Hkv, dh, left, right, sinks):
    """Queries in the middle of a cache: frames in front of the window, between the sinks and the window, and behind the last row's view may hold anything in the backward pass too."""
    q, k, v, dout = inputs(31, dtype, B, Tq, Tk, Hq, Hkv, dh)
    starts, lens = [Tk // 2 - 11 * b for b in range(B)], [Tk - 7 * b for b in range(B)]
    kw = dict(left=left, right=right, sinks=sinks, q_start=torch.tensor(starts, device=DEV), key_len=torch.tensor(lens, device=DEV))
    clean = check(q, k, v, dout, left, right, sinks, key_len=lens, q_start=starts)
    unseen = ~seen(Tq, Tk, kw["key_len"], kw["q_start"], left, right, sinks).any(1)
    assert unseen[:, sinks:starts[-1] - left].all() and unseen[:, starts[0] + Tq + right:].all()
    for bad in (math.inf, -math.inf, math.nan, torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[unseen], v2[unseen] = bad, bad
        dirty = run(q, k2, v2, dout, **kw)
        assert (dirty["dk"][unseen] == 0).all() and (dirty["dv"][unseen] == 0).all(), bad
        assert all(torch.equal(clean[n], dirty[n]) for n in clean), bad


@pytest.mark.parametrize("T,Hq,Hkv,dh,left,right,sinks,v_size,k_size", [(60, 4, 2, 64, 2, 0, 0, 2, 0.25), (200, 4, 2, 64, 31, 3, 2, 8, 0.125), (150, 2, 2, 128, 9, 0, 0, 4, 0.25)])
def test_large_fp16_gradients_stay_finite(T, Hq, Hkv, dh, left, right, sinks, v_size, k_size):
    """A scaled loss: P (dP - D) lies past fp16's 65504 while dS = scale P (dP - D) and every result lie below it.  (The bounds are the other tests'.)"""
    q, k, v, dout = (t * f for t, f in zip(inputs(41, torch.float16, 2, T, T, Hq, Hkv, dh), (k_size, k_size, v_size, 8000)))
    G, scale = Hq // Hkv, dh ** -0.5
    mask = seen(T, T, torch.full((2,), T, device=DEV), torch.zeros(2, dtype=torch.long, device=DEV), left, right, sinks)[:, None]
    Q, K, V, dO = (t.double().permute(0, 2, 1, 3) for t in (q, k, v, dout))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    P = torch.softmax((Q @ K.transpose(2, 3).contiguous() * scale).masked_fill(~mask, -math.inf), -1)
    raw = P * (dO @ V.transpose(2, 3).contiguous() - (dO * (P @ V)).sum(-1, keepdim=True))
    assert raw.abs().max() > 1.5 * 65504 and scale * raw.abs().max() < 65504
    check(q, k, v, dout, left, right, sinks)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Tq", [3, 40])
@pytest.mark.parametrize("left,right", [(-1, 0), (-1, -1), (0, -1), (7, -1), (2 ** 29 + 10, 0), (2 ** 30 + 7, 2 ** 30), (2 ** 31 - 1, 3), (5, 2 ** 31 - 2), (2 ** 31 - 2, 2 ** 31 - 2)])
def test_positions_far_away(dtype, Tq, left, right):
    """Positions, and limits, up to the ends of 32 bits: a row far behind all keys sees them exactly when its limit reaches back that far."""
    starts = [2 ** 31 - 1, 2 ** 30 + 5, 2 ** 29 + 15, 2 ** 29 - 3, 0, -1, -2 ** 29 + 1, -2 ** 29 - 40, -2 ** 30 - 2, -2 ** 31]
    q, k, v, dout = inputs(51, dtype, len(starts), Tq, 50, 4, 2, 32)
    check(q, k, v, dout, -1 if left >= 2 ** 31 - 1 else left, right, 2 if right == 0 else 0, q_start=starts)
    want = run(q, k, v, dout, left=-1 if left >= 2 ** 31 - 1 else left, right=right, q_start=torch.tensor(starts, device=DEV))
    got = run(q, k, v, dout, left=left, right=right, q_start=torch.tensor(starts, device=DEV))
    assert all(torch.equal(want[n], got[n]) for n in want)
