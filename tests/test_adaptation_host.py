"""CPU: what window attention, adapter projections and the many-tensor AdamW refuse -- in Python and at the C entries, which check before any launch."""
import ctypes as C

import pytest
import torch

from fithubert_amd import _lib as L
from fithubert_amd.adapters import adapter_linear
from fithubert_amd.optim import ManyAdamW, adamw_many, adamw_moments, moment_blocks
from fithubert_amd.window_attention import window_attention

P = 4096   # an aligned address that no refused call may touch


def _win(**kw):
    d = L.WindowAttentionC()
    for n, x in dict(dict(B=1, Tq=4, Tk=4, Hq=2, Hkv=1, dh=64, left=2, right=0, sinks=0, scale=0.125, q_bs=512, q_ts=128, q_hs=64, k_bs=256, k_ts=64, k_hs=64,
                          v_bs=256, v_ts=64, v_hs=64), **kw).items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("dtype,bad", [(3, {}), (-1, {}), (1, dict(B=-1)), (1, dict(Tq=-1)), (1, dict(Tk=-4)), (1, dict(Hq=3, Hkv=2)), (1, dict(Hkv=0)), (1, dict(dh=12)), (1, dict(dh=136)), (1, dict(dh=0)),
                                       (1, dict(scale=0.0)), (1, dict(scale=-1.0)), (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (1, dict(q_ts=129)), (2, dict(k_hs=4)), (0, dict(v_bs=2)),
                                       (1, dict(B=70000)), (1, dict(Tq=1 << 29)), (1, dict(Tk=1 << 29)), (1, dict(Tq=1 << 28, Hq=8, Hkv=1))])
def test_window_attention_entries_refuse(dtype, bad):
    lib, d = L.lib(), _win(**bad)
    assert lib.fh_window_attention_scratch_bytes(dtype, C.byref(d), 0) == -1
    assert lib.fh_window_attention_forward(dtype, C.byref(d), P, P, P, P, None, P, None) < 0
    assert lib.fh_window_attention_backward(dtype, C.byref(d), P, P, P, P, P, P, P, P, P, P, None) < 0


def test_window_attention_entries_refuse_pointers():
    lib, d = L.lib(), _win()
    assert lib.fh_window_attention_forward(1, None, P, P, P, P, None, None, None) < 0
    for i in range(4):
        for bad in (None, P + 8):
            ptrs = [P] * 4
            ptrs[i] = bad
            assert lib.fh_window_attention_forward(1, C.byref(d), *ptrs, None, None, None) < 0
    for i in range(10):
        for bad in (None,) if i == 5 else (None, P + 8):
            ptrs = [P] * 10
            ptrs[i] = bad
            assert lib.fh_window_attention_backward(1, C.byref(d), *ptrs, None) < 0, i
    far = _win(Tq=1, Tk=100000, left=-1)                   # split over the keys: not without its scratch
    assert lib.fh_window_attention_scratch_bytes(1, C.byref(far), 0) > 0
    assert lib.fh_window_attention_forward(1, C.byref(far), P, P, P, P, None, None, None) < 0
    assert lib.fh_window_attention_forward(1, C.byref(_win(B=0)), None, None, None, None, None, None, None) == 0
    assert lib.fh_window_attention_forward(1, C.byref(_win(Tq=0)), None, None, None, None, None, None, None) == 0


def test_window_attention_refuses():
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    q, k = t(2, 5, 4, 16), t(2, 5, 2, 16)
    for args, kw in [((q[0], k, k), {}), ((q, k, t(2, 6, 2, 16)), {}), ((q, t(1, 5, 2, 16), t(1, 5, 2, 16)), {}), ((q, t(2, 5, 2, 8), t(2, 5, 2, 8)), {}),
                     ((q, k.half(), k), {}), ((q.double(), k.double(), k.double()), {}), ((q, k, k), {}),                     # (the last: not on a GPU)
                     ((q, t(2, 5, 3, 16), t(2, 5, 3, 16)), {}), ((t(2, 5, 4, 12), t(2, 5, 2, 12), t(2, 5, 2, 12)), {})]:
        with pytest.raises(ValueError):
            window_attention(*args, left=3, **kw)


def _ad(**kw):
    d = L.AdapterC()
    for n, x in dict(dict(M=4, K=64, N=64, R=8, n_adapters=2, n_segments=1, seg_start=P, seg_adapter=P, scaling=P), **kw).items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("dtype,bad", [(3, {}), (-1, {}), (1, dict(M=-1)), (1, dict(K=12)), (1, dict(N=0)), (1, dict(N=20)), (1, dict(R=4)), (1, dict(R=136)), (1, dict(R=0)), (1, dict(n_adapters=0)),
                                       (1, dict(n_segments=-1)), (1, dict(seg_start=None)), (1, dict(seg_adapter=None)), (1, dict(scaling=None))])
def test_adapter_entries_refuse(dtype, bad):
    lib, d = L.lib(), _ad(**bad)
    assert lib.fh_adapter_scratch_bytes(dtype, C.byref(d), 1) == -1
    assert lib.fh_adapter_linear_forward(dtype, C.byref(d), P, P, P, P, P, P, P, P, None) < 0
    assert lib.fh_adapter_linear_backward(dtype, C.byref(d), P, P, P, P, P, P, P, P, P, P, None) < 0


def test_adapter_entries_refuse_pointers():
    lib, d = L.lib(), _ad()
    assert lib.fh_adapter_linear_forward(1, None, P, P, P, P, P, P, P, P, None) < 0
    for i in (0, 1, 3, 4, 5, 6):
        for bad in (None, P + 2):
            ptrs = [P] * 8
            ptrs[i] = bad
            assert lib.fh_adapter_linear_forward(1, C.byref(d), *ptrs, None) < 0, i
    for i in range(10):
        for bad in ((P + 2,) if 6 <= i <= 8 else (None, P + 2)):
            ptrs = [P] * 10
            ptrs[i] = bad
            assert lib.fh_adapter_linear_backward(1, C.byref(d), *ptrs, None) < 0, i
    assert lib.fh_adapter_linear_backward(1, C.byref(d), *[P] * 6, None, None, None, None, None) == 0       # no gradient is wanted
    assert lib.fh_adapter_linear_forward(1, C.byref(_ad(M=0)), *[None] * 8, None) == 0


def test_adapter_linear_refuses():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ok = dict(x=torch.zeros(4, 16), weight=torch.zeros(24, 16), bias=torch.zeros(24), lora_a=torch.zeros(2, 8, 16), lora_b=torch.zeros(2, 24, 8), scaling=torch.ones(2), seg_start=i32(0, 4), seg_adapter=i32(0))
    for bad in [dict(x=torch.zeros(4, 8)), dict(x=torch.zeros(16)), dict(weight=torch.zeros(24, 16).half()), dict(lora_a=torch.zeros(3, 8, 16)), dict(lora_b=torch.zeros(2, 24, 4)), dict(bias=torch.zeros(8)), dict(bias=torch.zeros(24).half()),
                dict(scaling=torch.ones(3)), dict(scaling=torch.ones(2).double()), dict(seg_start=i32(0)), dict(seg_start=torch.tensor([0, 4])), dict(seg_adapter=torch.tensor([0])), dict(seg_adapter=i32(0, 1)),
                dict(weight=torch.zeros(20, 16), bias=None, lora_b=torch.zeros(2, 20, 8)), dict(lora_a=torch.zeros(2, 130, 16), lora_b=torch.zeros(2, 24, 130)), dict(lora_a=torch.zeros(0, 8, 16), lora_b=torch.zeros(0, 24, 8), scaling=torch.ones(0)),
                {}]:                                       # (the last: not on a GPU)
        with pytest.raises(ValueError):
            adapter_linear(**dict(ok, **bad))


def test_adamw_entry_refuses():
    lib = L.lib()
    arr = lambda t, *x: (t * len(x))(*x)  # noqa: E731

    def call(pdt=0, gdt=0, p=(P,), g=(P,), n=(300,), count=1, bits=8, m=P, ms=P, v=P, vs=P, lr=1e-3, b1=0.9, b2=0.99, step=1):
        return lib.fh_adamw_many(pdt, gdt, arr(C.c_void_p, *p) if p else None, arr(C.c_void_p, *g) if g else None, arr(C.c_long, *n) if n else None, count, bits, m, ms, v, vs, lr, b1, b2, 1e-8, 0.0, step, 1.0, 0, None)
    for bad in [dict(pdt=3), dict(gdt=-1), dict(bits=16), dict(count=-1), dict(step=0), dict(p=None), dict(g=None), dict(n=None), dict(n=(-1,)), dict(p=(None,)), dict(p=(P + 2,)), dict(g=(P + 1,)), dict(m=None), dict(ms=None), dict(v=None), dict(vs=None),
                dict(m=P + 4), dict(v=P + 8), dict(b1=1.0), dict(b2=-0.1), dict(b1=float("nan")), dict(n=(1 << 39,), bits=32)]:
        assert call(**bad) < 0, bad
    assert call(count=0, p=None, g=None, n=None) == 0 and call(n=(0,)) == 0
    assert lib.fh_adamw_many_blocks(arr(C.c_long, 1, 256, 257, 0), 4) == 4 == moment_blocks([1, 256, 257, 0])
    assert lib.fh_adamw_many_blocks(arr(C.c_long, -1), 1) == -1


def test_adamw_refuses():
    p = [torch.zeros(300), torch.zeros(7)]
    m = adamw_moments(p, 8)
    assert [t.numel() for t in m] == [768, 3, 768, 3] and m[0].dtype == torch.float8_e4m3fn
    assert [t.numel() for t in adamw_moments(p)] == [768, 768]
    for args in [(p, [p[0]], m), (p, [torch.zeros(300), torch.zeros(7)], m)]:      # (the last: not on a GPU)
        with pytest.raises(ValueError):
            adamw_many(*args, step=1, lr=1e-3)
    for bits in (4, 16):
        with pytest.raises(ValueError):
            adamw_moments(p, bits)
        with pytest.raises(ValueError):
            ManyAdamW([torch.zeros(3, requires_grad=True)], bits=bits)
    with pytest.raises(ValueError):
        adamw_moments([])
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            ManyAdamW([torch.zeros(3, requires_grad=True)], **bad)


@pytest.mark.parametrize("bad", [dict(q_ts=(1 << 23) + 8), dict(k_hs=(1 << 23) + 8), dict(k_ts=-64), dict(q_bs=-512), dict(Hq=1 << 18, dh=64)])
def test_window_attention_entries_refuse_strides(bad):
    lib, d = L.lib(), _win(**bad)
    assert lib.fh_window_attention_scratch_bytes(1, C.byref(d), 1) == -1
    assert lib.fh_window_attention_forward(1, C.byref(d), P, P, P, P, None, P, None) < 0
    assert lib.fh_window_attention_backward(1, C.byref(d), P, P, P, P, P, P, P, P, P, P, None) < 0


@pytest.mark.parametrize("K,N", [(0, 24), (16, 0)])
def test_adapter_linear_refuses_no_channels(K, N):
    with pytest.raises(ValueError, match="multiples of 8"):
        adapter_linear(torch.zeros(4, K), torch.zeros(N, K), None, torch.zeros(2, 8, K), torch.zeros(2, N, 8), torch.ones(2), torch.tensor([0, 4], dtype=torch.int32), torch.tensor([0], dtype=torch.int32))


def test_window_attention_refuses_limits():
    q = torch.zeros(2, 5, 4, 16)
    for kw in (dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            window_attention(q, q, q, **kw)


def test_native_calls_refuse_what_cannot_see_them():
    """Forward-mode derivatives and recorded programs: a native call would drop the one and leave the other with an output that nothing writes."""
    import torch.autograd.forward_ad as fwAD
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.ones(3)

    def f(t):
        L.native_call("f", (t, None))
        return t.new_empty(3).fill_(2)
    assert (f(x) == 2).all()
    with fwAD.dual_level():
        assert (f(x) == 2).all()
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(fwAD.make_dual(x, x))
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(f, (x,), check_trace=False)
    for kw in ({}, dict(tracing_mode="fake"), dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(f, **kw)(x)
    assert (f(x) == 2).all()
    p = [torch.zeros(300)]
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        adamw_many([fwAD.make_dual(p[0], p[0])], p, adamw_moments(p), step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(lambda t: adamw_many([t], [t], adamw_moments([t]), step=1, lr=1e-3))(p[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_do_not_start_anew_under_a_running_count(bits):
    """Parameters that change type after their first step keep no moments that fit: going on with zeros and the old step number would multiply the step."""
    layer = torch.nn.Linear(20, 30)
    opt = ManyAdamW(layer.parameters(), bits=bits)
    group = opt.param_groups[0]
    list(opt._sets(0, group))                              # (what the first step does ...)
    layer.double()                                         # nothing is lost before it has counted
    layer.float()
    list(opt._sets(0, group))
    group["steps"] = 1                                     # (... and counts)
    opt._moments[next(iter(opt._moments))][1][-1].fill_(3)
    saved = opt.state_dict()
    layer.bfloat16()
    with pytest.raises(RuntimeError, match="changed"):
        list(opt._sets(0, group))
    with pytest.raises(RuntimeError, match="changed"):
        opt.state_dict()
    layer.float()
    assert (list(opt._sets(0, group))[0][1][-1] == 3).all()
    layer.bfloat16()
    other = ManyAdamW(layer.parameters(), bits=bits)       # the way over: an optimizer of the new parameters that loads the state
    other.load_state_dict(saved)
    assert other.param_groups[0]["steps"] == 1 and (list(other._sets(0, other.param_groups[0]))[0][1][-1] == 3).all()


@pytest.mark.parametrize("sinks", [1, 64, 1000, 30001])
@pytest.mark.parametrize("B,Hq,Hkv,T", [(1, 16, 4, 30001), (8, 16, 16, 30001), (64, 12, 12, 1500), (2, 12, 12, 499)])
def test_window_attention_workspace_stays_in_proportion(B, Hq, Hkv, T, sinks):
    """The sink blocks' partial sums: no more workgroups than fill the chip share them, so the workspace is at most 1024 blocks of 128 keys (dk and dv, fp32) beside D,
    and nothing where no block is shared."""
    sinks = min(sinks, T)
    for dtype in (0, 1, 2):
        d = _win(B=B, Tq=T, Tk=T, Hq=Hq, Hkv=Hkv, left=1023, sinks=sinks, q_bs=T * Hq * 64, q_ts=Hq * 64, k_bs=T * Hkv * 64, k_ts=Hkv * 64, v_bs=T * Hkv * 64, v_ts=Hkv * 64)
        n = L.lib().fh_window_attention_scratch_bytes(dtype, C.byref(d), 1)
        rows = B * T * Hq * 4
        blocks = B * Hkv * -(-sinks // 64)
        assert rows <= n <= rows + 16 + (1024 + blocks) * 128 * 2 * 64 * 4, (dtype, n)
        if blocks >= 1024 * 2 or T * (Hq // Hkv) <= 1024:
            assert n <= rows + 16, (dtype, n)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_state_leaves_the_optimizer(bits):
    make = lambda *sizes: ManyAdamW([{"params": [torch.nn.Parameter(torch.zeros(n)) for n in s]} for s in sizes], bits=bits)  # noqa: E731
    opt, other = make((300, 7), (600,)), make((300, 7), (900,))
    for o, x in ((opt, 3), (other, 4)):
        for k, group in enumerate(o.param_groups):
            for _, moments in list(o._sets(k, group)):
                moments[-1].fill_(x)
            group["steps"] = x
    with pytest.raises(ValueError):
        opt.load_state_dict(other.state_dict())
    without = {k: v for k, v in other.state_dict().items() if k != "moments"}
    with pytest.raises(ValueError):                        # (torch.optim.AdamW's, say)
        opt.load_state_dict(without)
    assert [g["steps"] for g in opt.param_groups] == [3, 3]
    for k, group in enumerate(opt.param_groups):
        assert all((m[-1] == 3).all() for _, m in opt._sets(k, group))
