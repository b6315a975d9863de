"""GPU: one AdamW step over many tensors (fithubert_amd.optim) against its formulas in 64 bits.

Tolerances: every fp32 operation is off by 2^-24 of its result.  m is two products and a sum (4 2^-24 of |b1 m| + |(1 - b1) g|), v the same (6 2^-24 v),
the update a square root, a product, a sum and two divisions more (16 2^-24 of its value), the parameter's own products and difference 4 2^-24 |p|, and
one rounding to its type, u = eps / 2.  8-bit moments: a code may be either neighbour of the exact value, so it is off by less than
one spacing: 1/8 of the value, or 2^-9 of the scale where codes are subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fithubert_amd.optim import BLOCK, ManyAdamW, adamw_many, adamw_moments  # noqa: E402

DEV = "cuda"
E = 2.0 ** -24
H = dict(step=3, lr=2e-3, betas=(0.9, 0.98), eps=1e-6, weight_decay=0.05)


def tensors(seed, sizes, dtype, gdtype, misalign=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ps, gs = [], []
    for i, n in enumerate(sizes):
        k = 1 + i % 3 if misalign else 0
        ps.append((torch.randn(n + k, device=DEV, generator=g) * 0.1).to(dtype)[k:])
        gs.append((torch.randn(n + k, device=DEV, generator=g) * 10.0 ** -(i % 5)).to(gdtype)[k:])
    return ps, gs


def pieces(moments, sizes):
    """(m, v) of each tensor in 64 bits"""
    at, got = 0, []
    for n in sizes:
        pad = -(-n // BLOCK) * BLOCK
        if len(moments) == 2:
            got.append(tuple(t[at:at + n].double() for t in moments))
        else:
            m, r = ((moments[i][at:at + pad].double().view(-1, BLOCK) * moments[i + 1][at // BLOCK:(at + pad) // BLOCK, None].double()).view(-1)[:n] for i in (0, 2))
            got.append((m, r * r))
        at += pad
    return got


def expect(p, g, m, v, grad_scale=1.0, step=3, lr=2e-3, betas=(0.9, 0.98), eps=1e-6, weight_decay=0.05):
    u = torch.finfo(p.dtype).eps / 2 if p.dtype != torch.float32 else E
    p, g = p.double(), g.double() * grad_scale
    (b1, b2) = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em, ev = 6 * E * (b1 * m.abs() + (1 - b1) * g.abs()), 10 * E * v1
    den = (v1 / (1 - b2 ** step)).sqrt() + eps
    step_ = lr / (1 - b1 ** step) * m1 / den
    new = p * (1 - lr * weight_decay) - step_
    bound = 4 * E * p.abs() + 20 * E * step_.abs() + lr / (1 - b1 ** step) * em / den + u * new.abs() + (2.0 ** -25 if u == 2.0 ** -11 else 0)
    return new, bound, m1, em, v1, ev


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,misalign", [([1], False), ([255, 256, 257, 1, 4096, 5000], False), ([3, 1027, 0, 7, 64, 300], True), ([17 * (i % 9) + i for i in range(333)], False)])
def test_two_steps(bits, dtype, gdtype, sizes, misalign):
    ps, gs = tensors(len(sizes), sizes, dtype, gdtype, misalign)
    moments = adamw_moments(ps, bits)
    for k in range(2):
        before, old = pieces(moments, sizes), [p.clone() for p in ps]
        adamw_many(ps, gs, moments, grad_scale=0.25, seed=k, **H)
        at = 0
        for p, o, g, (m, v), (m2, v2), n in zip(ps, old, gs, before, pieces(moments, sizes), sizes):
            new, bound, m1, em, v1, ev = expect(o, g, m, v, 0.25, **H)
            assert ((p.double() - new).abs() <= bound).all()
            if bits == 32:
                assert ((m2 - m1).abs() <= em).all() and ((v2 - v1).abs() <= ev).all()
            elif n:
                blocks = -(-n // BLOCK)
                for got, want, scale in ((m2, m1, moments[1]), (v2.sqrt(), v1.sqrt(), moments[3])):
                    pad = torch.nn.functional.pad(want, (0, blocks * BLOCK - n)).view(-1, BLOCK)
                    sc = scale[at:at + blocks].double()
                    top = pad.abs().amax(1).clamp_min(1e-30)
                    assert ((sc * 448 - top).abs() <= 20 * E * top).all()
                    near = torch.maximum(want.abs() * (0.125 + 1e-5), sc.repeat_interleave(BLOCK)[:n] * 2.0 ** -9 * 1.0001)
                    assert ((got - want).abs() <= near).all()
                    assert ((got == 0) | (got.sign() == want.sign())).all()
                assert (m2[m1 == 0] == 0).all() and (v2[v1 > 0] > 0).all()
            at += -(-n // BLOCK)
    for t in moments:      # what pads the last block stays zero
        if t.dtype != torch.float32 or bits == 32:
            at = 0
            for n in sizes:
                pad = -(-n // BLOCK) * BLOCK
                assert (t[at + n:at + pad].float() == 0).all()
                at += pad


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def test_codes_are_the_formulas_codes():
    """the rounding, restated in fp32: every code is equal, so a step can be repeated from its seed"""
    n, seed = 40 * BLOCK, 12345
    ps, gs = tensors(1, [n], torch.float32, torch.float32)
    gs[0] *= torch.logspace(-6, 0, n, device=DEV)
    moments = adamw_moments(ps, 8)
    adamw_many(ps, gs, moments, seed=seed, **H)
    h = _mix(torch.arange(n, device=DEV) ^ _mix(torch.tensor([(seed * 0x9E3779B9 + 0x27D4EB2F) & 0xFFFFFFFF], device=DEV)))
    m = gs[0] * (1 - 0.9)
    r = ((gs[0] * gs[0]) * (1 - 0.98)).sqrt()
    for t, draw, i in ((m, h & 0xFFFF, 0), (r, h >> 16, 2)):
        x = t.view(-1, BLOCK)
        top = x.abs().amax(1).clamp_min(1e-30)
        a = (x.abs() * (torch.reciprocal(top) * 448.0)[:, None])
        q = torch.exp2((torch.frexp(a).exponent - 1).clamp_min(-6).float() - 3)
        code = (torch.floor(a / q + (draw.float() / 65536).view(-1, BLOCK)) * q).clamp_max(448.0)
        if i == 2:
            code = torch.where((a > 0) & (code == 0), 2.0 ** -9, code)
        want = (code * torch.where(x < 0, -1.0, 1.0)).to(torch.float8_e4m3fn)
        assert torch.equal(want.float().view(-1), moments[i].float())
        assert torch.equal(top * (1 / 448.0), moments[i + 1])


def test_rounding_by_chance_keeps_the_average():
    """a small change per step, far below a code's spacing, arrives on average: 400 steps of a constant gradient bring the root to |g|"""
    n = 64 * BLOCK
    p = [torch.zeros(n, device=DEV)]
    g = torch.full((n,), 1e-3, device=DEV)
    g[::BLOCK] = 1.0                                     # each block's scale belongs to another element
    moments = adamw_moments(p, 8)
    for k in range(1, 401):
        adamw_many(p, [g], moments, step=k, lr=0.0, betas=(0.9, 0.99), seed=k)
    m, v = pieces(moments, [n])[0]
    small = torch.ones(n, dtype=torch.bool, device=DEV)
    small[::BLOCK] = False
    # the mean over 16320 elements, each off by at most one spacing (1/8) with a memory of 1 / (1 - beta) = 100 (10) steps of independent draws
    assert abs(m[small].mean().item() / 1e-3 - 1) < 0.02
    want = (1 - 0.99 ** 400) * 1e-6
    assert abs(v[small].mean().item() / want - 1) < 0.10


def test_not_finite_harms_itself_alone():
    for bits in (8, 32):
        n = 600
        ps, gs = tensors(2, [n, 70], torch.float32, torch.float32)
        ref = [p.clone() for p in ps]
        g2 = [g.clone() for g in gs]
        g2[0][5], g2[0][300] = math.inf, math.nan
        ma, mb = adamw_moments(ps, bits), adamw_moments(ps, bits)
        for k in range(2):
            adamw_many(ref, gs, ma, seed=k, **H)
            adamw_many(ps, g2, mb, seed=k, **H)
        bad = torch.zeros(n, dtype=torch.bool, device=DEV)
        bad[5] = bad[300] = True
        assert torch.isnan(ps[0][bad]).all() and torch.equal(ps[1], ref[1])
        blocks_hit = torch.zeros(n, dtype=torch.bool, device=DEV)
        blocks_hit[:512] = True                          # (their blocks' scales may have lost their largest element: codes differ)
        assert torch.equal(ps[0][~blocks_hit], ref[0][~blocks_hit]) and torch.isfinite(ps[0][~bad]).all()
        if bits == 8:
            assert torch.isnan(mb[0][:n].float()[bad]).all() and torch.isfinite(mb[0][:n].float()[~bad]).all() and torch.isfinite(mb[1]).all()


def test_no_gradient_no_step():
    for bits in (8, 32):
        ps, gs = tensors(3, [300, 500, 20], torch.bfloat16, torch.float32)
        a, b = [p.clone() for p in ps], [p.clone() for p in ps]
        ma, mb = adamw_moments(ps, bits), adamw_moments(ps, bits)
        adamw_many(a, gs, ma, seed=1, **H)
        adamw_many(b, [gs[0], None, gs[2]], mb, seed=1, **H)
        assert torch.equal(b[1], ps[1]) and torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
        assert all((t[512:1024].float() == 0).all() for t in mb[:1])
        adamw_many(b, [None] * 3, mb, seed=1, **H)
        assert torch.equal(a[0], b[0])


def test_optimizer_follows_torch():
    shapes = [(40, 33), (1,), (7, 5, 3), (1000,)]
    for bits in (32, 8):
        g = torch.Generator(device=DEV).manual_seed(5)
        mine = [torch.randn(s, device=DEV, generator=g).requires_grad_(True) for s in shapes]
        theirs = [p.detach().clone().requires_grad_(True) for p in mine]
        groups = lambda ps: [{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.0}]  # noqa: E731
        a = ManyAdamW(groups(mine), lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1, bits=bits)
        b = torch.optim.AdamW(groups(theirs), lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1)
        sched = torch.optim.lr_scheduler.LambdaLR(a, lambda k: 1 / (k + 1)), torch.optim.lr_scheduler.LambdaLR(b, lambda k: 1 / (k + 1))
        for k in range(6):
            for p, t in zip(mine, theirs):
                p.grad = torch.randn(p.shape, device=DEV, generator=g)
                t.grad = p.grad.clone()
            v0 = mine[0]._version
            a.step()
            b.step()
            assert mine[0]._version > v0
            for s in sched:
                s.step()
            if k == 2:      # a state that is saved and loaded goes on as if nothing had happened
                c = ManyAdamW(groups([p.detach().clone().requires_grad_(True) for p in mine]), bits=bits)
                c.load_state_dict(a.state_dict())
                held = c, [p for gr in c.param_groups for p in gr["params"]]
            if k == 3:
                c, ps = held
                c.param_groups[0]["lr"], c.param_groups[1]["lr"] = 1e-2 / 4, 1e-3 / 4
                for p, t in zip(ps, mine):
                    p.grad = t.grad
                c.step()
                assert all(torch.equal(p, t) for p, t in zip(ps, mine))
        for p, t in zip(mine, theirs):
            if bits == 32:      # six steps of at most lr each, off by 2^-24 a few times over
                assert torch.allclose(p, t, rtol=0, atol=2e-6)
            else:               # six steps of at most 3 lr; m and r each off by at most an eighth per step
                assert (p - t).abs().max() < 6 * 3e-2


def test_streams_and_a_captured_step():
    ps, gs = tensors(6, [1000, 77, 4096], torch.float32, torch.float32)
    qs = [p.clone() for p in ps]
    ma, mb = adamw_moments(ps, 8), adamw_moments(qs, 8)
    st = torch.cuda.Stream()
    for _ in range(4):
        adamw_many(ps, gs, ma, seed=9, **H)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        adamw_many(qs, gs, mb, seed=9, **H)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        adamw_many(qs, gs, mb, seed=9, **H)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ps, qs)) and all(torch.equal(a.float(), b.float()) for a, b in zip(ma, mb))
    opt = ManyAdamW(ps, bits=8)
    for p in ps:
        p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_carry_the_moments_and_a_refused_step_counts_nothing(bits):
    import copy
    g = torch.Generator(device=DEV).manual_seed(6)
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV, generator=g)) for n in (300, 7)]
    opt = ManyAdamW(ps, lr=1e-2, bits=bits)
    grads = [torch.randn(p.shape, device=DEV, generator=g) for p in ps]

    def step(o):
        for p, t in zip(o.param_groups[0]["params"], grads):
            p.grad = t.clone()
        o.step()
    step(opt)
    twin = copy.deepcopy(opt)
    held = [p.detach().clone() for p in ps]
    step(twin)
    assert all(torch.equal(p, h) for p, h in zip(ps, held)) and twin.param_groups[0]["params"][0] is not ps[0]
    ps[1].data, was = ps[1].data.repeat(2)[::2], ps[1].data       # no longer contiguous: refused before anything is written
    ps[1].grad = None
    with pytest.raises(ValueError):
        opt.step()
    ps[1].data = was
    step(opt)
    assert all(torch.equal(a, b) for a, b in zip(ps, twin.param_groups[0]["params"])) and opt.param_groups[0]["steps"] == 2


def test_a_step_after_a_change_of_type_is_refused():
    layer = torch.nn.Linear(20, 30).to(DEV)
    opt = ManyAdamW(layer.parameters(), lr=1e-2)

    def step():
        for p in layer.parameters():
            p.grad = torch.ones_like(p)
        opt.step()
    step()
    layer.half()
    held = [p.detach().clone() for p in layer.parameters()]
    with pytest.raises(RuntimeError, match="changed"):
        step()
    assert all(torch.equal(p, h) for p, h in zip(layer.parameters(), held)) and opt.param_groups[0]["steps"] == 1
    layer.float()
    step()
    assert opt.param_groups[0]["steps"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_step_writes_nothing(bits):
    """Several types of parameters and gradients, several groups: a refusal in any of them comes before the first launch."""
    g = torch.Generator(device=DEV).manual_seed(16)
    make = lambda n, dt: torch.nn.Parameter(torch.randn(n, device=DEV, generator=g).to(dt))  # noqa: E731
    ps = [make(300, torch.float32), make(70, torch.bfloat16), make(600, torch.float32), make(40, torch.float32), make(50, torch.bfloat16)]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = (ManyAdamW([{"params": t[:3]}, {"params": t[3:], "lr": 1e-3}], lr=1e-2, bits=bits) for t in (ps, twins))
    grads = [torch.randn(p.shape, device=DEV, generator=g).to(p.dtype) for p in ps]

    def step(opt, params):
        for p, t in zip(params, grads):
            p.grad = t.clone()
        opt.step()
    step(a, ps)
    step(b, twins)
    for i in (4, 2, 1):
        held, moments = [p.detach().clone() for p in ps], a.state_dict()["moments"]
        was = ps[i].data
        ps[i].data = was.repeat_interleave(2)[::2]           # the same values, not contiguous
        ps[i].grad = None
        with pytest.raises(ValueError):
            step(a, ps)
        assert all(torch.equal(p, h) for p, h in zip(ps, held)) and [x["steps"] for x in a.param_groups] == [1, 1]
        now = a.state_dict()["moments"]
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for k in range(2) for m, n in zip(moments[k], now[k]) for x, y in zip(m, n))
        ps[i].grad = None
        ps[i].data = was
    step(a, ps)
    step(b, twins)
    assert all(torch.equal(p, t) for p, t in zip(ps, twins)) and [x["steps"] for x in a.param_groups] == [2, 2]


def test_one_tensor_is_not_two_moments():
    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    for bits in (32, 8):
        m = adamw_moments([p], bits)
        for bad in (dict(step=0), dict(step=1, betas=(0.9, 1.0)), dict(step=1, betas=(-0.1, 0.9)), dict(step=1, moments=m[:len(m) // 2] * 2)):
            with pytest.raises(ValueError):
                adamw_many([p], [g], lr=1e-3, **dict(dict(moments=m), **bad))
        assert (p == 1).all() and all((t.view(torch.uint8) == 0).all() for t in m)


def test_optimizer_with_8_bit_moments_moves_as_torch_does():
    """The first step reads no code (its moments are zero): as torch's but for fp32 roundings.  Each later one reads m and r = sqrt(v) as e4m3 codes, rounded by chance: off by at most half
    a code's spacing of 2^-3 in rms, 1/16.  m carries 5 such errors, each weighed by 0.9 a step: 0.106 of it; r's reach v doubled, 5 of them: 0.28 of v, 0.14 of r; together 0.18 of
    each step.  The gradients keep their direction, so the steps add up and the movement |t - start| is off by no more than that in norm; 0.25 is allowed.  (No step at all: 1.  The wrong way: 2.  A rate
    1.3 times too large: 0.3.)"""
    shapes = [(40, 33), (300,), (7, 5, 13), (1000,)]
    g = torch.Generator(device=DEV).manual_seed(5)
    start = [torch.randn(s, device=DEV, generator=g) for s in shapes]
    mine, theirs = ([p.clone().requires_grad_(True) for p in start] for _ in range(2))
    groups = lambda ps: [{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.0}]  # noqa: E731
    a = ManyAdamW(groups(mine), lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1, bits=8)
    b = torch.optim.AdamW(groups(theirs), lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1)
    sched = [torch.optim.lr_scheduler.LambdaLR(o, lambda k: 1 / (k + 1)) for o in (a, b)]
    base = [torch.randn(s, device=DEV, generator=g) for s in shapes]
    for k in range(6):
        for p, t, d in zip(mine, theirs, base):
            p.grad = d + 0.3 * torch.randn(d.shape, device=DEV, generator=g)
            t.grad = p.grad.clone()
        rates = [group["lr"] for group in a.param_groups]
        a.step()
        b.step()
        for s in sched:
            s.step()
        for i, (p, t, s) in enumerate(zip(mine, theirs, start)):
            p, t, s = p.detach().double(), t.detach().double(), s.double()
            if k == 0:   # the decay and the sum round p twice each, the quotient and the rate 16 times 2^-24 of the step
                assert ((p - t).abs() <= 4 * 2.0 ** -24 * s.abs() + 32 * 2.0 ** -24 * rates[i // 2]).all(), i
            else:
                assert (p - t).norm() < 0.25 * (t - s).norm(), (k, i)
