"""GPU: adapter projections (fithubert_amd.adapters) against their definition in 64 bits, forward and backward.

Tolerances are elementwise (u = eps / 2 of the element type; a sum of n products in fp32 is off by at most n 2^-24 of the sum of their magnitudes):
  h, G   (K or N) 2^-24 of their magnitude sums + u |h|, and the scaling's own rounding 2^-24
  y, dx  n 2^-24 of the magnitude sum of both products + the error of h (G) times |B| (|A|) + u |y|; the adapter's part may be rounded once on its
         way to the sum (short requests): + u |part|
  da, db rows 2^-24 of the magnitude sum + the error of G (h) times |x| (|dy|); rounded once to the factor's type: + u
fp16 adds half its smallest spacing, 2^-25, to every rounded value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from fithubert_amd.adapters import adapter_linear  # noqa: E402

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(seed, dtype, M, K, N, R, n, start, which, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, f=1.0: (torch.randn(*s, device=DEV, generator=g) * f).to(dtype)  # noqa: E731
    return dict(x=r(M, K), weight=r(N, K, f=K ** -0.5), bias=torch.randn(N, device=DEV, generator=g) if bias else None, a=r(n, R, K, f=K ** -0.5), b=r(n, N, R, f=R ** -0.5),
                scaling=torch.rand(n, device=DEV, generator=g) + 0.5, start=torch.tensor(start, dtype=torch.int32, device=DEV),
                which=torch.tensor(which, dtype=torch.int32, device=DEV), dy=r(M, N))


def reference(s):
    dtype = s["x"].dtype
    e = 2.0 ** -24
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else e
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    x, w, a, b, dy = (s[n].double() for n in ("x", "weight", "a", "b", "dy"))
    (M, K), N = x.shape, w.shape[0]
    n, R = a.shape[:2]
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros(N, device=DEV, dtype=torch.float64)
    y, ym = x @ w.T + bias, (x.abs() @ w.abs().T + bias.abs()) * (K + 8) * e
    dx, dxm = dy @ w, dy.abs() @ w.abs() * (N + 8) * e
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    dam, dbm = torch.zeros_like(a), torch.zeros_like(b)
    for i, j, k in zip(s["start"].tolist(), s["start"].tolist()[1:], s["which"].tolist()):
        i, j = max(0, min(M, i)), max(0, min(M, j))
        if j <= i or not 0 <= k < n:
            continue
        f = s["scaling"][k].item()
        X, Y = x[i:j], dy[i:j]
        h, G = f * X @ a[k].T, f * Y @ b[k]
        eh = (K + 8) * e * f * (X.abs() @ a[k].abs().T) + u * h.abs() + tiny
        eG = (N + 8) * e * f * (Y.abs() @ b[k].abs()) + u * G.abs() + tiny
        part, parx = h @ b[k].T, G @ a[k]
        y[i:j] += part
        ym[i:j] += (eh + (R + 8) * e * h.abs()) @ b[k].abs().T + u * part.abs() + tiny
        dx[i:j] += parx
        dxm[i:j] += (eG + (R + 8) * e * G.abs()) @ a[k].abs() + u * parx.abs() + tiny
        da[k] += G.T @ X
        dam[k] += (eG + (M + 8) * e * G.abs()).T @ X.abs()
        db[k] += Y.T @ h
        dbm[k] += Y.abs().T @ (eh + (M + 8) * e * h.abs())
    return {"y": (y, ym + u * y.abs() + tiny), "dx": (dx, dxm + u * dx.abs() + tiny), "da": (da, dam + u * da.abs() + tiny), "db": (db, dbm + u * db.abs() + tiny)}


def run(s):
    x, a, b = (s[n].detach().requires_grad_(True) for n in ("x", "a", "b"))
    y = adapter_linear(x, s["weight"], s["bias"], a, b, s["scaling"], s["start"], s["which"])
    dx, da, db = torch.autograd.grad(y, (x, a, b), s["dy"])
    return {"y": y.detach(), "dx": dx, "da": da, "db": db}


def check(s):
    got, ref = run(s), reference(s)
    for n, (value, bound) in ref.items():
        off = (got[n].double() - value).abs()
        assert torch.isfinite(got[n]).all(), n
        assert got[n].dtype == s["x"].dtype and (off <= bound * 1.0001 + 1e-30).all(), f"{n}: {(off / bound.clamp_min(1e-300)).max().item():.2f} times its bound"
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R,n,start,which", [
    (1, 8, 8, 8, 1, [0, 1], [0]),
    (1, 768, 768, 16, 3, [0, 1], [2]),
    (17, 480, 1440, 8, 2, [0, 5, 17], [1, 0]),
    (32, 768, 512, 16, 8, list(range(33)), [(5 * i) % 8 for i in range(32)]),          # a frame each
    (130, 40, 72, 24, 3, [0, 0, 64, 65, 65, 130], [0, 1, 2, 0, 1]),                     # empty requests
    (300, 512, 264, 64, 2, [3, 100, 290], [0, 1]),                                      # rows in front of and behind them
    (257, 488, 480, 128, 4, [0, 90, 200, 257], [3, -1, 3]),                             # none, and one adapter twice
    (515, 136, 1000, 32, 5, [0, 250, 515], [7, 1]),                                     # a number that is no adapter's
    (700, 96, 104, 40, 70, [10 * i for i in range(71)], list(range(70))),
    (2100, 480, 480, 16, 2, [0, 1500, 2100], [0, 1]),
    (1000, 1024, 256, 8, 1, [0], []),
    (513, 72, 200, 16, 4, [0, 300, 513], [3, 0]),                                        # behind the few-row kernel's last row
    (511, 200, 72, 8, 70, [7 * i for i in range(74)], list(range(73))),                  # more than 64 requests in it
    (17000, 72, 40, 56, 3, [0, 5000, 5001, 16990], [1, 0, 2]),                          # 32-row tiles
    # the 256-tile loop: rows and columns that end inside a tile, a wave's rows, 64 columns
    (9973, 480, 1440, 8, 12, [0, 82, 327, 736, 4900, 9900], [1, 6, -1, 11, 4]),
    (2561, 136, 2568, 24, 3, [100, 1000, 2000, 2550], [0, 2, 1]),
    (6200, 1448, 1096, 40, 2, [0, 3100, 6200], [1, 0])])                                                   # no request at all
def test_forward_and_backward(dtype, M, K, N, R, n, start, which):
    check(make(M + K, dtype, M, K, N, R, n, start, which, bias=M % 2 == 0))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_requests_of_one_adapter(dtype):
    M, S = 1500, 300
    check(make(4, dtype, M, 128, 128, 16, 3, [M * i // S for i in range(S + 1)], [1 if i % 3 else -1 for i in range(S)]))


@pytest.mark.parametrize("dtype", TYPES)
def test_requests_past_the_last_row_are_clipped(dtype):
    s = make(5, dtype, 50, 64, 64, 8, 2, [0, 20, 80, 90], [0, 1, 0])
    a = check(s)
    s["start"][2:] = 50
    b = run(s)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [1, 4, 12])
def test_other_ranks_are_padded(dtype, R):
    check(make(6, dtype, 90, 64, 96, R, 2, [0, 40, 90], [0, 1]))


def test_leading_axes_slices_and_partial_gradients():
    s = make(7, torch.bfloat16, 60, 64, 96, 16, 2, [0, 25, 60], [1, 0])
    want = run(s)
    wide = torch.zeros(3, 20, 70, device=DEV, dtype=torch.bfloat16)
    wide[..., 3:67] = s["x"].view(3, 20, 64)
    a = s["a"].detach().requires_grad_(True)
    y = adapter_linear(wide[..., 3:67], s["weight"], s["bias"], a, s["b"], s["scaling"], s["start"], s["which"])
    assert y.shape == (3, 20, 96) and torch.equal(y.view(60, 96), want["y"])
    assert torch.equal(torch.autograd.grad(y, a, s["dy"].view(3, 20, 96))[0], want["da"])
    with torch.no_grad():
        assert torch.equal(adapter_linear(s["x"], s["weight"], s["bias"], a, s["b"], s["scaling"], s["start"], s["which"]), want["y"])
    none = adapter_linear(s["x"][:0], s["weight"], s["bias"], a, s["b"].detach().requires_grad_(True), s["scaling"], s["start"], s["which"])
    assert none.shape == (0, 96) and (torch.autograd.grad(none.sum(), a)[0] == 0).all()


def test_padding_rows_may_be_anything():
    s = make(8, torch.float16, 40, 64, 64, 8, 2, [0, 10, 30], [0, 1])
    s["dy"][30:] = 0
    want = run(s)
    for bad in (float("nan"), float("inf")):
        s["x"][30:] = bad
        got = run(s)
        assert torch.equal(got["y"][:30], want["y"][:30]) and torch.equal(got["da"], want["da"]) and torch.equal(got["db"], want["db"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,start", [(90, 64, 96, [0, 37, 80]), (900, 64, 96, [0, 437, 880]), (900, 64, 96, [10 * i for i in range(91)]), (9000, 136, 1096, [0, 4437, 8880])])
def test_an_adapter_of_infinities_stays_with_its_own_rows(dtype, M, K, N, start):
    s = make(11, dtype, M, K, N, 16, 2, start, [i % 2 for i in range(len(start) - 1)])
    want = run(s)
    theirs = torch.ones(M, dtype=torch.bool, device=DEV)
    for i, (b, e) in enumerate(zip(start, start[1:])):
        theirs[b:e] = i % 2 == 0
    for n in ("a", "b"):
        for bad in (float("nan"), float("inf")):
            t = dict(s, **{n: s[n].clone()})
            t[n][1] = bad
            got = run(t)
            assert torch.equal(got["y"][theirs], want["y"][theirs]) and torch.equal(got["dx"][theirs], want["dx"][theirs])
            assert torch.equal(got["da"][0], want["da"][0]) and torch.equal(got["db"][0], want["db"][0])


def test_gradients_against_differences():
    s = make(9, torch.float32, 50, 48, 56, 8, 2, [0, 21, 50], [0, 1])
    got = run(s)
    g = torch.Generator(device=DEV).manual_seed(2)
    for n, d in (("x", "dx"), ("a", "da"), ("b", "db")):
        v = torch.randn(s[n].shape, device=DEV, generator=g)
        vals = []
        for h in (0.125, -0.125):          # the function is linear in each of the three: the difference is exact but for fp32
            t = dict(s, **{n: s[n] + h * v})
            vals.append((adapter_linear(t["x"], t["weight"], t["bias"], t["a"], t["b"], t["scaling"], t["start"], t["which"]).double() * s["dy"].double()).sum().item())
        diff = (vals[0] - vals[1]) / 0.25
        assert abs(diff - (got[d].double() * v.double()).sum().item()) < 1e-3 * max(10.0, abs(diff)), n


def test_equal_calls_give_equal_bits_on_any_stream_and_captured():
    s = make(10, torch.bfloat16, 900, 256, 320, 16, 3, [0, 100, 101, 600, 890], [0, 2, 1, 0])
    want = run(s)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = run(s)
        run(s)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(want[n], got[n]) for n in want)
    leaves = {n: s[n].clone().requires_grad_(True) for n in ("x", "a", "b")}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = adapter_linear(leaves["x"], s["weight"], s["bias"], leaves["a"], leaves["b"], s["scaling"], s["start"], s["which"])
        grads = torch.autograd.grad(y, (leaves["x"], leaves["a"], leaves["b"]), s["dy"])
    for _ in range(3):
        for t in (y,) + grads:
            t.detach().zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(want[n], t) for n, t in zip(("y", "dx", "da", "db"), (y,) + grads))
        torch.ones(500, 500, device=DEV).cumsum(0).sum().item()
    s["which"].copy_(torch.tensor([1, 1, -1, 2], device=DEV))     # other adapters for the captured requests
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(run(s)[n], t) for n, t in zip(("y", "dx", "da", "db"), (y,) + grads))


def test_saved_tensors_that_come_back_elsewhere():
    """Activations parked in host memory between the passes, and hooks that give back other strides."""
    s = make(12, torch.bfloat16, 90, 64, 96, 16, 2, [0, 37, 80], [1, 0])
    want = run(s)
    other = lambda t: torch.empty((2,) + t.shape, dtype=t.dtype, device=t.device).permute(*range(1, t.dim() + 1), 0)[..., 0].copy_(t)  # noqa: E731
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), other)):
        x, a, b = (s[n].detach().requires_grad_(True) for n in ("x", "a", "b"))
        with hooks:
            y = adapter_linear(x, s["weight"], s["bias"], a, b, s["scaling"], s["start"].clone(), s["which"].clone())
        got = torch.autograd.grad(y, (x, a, b), s["dy"])
        assert all(torch.equal(want[n], t) for n, t in zip(("dx", "da", "db"), got))


def test_under_the_gemm_tuner():
    """The tuner runs a launch several times: the sum that lies in the output already must not be taken again."""
    from fithubert_amd import _lib as L
    s = make(13, torch.bfloat16, 900, 256, 320, 16, 3, [10 * i for i in range(91)], [i % 3 for i in range(90)])
    want = run(s)
    L.lib().fh_gemm_tune(1)
    try:
        got = run(s)
    finally:
        L.lib().fh_gemm_tune(0)
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_refusals_on_the_gpu():
    s = make(14, torch.bfloat16, 20, 64, 64, 8, 2, [0, 20], [1])
    args = [s[n] for n in ("x", "weight", "bias", "a", "b", "scaling", "start", "which")]
    for i in (1, 2, 5):                                      # the projection and the scalings are frozen
        bad = list(args)
        bad[i] = bad[i].clone().requires_grad_(True)
        with pytest.raises(ValueError):
            adapter_linear(*bad)
        with torch.no_grad():
            assert torch.equal(adapter_linear(*bad), adapter_linear(*args))
    for i in (2, 6, 7):                                      # not on the GPU
        bad = list(args)
        bad[i] = bad[i].cpu()
        with pytest.raises(ValueError):
            adapter_linear(*bad)


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_inputs_and_one_leaf_twice(dtype):
    """A row that stands for many, and both factors out of one tensor: the gradients are the sums."""
    s = make(15, dtype, 40, 64, 64, 8, 2, [0, 20, 40], [1, 0])
    s["x"] = s["x"][:1].expand(40, -1)
    s["b"] = s["a"].transpose(1, 2)
    check(s)
    row = s["x"][:1].clone().requires_grad_(True)
    one = s["a"].clone().requires_grad_(True)
    y = adapter_linear(row.expand(40, -1), s["weight"], s["bias"], one, one.transpose(1, 2), s["scaling"], s["start"], s["which"])
    dx, da = torch.autograd.grad(y, (row, one), s["dy"])
    want = run(s)
    assert torch.equal(dx, want["dx"].sum(0, keepdim=True)) and torch.equal(da, want["da"] + want["db"].transpose(1, 2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,R", [(1024, 512, 1024, 8), (4096, 1536, 1536, 8), (4096, 1536, 1536, 40), (40, 512, 512, 24), (300, 512, 512, 8)])
def test_a_product_past_the_type_gives_infinity_in_its_row(dtype, M, K, N, R):
    """h (backward: G) of one row overflows: its row of y (dx) is infinite, as infinity times positive factors is, not NaN; no other row notices."""
    s = make(61, dtype, M, K, N, R, 2, [0, M // 3, M], [0, 1])
    s["a"], s["b"] = s["a"].abs() + 0.25, s["b"].abs() + 0.25
    clean = run(s)
    big = 6e4 if dtype == torch.float16 else 2e37   # (times 0.25 K or 0.25 N: past either type; the projection's own sum stays inside 32 bits)
    for row in (5, M // 3 + 4):
        s2 = dict(s, x=s["x"].clone(), dy=s["dy"].clone())
        s2["x"][row], s2["dy"][row] = big, big
        dirty = run(s2)
        for n in ("y", "dx"):
            assert (dirty[n][row] == float("inf")).all(), n
            assert torch.equal(dirty[n][:row], clean[n][:row]) and torch.equal(dirty[n][row + 1:], clean[n][row + 1:]), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N,R,S", [(900, 480, 1440, 8, 6), (9973, 480, 1440, 8, 40), (257, 488, 480, 16, 3), (600, 768, 2304, 16, 4), (3000, 1024, 1024, 16, 8), (70, 480, 480, 8, 10), (40, 512, 768, 16, 40)])
def test_both_results_are_rounded_once(dtype, M, K, N, R, S):
    """y and dx are off by half a step from their products with h and G as rounded to the element type -- the adapter's part is added before that rounding, not rounded on its way.  (A
    quarter more and 1 % of the elements are allowed to an h or G that the fp32 sum rounds the other way; a part rounded on its own misses by more in 2.5 to 6 % of them.)"""
    s = make(71, dtype, M, K, N, R, 2, [M * i // S for i in range(S + 1)], [i % 2 for i in range(S)])
    got = run(s)
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    x, w, a, b, dy = (s[n].double() for n in ("x", "weight", "a", "b", "dy"))
    y, dx = x @ w.T + s["bias"].double(), dy @ w
    noise = {"y": (x.abs() @ w.abs().T) * (K + R + 8) * e, "dx": (dy.abs() @ w.abs()) * (N + R + 8) * e}
    for i, j, k in zip(s["start"].tolist(), s["start"].tolist()[1:], s["which"].tolist()):
        f = s["scaling"][k].item()
        y[i:j] += (f * x[i:j] @ a[k].T).to(dtype).double() @ b[k].T
        dx[i:j] += (f * dy[i:j] @ b[k]).to(dtype).double() @ a[k]
    for n, exact in (("y", y), ("dx", dx)):
        off = (got[n].double() - exact).abs() > 1.25 * u * exact.abs() + noise[n] + 2.0 ** -25
        assert off.double().mean() < 0.01, (n, off.double().mean().item())
