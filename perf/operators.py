"""Cases for the operators that adapt the distilled encoder to long recordings and to many tasks at once:

* ``attention``: attention inside a sliding window with a few first frames that stay visible, forward and backward
  (``fithubert_amd.window_attention``) -- an encoder or a streaming front end over recordings of minutes;
* ``adapter``: low-rank adapters of many requests beside one frozen projection, forward and backward
  (``fithubert_amd.adapters``) -- one upstream encoder that serves, or trains, several downstream tasks;
* ``adamw``: one AdamW step over a list of tensors, its moments in 32 or in 8 bits (``fithubert_amd.optim``) -- the adapters'
  optimizer, or a whole encoder's.

``run`` computes them from elementary torch operations, or with ``own`` set by the framework's kernels.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256          # elements that share one scale in the 8-bit moments
E4M3_MAX = 448.0
TINY = 1e-30


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one layer of the 12 x 40 student on a ragged batch of 15 s utterances behind its time reduction, a local window on both sides
        {"name": "attn-student-bf16", "op": "attention", "train": True, "dtype": "bf16", "B": 8, "Tq": 375, "Tk": 375, "Hq": 12, "Hkv": 12, "dh": 40,
         "left": 64, "right": 64, "sinks": 0, "ragged": True},
        # one layer of a 12 x 64 encoder in the fp32 parity mode: 10 s clips, a window with some look-ahead and four first frames
        {"name": "attn-base-fp32", "op": "attention", "train": True, "dtype": "fp32", "B": 2, "Tq": 499, "Tk": 499, "Hq": 12, "Hkv": 12, "dh": 64,
         "left": 100, "right": 20, "sinks": 4, "ragged": True},
        # a causal layer with shared key heads over ten minutes of audio (50 frames a second)
        {"name": "attn-ten-minutes-bf16", "op": "attention", "train": True, "dtype": "bf16", "B": 1, "Tq": 30001, "Tk": 30001, "Hq": 16, "Hkv": 4, "dh": 64,
         "left": 1023, "right": 0, "sinks": 16, "ragged": False},
        # 64 live streams, one new frame each, against their caches
        {"name": "attn-stream-token-fp16", "op": "attention", "train": False, "dtype": "fp16", "B": 64, "Tq": 1, "Tk": 8192, "Hq": 16, "Hkv": 4, "dh": 64,
         "left": 1023, "right": 0, "sinks": 4, "ragged": True},
        # one recording's last frames against all that came before
        {"name": "attn-stream-chunk-bf16", "op": "attention", "train": False, "dtype": "bf16", "B": 1, "Tq": 16, "Tk": 65536, "Hq": 16, "Hkv": 2, "dh": 128,
         "left": 65536, "right": 0, "sinks": 0, "ragged": False},
        # 32 live requests of one frame, eight adapters, a 768-wide projection
        {"name": "adapter-token-fp16", "op": "adapter", "train": False, "dtype": "fp16", "rows": 32, "K": 768, "N": 768, "R": 16, "adapters": 8, "requests": 32},
        # 40 utterances of uneven length through the 480-wide student's q|k|v projection
        {"name": "adapter-student-bf16", "op": "adapter", "train": False, "dtype": "bf16", "rows": 9973, "K": 480, "N": 1440, "R": 8, "adapters": 12, "requests": 40},
        # training four tasks' adapters beside a 1024 -> 4096 projection
        {"name": "adapter-train-bf16", "op": "adapter", "train": True, "dtype": "bf16", "rows": 16384, "K": 1024, "N": 4096, "R": 16, "adapters": 4, "requests": 32},
        # the same in the fp32 parity mode, at the student's width
        {"name": "adapter-train-fp32", "op": "adapter", "train": True, "dtype": "fp32", "rows": 1497, "K": 480, "N": 480, "R": 32, "adapters": 3, "requests": 6},
        # the optimizer step of the adapters: 12 layers, four projections, three tasks, each factor a tensor
        {"name": "adamw-adapters-32", "op": "adamw", "dtype": "fp32", "grad": "fp32", "bits": 32, "tensors": 144, "size": 7680, "spread": 4},
        # the student (about 30 M parameters in 200 tensors) with 8-bit moments
        {"name": "adamw-student-8", "op": "adamw", "dtype": "fp32", "grad": "fp32", "bits": 8, "tensors": 200, "size": 19000, "spread": 64},
        # an encoder of 300 M parameters held in bf16, with 8-bit moments
        {"name": "adamw-large-8", "op": "adamw", "dtype": "bf16", "grad": "bf16", "bits": 8, "tensors": 380, "size": 100000, "spread": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "adapter", "adapter", "adamw"))
    dtype = rng.choice(("bf16", "fp16", "bf16", "fp32"))
    if op == "attention":
        hkv = rng.choice((1, 2, 4, 8, 12))
        g = rng.choice((1, 1, 2, 4))
        dh = rng.choice((40, 64, 64, 80, 96, 128))
        sinks = rng.choice((0, 0, 1, 4, 16, 33))
        if rng.random() < 0.4:        # serving: a few new frames against a cache
            tk = _log(rng, 200, 40000)
            tq = rng.choice((1, 1, 2, 7, 16, 33))
            return {"op": op, "train": False, "dtype": dtype, "B": max(1, min(_log(rng, 1, 64), 400000 // tk)), "Tq": tq, "Tk": tk, "Hq": hkv * g, "Hkv": hkv, "dh": dh,
                    "left": _log(rng, 32, tk), "right": rng.choice((0, 0, 8)), "sinks": sinks, "ragged": rng.random() < 0.7}
        b, t, left, right = _log(rng, 1, 16), _log(rng, 60, 12000), _log(rng, 16, 1000), rng.choice((0, 0, 16, 100))
        most = (4e9 if dtype == "fp32" else 2.5e10) / (hkv * g * dh * (left + right + sinks + 1))     # rows, within the largest listed case's work
        t = int(min(t, most))
        return {"op": op, "train": rng.random() < 0.8, "dtype": dtype, "B": max(1, min(b, int(most) // t)), "Tq": t, "Tk": t, "Hq": hkv * g, "Hkv": hkv, "dh": dh,
                "left": left, "right": right, "sinks": sinks, "ragged": rng.random() < 0.6}
    if op == "adapter":
        train = rng.random() < 0.6
        requests = _log(rng, 1, 64)
        rows = _log(rng, 16, 16000) if train else _log(rng, 1, 16000)
        if dtype == "fp32":
            rows = min(rows, 2000)
        return {"op": op, "train": train, "dtype": dtype, "rows": max(rows, requests), "K": rng.choice((480, 512, 768, 1024, 1536)), "N": rng.choice((480, 768, 1024, 1440, 2304)),
                "R": rng.choice((8, 16, 24, 32, 64)), "adapters": rng.choice((1, 2, 5, 8, 16)), "requests": requests}
    return {"op": op, "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16")), "grad": rng.choice(("fp32", "bf16")), "bits": rng.choice((8, 8, 32)),
            "tensors": _log(rng, 1, 300), "size": _log(rng, 300, 40000), "spread": rng.choice((1, 4, 64))}


# ------------------------------------------------------------------------------------------------ what a user's program has in hand
def _key_len(c):
    """valid keys of each entry: all of them, or down to about a third, odd values among them"""
    tk, b = c["Tk"], c["B"]
    if not c["ragged"]:
        return [tk] * b
    return [max(1, tk - (2 * i * tk) // (3 * b)) for i in range(b)]


def _q_start(c):
    """position of each entry's first query: the last Tq valid frames, or the beginning where queries and keys are the same frames"""
    if c["Tq"] == c["Tk"]:
        return [0] * c["B"]
    return [max(0, n - c["Tq"]) for n in _key_len(c)]


def _segments(c):
    """rows where each request begins (uneven, one row at least; where there are many, padding rows lie behind the last one) and its adapter (-1: none)"""
    n, rows = c["requests"], c["rows"]
    spare = rows - n - (rows // 64 if n > 4 and rows > 2 * n else 0)
    weight = [1 + (7 * i) % 5 for i in range(n)]
    total, acc, start = sum(weight), 0, [0]
    for i in range(n):
        acc += weight[i]
        start.append(i + 1 + spare * acc // total)
    return start, [-1 if n > 4 and i % 9 == 4 else (5 * i + 1) % c["adapters"] for i in range(n)]


def _sizes(c):
    """element counts of the tensors: a few large ones, many small ones, odd ones among them"""
    got = []
    for i in range(c["tensors"]):
        f = c["spread"] ** (((i * 37) % 101) / 100.0 * 2 - 1)
        got.append(max(1, int(c["size"] * f) + (i % 3 if i % 5 == 0 else 0)))
    return got


def _starts(sizes):
    """where each tensor begins in the one buffer that holds them, as an encoder with a flat parameter keeps them: at multiples of 64 elements"""
    got = [0]
    for n in sizes:
        got.append(got[-1] + -(-n // 64) * 64)
    return got


def prepare(case, seed):
    c, dev = case, "cuda"
    dt = DTYPES[c["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device=dev, generator=gen) * scale).to(dtype)

    if c["op"] == "attention":
        s = {"case": c, "q": normal(c["B"], c["Tq"], c["Hq"], c["dh"]), "k": normal(c["B"], c["Tk"], c["Hkv"], c["dh"]), "v": normal(c["B"], c["Tk"], c["Hkv"], c["dh"]),
             "key_len": torch.tensor(_key_len(c), dtype=torch.int32, device=dev), "q_start": torch.tensor(_q_start(c), dtype=torch.int32, device=dev)}
        if c["train"]:
            s["dout"] = normal(c["B"], c["Tq"], c["Hq"], c["dh"])
            for n in "qkv":
                s[n].requires_grad_(True)
        return s
    if c["op"] == "adapter":
        start, which = _segments(c)
        s = {"case": c, "x": normal(c["rows"], c["K"]), "weight": normal(c["N"], c["K"], scale=c["K"] ** -0.5), "bias": normal(c["N"], scale=0.1, dtype=torch.float32),
             "a": normal(c["adapters"], c["R"], c["K"], scale=c["K"] ** -0.5), "b": normal(c["adapters"], c["N"], c["R"], scale=c["R"] ** -0.5),
             "scaling": torch.rand(c["adapters"], device=dev, generator=gen) + 0.5, "start": torch.tensor(start, dtype=torch.int32, device=dev),
             "which": torch.tensor(which, dtype=torch.int32, device=dev)}
        if c["train"]:
            s["dy"] = normal(c["rows"], c["N"])
            for n in ("x", "a", "b"):
                s[n].requires_grad_(True)
        return s
    sizes = _sizes(c)
    starts = _starts(sizes)
    flat, grad = normal(starts[-1], scale=0.05), normal(starts[-1], scale=1e-3, dtype=DTYPES[c["grad"]])
    s = {"case": c, "seed": seed % 65521, "flat": flat, "params": [flat[i:i + n] for i, n in zip(starts, sizes)], "grads": [grad[i:i + n] for i, n in zip(starts, sizes)]}
    padded = sum(-(-n // BLOCK) for n in sizes) * BLOCK
    m = torch.randn(padded, device=dev, generator=gen) * 3e-4
    r = torch.rand(padded, device=dev, generator=gen) * 1e-3 + 1e-4
    live = torch.cat([(torch.arange(-(-n // BLOCK) * BLOCK, device=dev) < n) for n in sizes])
    m, r = m * live, r * live
    if c["bits"] == 32:
        s["moments"] = [m, r * r]
    else:
        s["moments"] = []
        for t in (m, r):
            scale = t.view(-1, BLOCK).abs().amax(1).clamp_min(TINY) / E4M3_MAX
            s["moments"] += [(t.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1), scale]
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    return {"attention": _attention, "adapter": _adapter, "adamw": _adamw}[c["op"]](state, c)


def _attention(s, c):
    if own:
        from fithubert_amd.window_attention import window_attention
        if not c["train"]:
            return window_attention(s["q"], s["k"], s["v"], left=c["left"], right=c["right"], sinks=c["sinks"], key_len=s["key_len"], q_start=s["q_start"])
        out = window_attention(s["q"], s["k"], s["v"], left=c["left"], right=c["right"], sinks=c["sinks"], key_len=s["key_len"], q_start=s["q_start"])
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if not c["train"]:
        return _attend(s["q"], s["k"], s["v"], s["key_len"], s["q_start"], c).to(s["q"].dtype)
    out = _attend(s["q"], s["k"], s["v"], s["key_len"], s["q_start"], c)
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"].float())
    return {"out": out.detach().to(s["q"].dtype), "dq": dq, "dk": dk, "dv": dv}


def _attend(q, k, v, key_len, q_start, c):
    """softmax over the visible keys in 32 bits: blocks of queries against the keys of their common window, and the first keys beside it"""
    B, Tq, Hq, dh = q.shape
    Tk, Hkv, G = k.shape[1], k.shape[2], q.shape[2] // k.shape[2]
    left, right, sinks, dev = min(c["left"], Tk + Tq), c["right"], min(c["sinks"], Tk), q.device
    n = min(Tq, 128)
    blocks = -(-Tq // n)
    q32 = torch.nn.functional.pad(q.float() * dh ** -0.5, (0, 0, 0, 0, 0, blocks * n - Tq)).view(B, blocks, n, Hkv, G, dh)
    first = q_start.long()[:, None] + torch.arange(blocks, device=dev) * n                                      # B, blocks
    pos = (first[:, :, None] + torch.arange(n, device=dev))[..., None]                                          # B, blocks, n, 1
    width = min(left + n + right, Tk)
    lo = (first - left).clamp(0, Tk - width)
    at = lo[:, :, None] + torch.arange(width, device=dev)                                                       # B, blocks, width
    sink = torch.arange(sinks, device=dev).expand(B, blocks, sinks)
    in_band = (at[:, :, None] >= pos - left) & (at[:, :, None] <= pos + right)
    in_sink = (sink[:, :, None] < pos - left) & (sink[:, :, None] <= pos + right)
    at, seen = torch.cat((sink, at), 2), torch.cat((in_sink, in_band), 3)
    seen = seen & (at[:, :, None] < key_len.long()[:, None, None, None])
    entry = torch.arange(B, device=dev)[:, None, None]
    kw = k.float()[entry, at].permute(0, 1, 3, 4, 2).unsqueeze(3)                                               # B, blocks, Hkv, 1, dh, width
    vw = v.float()[entry, at].permute(0, 1, 3, 2, 4).unsqueeze(3)                                               # B, blocks, Hkv, 1, width, dh
    w = torch.matmul(q32.permute(0, 1, 3, 4, 2, 5).reshape(B, blocks, Hkv, 1, G * n, dh), kw).view(B, blocks, Hkv, G, n, -1)
    w = w.masked_fill(~seen[:, :, None, None], -math.inf)
    top = w.detach().amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-37)
    out = torch.matmul(w.view(B, blocks, Hkv, 1, G * n, -1), vw).view(B, blocks, Hkv, G, n, dh)
    return out.permute(0, 1, 4, 2, 3, 5).reshape(B, blocks * n, Hq, dh)[:, :Tq]


def _adapter(s, c):
    if own:
        from fithubert_amd.adapters import adapter_linear
        y = adapter_linear(s["x"], s["weight"], s["bias"], s["a"], s["b"], s["scaling"], s["start"], s["which"])
        if not c["train"]:
            return y
        dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "da": da, "db": db}
    y = _project(s, c)
    if not c["train"]:
        return y.to(s["x"].dtype)
    dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"].float())
    return {"y": y.detach().to(s["x"].dtype), "dx": dx, "da": da, "db": db}


def _project(s, c):
    """x W^T + bias, and every adapter's product with the rows of other adapters set to nought, in 32 bits"""
    rows, R, n = c["rows"], c["R"], c["adapters"]
    x = s["x"].float()
    at = torch.searchsorted(s["start"][1:].contiguous(), torch.arange(rows, device=x.device, dtype=torch.int32), right=True)
    which = torch.cat((s["which"], s["which"].new_full((1,), -1)))[at]                                          # rows; -1: no adapter
    share = (which[:, None] == torch.arange(n, device=x.device)) * s["scaling"]                                 # rows, adapters
    h = (x @ s["a"].float().view(n * R, -1).t()).view(rows, n, R) * share[:, :, None]
    return x @ s["weight"].float().t() + s["bias"] + h.view(rows, n * R) @ s["b"].float().permute(0, 2, 1).reshape(n * R, -1)


HYPER = {"step": 7, "lr": 5e-4, "beta1": 0.9, "beta2": 0.98, "eps": 1e-6, "weight_decay": 0.01, "grad_scale": 0.5}


def _adamw(s, c):
    if own:
        from fithubert_amd.optim import adamw_many
        h = HYPER
        adamw_many(s["params"], s["grads"], s["moments"], step=h["step"], lr=h["lr"], betas=(h["beta1"], h["beta2"]), eps=h["eps"], weight_decay=h["weight_decay"],
                   grad_scale=h["grad_scale"], seed=s["seed"])
    else:
        _step(s["params"], s["grads"], s["moments"], s["seed"], **HYPER)
    return {"params": s["flat"], "moments": s["moments"]}


def _step(params, grads, moments, seed, step, lr, beta1, beta2, eps, weight_decay, grad_scale):
    """the step on one flat copy, every tensor padded to whole blocks"""
    sizes = [p.numel() for p in params]
    blocks = [-(-n // BLOCK) * BLOCK for n in sizes]
    flat = lambda ts: torch.cat([torch.nn.functional.pad(t.float().view(-1), (0, b - n)) for t, n, b in zip(ts, sizes, blocks)])  # noqa: E731
    p, g = flat(params), flat(grads) * grad_scale
    if len(moments) == 2:
        m, v = moments
    else:
        m = (moments[0].float().view(-1, BLOCK) * moments[1][:, None]).view(-1)
        r = (moments[2].float().view(-1, BLOCK) * moments[3][:, None]).view(-1)
        v = r * r
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + (g * g) * (1 - beta2)
    r = v.sqrt()
    p = p * (1 - lr * weight_decay) - (lr / (1 - beta1 ** step)) * (m / (r * (1 / math.sqrt(1 - beta2 ** step)) + eps))
    if len(moments) == 2:
        moments[0].copy_(m)
        moments[1].copy_(v)
    else:
        low, high = _dither(m.numel(), seed, m.device)
        for k, (t, u) in enumerate(((m, low), (r, high))):
            code, scale = _to_e4m3(t, u, keep=k == 1)
            moments[2 * k].copy_(code)
            moments[2 * k + 1].copy_(scale)
    torch._foreach_copy_(params, [x[:n].view_as(t) for x, n, t in zip(p.split(blocks), sizes, params)])


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(n, seed, dev):
    """two fractions in [0, 1) of each place: 16 bits each of one hash of the seed and the place"""
    key = _mix(torch.tensor([(seed * 0x9E3779B9 + 0x27D4EB2F) & 0xFFFFFFFF], device=dev))
    h = _mix(torch.arange(n, device=dev) ^ key)
    return (h & 0xFFFF).float() / 65536, (h >> 16).float() / 65536


def _to_e4m3(t, u, keep):
    """blocks of `t` over their largest value, each rounded up with the probability of its fraction; `keep`: what is not nought stays so"""
    x = t.view(-1, BLOCK)
    top = x.abs().amax(1).clamp_min(TINY)
    a = x.abs() * (torch.reciprocal(top) * E4M3_MAX)[:, None]
    step = torch.exp2((torch.frexp(a).exponent - 1).clamp_min(-6).float() - 3)
    code = (torch.floor(a / step + u.view(-1, BLOCK)) * step).clamp_max(E4M3_MAX)
    if keep:
        code = torch.where((a > 0) & (code == 0), 2.0 ** -9, code)
    return (code * torch.where(x < 0, -1.0, 1.0)).to(torch.float8_e4m3fn).view(-1), top * (1 / E4M3_MAX)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(c):
    """(query, key) pairs that see each other, over all entries, and keys that some query sees"""
    pairs = keys = 0
    for n, q0 in zip(_key_len(c), _q_start(c)):
        seen = [False] * n
        for p in range(q0, q0 + c["Tq"]):
            lo, hi = max(0, p - c["left"]), min(n, p + c["right"] + 1)
            pairs += max(0, hi - lo) + max(0, min(c["sinks"], lo, hi, n))
            if c["Tq"] != c["Tk"] and hi > lo:
                seen[lo:hi] = [True] * (hi - lo)
        keys += n if c["Tq"] == c["Tk"] else sum(seen) + min(c["sinks"], n - sum(seen))
    return pairs, keys


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "attention":
        pairs, keys = _pairs(c)
        rows, kv = c["B"] * c["Tq"] * c["Hq"] * c["dh"], keys * c["Hkv"] * c["dh"]
        if c["train"]:
            return {"bytes": e * (4 * rows + 4 * kv), "flops": 14 * pairs * c["Hq"] * c["dh"]}
        return {"bytes": e * (2 * rows + 2 * kv), "flops": 4 * pairs * c["Hq"] * c["dh"]}
    if c["op"] == "adapter":
        M, K, N, R = c["rows"], c["K"], c["N"], c["R"]
        start, which = _segments(c)
        held = sum(start[i + 1] - start[i] for i, w in enumerate(which) if w >= 0)
        used = len({w for w in which if w >= 0})
        low = used * R * (K + N)
        if c["train"]:
            return {"bytes": e * (2 * M * K + 2 * M * N + N * K + 2 * low), "flops": 4 * M * K * N + 6 * held * R * (K + N)}
        return {"bytes": e * (M * K + M * N + N * K + low), "flops": 2 * M * K * N + 2 * held * R * (K + N)}
    n, blocks = sum(_sizes(c)), sum(-(-k // BLOCK) for k in _sizes(c))
    moments = 16 * n if c["bits"] == 32 else 4 * n + 16 * blocks
    return {"bytes": n * (2 * e + (4 if c["grad"] == "fp32" else 2)) + moments, "flops": 14 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "attention":
        return _exact_attention(s, c)
    if c["op"] == "adapter":
        return _exact_adapter(s, c)
    return _exact_adamw(s, c)


@torch.no_grad()
def _exact_attention(s, c):
    q, k, v = (s[n].double() for n in "qkv")
    B, Tq, Hq, dh = q.shape
    Tk, Hkv = k.shape[1:3]
    G, scale = Hq // Hkv, 1 / math.sqrt(dh)
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for b in range(B):
        for lo in range(0, Tq, 2048):
            hi = min(Tq, lo + 2048)
            p = (int(s["q_start"][b]) + torch.arange(lo, hi, device=q.device))[:, None]
            # the columns that any of these rows can see: the first keys, and from the first row's window to the last row's
            k1 = min(int(s["key_len"][b]), int(p[-1]) + c["right"] + 1)
            k0 = max(0, int(p[0]) - c["left"])
            cols = torch.cat((torch.arange(0, min(c["sinks"], k0, max(0, k1)), device=q.device), torch.arange(k0, max(k0, k1), device=q.device)))
            if not len(cols):
                continue
            hidden = ((cols < p - c["left"]) & (cols >= c["sinks"])) | (cols > p + c["right"])
            for h in range(Hkv):
                kk, vv = k[b, cols, h], v[b, cols, h]
                for g in range(h * G, h * G + G):
                    x = (q[b, lo:hi, g] @ kk.T) * scale
                    x[hidden] = -math.inf
                    x = torch.exp(x - x.max(1, keepdim=True).values.nan_to_num(neginf=0.0))
                    total = x.sum(1, keepdim=True)
                    x = torch.where(total > 0, x / total, 0.0)
                    o = x @ vv
                    out[b, lo:hi, g] = o
                    if not c["train"]:
                        continue
                    do = s["dout"][b, lo:hi, g].double()
                    dv[b].index_put_((cols, torch.tensor(h, device=q.device)), x.T @ do, accumulate=True)
                    ds = x * (do @ vv.T - (do * o).sum(1, keepdim=True)) * scale
                    dq[b, lo:hi, g] = ds @ kk
                    dk[b].index_put_((cols, torch.tensor(h, device=q.device)), ds.T @ q[b, lo:hi, g], accumulate=True)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if c["train"] else out


@torch.no_grad()
def _exact_adapter(s, c):
    x, w, a, b = (s[n].double() for n in ("x", "weight", "a", "b"))
    y = torch.addmm(s["bias"].double(), x, w.T)
    start, which = s["start"].tolist(), s["which"].tolist()
    parts = [(i, j, n, float(s["scaling"][n])) for i, j, n in zip(start, start[1:], which) if n >= 0 and j > i]
    for i, j, n, f in parts:
        y[i:j] += f * ((x[i:j] @ a[n].T) @ b[n].T)
    if not c["train"]:
        return y
    dy = s["dy"].double()
    dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    for i, j, n, f in parts:
        low = f * (dy[i:j] @ b[n])
        dx[i:j] += low @ a[n]
        da[n] += low.T @ x[i:j]
        db[n] += f * (dy[i:j].T @ (x[i:j] @ a[n].T))
    return {"y": y, "dx": dx, "da": da, "db": db}


@torch.no_grad()
def _exact_adamw(s, c):
    """parameters and 32-bit moments; what a rounding by chance leaves of the 8-bit ones has no value in 64 bits but its scales"""
    h, moments = HYPER, s["moments"]
    new, at = s["flat"].double(), 0
    views = [new[i:i + t.numel()] for i, t in zip(_starts([t.numel() for t in s["params"]]), s["params"])]
    scales = [torch.empty_like(t, dtype=torch.float64) for t in moments[1::2]] if c["bits"] == 8 else [torch.zeros_like(t, dtype=torch.float64) for t in moments]
    for p, g in zip(views, s["grads"]):
        n = p.numel()
        padded = -(-n // BLOCK) * BLOCK
        if c["bits"] == 8:
            per = [(moments[i][at:at + padded].double().view(-1, BLOCK) * moments[i + 1][at // BLOCK:(at + padded) // BLOCK, None].double()).view(-1)[:n] for i in (0, 2)]
            m, v = per[0], per[1] ** 2
        else:
            m, v = (t[at:at + n].double() for t in moments)
        g = g.double() * h["grad_scale"]
        m = h["beta1"] * m + (1 - h["beta1"]) * g
        v = h["beta2"] * v + (1 - h["beta2"]) * g ** 2
        hat_m, hat_v = m / (1 - h["beta1"] ** h["step"]), v / (1 - h["beta2"] ** h["step"])
        p -= h["lr"] * h["weight_decay"] * p + h["lr"] * hat_m / (hat_v.sqrt() + h["eps"])
        for k, t in enumerate((m, v.sqrt() if c["bits"] == 8 else v)):
            if c["bits"] == 8:
                top = torch.nn.functional.pad(t, (0, padded - n)).view(-1, BLOCK).abs().amax(1)
                scales[k][at // BLOCK:(at + padded) // BLOCK] = top.clamp_min(TINY) / E4M3_MAX
            else:
                scales[k][at:at + n] = t
        at += padded
    return {"params": new, "moments": [None, scales[0], None, scales[1]] if c["bits"] == 8 else scales}
