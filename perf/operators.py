"""Workloads of the operators around the fused linears: each in a plain PyTorch form and as a call of this package.

``own`` selects which one ``run`` computes.  The plain form uses elementary torch operations in 32 bits (integers of 64
bits for the dropout generator) and rounds once at the end; ``exact`` evaluates the definitions in 64 bits.

Kinds of cases:

* ``ce``        softmax cross entropy behind a projection onto a large vocabulary, loss alone or with its two gradients
* ``norm``      (residual + dropout(x)) and its RMS norm, forward and backward; or the norm alone
* ``norm8``     the same rows in inference, leaving as e4m3 values with one scale a row
* ``linear8``   a projection of e4m3 rows by an e4m3 weight, from rows already in 8 bits or from bf16 rows
* ``dropout``   counter-based dropout, forward and backward
"""

import functools
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5
_IGNORE = -100
_E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the loss of a training step at an 8B model's shapes: the repository's cross-entropy benchmark
        {"name": "ce_step", "kind": "ce", "rows": 8192, "dim": 4096, "vocab": 128256, "grad": True, "reduction": "mean", "ignored": 0.05},
        # a short packed batch of a small model: odd vocabulary, odd row count, a third of the labels masked
        {"name": "ce_step_ragged", "kind": "ce", "rows": 1003, "dim": 1032, "vocab": 32003, "grad": True, "reduction": "sum", "ignored": 0.3},
        # validation loss: no gradient
        {"name": "ce_eval", "kind": "ce", "rows": 2048, "dim": 2048, "vocab": 50257, "grad": False, "reduction": "mean", "ignored": 0.05},
        # a sublayer's end in a training step: dropout, residual addition, norm, and all gradients
        {"name": "norm_step", "kind": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "p": 0.1, "residual": True},
        # the same in half precision at a width that is no multiple of anything, without dropout
        {"name": "norm_step_ragged", "kind": "norm", "rows": 1777, "cols": 1531, "dtype": "fp16", "p": 0.0, "residual": True},
        # a prompt on its way into an 8-bit projection
        {"name": "norm8_prompt", "kind": "norm8", "rows": 8192, "cols": 5120, "dtype": "bf16", "residual": True},
        # one token on the same way: latency
        {"name": "norm8_token", "kind": "norm8", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True},
        # gate and up projection of a prompt, rows already in 8 bits
        {"name": "linear8_prompt", "kind": "linear8", "rows": 8192, "dim": 4096, "out": 28672, "quantize": False},
        # q, k and v of one token, from a bf16 row
        {"name": "linear8_token", "kind": "linear8", "rows": 1, "dim": 4096, "out": 6144, "quantize": True},
        # a small mixed batch
        {"name": "linear8_ragged", "kind": "linear8", "rows": 333, "dim": 1552, "out": 2056, "quantize": True},
        # dropout on an MLP's hidden activations in a training step
        {"name": "dropout_step", "kind": "dropout", "rows": 16384, "cols": 14336, "dtype": "bf16", "p": 0.1},
        # odd rows in single precision
        {"name": "dropout_ragged", "kind": "dropout", "rows": 4097, "cols": 1023, "dtype": "fp32", "p": 0.5},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "norm", "norm", "norm8", "linear8", "linear8", "dropout"])
    if kind == "ce":
        grad = rng.random() < 0.7
        return {"kind": kind, "rows": _log(rng, 1, 8192), "dim": 8 * _log(rng, 8, 512), "vocab": _log(rng, 1000, 128256), "grad": grad,
                "reduction": rng.choice(["mean", "sum"]), "ignored": rng.choice([0.0, 0.05, 0.3])}
    if kind == "linear8":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "dim": 16 * _log(rng, 8, 256), "out": 8 * _log(rng, 16, 3584),
                "quantize": rng.random() < 0.5}
    case = {"kind": kind, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 14336 if kind == "dropout" else 8192)}
    if rng.random() < 0.5:
        case["cols"] = max(64, case["cols"] // 64 * 64)
    case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "dropout":
        case["p"] = rng.choice([0.05, 0.1, 0.5])
    else:
        case["residual"] = rng.random() < 0.75
        if kind == "norm":
            case["p"] = rng.choice([0.0, 0.1, 0.2]) if case["residual"] else 0.0
    return case


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    kind = case["kind"]
    if kind == "ce":
        m, k, v = case["rows"], case["dim"], case["vocab"]
        s["x"] = normal(m, k).requires_grad_(case["grad"])
        s["weight"] = normal(v, k, std=k**-0.5).requires_grad_(case["grad"])
        target = torch.randint(0, v, (m,), generator=g, device="cuda", dtype=torch.int32)
        masked = torch.rand(m, generator=g, device="cuda") < case["ignored"]
        masked[0] = False  # a batch has a label
        s["target"] = torch.where(masked, torch.full_like(target, _IGNORE), target)
        return s
    if kind == "linear8":
        m, k, n = case["rows"], case["dim"], case["out"]
        w = normal(n, k, std=k**-0.5, dtype=torch.float32)
        s["w_scale"] = w.abs().amax(1) / _E4M3_MAX
        s["w8"] = (w / s["w_scale"][:, None]).to(torch.float8_e4m3fn)
        s["x"] = normal(m, k)
        if not case["quantize"]:
            x = s.pop("x").float()
            s["x_scale"] = x.abs().amax(1) / _E4M3_MAX
            s["x8"] = (x / s["x_scale"][:, None]).to(torch.float8_e4m3fn)
        return s
    m, n, dtype = case["rows"], case["cols"], _DTYPES[case["dtype"]]
    train = kind in ("norm", "dropout")
    s["x"] = normal(m, n, dtype=dtype).requires_grad_(train)
    if kind == "dropout":
        s["dout"] = normal(m, n, dtype=dtype)
    else:
        s["weight"] = normal(n, std=0.1, mean=1.0, dtype=dtype).requires_grad_(train)
        if case["residual"]:
            s["residual"] = normal(m, n, dtype=dtype).requires_grad_(train)
        if train:
            s["dout"] = normal(m, n, dtype=dtype)
            if case["residual"]:
                s["dh"] = normal(m, n, dtype=dtype)
    if case.get("p"):
        s["rng"] = torch.tensor([(seed * 0x9E3779B1 + 12345) % 2**62, seed % 1000], dtype=torch.int64, device="cuda")  # seed, step
        s["stream"] = seed % 64
    return s


# ------------------------------------------------------------------------------------------------ the calls of this package
def _run_own(s):
    import coda_kernels_b200 as ck

    case = s["case"]
    kind = case["kind"]
    if kind == "ce":
        loss = ck.linear_cross_entropy_pieces(s["x"], s["weight"], s["target"], ignore_index=_IGNORE, reduction=case["reduction"])
        if not case["grad"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (s["x"], s["weight"]))
        return {"loss": loss.detach(), "dx": dx, "dweight": dw}
    if kind == "norm":
        if not case["residual"]:
            out = ck.rms_norm(s["x"], s["weight"], _EPS)
            dx, dw = torch.autograd.grad(out, (s["x"], s["weight"]), s["dout"])
            return {"out": out.detach(), "dx": dx, "dweight": dw}
        out, h = ck.add_rms_norm(s["x"], s["residual"], s["weight"], _EPS, p=case["p"], rng=s.get("rng"), stream=s.get("stream", 0))
        dx, dres, dw = torch.autograd.grad((out, h), (s["x"], s["residual"], s["weight"]), (s["dout"], s["dh"]))
        return {"out": out.detach(), "h": h.detach(), "dx": dx, "dresidual": dres, "dweight": dw}
    if kind == "norm8":
        if not case["residual"]:
            q, scale = ck.rms_norm_e4m3(s["x"], s["weight"], _EPS)
            return {"q": q, "scale": scale}
        q, scale, h = ck.add_rms_norm_e4m3(s["x"], s["residual"], s["weight"], _EPS)
        return {"q": q, "scale": scale, "h": h}
    if kind == "linear8":
        if case["quantize"]:
            q, scale = ck.quantize_e4m3(s["x"])
            return {"q": q, "scale": scale, "out": ck.linear_e4m3(q, scale, s["w8"], s["w_scale"])}
        return {"out": ck.linear_e4m3(s["x8"], s["x_scale"], s["w8"], s["w_scale"])}
    out = ck.dropout(s["x"], case["p"], s["rng"], stream=s["stream"])
    return {"out": out.detach(), "dx": torch.autograd.grad(out, s["x"], s["dout"])[0]}


# ------------------------------------------------------------------------------------------------ plain forms
def _philox_round(state, i):
    """One round of Philox4x32 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, SC'11) on int64 holding 32-bit words."""
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    k0, k1 = (k0 + i * 0x9E3779B9) & 0xFFFFFFFF, (k1 + i * 0xBB67AE85) & 0xFFFFFFFF
    hi_a, hi_b = (a >> 32) & 0xFFFFFFFF, (b >> 32) & 0xFFFFFFFF
    return hi_b ^ c1 ^ k0, b & 0xFFFFFFFF, hi_a ^ c3 ^ k1, a & 0xFFFFFFFF, state[4], state[5]


def _keep(rows, cols, p, rng, stream):
    """Which elements stay: word c % 4 of the block whose counter is (r * ceil(cols / 4) + c // 4, step, stream)."""
    blocks = -(-cols // 4)
    b = torch.arange(rows * blocks, dtype=torch.int64, device=rng.device)
    seed, step = rng[0], rng[1] & 0xFFFFFFFF
    zero = torch.zeros_like(b)
    start = (b & 0xFFFFFFFF, b >> 32, zero + step, zero + stream, seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    words = functools.reduce(_philox_round, range(10), start)[:4]
    u = torch.stack(words, dim=1).view(rows, blocks * 4)[:, :cols]
    return u >= round(p * 2**32)


def _dropped(x, keep, p):
    return torch.where(keep, x * (1.0 / (1.0 - p)), torch.zeros_like(x))


def _rows_to_e4m3(out):
    scale = (out.abs().amax(1) / _E4M3_MAX).clamp_min(2.0**-126)
    return (out / scale[:, None]).to(torch.float8_e4m3fn), scale


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "ce":
        x, w, t = s["x"].detach().float(), s["weight"].detach().float(), s["target"].long()
        z = x @ w.t()
        top = z.amax(1, keepdim=True)
        e = (z - top).exp()
        total = e.sum(1, keepdim=True)
        valid = t != _IGNORE
        label = torch.where(valid, t, torch.zeros_like(t))[:, None]
        rows = torch.where(valid, (top + total.log() - z.gather(1, label))[:, 0], torch.zeros_like(top[:, 0]))
        alpha = 1.0 / valid.sum() if case["reduction"] == "mean" else torch.ones((), device=x.device)
        loss = rows.sum() * alpha
        if not case["grad"]:
            return {"loss": loss}
        del z
        g = e.div_(total)
        g.scatter_add_(1, label, torch.full_like(total, -1.0))
        g.mul_(torch.where(valid, alpha, torch.zeros_like(alpha))[:, None])
        dtype = s["x"].dtype
        return {"loss": loss, "dx": (g @ w).to(dtype), "dweight": (g.t() @ x).to(dtype)}
    if kind == "linear8":
        if case["quantize"]:
            q, scale = _rows_to_e4m3(s["x"].float())
        else:
            q, scale = s["x8"], s["x_scale"]
        out = ((q.float() @ s["w8"].float().t()) * scale[:, None] * s["w_scale"]).to(torch.bfloat16)
        return {"q": q, "scale": scale, "out": out} if case["quantize"] else {"out": out}
    x = s["x"].detach().float()
    dtype = s["x"].dtype
    p = case.get("p", 0.0)
    keep = _keep(x.shape[0], x.shape[1], p, s["rng"], s["stream"]) if p else None
    if kind == "dropout":
        return {"out": _dropped(x, keep, p).to(dtype), "dx": _dropped(s["dout"].float(), keep, p).to(dtype)}
    w = s["weight"].detach().float()
    h = _dropped(x, keep, p) if p else x
    if case["residual"]:
        h = h + s["residual"].detach().float()
    r = (h.square().mean(1, keepdim=True) + _EPS).rsqrt()
    xh = h * r
    out = xh * w
    if kind == "norm8":
        q, scale = _rows_to_e4m3(out)
        return {"q": q, "scale": scale, "h": h.to(dtype)} if case["residual"] else {"q": q, "scale": scale}
    dout = s["dout"].float()
    gw = dout * w
    dh = r * (gw - xh * (gw * xh).mean(1, keepdim=True))
    dw = (dout * xh).sum(0)
    if not case["residual"]:
        return {"out": out.to(dtype), "dx": dh.to(dtype), "dweight": dw.to(dtype)}
    dh = dh + s["dh"].float()
    dx = _dropped(dh, keep, p) if p else dh
    return {"out": out.to(dtype), "h": h.to(dtype), "dx": dx.to(dtype), "dresidual": dh.to(dtype), "dweight": dw.to(dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "ce":
        m, k, v = case["rows"], case["dim"], case["vocab"]
        tensors = 2 * (m * k + v * k)
        # logits; with gradients also their products with the weight and with the rows.  dloss multiplies at the end.
        return {"bytes": tensors * (2 if case["grad"] else 1) + 4 * m, "flops": (6 if case["grad"] else 2) * m * v * k}
    if kind == "linear8":
        m, k, n = case["rows"], case["dim"], case["out"]
        return {"bytes": m * k * (3 if case["quantize"] else 1) + n * k + 4 * (m + n) + 2 * m * n, "flops": 2 * m * n * k}
    m, n, s = case["rows"], case["cols"], _DTYPES[case["dtype"]].itemsize
    if kind == "dropout":
        return {"bytes": 4 * m * n * s, "flops": 2 * m * n}
    if kind == "norm8":
        return {"bytes": m * n * s * (3 if case["residual"] else 1) + m * n + 4 * m + n * s, "flops": 7 * m * n}
    # forward: x (, residual) -> out (, h).  Backward, which comes later: dout (, dh) and h again -> dx (, dresidual), dweight.
    return {"bytes": m * n * s * (9 if case["residual"] else 5) + 3 * n * s, "flops": 17 * m * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def _mul_words(a, b):
    """(high, low) 32-bit words of a * b for 32-bit words in int64, from 16-bit halves."""
    al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    low = al * bl
    mid = ah * bl + (low >> 16)
    mid2 = al * bh + (mid & 0xFFFF)
    return ah * bh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_keep(rows, cols, p, rng, stream):
    seed, step = (int(v) for v in rng.tolist())
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    col = torch.arange(-(-cols // 4), device="cuda")
    kept = torch.empty(rows, cols, dtype=torch.bool, device="cuda")
    for first in range(0, rows, 2048):
        row = torch.arange(first, min(rows, first + 2048), device="cuda")
        block = row[:, None] * col.numel() + col
        c = [block % 2**32, block // 2**32, torch.full_like(block, step % 2**32), torch.full_like(block, stream)]
        k = list(key)
        for _ in range(10):
            h0, l0 = _mul_words(c[0], 0xD2511F53)
            h1, l1 = _mul_words(c[2], 0xCD9E8D57)
            c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
            k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
        for j in range(min(4, cols)):
            mine = kept[first:first + row.numel(), j::4]
            mine.copy_(c[j][:, :mine.shape[1]] >= round(p * 2**32))
    return kept


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point() and k != "rng"}
    kind = case["kind"]
    if kind == "ce":
        x, w, t = d["x"], d["weight"], s["target"].long()
        m = x.shape[0]
        count = int((t >= 0).sum())
        a = 1.0 / count if case["reduction"] == "mean" else 1.0
        loss, dx, dw = 0.0, torch.empty_like(x), torch.zeros_like(w)
        for i in range(0, m, 2048):
            rows = slice(i, min(m, i + 2048))
            z = x[rows] @ w.T
            lse = torch.logsumexp(z, 1)
            at = (t[rows] >= 0).nonzero()[:, 0]
            loss = loss + (lse[at] - z[at, t[rows][at]]).sum() * a
            if case["grad"]:
                soft = torch.exp(z - lse[:, None]) * (t[rows] >= 0)[:, None]
                soft[at, t[rows][at]] -= 1.0
                dx[rows] = soft @ w * a
                dw += soft.T @ x[rows] * a
        loss = torch.as_tensor(loss, dtype=torch.float64, device="cuda")
        return {"loss": loss, "dx": dx, "dweight": dw} if case["grad"] else {"loss": loss}

    def rows8(v):
        scale = torch.clamp(v.abs().max(1).values / 448.0, min=2.0**-126)
        return v / scale[:, None], scale

    if kind == "linear8":
        if not case["quantize"]:
            x = s["x8"].double() * s["x_scale"].double()[:, None]
            return {"out": x @ (s["w8"].double() * s["w_scale"].double()[:, None]).T}
        q, scale = rows8(d["x"])
        x = q.to(torch.float8_e4m3fn).double() * scale[:, None]
        return {"q": q, "scale": scale, "out": x @ (s["w8"].double() * s["w_scale"].double()[:, None]).T}
    p = case.get("p", 0.0)
    keep = _exact_keep(case["rows"], case["cols"], p, s["rng"], s["stream"]) if p else torch.ones((), dtype=torch.bool, device="cuda")
    if kind == "dropout":
        return {"out": d["x"] * keep / (1 - p), "dx": d["dout"] * keep / (1 - p)}
    h = d["x"] * keep / (1 - p) + d.get("residual", 0.0)
    n = h.shape[1]
    rms = torch.sqrt((h * h).sum(1) / n + _EPS)[:, None]
    out = h / rms * d["weight"]
    if kind == "norm8":
        q, scale = rows8(out)
        return {"q": q, "scale": scale, "h": h} if case["residual"] else {"q": q, "scale": scale}
    gw = d["dout"] * d["weight"]
    dh = gw / rms - h * (gw * h).sum(1, keepdim=True) / (n * rms**3) + d.get("dh", 0.0)
    dw = (d["dout"] * h / rms).sum(0)
    if not case["residual"]:
        return {"out": out, "dx": dh, "dweight": dw}
    return {"out": out, "h": h, "dx": dh * keep / (1 - p), "dresidual": dh, "dweight": dw}
