"""Timed calls of the training-step operators that stand around attention: the plain form of each, and the framework's.

Three operators in both directions:

* layer norm over rows, with the rows' statistics, and its gradients (input, scale and shift);
* rotary positions on query and key heads, and the inverse rotation (its gradient);
* the cross entropy of a linear head, from hidden states and the head's weight, and its gradients.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass in the
plain form (elementary torch operations in 32 bits, rounded once) or, with ``own``, through ``pdum_dsl_b200.kernels``,
``work`` counts what a pass cannot do without, and ``exact`` evaluates the definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
EPS = 1e-5
IGNORE = -100


def _kernels():
    from pdum_dsl_b200 import kernels

    return kernels


# ---- the cases ------------------------------------------------------------------------------------------------------
def _norm(name, back, rows, cols, dtype, params):
    return {"name": name, "op": "norm", "back": back, "rows": rows, "cols": cols, "dtype": dtype, "params": params}


def _rotary(name, back, batch, heads_q, heads_k, length, head_dim, rotary_dim, layout, interleaved, dtype, first, scaling):
    return {"name": name, "op": "rotary", "back": back, "batch": batch, "heads_q": heads_q, "heads_k": heads_k,
            "length": length, "head_dim": head_dim, "rotary_dim": rotary_dim, "layout": layout,
            "interleaved": interleaved, "dtype": dtype, "first": first, "scaling": scaling}


def _loss(name, back, tokens, vocab, width, ignored):
    return {"name": name, "op": "loss", "back": back, "tokens": tokens, "vocab": vocab, "width": width, "ignored": ignored}


def listed():
    return [
        # one token's row while generating: nothing but latency
        _norm("norm_one_row", False, 1, 4096, "bf16", "f32"),
        # a training batch's activations (the benchmark's row-statistics matrix, in the training type)
        _norm("norm_batch", False, 8192, 4096, "bf16", "f32"),
        # the same matrix's gradient in 32 bits
        _norm("norm_grad_f32", True, 8192, 4096, "f32", "f32"),
        # a ragged batch at an odd width: rows that no 16-byte access fits
        _norm("norm_grad_ragged", True, 4099, 1001, "bf16", "bf16"),
        # norms of every head's queries: very many short rows
        _norm("norm_grad_heads", True, 262144, 128, "bf16", "f32"),
        # one new token for each of 64 sequences, far into a long context
        _rotary("rotary_decode", False, 64, 32, 8, 1, 128, 128, "bthd", False, "bf16", 1_000_000, "by_parts"),
        # a training batch with grouped keys (the benchmark's attention shape)
        _rotary("rotary_batch", False, 8, 32, 8, 4096, 128, 128, "bhtd", False, "bf16", 0, "none"),
        # its gradient where part of the head turns, interleaved pairs, 32 bits, an odd length
        _rotary("rotary_grad_part", True, 4, 16, 16, 2047, 80, 48, "bthd", True, "f32", 8192, "linear"),
        # the loss of one sequence's last token: reading the head's weight once
        _loss("loss_one_token", False, 1, 32000, 2048, 0.0),
        # a batch's loss alone (evaluation)
        _loss("loss_batch", False, 4096, 65536, 2048, 0.1),
        # a ragged batch's gradient over an odd vocabulary
        _loss("loss_grad_ragged", True, 1021, 50021, 1000, 0.3),
        # a training step's gradient over a large vocabulary
        _loss("loss_grad_batch", True, 8192, 128000, 4096, 0.1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "loss"])
    back = rng.random() < 0.5
    if op == "norm":
        cols = _log(rng, 32, 16384)
        if rng.random() < 0.5:
            cols = max(32, cols // 64 * 64)
        rows = _log(rng, 1, min(262144, (1 << 25) // cols))
        dtype = rng.choice(["bf16", "f32"])
        c = _norm("", back, rows, cols, dtype, rng.choice(["f32", dtype]))
    elif op == "rotary":
        head_dim = rng.choice([32, 64, 80, 96, 128, 192, 256, 2 * rng.randint(8, 128)])
        rotary_dim = head_dim if rng.random() < 0.6 else 2 * rng.randint(1, head_dim // 2)
        heads_k = rng.choice([1, 2, 4, 8, 16])
        heads_q = heads_k * rng.choice([1, 1, 2, 4])
        length = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(64, (1 << 27) // (length * (heads_q + heads_k) * head_dim))))
        c = _rotary("", back, batch, heads_q, heads_k, length, head_dim, rotary_dim, rng.choice(["bhtd", "bthd"]),
                    rng.random() < 0.5, rng.choice(["bf16", "f32"]), rng.choice([0, _log(rng, 1, 4_000_000)]),
                    rng.choice(["none", "linear", "by_parts"]))
    else:
        width = 8 * _log(rng, 8, 512)
        vocab = _log(rng, 500, 128000)
        tokens = _log(rng, 1, 8192)
        c = _loss("", back, tokens, vocab, width, rng.choice([0.0, 0.1, 0.5]))
    del c["name"]
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians per position of each rotated pair, in 64 bits; and the factor on cos and sin."""
    r = case["rotary_dim"]
    f = 10000.0 ** (-np.arange(0, r, 2, dtype=np.float64) / r)
    if case["scaling"] == "linear":  # every position divided by 4
        return f / 4.0, 1.0
    if case["scaling"] == "by_parts":  # factor 16 on a context of 4096: slow pairs interpolated, fast ones kept
        turns = 4096.0 * f / (2.0 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * keep + f / 16.0 * (1.0 - keep), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _draw_like(shape, gen, dtype):
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "norm":
        dtype, ptype = _TYPES[case["dtype"]], _TYPES[case["params"]]
        rows, cols = case["rows"], case["cols"]
        # activations: every channel with a size and an offset of its own, a few of them large
        size = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
        x = torch.randn((rows, cols), device="cuda", generator=gen) * size
        x += 0.3 * torch.randn(cols, device="cuda", generator=gen) + 0.1
        s = {"case": case, "x": x.to(dtype)}
        s["gamma"] = (1.0 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).to(ptype)
        s["beta"] = (0.1 * torch.randn(cols, device="cuda", generator=gen)).to(ptype)
        if case["back"]:
            s["dout"] = _draw_like((rows, cols), gen, dtype)
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + EPS)
        return s
    if case["op"] == "rotary":
        dtype = _TYPES[case["dtype"]]

        def heads(n):
            b, t, d = case["batch"], case["length"], case["head_dim"]
            if case["layout"] == "bthd":  # as a projection leaves them: a view with the heads moved up
                return _draw_like((b, t, n, d), gen, dtype).transpose(1, 2)
            return _draw_like((b, n, t, d), gen, dtype)

        inv_freq, amplitude = _frequencies(case)
        # sequences that begin at positions of their own
        at = torch.randint(0, 1000, (case["batch"], 1), device="cuda", generator=gen) + case["first"]
        positions = at + torch.arange(case["length"], device="cuda")
        return {"case": case, "q": heads(case["heads_q"]), "k": heads(case["heads_k"]), "inv_freq": inv_freq,
                "amplitude": amplitude, "positions": positions, "on_gpu": torch.from_numpy(inv_freq).to("cuda")}
    n, v, d = case["tokens"], case["vocab"], case["width"]
    w = torch.randn((v, d), device="cuda", generator=gen).mul_(1.5 / math.sqrt(d)).to(torch.bfloat16)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = torch.randn((n, d), device="cuda", generator=gen)
    # every second token leans towards its target
    x[1::2] += w[target[1::2]].float() * (4.0 / 2.25)
    skip = torch.rand(n, device="cuda", generator=gen) < case["ignored"]
    skip[0] = False
    s = {"case": case, "x": x.to(torch.bfloat16), "w": w, "target": torch.where(skip, IGNORE, target)}
    if case["back"]:
        s["dloss"] = torch.full((n,), 1.0 / int((~skip).sum()), device="cuda")
        s["lse"] = torch.logsumexp(s["x"].float() @ w.float().t(), 1)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    x = s["x"].float()
    c = x.shape[1]
    g = s["gamma"].float()
    if not s["case"]["back"]:
        mean = x.sum(1, keepdim=True) / c
        z = x - mean
        rstd = 1.0 / torch.sqrt((z * z).sum(1, keepdim=True) / c + EPS)
        return (z * rstd * g + s["beta"].float()).to(s["x"].dtype), mean[:, 0], rstd[:, 0]
    rstd = s["rstd"][:, None]
    z = (x - s["mean"][:, None]) * rstd
    dy = s["dout"].float()
    dz = dy * g
    dx = rstd * (dz - dz.sum(1, keepdim=True) / c - z * ((dz * z).sum(1, keepdim=True) / c))
    p = s["gamma"].dtype
    return dx.to(s["x"].dtype), (dy * z).sum(0).to(p), dy.sum(0).to(p)


def _plain_rotary(s):
    case = s["case"]
    r = case["rotary_dim"]
    # the angles of far positions lose their digits in 32 bits
    angle = s["positions"].double()[:, None, :, None] * s["on_gpu"]
    cos, sin = (torch.cos(angle) * s["amplitude"]).float(), (torch.sin(angle) * s["amplitude"]).float()
    if case["back"]:
        sin = -sin

    def turn(t):
        x = t.float()
        y = x.clone()
        a, b = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(t.dtype)

    return turn(s["q"]), turn(s["k"])


def _plain_loss(s):
    x, w, t = s["x"].float(), s["w"].float(), s["target"]
    valid = t != IGNORE
    at = t.clamp(min=0)[:, None]
    logits = x @ w.t()
    if not s["case"]["back"]:
        m = logits.max(1, keepdim=True).values
        lse = (m + torch.log(torch.exp(logits - m).sum(1, keepdim=True)))[:, 0]
        return torch.where(valid, lse - logits.gather(1, at)[:, 0], 0.0), lse
    p = torch.exp(logits - s["lse"][:, None])
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p *= (s["dloss"] * valid)[:, None]
    return (p @ w).to(torch.bfloat16), (p.t() @ x).to(torch.bfloat16)


def run(state):
    s, case = state, state["case"]
    if own:
        k = _kernels()
        if case["op"] == "norm":
            if case["back"]:
                return k.layernorm_backward(s["dout"], s["x"], s["mean"], s["rstd"], s["gamma"])
            return k.layernorm(s["x"], s["gamma"], s["beta"], eps=EPS, return_stats=True)
        if case["op"] == "rotary":
            return k.rotary(s["q"], s["k"], inv_freq=s["inv_freq"], positions=s["positions"],
                            interleaved=case["interleaved"], amplitude=s["amplitude"], inverse=case["back"])
        if case["back"]:
            return k.linear_cross_entropy_backward(s["x"], s["w"], s["target"], s["dloss"], s["lse"], ignore_index=IGNORE)
        return k.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE, return_lse=True)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "loss": _plain_loss}[case["op"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        rows, cols, e, p = case["rows"], case["cols"], _SIZE[case["dtype"]], _SIZE[case["params"]]
        if case["back"]:  # x, dout -> dx; the statistics and gamma in, two gradients out
            return {"bytes": 3 * rows * cols * e + 8 * rows + 3 * cols * p, "flops": 12 * rows * cols}
        return {"bytes": 2 * rows * cols * e + 8 * rows + 2 * cols * p, "flops": 7 * rows * cols}
    if case["op"] == "rotary":
        heads = case["batch"] * case["length"] * (case["heads_q"] + case["heads_k"])
        return {"bytes": 2 * heads * case["head_dim"] * _SIZE[case["dtype"]] + 8 * case["batch"] * case["length"],
                "flops": 3 * heads * case["rotary_dim"]}
    n, v, d = case["tokens"], case["vocab"], case["width"]
    if case["back"]:  # the logits again, then the two gradients
        return {"bytes": 4 * (n * d + v * d) + 16 * n, "flops": 6 * n * v * d}
    return {"bytes": 2 * (n * d + v * d) + 16 * n, "flops": 2 * n * v * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _exact_norm(s):
    x, g, b = s["x"].double(), s["gamma"].double(), s["beta"].double()
    if not s["case"]["back"]:
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS).rsqrt()
        return g * (x - mean.unsqueeze(1)) * rstd.unsqueeze(1) + b, mean, rstd
    mean, rstd, dy = s["mean"].double(), s["rstd"].double(), s["dout"].double()
    z = torch.einsum("rc,r->rc", x - mean.unsqueeze(1), rstd)
    dgamma = torch.einsum("rc,rc->c", dy, z)
    up = dy * g
    along = torch.einsum("rc,rc->r", up, z) / x.shape[1]
    dx = (up - up.mean(dim=1, keepdim=True) - z * along.unsqueeze(1)) * rstd.unsqueeze(1)
    return dx, dgamma, dy.sum(dim=0)


def _exact_rotary(s):
    case = s["case"]
    half = case["rotary_dim"] // 2
    radians = torch.einsum("bt,j->btj", s["positions"].double(), s["on_gpu"])
    factor = torch.polar(torch.full_like(radians, s["amplitude"]), -radians if case["back"] else radians)[:, None]

    def turn(t):
        head, rest = t.double().split([2 * half, case["head_dim"] - 2 * half], dim=-1)
        if case["interleaved"]:
            pairs = head.unflatten(-1, (half, 2))
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * factor).flatten(-2)
        else:
            z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * factor
            turned = torch.cat([z.real, z.imag], dim=-1)
        return torch.cat([turned, rest], dim=-1)

    return turn(s["q"]), turn(s["k"])


def _exact_loss(s):
    x, w, t = s["x"].double(), s["w"].double(), s["target"]
    logits = x @ w.mT
    rows = torch.nonzero(t != IGNORE)[:, 0]
    if not s["case"]["back"]:
        lse = torch.logsumexp(logits, dim=1)
        loss = torch.zeros(len(t), dtype=torch.float64, device="cuda")
        loss[rows] = lse[rows] - logits[rows, t[rows]]
        return loss, lse
    up = torch.zeros(len(t), dtype=torch.float64, device="cuda")
    up[rows] = s["dloss"].double()[rows]
    g = logits.sub_(s["lse"].double().unsqueeze(1)).exp_()
    g[rows, t[rows]] -= 1.0
    g *= up.unsqueeze(1)
    return g @ w, g.mT @ x


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "loss": _exact_loss}[case["op"]](s)
