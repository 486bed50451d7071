"""The training operators in a row, as a step of an attention block uses them: layer norm -> projections -> rotary
positions -> attention -> projection and residual -> layer norm -> the head's cross entropy over a padded batch, and all
the way back, against the same step in 64 bits under torch's autograd.

Tolerance.  Between an input and a gradient lie at most 16 tensors that are rounded to bf16 (the normed rows, q / k / v,
the turned q / k, the probabilities, the attention's output and projection, the residual sum, the normed rows, G, and
their gradients on the way back), each off by at most 2^-8 of itself; norms, turns, softmax and projections are, in the
2-norm, no more sensitive than to pass that on once: 16 * 2^-8 of the gradient's 2-norm.
"""

import pytest

pytestmark = pytest.mark.gpu

B, T, H, HKV, D, V = 2, 97, 4, 2, 64, 1003
W = H * D
IGN = -100
BOUND = 16 * 2.0 ** -8


def _inputs(dev, seed):
    import torch

    g = torch.Generator(device="cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    p = {"x": r(B * T, W), "wq": r(W, W) / W ** 0.5, "wk": r(HKV * D, W) / W ** 0.5, "wv": r(HKV * D, W) / W ** 0.5,
         "wo": r(W, W) / W ** 0.5, "head": r(V, W) / W ** 0.5, "g1": 1 + 0.1 * r(W), "b1": 0.1 * r(W), "g2": 1 + 0.1 * r(W),
         "b2": 0.1 * r(W)}
    p = {k: t.to(dev) if k[0] in "gb" else t.to(torch.bfloat16).to(dev) for k, t in p.items()}
    target = torch.randint(0, V, (B, T), generator=g)
    target[1, 60:] = IGN  # the second sequence ends here
    return p, target.to(dev)


def _step(p, target, freq):
    """The step on the framework's operators; its matrix products are kernels.contract's."""
    import torch

    from pdum_dsl_b200 import kernels as K

    # a b^T; rows of the operands are multiples of 16 bytes
    pad = lambda t: torch.nn.functional.pad(t, (0, -t.shape[1] % 8))
    mm = lambda a, b: K.contract(pad(a)[None], pad(b)[None])[0]
    heads = lambda t, n: t.view(B, T, n, D).transpose(1, 2)         # (B, n, T, D) views of the projections
    flat = lambda t: t.transpose(1, 2).reshape(B * T, -1)
    a, m1, r1 = K.layernorm(p["x"], p["g1"], p["b1"], return_stats=True)
    q, k, v = heads(mm(a, p["wq"]), H), heads(mm(a, p["wk"]), HKV), heads(mm(a, p["wv"]), HKV)
    qr, kr = K.rotary(q, k, inv_freq=freq, start=1000)
    o, lse = K.flash_attention(qr, kr, v, causal=True, return_lse=True)
    of = flat(o)
    res = p["x"] + mm(of, p["wo"])
    c, m2, r2 = K.layernorm(res, p["g2"], p["b2"], return_stats=True)
    t = target.view(-1)
    loss, hl = K.linear_cross_entropy(c, p["head"], t, return_lse=True)
    count = (t != IGN).sum().float()
    mean = loss.sum() / count
    # back
    d = {}
    dc, d["head"] = K.linear_cross_entropy_backward(c, p["head"], t, (1 / count), hl)
    dres, d["g2"], d["b2"] = K.layernorm_backward(dc, res, m2, r2, p["g2"])
    tr = lambda t: t.t().contiguous()
    d["wo"] = mm(tr(dres), tr(of))
    do = heads(mm(dres, tr(p["wo"])), H)
    dqr, dkr, dv = K.flash_attention_backward(qr, kr, v, o, do, lse, causal=True)
    dq, dk = K.rotary(dqr, dkr, inv_freq=freq, start=1000, inverse=True)
    dq, dk, dv = flat(dq), flat(dk), flat(dv)
    for n, t in (("wq", dq), ("wk", dk), ("wv", dv)):
        d[n] = mm(tr(t), tr(a))
    da = mm(dq, tr(p["wq"])) + mm(dk, tr(p["wk"])) + mm(dv, tr(p["wv"]))
    dx, d["g1"], d["b1"] = K.layernorm_backward(da, p["x"], m1, r1, p["g1"])
    d["x"] = dx + dres
    return mean, d


def _step64(p, target, freq):
    import numpy as np
    import torch

    q = {k: t.double().requires_grad_() for k, t in p.items()}

    def norm(x, g, b):
        z = x - x.mean(1, keepdim=True)
        return z / (z.square().mean(1, keepdim=True) + 1e-5).sqrt() * g + b

    ang = torch.from_numpy((1000 + np.arange(T))[:, None] * freq).to(p["x"].device)

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

    heads = lambda t, n: t.view(B, T, n, D).transpose(1, 2)
    a = norm(q["x"], q["g1"], q["b1"])
    qq, kk, vv = heads(a @ q["wq"].T, H), heads(a @ q["wk"].T, HKV), heads(a @ q["wv"].T, HKV)
    kk, vv = (t.repeat_interleave(H // HKV, 1) for t in (turn(kk), vv))
    s = turn(qq) @ kk.transpose(-1, -2) / D ** 0.5
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
    o = (torch.softmax(s, -1) @ vv).transpose(1, 2).reshape(B * T, W)
    c = norm(q["x"] + o @ q["wo"].T, q["g2"], q["b2"])
    loss = torch.nn.functional.cross_entropy(c @ q["head"].T, target.view(-1), ignore_index=IGN)
    loss.backward()
    return loss.detach(), {k: t.grad for k, t in q.items()}


def test_gradients_of_a_step(cuda):
    from pdum_dsl_b200 import kernels as K

    freq, _ = K.rotary_frequencies(D)
    p, target = _inputs(cuda, 0)
    loss, d = _step(p, target, freq)
    K.check_device_errors()
    ref, dr = _step64(p, target, freq)
    assert abs(loss.double() - ref) <= BOUND * ref.abs()
    assert d.keys() == dr.keys()
    for name, g in dr.items():
        err = ((d[name].double() - g).norm() / g.norm()).item()
        assert err <= BOUND, (name, err)


def test_a_captured_step_is_the_same(cuda):
    """Captured once and replayed on other data: the same bits as the calls one by one."""
    import torch

    from pdum_dsl_b200 import kernels as K

    freq, _ = K.rotary_frequencies(D)
    p, target = _inputs(cuda, 1)
    _step(p, target, freq)  # the first call of every kernel is not captured
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, d = _step(p, target, freq)
    for seed in (2, 3):
        p2, t2 = _inputs(cuda, seed)
        for k in p:
            p[k].copy_(p2[k])
        target.copy_(t2)
        graph.replay()
        want, dw = _step(p2, t2, freq)
        assert torch.equal(loss, want)
        for k in d:
            # the attention's dq adds its parts in an order that varies, and x / wq / g1 / b1 lie behind it
            if k in ("x", "wq", "wk", "g1", "b1"):
                assert ((d[k].double() - dw[k].double()).norm() <= BOUND * dw[k].double().norm()), k
            else:
                assert torch.equal(d[k], dw[k]), k


def test_single_tokens_agree_with_the_whole_sequence(cuda):
    """One token at a time, as in generation: each operator gives for a position what it gives within the sequence."""
    import torch

    from pdum_dsl_b200 import kernels as K

    freq, m = K.rotary_frequencies(D, scaling="by_parts", factor=4.0, context=64)
    p, target = _inputs(cuda, 4)
    a = K.layernorm(p["x"], p["g1"], p["b1"])
    q = a.view(B, T, H, D).transpose(1, 2)
    turned = K.rotary(q, inv_freq=freq, amplitude=m, start=7)
    loss, lse = K.linear_cross_entropy(a, p["head"], target.view(-1), return_lse=True)
    for t in (0, 1, 50, T - 1):
        rows = torch.tensor([t, T + t], device=cuda)
        one = K.layernorm(p["x"][rows], p["g1"], p["b1"])
        assert torch.equal(one, a[rows])
        at = torch.tensor([[7 + t], [7 + t]], device=cuda)
        assert torch.equal(K.rotary(q[:, :, t:t + 1], inv_freq=freq, amplitude=m, positions=at), turned[:, :, t:t + 1])
        l1, e1 = K.linear_cross_entropy(one, p["head"], target.view(-1)[rows], return_lse=True)
        # other tiles, the same 32-bit sums in another order
        assert ((e1 - lse[rows]).abs() <= 2.0 ** -20 * (1 + lse[rows].abs())).all()
        assert ((l1 - loss[rows]).abs() <= 2.0 ** -19 * (1 + lse[rows].abs())).all()


def test_on_a_stream_of_its_own_next_to_another(cuda):
    """Two steps at once on two streams, each on data made there: what each gives alone."""
    import torch

    from pdum_dsl_b200 import kernels as K

    freq, _ = K.rotary_frequencies(D)
    alone = []
    for seed in (5, 6):
        p, target = _inputs(cuda, seed)
        alone.append(_step(p, target, freq))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for seed, s in zip((5, 6), streams):
        with torch.cuda.stream(s):
            p, target = _inputs(cuda, seed)
            got.append(_step(p, target, freq))
    torch.cuda.synchronize()
    K.check_device_errors()
    for (loss, d), (want, dw) in zip(got, alone):
        assert torch.equal(loss, want)
        for k in d:  # as above: the attention's dq varies in its last bits
            if k in ("x", "wq", "wk", "g1", "b1"):
                assert ((d[k].double() - dw[k].double()).norm() <= BOUND * dw[k].double().norm()), k
            else:
                assert torch.equal(d[k], dw[k]), k
