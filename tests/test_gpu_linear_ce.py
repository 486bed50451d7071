"""The linear head's cross entropy and its gradients against the formulas in 64 bits.

Tolerances, u = 2^-24.  A logit, a dot product of `width` bf16 products summed in f32, is off by at most
e = (width + 16) u sum|x w|.  exp takes an approximation of 2^-22 and a rounded argument of 2 u |logit|; a row's sum
of `vocab` positive terms takes at most 8 + vocab / 4096 + 140 steps, so lse is off by
e + 2^-21 + (150 + vocab / 4096) u + 4 u |lse|.  G is rounded to the operands' type (half a step: bf16 2^-8 of itself,
f32 u) after a probability with the same relative error; the products that follow sum in f32 and round once more.
"""

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGN = -100


def _inputs(dev, N, V, W, seed, ignored=0.2, spread=1.5, dtype="bfloat16"):
    import torch

    g = torch.Generator(device="cpu").manual_seed(seed)
    x = torch.randn(N, W, generator=g)
    w = torch.randn(V, W, generator=g) * spread / W ** 0.5
    t = torch.randint(0, V, (N,), generator=g)
    x[::2] += 1.5 * w[t[::2]]
    t[torch.rand(N, generator=g) < ignored] = IGN
    dl = torch.randn(N, generator=g) / max(N, 1)
    dtype = getattr(torch, dtype)
    return x.to(dtype).to(dev), w.to(dtype).to(dev), t.to(dev), dl.to(dev)


def _logits(x, w):
    """Logits and their possible error, in 64 bits."""
    xd, wd = x.double(), w.double()
    e = (x.shape[1] + 16) * U * (xd.abs() @ wd.abs().T).amax(1)
    return xd @ wd.T, e


def _check_forward(x, w, t, loss, lse):
    import torch

    z, e = _logits(x, w)
    ref = torch.logsumexp(z, 1)
    tol = e + 2.0 ** -21 + (150 + w.shape[0] / 4096) * U + 4 * U * ref.abs()
    assert ((lse.double() - ref).abs() <= tol).all(), ((lse.double() - ref).abs() / tol).max()
    valid = t != IGN
    want = torch.where(valid, ref - z.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    err = (loss.double() - want).abs()
    assert (err <= (tol + e + 2 * U * ref.abs()) * valid).all(), (err / tol).max()


def _check_backward(x, w, t, dl, lse, dx, dw):
    import torch

    N, W = x.shape
    V = w.shape[0]
    half = torch.finfo(x.dtype).eps / 2
    assert all(t is None or t.dtype == x.dtype for t in (dx, dw))
    z, e = _logits(x, w)
    valid = t != IGN
    up = (dl.double() * valid)[:, None]
    p = torch.exp(z - lse.double()[:, None])
    rel = e[:, None] + 2.0 ** -21 + 6 * U * z.abs().amax(1, keepdim=True)
    perr = p * rel * (1 + rel)
    G = p.clone()
    G.scatter_add_(1, t.clamp(min=0)[:, None], torch.full((N, 1), -1.0, dtype=torch.float64, device=x.device))
    G *= up
    gerr = up.abs() * (perr + 3 * U) * 1.01 + half * G.abs()
    wd, xd = w.double(), x.double()
    if dx is not None:
        ref = G @ wd
        tol = (gerr + (V + 16) * U * G.abs()) @ wd.abs() * 1.01 + half * ref.abs() + 1e-38
        assert ((dx.double() - ref).abs() <= tol).all(), ((dx.double() - ref).abs() / tol).max()
        assert (dx[~valid] == 0).all()
    if dw is not None:
        ref = G.T @ xd
        tol = (gerr + (N + 16) * U * G.abs()).T @ xd.abs() * 1.01 + half * ref.abs() + 1e-38
        assert ((dw.double() - ref).abs() <= tol).all(), ((dw.double() - ref).abs() / tol).max()


SHAPES = [(1, 1, 8), (1, 500, 64), (3, 257, 72), (130, 1000, 128), (257, 256, 64), (256, 255, 256), (300, 777, 1000),
          (512, 4099, 256), (1021, 2000, 520), (5, 33000, 16), (2048, 300, 64), (4100, 511, 40), (64, 20000, 2048)]


@pytest.mark.parametrize("N,V,W", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_loss_and_gradients(cuda, N, V, W, dtype):
    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, N, V, W, N + V + W, ignored=0.2 if N > 1 else 0.0, dtype=dtype)
    loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    kernels.check_device_errors()
    _check_forward(x, w, t, loss, lse)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    kernels.check_device_errors()
    _check_backward(x, w, t, dl, lse, dx, dw)


@pytest.mark.parametrize("N,dtype", [(8192, "bfloat16"), (4096, "float32")])
def test_several_pieces(cuda, N, dtype):
    """A vocabulary that one piece of the gradient's workspace does not hold."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, N, 70001, 16, 1, dtype=dtype)
    loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    _check_forward(x, w, t, loss, lse)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    kernels.check_device_errors()
    _check_backward(x, w, t, dl, lse, dx, dw)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_one_gradient_alone_and_lse_recomputed(cuda, dtype):
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 200, 900, 128, 2, dtype=dtype)
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    a, none = kernels.linear_cross_entropy_backward(x, w, t, dl, need_dweight=False)
    assert none is None and torch.equal(a, dx)
    none, b = kernels.linear_cross_entropy_backward(x, w, t, dl, need_dx=False)
    assert none is None and torch.equal(b, dw)
    assert kernels.linear_cross_entropy_backward(x, w, t, dl, lse, need_dx=False, need_dweight=False) == (None, None)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_mean_leading_dims_and_strides(cuda, dtype):
    """One dloss for all tokens; (batch, row) tokens; rows of wider matrices, aligned or not; any ignore index."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, _ = _inputs(cuda, 66, 400, 136, 3, dtype=dtype)
    lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)[1]
    mean = torch.full((), 1 / 50, device=cuda)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, mean, lse)
    _check_backward(x, w, t, mean.expand(66), lse, dx, dw)
    l3, e3 = kernels.linear_cross_entropy(x.view(6, 11, 136), w, t.view(6, 11), return_lse=True)
    assert l3.shape == (6, 11) and torch.equal(e3.view(-1), lse)
    d3, w3 = kernels.linear_cross_entropy_backward(x.view(6, 11, 136), w, t.view(6, 11), mean, e3)
    assert torch.equal(d3.view(66, 136), dx) and torch.equal(w3, dw)
    for lo, hi in ((0, 128), (8, 136), (1, 129), (4, 132)):
        xs, ws = x[:, lo:hi], w[:, lo:hi]
        ls, es = kernels.linear_cross_entropy(xs, ws, t, return_lse=True)
        _check_forward(xs, ws, t, ls, es)
        gx, gw = kernels.linear_cross_entropy_backward(xs, ws, t, mean, es)
        _check_backward(xs, ws, t, mean.expand(66), es, gx, gw)
    t0 = t.clone()
    t0[t == IGN] = 7  # an entry of the vocabulary as the index that is ignored
    keep = t0 != 7
    l0 = kernels.linear_cross_entropy(x, w, t0, ignore_index=7)
    assert (l0[~keep] == 0).all() and torch.equal(l0[keep], kernels.linear_cross_entropy(x, w, t)[keep])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_nothing_to_do(cuda, dtype):
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 40, 300, 64, 4, dtype=dtype)
    t[:] = IGN
    loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    assert (loss == 0).all()
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    assert (dx == 0).all() and (dw == 0).all()
    x[3] = float("inf")  # in an ignored row: no gradient still
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    assert (dx == 0).all() and (dw == 0).all()
    none = x[:0]
    loss, lse = kernels.linear_cross_entropy(none, w, t[:0], return_lse=True)
    dx, dw = kernels.linear_cross_entropy_backward(none, w, t[:0], dl[:0], lse)
    assert loss.shape == (0,) and dx.shape == (0, 64) and dw.shape == w.shape and (dw == 0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_targets_outside_the_vocabulary_give_nan(cuda, dtype):
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 40, 300, 64, 5, ignored=0.0, dtype=dtype)
    good = kernels.linear_cross_entropy(x, w, t)
    for bad in (300, -1, 2 ** 40, -(2 ** 62)):
        t2 = t.clone()
        t2[11] = bad
        loss, lse = kernels.linear_cross_entropy(x, w, t2, return_lse=True)
        assert loss[11].isnan() and torch.equal(loss[:11], good[:11]) and torch.equal(loss[12:], good[12:])
        dx, _ = kernels.linear_cross_entropy_backward(x, w, t2, dl, lse, need_dweight=False)
        assert dx[11].isnan().all() and dx[:11].isfinite().all() and dx[12:].isfinite().all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_large_logits(cuda, dtype):
    """Logits of hundreds, one entry holding all of a row's probability; nothing overflows."""
    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 129, 600, 64, 6, spread=150.0, dtype=dtype)
    loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    _check_forward(x, w, t, loss, lse)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    _check_backward(x, w, t, dl, lse, dx, dw)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_same_bits_every_time_on_two_streams_and_in_a_graph(cuda, dtype):
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 700, 5000, 256, 7, dtype=dtype)

    def both():
        loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
        return (loss, lse, *kernels.linear_cross_entropy_backward(x, w, t, dl, lse))

    first = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(both())
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    x2, _, t2, dl2 = _inputs(cuda, 700, 5000, 256, 8, dtype=dtype)
    x.copy_(x2), t.copy_(t2), dl.copy_(dl2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, both()))


def test_gradient_against_differences(cuda):
    """<dx, a> + <dw, b> against a central difference of sum(dloss * loss) along (a, b), evaluated in 64 bits."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 50, 90, 32, 9)
    a, b, _, _ = _inputs(cuda, 50, 90, 32, 10)
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    valid = t != IGN

    def at(h):
        z = (x.double() + h * a.double()) @ (w.double() + h * b.double()).T
        loss = torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0]
        return (dl.double() * loss * valid).sum()

    h = 1e-4
    slope = (at(h) - at(-h)) / (2 * h)
    got = (dx.double() * a.double()).sum() + (dw.double() * b.double()).sum()
    # each gradient element is off by at most 2^-8 of itself and 2^-8 of the |G| |operand| sums behind it
    p = torch.softmax(x.double() @ w.double().T, 1)
    p.scatter_add_(1, t.clamp(min=0)[:, None], torch.ones(50, 1, dtype=torch.float64, device=cuda))
    G = p * (dl.double().abs() * valid)[:, None]
    size = ((G @ w.double().abs()) * a.double().abs()).sum() + ((G.T @ x.double().abs()) * b.double().abs()).sum()
    assert abs(got - slope) <= (2.0 ** -7 * 1.1 + 100 * h * h) * size


@pytest.mark.parametrize("n", [1, 3, 7373])
def test_a_mean_does_not_scale_the_gradient(cuda, n):
    """Under a mean, all targets' entries of G are almost the same number; its rounding must not scale the gradient.
    The regression of dx on its exact value is 1 up to 4 sigma of dx's own rounding, 2^-8 / sqrt(elements) at most,
    and 1 / vocab from a target's 1 - p, with p near 1 / vocab in every row, rounded to 1."""
    import torch

    from pdum_dsl_b200 import kernels

    g = torch.Generator(device="cpu").manual_seed(11)
    x = (torch.randn(512, 64, generator=g) * 1e-3).to(torch.bfloat16).to(cuda)
    w = torch.randn(20000, 64, generator=g).to(torch.bfloat16).to(cuda)
    t = torch.randint(0, 20000, (512,), generator=g).to(cuda)
    dl = torch.full((512,), 1.0 / n, device=cuda)
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    dx, _ = kernels.linear_cross_entropy_backward(x, w, t, dl, lse, need_dweight=False)
    p = torch.exp(x.double() @ w.double().T - lse.double()[:, None])
    ref = (p @ w.double() - w[t].double()) / n
    slope = (dx.double() * ref).sum() / (ref * ref).sum()
    assert abs(slope - 1) <= 4 * 2.0 ** -8 / (512 * 64) ** 0.5 + 1 / 20000


@pytest.mark.parametrize("N,V,W,count", [(300, 700, 72, 1), (300, 700, 72, 33), (300, 700, 72, 64), (300, 700, 72, 299),
                                         (513, 20000, 256, 255), (2000, 300, 64, 129), (700, 40000, 40, 350), (40, 700, 64, 7)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_ignored_tokens_hold_anything(cuda, N, V, W, count, dtype):
    """Infinities and NaN in the rows, lse and dloss of ignored tokens (a padded batch) reach no gradient, for counts that
    end inside and on the products' blocks; the gradients are those of the remaining tokens alone."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, N, V, W, N + count, ignored=0.0, dtype=dtype)
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    keep = torch.zeros(N, dtype=torch.bool, device=cuda)
    keep[torch.randperm(N, generator=torch.Generator().manual_seed(count))[:count].to(cuda)] = True
    t = torch.where(keep, t, IGN)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    _check_backward(x, w, t, dl, lse, dx, dw)
    x2, lse2, dl2 = x.clone(), lse.clone(), dl.clone()
    for value in (float("nan"), float("inf"), -float("inf")):
        x2[~keep], lse2[~keep], dl2[~keep] = value, value, value
        dx2, dw2 = kernels.linear_cross_entropy_backward(x2, w, t, dl2, lse2)
        assert torch.equal(dx2, dx) and torch.equal(dw2, dw)
    loss = kernels.linear_cross_entropy(x2, w, t)
    assert (loss[~keep] == 0).all() and loss.isfinite().all()
    kernels.check_device_errors()


def test_ignored_tokens_over_several_pieces(cuda):
    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 8200, 70001, 24, 12, ignored=0.4)
    _, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
    kernels.check_device_errors()
    _check_backward(x, w, t, dl, lse, dx, dw)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_that_lie_beyond_32_bits(cuda, dtype):
    """Rows of x 2^31 and of the weight 2^24 elements apart: offsets pass 2^32 elements."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 3, 300, 72, 13, ignored=0.0, dtype=dtype)
    far = torch.empty(299 * 2 ** 24 + 2 ** 20, dtype=x.dtype, device=cuda)
    xs, ws = far[1024:].as_strided((3, 72), (2 ** 31, 1)), far.as_strided((300, 72), (2 ** 24, 1))
    xs.copy_(x), ws.copy_(w)
    for t in (t, torch.tensor([IGN, 299, 0], device=cuda)):
        loss, lse = kernels.linear_cross_entropy(xs, ws, t, return_lse=True)
        _check_forward(x, w, t, loss, lse)
        dx, dw = kernels.linear_cross_entropy_backward(xs, ws, t, dl, lse)
        kernels.check_device_errors()
        _check_backward(x, w, t, dl, lse, dx, dw)


@pytest.mark.parametrize("lowest", [True, False])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_masked_entries(cuda, dtype, lowest):
    """Entries whose logits are the type's lowest value, or minus infinity (forward alone: its gradient multiplies them),
    whole tiles of them: the loss and the gradients are those of the other entries alone."""
    import torch

    from pdum_dsl_b200 import kernels

    x, w, t, dl = _inputs(cuda, 150, 1000, 72, 14, dtype=dtype)
    live = torch.zeros(1000, dtype=torch.bool, device=cuda)
    live[300:420] = live[999] = True
    x[:, 0] = 1.0
    w[:, 0] = torch.where(live, 0.0, torch.finfo(w.dtype).min if lowest else -float("inf"))
    few = torch.where(t == IGN, IGN, t % 121)  # among the entries that count, and in the whole vocabulary
    t = torch.where(few == IGN, IGN, torch.where(few == 120, 999, few + 300))
    loss, lse = kernels.linear_cross_entropy(x, w, t, return_lse=True)
    _check_forward(x, w[live], few, loss, lse)
    if lowest:
        dx, dw = kernels.linear_cross_entropy_backward(x, w, t, dl, lse)
        _check_backward(x, w[live], few, dl, lse, dx, dw[live])
        assert (dw[~live] == 0).all()
    kernels.check_device_errors()
