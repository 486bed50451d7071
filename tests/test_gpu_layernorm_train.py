"""Layer norm with statistics and its gradients, f32 and bf16, against the formulas in 64 bits.

Tolerances.  u = 2^-24 is f32's half step; an output rounded to type t is off by at most
eps(t) / 2 relative to itself.  A sum in n sequential or tree steps is off by at most
n u sum|terms| (first order).  A row's sums take at most 32 steps in a thread, 5 in its
warp and 32 over the warps, or cols / 512 + 21 where the row is looped over, so
n = 70 + cols / 512; a dozen further roundings give K = 82 + cols / 512 steps on the
magnitudes that enter an output.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _types():
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}


def _half(t):
    import torch

    return torch.finfo(t).eps / 2


def _within(got, ref, out_type, slack, what):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    tol = _half(out_type) * ref.abs() + slack * (1 + _half(out_type))
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {((got - ref).abs() / tol.clamp(min=1e-300)).max():.2f} x tolerance"


def _inputs(dev, R, C, t, pt, seed):
    import torch

    g = torch.Generator(device="cpu").manual_seed(seed)
    x = (torch.randn(R, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + 0.3).to(t).to(dev)
    dy = torch.randn(R, C, generator=g).to(t).to(dev)
    gam = (1 + 0.1 * torch.randn(C, generator=g)).to(pt).to(dev)
    bet = (0.1 * torch.randn(C, generator=g)).to(pt).to(dev)
    return x, dy, gam, bet


def _check_forward(x, gam, bet, eps, y, mean, rstd):
    import torch

    C = x.shape[-1]
    K = (82 + C / 512) * U
    xd = x.double()
    mu = xd.mean(-1, keepdim=True)
    var = (xd - mu).square().mean(-1, keepdim=True)
    r = (var + eps).rsqrt()
    big = xd.abs().mean(-1, keepdim=True)
    dmu = K * big                                      # the mean's error
    # d var: 2 |x - mu| dmu averages to at most 2 sqrt(var) dmu (and dmu^2); its own K roundings
    dvar = K * (var + eps) + 2 * var.sqrt() * dmu + dmu * dmu
    drel = dvar / (2 * (var + eps)) + 4 * U            # relative error of rstd
    _within(mean, mu[..., 0], torch.float32, dmu[..., 0], "mean")
    _within(rstd, r[..., 0], torch.float32, (drel * r)[..., 0], "rstd")
    z = (xd - mu) * r
    gd = gam.double() if gam is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    bd = bet.double() if bet is not None else torch.zeros(C, dtype=torch.float64, device=x.device)
    ref = z * gd + bd
    slack = gd.abs() * (r * dmu + z.abs() * (drel + 4 * U) + 4 * U * r * xd.abs()) + 2 * U * (ref.abs() + bd.abs())
    _within(y, ref, y.dtype, slack, "y")


def _check_backward(x, dy, mean, rstd, gam, dx, dg, db):
    import torch

    R, C = x.shape[0], x.shape[-1]
    K = (82 + C / 512) * U
    xd, dyd, m, r = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    gd = gam.double() if gam is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    z = (xd - m) * r
    dz = dyd * gd
    m0, m1 = dz.mean(1, keepdim=True), (dz * z).mean(1, keepdim=True)
    zerr = 3 * U * (z.abs() + r * m.abs())              # of z, from a rounded difference
    e0 = K * dz.abs().mean(1, keepdim=True)
    e1 = K * (dz * z).abs().mean(1, keepdim=True) + (dz.abs() * zerr).mean(1, keepdim=True)
    slack = r * (e0 + z.abs() * e1 + zerr * m1.abs() + 6 * U * (dz.abs() + m0.abs() + (z * m1).abs()))
    _within(dx, r * (dz - m0 - z * m1), dx.dtype, slack, "dx")
    if dg is None:
        return
    # rows in sequence within a block, then the blocks: at most R steps in all, and 64 more
    n = (R + 64) * U
    _within(dg, (dyd * z).sum(0), dg.dtype, n * (dyd * z).abs().sum(0) + (dyd.abs() * zerr).sum(0), "dgamma")
    _within(db, dyd.sum(0), db.dtype, n * dyd.abs().sum(0), "dbeta")


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 4096), (300, 64), (1000, 128), (37, 1001), (257, 520), (301, 2048), (70, 4096),
          (9, 5000), (50, 9344), (33, 12001), (150, 20000), (7, 30001), (64, 1002), (200, 515), (20, 4099), (90, 16), (13, 8191), (700, 8192), (5, 8200), (3, 16384), (4, 32768), (2, 40003), (5000, 32),
          (3001, 57), (2000, 100)]


@pytest.mark.parametrize("R,C", SHAPES)
@pytest.mark.parametrize("t,pt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_forward_and_gradients(cuda, R, C, t, pt):
    from pdum_dsl_b200 import kernels

    T = _types()
    x, dy, gam, bet = _inputs(cuda, R, C, T[t], T[pt], R * 7 + C)
    y, mean, rstd = kernels.layernorm(x, gam, bet, eps=1e-5, return_stats=True)
    assert y.dtype == x.dtype and mean.shape == rstd.shape == (R,)
    _check_forward(x, gam, bet, 1e-5, y, mean, rstd)
    dx, dg, db = kernels.layernorm_backward(dy, x, mean, rstd, gam)
    assert dx.dtype == x.dtype and dg.dtype == db.dtype == gam.dtype
    _check_backward(x, dy, mean, rstd, gam, dx, dg, db)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_without_weights_strided_and_shaped(cuda, t):
    """No gamma / beta; rows of a wider matrix (aligned and not); leading dims; a broadcast dout."""
    import torch

    from pdum_dsl_b200 import kernels

    T = _types()[t]
    x, dy, _, bet = _inputs(cuda, 60, 1040, T, torch.float32, 5)
    for lo, hi in ((0, 1024), (3, 1000), (8, 1032)):
        xs, ds = x[:, lo:hi], dy[:, lo:hi]
        y, mean, rstd = kernels.layernorm(xs, None, None, return_stats=True)
        _check_forward(xs, None, None, 1e-5, y, mean, rstd)
        dx, dg, db = kernels.layernorm_backward(ds, xs, mean, rstd)
        _check_backward(xs, ds, mean, rstd, None, dx, dg, db)
        dx2, dg2, db2 = kernels.layernorm_backward(ds, xs, mean, rstd, weight_grads=False)
        assert dg2 is None and db2 is None and torch.equal(dx, dx2)
    for xo, do in ((3, 0), (0, 5), (3, 11)):  # rows that lie differently against 16 bytes; the last pair alike
        xs, ds = x[:, xo:xo + 999], dy[:, do:do + 999]
        y, mean, rstd = kernels.layernorm(xs, None, None, return_stats=True)
        _check_forward(xs, None, None, 1e-5, y, mean, rstd)
        dx, dg, db = kernels.layernorm_backward(ds, xs, mean, rstd)
        _check_backward(xs, ds, mean, rstd, None, dx, dg, db)
    for C in (700, 3001, 6000):  # y on other boundaries than x; longer rows, element by element
        wide, _, g2, b2 = _inputs(cuda, 11, C + 9, T, torch.float32, C)
        buf = torch.full((11, C + 9), 5.0, device=cuda, dtype=T)
        out = kernels.layernorm(wide[:, 1:C + 1], g2[:C], b2[:C], out=buf[:, 2:C + 2])
        _, mean, rstd = kernels.layernorm(wide[:, 1:C + 1], g2[:C], b2[:C], return_stats=True)
        _check_forward(wide[:, 1:C + 1], g2[:C], b2[:C], 1e-5, out, mean, rstd)
        assert (buf[:, :2] == 5).all() and (buf[:, C + 2:] == 5).all()
        xs, ds = wide[:, 1:C + 1], wide[:, 4:C + 4]
        dx, dg, db = kernels.layernorm_backward(ds, xs, mean, rstd, g2[:C])
        _check_backward(xs, ds, mean, rstd, g2[:C], dx, dg, db)
    x3, d3 = x.view(3, 20, 1040), dy[:20].expand(3, 20, 1040)
    y, mean, rstd = kernels.layernorm(x3, None, bet, return_stats=True)
    assert y.shape == x3.shape and mean.shape == (3, 20)
    dx, dg, db = kernels.layernorm_backward(d3, x3, mean, rstd)
    _check_backward(x, d3.reshape(60, 1040), mean.view(-1), rstd.view(-1), None, dx.view(60, 1040), dg, db)
    one = torch.ones(1, 1, device=cuda, dtype=T).expand(60, 1040)
    dx, dg, db = kernels.layernorm_backward(one, x, mean.view(-1), rstd.view(-1))
    _check_backward(x, one, mean.view(-1), rstd.view(-1), None, dx, dg, db)


def test_no_rows_and_untouched_neighbours(cuda):
    import torch

    from pdum_dsl_b200 import kernels

    x = torch.empty(0, 96, device=cuda, dtype=torch.bfloat16)
    y, mean, rstd = kernels.layernorm(x, return_stats=True)
    assert y.shape == (0, 96) and mean.numel() == 0
    dx, dg, db = kernels.layernorm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 96) and dg.abs().max() == 0 and db.abs().max() == 0
    buf = torch.full((5, 104), 7.0, device=cuda, dtype=torch.bfloat16)
    xin = torch.randn(5, 96, device=cuda).to(torch.bfloat16)
    kernels.layernorm(xin, out=buf[:, :96])
    assert (buf[:, 96:] == 7).all()
    assert torch.equal(buf[:, :96], kernels.layernorm(xin))


def test_values_that_are_not_finite_stay_in_their_row(cuda):
    import torch

    from pdum_dsl_b200 import kernels

    x = torch.randn(6, 512, device=cuda)
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    y, mean, rstd = kernels.layernorm(x, return_stats=True)
    assert y[2].isnan().all() and y[4].isnan().any() and mean[4] == float("inf")
    ok = [0, 1, 3, 5]
    _check_forward(x[ok], None, None, 1e-5, y[ok], mean[ok], rstd[ok])


def test_constant_rows(cuda):
    """A row of one value has no variance: z is 0 and rstd 1 / sqrt(eps)."""
    import torch

    from pdum_dsl_b200 import kernels

    x = torch.full((3, 256), 2.0, device=cuda)
    y, mean, rstd = kernels.layernorm(x, eps=1e-6, return_stats=True)
    assert (y == 0).all() and (mean == 2).all()
    assert ((rstd.double() - 1e3).abs() <= 4 * U * 1e3).all()


def test_the_same_bits_every_time_and_in_a_graph(cuda):
    import torch

    from pdum_dsl_b200 import kernels

    x, dy, gam, bet = _inputs(cuda, 4099, 1001, torch.bfloat16, torch.float32, 3)

    def both():
        y, mean, rstd = kernels.layernorm(x, gam, bet, return_stats=True)
        return (y, mean, rstd, *kernels.layernorm_backward(dy, x, mean, rstd, gam))

    first = [t.clone() for t in both()]
    for a, b in zip(first, both()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    x2, dy2, _, _ = _inputs(cuda, 4099, 1001, torch.bfloat16, torch.float32, 4)
    x.copy_(x2)
    dy.copy_(dy2)
    graph.replay()
    for a, b in zip(outs, both()):
        assert torch.equal(a, b)


def test_gradient_against_differences(cuda):
    """<dx, v> + <dgamma, p> + <dbeta, q> against a central difference of sum(dout * y) along (v, p, q), the
    forward evaluated in 64 bits."""
    import torch

    from pdum_dsl_b200 import kernels

    x, dy, gam, bet = _inputs(cuda, 33, 200, torch.float32, torch.float32, 8)
    v, _, p, q = _inputs(cuda, 33, 200, torch.float32, torch.float32, 9)
    y, mean, rstd = kernels.layernorm(x, gam, bet, return_stats=True)
    dx, dg, db = kernels.layernorm_backward(dy, x, mean, rstd, gam)

    def at(h):
        xx = x.double() + h * v.double()
        z = (xx - xx.mean(1, keepdim=True)) / (xx.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        return (dy.double() * (z * (gam.double() + h * p.double()) + bet.double() + h * q.double())).sum()

    h = 1e-4
    slope = ((at(h) - at(-h)) / (2 * h)).item()
    got = (dx.double() * v).sum() + (dg.double() * p).sum() + (db.double() * q).sum()
    # the difference is off by h^2/6 times a third derivative of order |terms|; the gradients by ~100 u
    size = ((dx.double() * v).abs().sum() + (dg.double() * p).abs().sum() + (db.double() * q).abs().sum()).item()
    assert abs(got.item() - slope) <= (200 * U + 10 * h * h) * size


@pytest.mark.parametrize("C", [96, 1001, 9000, 50000])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_in_place(cuda, C, t):
    """y over x; through the C ABI also dx over dout and over x, whichever kernels the width takes."""
    import ctypes as CT

    import torch

    from pdum_dsl_b200 import _lib, kernels

    x, dy, gam, bet = _inputs(cuda, 40, C, _types()[t], torch.float32, C)
    y, mean, rstd = kernels.layernorm(x, gam, bet, return_stats=True)
    z = x.clone()
    kernels.layernorm(z, gam, bet, out=z)
    assert torch.equal(z, kernels.layernorm(x, gam, bet))
    want = kernels.layernorm_backward(dy, x, mean, rstd, gam)
    lib = _lib.load()
    for over in ("dout", "x"):
        a, b = dy.clone(), x.clone()
        dx = a if over == "dout" else b
        dw = torch.empty(2, C, device=cuda)
        d = _lib.LayerNormBwdDesc(a.data_ptr(), b.data_ptr(), mean.data_ptr(), rstd.data_ptr(), gam.data_ptr(), dx.data_ptr(),
                                  dw[0].data_ptr(), dw[1].data_ptr(), None, 0, 40, C, C, C, C,
                                  _lib.PDB_BF16 if t == "bf16" else _lib.PDB_F32, _lib.PDB_F32)
        ws = torch.empty(lib.pdb_layernorm_bwd_workspace_size(CT.byref(d)), dtype=torch.uint8, device=cuda)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.pdb_layernorm_bwd(CT.byref(d), torch.cuda.current_stream().cuda_stream), "pdb_layernorm_bwd")
        assert torch.equal(dx, want[0]) and torch.equal(dw[0], want[1]) and torch.equal(dw[1], want[2])


@pytest.mark.parametrize("C", [512, 777])
def test_rows_that_lie_beyond_32_bits(cuda, C):
    """Five rows 2^30 + 1 elements apart: offsets pass 2^32 elements, and a row's place against 16 bytes changes."""
    import torch

    from pdum_dsl_b200 import kernels

    x, dy, gam, bet = _inputs(cuda, 5, C, torch.bfloat16, torch.float32, C)
    far = torch.empty(4 * (2 ** 30 + 1) + C, dtype=torch.bfloat16, device=cuda)
    for away in (2 ** 30 + 1, 2 ** 30):
        xs = far.as_strided((5, C), (away, 1))
        xs.copy_(x)
        y, mean, rstd = kernels.layernorm(xs, gam, bet, return_stats=True)
        _check_forward(xs, gam, bet, 1e-5, y, mean, rstd)
        dx, dg, db = kernels.layernorm_backward(dy, xs, mean, rstd, gam)
        _check_backward(xs, dy, mean, rstd, gam, dx, dg, db)
        out = kernels.layernorm(x, gam, bet, out=xs)
        assert torch.equal(out, kernels.layernorm(x, gam, bet)) and torch.equal(xs, out)


@pytest.mark.parametrize("C", [12000, 20000, 28001])
def test_long_rows_captured_first_and_called_twice_at_once(cuda, C):
    """Rows on clusters (3, 5 and 7 blocks of the gradients): captured before any other call of their width, replayed on
    new inputs, and two calls at once on two streams; all the same bits."""
    import torch

    from pdum_dsl_b200 import kernels

    x, dy, gam, bet = _inputs(cuda, 300, C, torch.bfloat16, torch.float32, C)
    sx, sdy = torch.zeros_like(x), torch.zeros_like(dy)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = kernels.layernorm(sx, gam, bet, return_stats=True)
        captured += kernels.layernorm_backward(sdy, sx, captured[1], captured[2], gam)
    sx.copy_(x), sdy.copy_(dy)
    graph.replay()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y, mean, rstd = kernels.layernorm(x, gam, bet, return_stats=True)
            results.append((y, mean, rstd) + kernels.layernorm_backward(dy, x, mean, rstd, gam))
    torch.cuda.synchronize()
    kernels.check_device_errors()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(captured, r))
    y, mean, rstd, dx, dg, db = results[0]
    _check_forward(x, gam, bet, 1e-5, y, mean, rstd)
    _check_backward(x, dy, mean, rstd, gam, dx, dg, db)


def _check_backward_given(x, dy, mean, rstd, gam, dx, dg, db):
    """As _check_backward, with the statistics taken as given: the difference from the mean is rounded once, to u of
    itself, and so is its product with rstd, so z is off by at most (1 + u)^2 - 1 <= 3 u of itself, however far the row
    lies from 0."""
    import torch

    R, C = x.shape
    K = (82 + C / 512) * U
    xd, dyd, m, r = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    gd = gam.double() if gam is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    z = (xd - m) * r
    dz = dyd * gd
    m0, m1 = dz.mean(1, keepdim=True), (dz * z).mean(1, keepdim=True)
    zerr = 3 * U * z.abs()
    e0 = K * dz.abs().mean(1, keepdim=True)
    e1 = (K + 3 * U) * (dz * z).abs().mean(1, keepdim=True)
    slack = r * (e0 + z.abs() * e1 + zerr * m1.abs() + 6 * U * (dz.abs() + m0.abs() + (z * m1).abs()))
    _within(dx, r * (dz - m0 - z * m1), dx.dtype, slack, "dx")
    n = (R + 64) * U
    _within(dg, (dyd * z).sum(0), dg.dtype, (n + 3 * U) * (dyd * z).abs().sum(0), "dgamma")
    _within(db, dyd.sum(0), db.dtype, n * dyd.abs().sum(0), "dbeta")


# (cols, elements by which x and dout lie behind a 16-byte boundary): in registers on 4 to 512 threads, ragged, element
# by element, on clusters (ragged too), and read again
OFFSET_ROWS = [(64, 0, 0), (96, 0, 0), (768, 0, 0), (4096, 0, 0), (8192, 0, 0), (57, 0, 0), (1001, 0, 0), (5003, 0, 0),
               (100, 1, 2), (1001, 1, 4), (6000, 3, 0), (12000, 0, 0), (20000, 0, 0), (28001, 0, 0), (50000, 0, 0)]


def _offset_inputs(dev, C, at, t, seed, offset, spread):
    import torch

    g = torch.Generator(device="cpu").manual_seed(seed)
    wide = torch.empty(13, C + 8, device=dev, dtype=t), torch.empty(13, C + 8, device=dev, dtype=t)
    x, dy = wide[0][:, at[0]:at[0] + C], wide[1][:, at[1]:at[1] + C]
    where = offset * (1 + torch.rand(13, 1, generator=g)) * torch.tensor([1.0, -1.0]).repeat(7)[:13, None]
    x.copy_(where + spread * torch.randn(13, C, generator=g))
    dy.copy_(torch.randn(13, C, generator=g))
    return x, dy, (1 + 0.1 * torch.randn(C, generator=g)).to(dev)


@pytest.mark.parametrize("C,at_x,at_dy", OFFSET_ROWS)
@pytest.mark.parametrize("t,offset", [("f32", 1e2), ("f32", 1e4), ("bf16", 1e2)])
def test_gradients_of_rows_far_from_zero(cuda, C, at_x, at_dy, t, offset):
    """Rows whose mean is 100 and 10 000 times their spread."""
    from pdum_dsl_b200 import kernels

    x, dy, gam = _offset_inputs(cuda, C, (at_x, at_dy), _types()[t], C, offset, 1.0)
    _, mean, rstd = kernels.layernorm(x, gam, return_stats=True)
    _check_backward_given(x, dy, mean, rstd, gam, *kernels.layernorm_backward(dy, x, mean, rstd, gam))


@pytest.mark.parametrize("C,at_x,at_dy", OFFSET_ROWS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_gradients_of_constant_rows(cuda, C, at_x, at_dy, t):
    """Rows of one value, which is their mean: z is 0, and so are the scale's gradients, exactly."""
    import torch

    from pdum_dsl_b200 import kernels

    x, dy, gam = _offset_inputs(cuda, C, (at_x, at_dy), _types()[t], C + 1, 1000.7, 0.0)
    mean, rstd = x[:, 0].float(), torch.full((13,), 1e-5 ** -0.5, device=cuda)
    dx, dg, db = kernels.layernorm_backward(dy, x, mean, rstd, gam)
    assert (dg == 0).all()
    _check_backward_given(x, dy, mean, rstd, gam, dx, dg, db)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_in_place_over_rows_of_another_stride_is_refused(cuda, t):
    import torch

    from pdum_dsl_b200 import kernels

    buf = torch.randn(4, 16, device=cuda).to(_types()[t])
    x, dense = buf[:, :8], buf.view(-1)[:32].view(4, 8)
    for stats in (False, True):
        for a, b in ((x, dense), (dense, x)):
            with pytest.raises(ValueError, match="over x"):
                kernels.layernorm(a, out=b, return_stats=stats)
    want = kernels.layernorm(x)
    assert kernels.layernorm(x, out=x).data_ptr() == buf.data_ptr() and torch.equal(x, want)
