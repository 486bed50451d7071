"""Rotary positions against the formula in 64 bits.

Tolerance.  The angle is exact up to position * 2^-54 of a turn (the frequency's 53 bits) and f32's
2^-25 of half a turn; cos and sin add 2 ulp and the amplitude one rounding, the turn two products and
a sum: at most 10 u (|a| + |b|) amplitude with u = 2^-24, and half a step of the output's type.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _reference(x, inv_freq, pos, interleaved, amplitude, inverse):
    """x (B, H, T, D) f64, pos (B, T) integers -> turned x, and |a| + |b| per feature."""
    import torch

    r = 2 * len(inv_freq)
    # angles in whole turns removed with integers, so far positions keep their digits
    turns = np.asarray(inv_freq, dtype=np.longdouble) / (2 * np.longdouble(math.pi) + np.longdouble(2.4492935982947064e-16))
    ang = np.asarray(pos.cpu().numpy(), dtype=np.longdouble)[..., None] * turns
    ang = np.asarray((ang - np.rint(ang)) * (2 * np.longdouble(math.pi)), dtype=np.float64)
    if inverse:
        ang = -ang
    c = torch.from_numpy(np.cos(ang)).to(x.device)[:, None] * amplitude
    s = torch.from_numpy(np.sin(ang)).to(x.device)[:, None] * amplitude
    y, size = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * amplitude
    return y, size


def _check(got, x, inv_freq, pos, interleaved=False, amplitude=1.0, inverse=False, far=0.0):
    import torch

    ref, size = _reference(x.double(), inv_freq, pos, interleaved, amplitude, inverse)
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + (1.01 * 10 * U + far) * size
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - ref).abs() <= tol).all()
    r = 2 * len(inv_freq)
    assert torch.equal(got[..., r:], x[..., r:])


def _draw(dev, shape, t, seed):
    import torch

    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(shape, generator=g).to(getattr(torch, t)).to(dev)


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,r", [(128, 128), (64, 64), (80, 48), (2, 2), (6, 2), (96, 20), (256, 256), (130, 130), (7, 6),
                                 (64, 0), (320, 256)])
def test_shapes(cuda, D, r, interleaved, t):
    import torch

    from pdum_dsl_b200 import kernels

    f, _ = kernels.rotary_frequencies(r)
    for B, H, HK, T in ((1, 1, 1, 1), (2, 6, 2, 33), (3, 1, 5, 7)):
        q, k = _draw(cuda, (B, H, T, D), t, D + T), _draw(cuda, (B, HK, T, D), t, D + T + 1)
        pos = torch.randint(-5, 70000, (B, T), generator=torch.Generator().manual_seed(T)).to(cuda)
        for inverse in (False, True):
            gq, gk = kernels.rotary(q, k, inv_freq=f, positions=pos, interleaved=interleaved, inverse=inverse)
            _check(gq, q, f, pos, interleaved, 1.0, inverse)
            _check(gk, k, f, pos, interleaved, 1.0, inverse)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_and_scalings(cuda, interleaved):
    """Positions up to 2^40: what the frequency's 53 bits leave, |position| 2^-54 turns, is allowed for."""
    import torch

    from pdum_dsl_b200 import kernels

    x = _draw(cuda, (1, 2, 6, 64), "float32", 0)
    pos = torch.tensor([[0, 1, 1_000_003, 2 ** 31 + 5, 2 ** 40 + 12345, -(2 ** 33) - 7]], device=cuda)
    far = 2 * math.pi * 2.0 ** 41 * 2.0 ** -53
    for kw in ({}, {"scaling": "linear", "factor": 8.0}, {"scaling": "ntk", "factor": 4.0},
               {"scaling": "by_parts", "factor": 16.0, "context": 4096}):
        f, m = kernels.rotary_frequencies(64, **kw)
        got = kernels.rotary(x, inv_freq=f, positions=pos, interleaved=interleaved, amplitude=m)
        _check(got, x, f, pos, interleaved, m, far=far)


def test_frequencies(cuda):
    from pdum_dsl_b200 import kernels

    f, m = kernels.rotary_frequencies(8, base=100.0)
    assert m == 1.0 and np.allclose(f, [1, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    g, _ = kernels.rotary_frequencies(8, base=100.0, scaling="ntk", factor=4.0)
    assert g[0] == 1.0 and np.isclose(g[-1], f[-1] / 4, rtol=1e-14)
    h, m = kernels.rotary_frequencies(128, scaling="by_parts", factor=8.0, context=4096)
    f, _ = kernels.rotary_frequencies(128)
    assert h[0] == f[0] and np.isclose(h[-1], f[-1] / 8, rtol=1e-15) and np.isclose(m, 0.1 * math.log(8) + 1)
    assert (h <= f).all() and (h >= f / 8 * (1 - 1e-15)).all()


def test_layouts_positions_and_in_place(cuda):
    """Transposed views, odd offsets, broadcast and implied positions, 2-D and 3-D inputs, in place, one tensor."""
    import torch

    from pdum_dsl_b200 import kernels

    f, _ = kernels.rotary_frequencies(32)
    wide = _draw(cuda, (2, 9, 3, 133), "bfloat16", 1)
    for lo in (0, 1, 4):  # 16-, 2- and 8-byte addresses
        x = wide[..., lo:lo + 64].transpose(1, 2)
        for inter in (False, True):
            got = kernels.rotary(x, inv_freq=f, start=11, interleaved=inter)
            pos = (torch.arange(9, device=cuda) + 11).expand(2, 9)
            _check(got, x, f, pos, inter)
            keep = wide.clone()
            y = keep[..., lo:lo + 64].transpose(1, 2)
            assert kernels.rotary(y, inv_freq=f, start=11, interleaved=inter, out=y) is y
            assert torch.equal(y, got)
            untouched = torch.ones(133, dtype=torch.bool, device=cuda)
            untouched[lo:lo + 32] = False
            assert torch.equal(keep[..., untouched], wide[..., untouched])
    x = _draw(cuda, (9, 64), "float32", 2)
    p32 = torch.arange(9, device=cuda, dtype=torch.int32) * 3
    one = kernels.rotary(x, inv_freq=f, positions=p32)
    _check(one[None, None], x[None, None], f, p32[None])
    three = kernels.rotary(x[None].expand(4, 9, 64), inv_freq=f, positions=p32.long())
    assert torch.equal(three, one.expand(4, 9, 64))
    q = _draw(cuda, (3, 2, 5, 64), "float32", 3)
    at = torch.tensor([[5], [6], [100000]], device=cuda)
    _check(kernels.rotary(q, inv_freq=f, positions=at), q, f, at.expand(3, 5))


def test_empty(cuda):
    import torch

    from pdum_dsl_b200 import kernels

    f, _ = kernels.rotary_frequencies(32)
    for shape in ((0, 2, 3, 32), (2, 0, 3, 32), (2, 2, 0, 32)):
        x = torch.empty(shape, device=cuda)
        assert kernels.rotary(x, inv_freq=f).shape == shape
    x, none = torch.randn(2, 2, 3, 32, device=cuda), torch.empty(2, 0, 3, 32, device=cuda)
    a, b = kernels.rotary(x, none, inv_freq=f)
    assert b.shape == none.shape and torch.equal(a, kernels.rotary(x, inv_freq=f))
    a, b = kernels.rotary(none, x, inv_freq=f)
    assert torch.equal(b, kernels.rotary(x, inv_freq=f))


def test_inverse_is_the_gradient(cuda):
    """<rotary(x), g> = <x, inverse(g)> for every x and g, since the turn is linear; and differences along a direction
    are exact for a linear map."""
    import torch

    from pdum_dsl_b200 import kernels

    f, m = kernels.rotary_frequencies(48, scaling="by_parts", factor=4.0, context=64)
    x, g = _draw(cuda, (2, 3, 65, 80), "float32", 4), _draw(cuda, (2, 3, 65, 80), "float32", 5)
    kw = dict(inv_freq=f, start=1000, amplitude=m)
    left = (kernels.rotary(x, **kw).double() * g.double()).sum()
    right = (x.double() * kernels.rotary(g, inverse=True, **kw).double()).sum()
    size = (x.double().abs() * (g.double().abs() + g.double().abs().roll(24, -1) + g.double().abs().roll(-24, -1))).sum()
    assert abs(left - right) <= 20 * U * m * size


def test_in_a_graph(cuda):
    import torch

    from pdum_dsl_b200 import kernels

    f, _ = kernels.rotary_frequencies(64)
    q, pos = _draw(cuda, (2, 4, 1, 64), "bfloat16", 6), torch.tensor([[3], [9]], device=cuda)
    kernels.rotary(q, inv_freq=f, positions=pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.rotary(q, inv_freq=f, positions=pos)
    for step in range(3):
        pos += 1
        graph.replay()
        assert torch.equal(out, kernels.rotary(q, inv_freq=f, positions=pos))


@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_that_lie_beyond_32_bits(cuda, interleaved):
    """Strides of 2^31 and 2^30 elements between batches, heads and rows, read and written in place."""
    import torch

    from pdum_dsl_b200 import kernels

    f, _ = kernels.rotary_frequencies(64)
    x = _draw(cuda, (2, 2, 3, 64), "bfloat16", 9)
    pos = torch.arange(3, device=cuda).expand(2, 3)
    far = torch.empty(2 ** 32 + 2 ** 31 + 4096, dtype=torch.bfloat16, device=cuda)
    for strides in ((2 ** 32, 2 ** 31, 64, 1), (64 * 3, 2 ** 32, 64, 1), (128, 64, 2 ** 31, 1)):
        xs = far.as_strided((2, 2, 3, 64), strides)
        xs.copy_(x)
        got = kernels.rotary(xs, inv_freq=f, interleaved=interleaved)
        _check(got, x, f, pos, interleaved)
        kernels.rotary(xs, inv_freq=f, interleaved=interleaved, out=xs)
        assert torch.equal(xs, got)


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_with_a_second_unit_stride(cuda, interleaved, t):
    """Windows that slide by one element along heads, rows or both, alone and as either of two tensors; the results
    are laid out with their features together whatever the input's strides."""
    import torch

    from pdum_dsl_b200 import kernels

    f, m = kernels.rotary_frequencies(8, scaling="by_parts", factor=4.0, context=64)
    flat = _draw(cuda, (400,), t, 11)
    pos = torch.tensor([[3, 70, 4000], [9, 11, 100]], device=cuda)
    plain = _draw(cuda, (2, 4, 3, 8), t, 12)
    for strides in ((100, 1, 20, 1), (100, 20, 1, 1), (50, 1, 1, 1), (1, 1, 1, 1)):
        x = flat.as_strided((2, 4, 3, 8), strides)
        kw = dict(inv_freq=f, positions=pos, interleaved=interleaved, amplitude=m)
        got = kernels.rotary(x, **kw)
        _check(got, x.contiguous(), f, pos, interleaved, m)
        a, b = kernels.rotary(x, plain, **kw)
        c, d = kernels.rotary(plain, x, **kw)
        assert torch.equal(a, got) and torch.equal(d, got) and torch.equal(b, c)
        _check(b, plain, f, pos, interleaved, m)
    three = flat.as_strided((4, 3, 8), (1, 20, 1))
    _check(kernels.rotary(three, inv_freq=f, interleaved=interleaved)[None], three.contiguous()[None], f,
           torch.arange(3, device=cuda)[None], interleaved)
