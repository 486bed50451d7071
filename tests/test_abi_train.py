"""Layer norm for training and rotary positions through the C ABI and the Python layer, without a GPU: descriptor
layouts, and the calls that are refused before anything is launched."""

import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest

from pdum_dsl_b200 import _lib
from tests.test_abi import REPO

_STRUCTS = {"pdb_layernorm_fwd_desc": "LayerNormFwdDesc", "pdb_layernorm_bwd_desc": "LayerNormBwdDesc",
            "pdb_rotary_desc": "RotaryDesc", "pdb_linear_ce_fwd_desc": "LinearCeFwdDesc",
            "pdb_linear_ce_bwd_desc": "LinearCeBwdDesc"}


def test_descriptor_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "pdb.h"', "int main(void) {"]
    for cname, pyname in _STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for fname, _ in getattr(_lib, pyname)._fields_:
            lines.append(f'printf("{cname}.{fname} %zu\\n", offsetof({cname}, {fname}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([cc, "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                          check=True).stdout.splitlines())
    for cname, pyname in _STRUCTS.items():
        st = getattr(_lib, pyname)
        assert int(got[cname]) == C.sizeof(st), cname
        for fname, _ in st._fields_:
            assert int(got[f"{cname}.{fname}"]) == getattr(st, fname).offset, f"{cname}.{fname}"


def _norm(rows=2, cols=8, dtype=_lib.PDB_BF16, param=_lib.PDB_F32, stride=8):
    return _lib.LayerNormFwdDesc(16, None, None, 16, None, None, rows, cols, stride, stride, 1e-5, dtype, param)


def _norm_bwd(rows=2, cols=8, dtype=_lib.PDB_BF16, param=_lib.PDB_F32, stride=8):
    return _lib.LayerNormBwdDesc(16, 16, 16, 16, None, 16, 16, 16, None, 0, rows, cols, stride, stride, stride, dtype, param)


def test_layernorm_refusals():
    lib = _lib.load()
    assert lib.pdb_layernorm_fwd(None, None) == _lib.PDB_ERR_ARG
    for kw, want in (({"rows": -1}, _lib.PDB_ERR_SHAPE), ({"cols": -1}, _lib.PDB_ERR_SHAPE),
                     ({"rows": 1 << 31}, _lib.PDB_ERR_SHAPE), ({"cols": (1 << 30) + 1, "stride": 1 << 31}, _lib.PDB_ERR_SHAPE),
                     ({"stride": 7}, _lib.PDB_ERR_SHAPE), ({"stride": 0}, _lib.PDB_ERR_SHAPE),
                     ({"dtype": 2}, _lib.PDB_ERR_UNSUPPORTED), ({"param": 2}, _lib.PDB_ERR_UNSUPPORTED),
                     ({"dtype": _lib.PDB_F32, "param": _lib.PDB_BF16}, _lib.PDB_ERR_UNSUPPORTED)):
        assert lib.pdb_layernorm_fwd(C.byref(_norm(**kw)), None) == want, kw
        assert lib.pdb_layernorm_bwd(C.byref(_norm_bwd(**kw)), None) == want, kw
    d = _norm()
    d.x = None
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_ERR_ARG
    for field in ("x", "y", "gamma", "beta"):
        d = _norm(dtype=_lib.PDB_BF16, param=_lib.PDB_BF16)
        setattr(d, field, 17)
        assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_ERR_ALIGN
    for field in ("x", "dout", "dx", "gamma", "dgamma", "dbeta", "workspace"):
        d = _norm_bwd()
        d.workspace, d.workspace_bytes = 16, 1 << 20
        setattr(d, field, 17)
        assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ALIGN
    d = _norm(cols=0)
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_OK
    d.mean = 16
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_ERR_SHAPE
    d = _norm_bwd()
    d.dbeta = None
    assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ARG
    d = _norm_bwd()
    need = lib.pdb_layernorm_bwd_workspace_size(C.byref(d))
    assert need == 2 * 10 * 8 * 4  # two rows: at most ten partial rows of each gradient
    d.workspace, d.workspace_bytes = 16, need - 1
    assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ARG
    assert b"workspace too small" in lib.pdb_last_error_string()
    d.mean = None
    assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ARG


def _rot(**kw):
    d = _lib.RotaryDesc()
    d.x[0] = d.y[0] = 16
    d.heads[0] = d.batch = d.seqlen = 2
    d.head_dim, d.rotary_dim, d.amplitude, d.dtype = 64, 64, 1.0, _lib.PDB_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_rotary_record_is_the_descriptor():
    """The packed record fills every field of the descriptor in order."""
    freq = np.arange(64, dtype=np.float64)
    assert _lib.ROTARY_PACK.size == C.sizeof(_lib.RotaryDesc)
    d = _lib.RotaryDesc.from_buffer_copy(_lib.ROTARY_PACK.pack(*range(1, 5), *range(5, 19), 19, *range(20, 27), 27.5,
                                                               freq.tobytes(), 1, 2, 3, 4))
    assert list(d.x) == [1, 2] and list(d.y) == [3, 4] and list(d.heads) == [5, 6]
    assert [list(s) for s in d.x_stride] == [[7, 8, 9], [10, 11, 12]]
    assert [list(s) for s in d.y_stride] == [[13, 14, 15], [16, 17, 18]]
    assert (d.positions, list(d.pos_stride), d.start) == (19, [20, 21], 22)
    assert (d.batch, d.seqlen, d.head_dim, d.rotary_dim, d.amplitude) == (23, 24, 25, 26, 27.5)
    assert list(d.inv_freq) == [*freq] + [0.0] * 64
    assert (d.interleaved, d.inverse, d.dtype, d.reserved) == (1, 2, 3, 4)


def test_rotary_refusals():
    lib = _lib.load()
    assert lib.pdb_rotary(None, None) == _lib.PDB_ERR_ARG
    for kw, want in (({"batch": -1}, _lib.PDB_ERR_SHAPE), ({"rotary_dim": 63}, _lib.PDB_ERR_SHAPE),
                     ({"rotary_dim": 66}, _lib.PDB_ERR_SHAPE), ({"rotary_dim": -2}, _lib.PDB_ERR_SHAPE),
                     ({"head_dim": 512, "rotary_dim": 258}, _lib.PDB_ERR_SHAPE),
                     ({"head_dim": 1 << 21}, _lib.PDB_ERR_SHAPE), ({"dtype": 5}, _lib.PDB_ERR_UNSUPPORTED),
                     ({"batch": 1 << 30, "seqlen": 1 << 30}, _lib.PDB_ERR_SHAPE), ({"batch": 0}, _lib.PDB_OK)):
        assert lib.pdb_rotary(C.byref(_rot(**kw)), None) == want, kw
    for f in (float("nan"), float("inf"), 1e12):
        d = _rot()
        d.inv_freq[3] = f
        assert lib.pdb_rotary(C.byref(d), None) == _lib.PDB_ERR_ARG
        assert b"inv_freq[3]" in lib.pdb_last_error_string()
    d = _rot()
    d.x[0] = 17
    assert lib.pdb_rotary(C.byref(d), None) == _lib.PDB_ERR_ALIGN
    d = _rot()
    d.heads[1] = 1
    assert lib.pdb_rotary(C.byref(d), None) == _lib.PDB_ERR_ARG
    # in place with other strides, and results that are another tensor
    d = _rot()
    d.x_stride[0][:], d.y_stride[0][:] = (256, 64, 128), (256, 128, 64)
    assert lib.pdb_rotary(C.byref(d), None) == _lib.PDB_ERR_ARG
    assert b"in place" in lib.pdb_last_error_string()
    for x, y in (((16, 16), (16, 16)), ((16, 4096), (8192, 8192)), ((16, 4096), (4096, 8192)), ((16, 4096), (8192, 16))):
        d = _rot()
        d.heads[1] = 2
        d.x[:], d.y[:] = x, y
        assert lib.pdb_rotary(C.byref(d), None) == _lib.PDB_ERR_ARG
        assert b"overlaps" in lib.pdb_last_error_string()


def _ce(**kw):
    d = _lib.LinearCeFwdDesc(16, 16, 16, 16, 16, None, 0, 4, 300, 64, 64, 64, -100, _lib.PDB_BF16, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _ce_bwd(**kw):
    d = _lib.LinearCeBwdDesc(16, 16, 16, 16, 16, 16, 16, None, 0, 4, 300, 64, 64, 64, 64, 64, 1, -100, _lib.PDB_BF16, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_linear_cross_entropy_refusals():
    lib = _lib.load()
    assert lib.pdb_linear_ce_fwd(None, None) == lib.pdb_linear_ce_bwd(None, None) == _lib.PDB_ERR_ARG
    assert lib.pdb_linear_ce_fwd_workspace_size(None) == lib.pdb_linear_ce_bwd_workspace_size(None) == 0
    for kw, want in (({"tokens": -1}, _lib.PDB_ERR_SHAPE), ({"vocab": 0}, _lib.PDB_ERR_SHAPE),
                     ({"width": 0}, _lib.PDB_ERR_SHAPE), ({"tokens": (1 << 24) + 1}, _lib.PDB_ERR_SHAPE),
                     ({"vocab": 1 << 40}, _lib.PDB_ERR_SHAPE), ({"width": 1 << 17, "x_stride": 1 << 17}, _lib.PDB_ERR_SHAPE),
                     ({"width": 60}, _lib.PDB_ERR_ALIGN), ({"x_stride": 68}, _lib.PDB_ERR_ALIGN),
                     ({"w_stride": 56}, _lib.PDB_ERR_ALIGN), ({"dtype": 2}, _lib.PDB_ERR_UNSUPPORTED),
                     ({"dtype": _lib.PDB_F32, "width": 62}, _lib.PDB_ERR_ALIGN),
                     ({"dtype": _lib.PDB_F32, "x_stride": 66}, _lib.PDB_ERR_ALIGN),
                     ({"x": None}, _lib.PDB_ERR_ARG), ({"target": None}, _lib.PDB_ERR_ARG)):
        for d, run, size in ((_ce(**kw), lib.pdb_linear_ce_fwd, lib.pdb_linear_ce_fwd_workspace_size),
                             (_ce_bwd(**kw), lib.pdb_linear_ce_bwd, lib.pdb_linear_ce_bwd_workspace_size)):
            assert run(C.byref(d), None) == want, kw
            if want != _lib.PDB_ERR_ARG:
                assert size(C.byref(d)) == 0
    assert lib.pdb_linear_ce_fwd(C.byref(_ce(loss=None, lse=None)), None) == _lib.PDB_ERR_ARG
    assert lib.pdb_linear_ce_bwd(C.byref(_ce_bwd(dx=None, dw=None)), None) == _lib.PDB_ERR_ARG
    for kw in ({"x": 8}, {"w": 40}):
        assert lib.pdb_linear_ce_fwd(C.byref(_ce(**kw)), None) == _lib.PDB_ERR_ALIGN, kw
    for kw in ({"x": 8}, {"w": 40}, {"dx": 8}, {"dw": 8}, {"dx_stride": 68}, {"dw_stride": 56}):
        assert lib.pdb_linear_ce_bwd(C.byref(_ce_bwd(**kw)), None) == _lib.PDB_ERR_ALIGN, kw
    for d, run, size in ((_ce(), lib.pdb_linear_ce_fwd, lib.pdb_linear_ce_fwd_workspace_size),
                         (_ce_bwd(), lib.pdb_linear_ce_bwd, lib.pdb_linear_ce_bwd_workspace_size)):
        need = size(C.byref(d))
        assert need > 0
        d.workspace, d.workspace_bytes = 256, need - 1
        assert run(C.byref(d), None) == _lib.PDB_ERR_ARG
        d.workspace, d.workspace_bytes = 264, need
        assert run(C.byref(d), None) == _lib.PDB_ERR_ARG
        assert b"workspace" in lib.pdb_last_error_string()


def test_linear_cross_entropy_without_tokens():
    """No division by the number of tiles there are not."""
    lib = _lib.load()
    d, b = _ce(tokens=0), _ce_bwd(tokens=0, dw=None)
    assert lib.pdb_linear_ce_fwd_workspace_size(C.byref(d)) == lib.pdb_linear_ce_bwd_workspace_size(C.byref(b)) == 0
    assert lib.pdb_linear_ce_fwd(C.byref(d), None) == lib.pdb_linear_ce_bwd(C.byref(b), None) == _lib.PDB_OK


def test_linear_cross_entropy_workspaces():
    """The gradient's workspace is one piece of G (at most 512 MiB, or 256 columns) and f32 sums of dx, where they are
    shared or in pieces; the largest sizes stay within 64 bits."""
    lib = _lib.load()
    al = lambda n: (n + 255) // 256 * 256

    def need(tokens, vocab, width):
        kw = dict(tokens=tokens, vocab=vocab, width=width, x_stride=width, w_stride=width)
        assert lib.pdb_linear_ce_fwd_workspace_size(C.byref(_ce(**kw))) >= 8 * -(-vocab // 256) * tokens
        return lib.pdb_linear_ce_bwd_workspace_size(C.byref(_ce_bwd(dx_stride=width, dw_stride=width, **kw)))

    def rows(tokens, width):  # the packed tokens: rows of x, target, lse, dloss and index, behind count and unit
        return 512 + al(tokens * ((width + 63) // 64) * 128) + al(tokens * 8) + 3 * al(tokens * 4)

    assert need(8192, 128000, 4096) == 8192 * 32000 * 2 + rows(8192, 4096) + 4 * 8192 * 4096  # four pieces of 32000
    assert need(8192, 32000, 4096) == 8192 * 32000 * 2 + rows(8192, 4096)  # one
    assert need(1 << 24, 1 << 24, 1 << 16) == (1 << 24) * 256 * 2 + rows(1 << 24, 1 << 16) + 4 * (1 << 40)
    assert need(1, 1, 8) == 256 + 512 + 5 * 256


def test_host_tensors_are_refused():
    import torch

    from pdum_dsl_b200 import kernels

    x, v = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.layernorm(x, return_stats=True)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.layernorm_backward(x, x, v, v)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.rotary(x, inv_freq=[1.0])
    b, t = x.bfloat16(), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.linear_cross_entropy(b, b, t)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.linear_cross_entropy_backward(b, b, t, v)


def test_frequency_refusals():
    from pdum_dsl_b200 import kernels

    for args, kw in (((7,), {}), ((258,), {}), ((-2,), {}), ((8,), {"base": 0.0}), ((8,), {"scaling": "other"}),
                     ((8,), {"scaling": "by_parts", "factor": 2.0}), ((2,), {"scaling": "ntk", "factor": 2.0}),
                     ((8,), {"scaling": "linear", "factor": 0.0}),
                     ((8,), {"scaling": "by_parts", "factor": 2.0, "context": 64, "fast": 1.0, "slow": 1.0})):
        with pytest.raises(ValueError):
            kernels.rotary_frequencies(*args, **kw)
    f, m = kernels.rotary_frequencies(0)
    assert len(f) == 0 and m == 1.0
    assert np.array_equal(kernels.rotary_frequencies(2)[0], [1.0])


def test_row_reduction_runners_are_f32():
    """A row-reduction region has an f32 kernel only: its runner refuses device tensors of another type."""
    import torch

    from pdum_dsl_b200.recognize import RowSpec
    from pdum_dsl_b200.tile import _Runner

    for kind in ("softmax", "layernorm"):
        run = object.__new__(_Runner)
        run.dtype = "f32"
        run.spec = RowSpec(kind, 0, None, None, 1e-5, "c", ("r", "c"), ("r", "c"))
        for t in (torch.bfloat16, torch.float64):
            with pytest.raises(TypeError, match="float32"):
                run.run_t(torch.zeros(2, 8, dtype=t))
        with pytest.raises(ValueError, match="CUDA"):
            run.run_t(torch.zeros(2, 8))


def test_layernorm_in_place_needs_one_row_stride():
    """y over x, dx over x or over dout: a row's result lies where the row does, or the call is refused."""
    lib = _lib.load()
    d = _norm()
    d.y_row_stride = 16
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_ERR_ARG
    assert b"in place" in lib.pdb_last_error_string()
    for dx in ("x", "dout"):
        d = _norm_bwd()
        d.workspace, d.workspace_bytes = 16, 1 << 20
        d.x, d.dout, d.dx = 1 << 20, 1 << 21, 1 << (20 if dx == "x" else 21)
        setattr(d, f"{dx}_row_stride", 16)
        assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ARG
        assert b"in place" in lib.pdb_last_error_string()


def test_layernorm_out_over_x_needs_its_row_stride():
    """The same in Python, before the kernels of either kind are called."""
    import torch

    from pdum_dsl_b200 import kernels

    buf = torch.zeros(4, 16)
    x, dense = buf[:, :8], buf.view(-1)[:32].view(4, 8)
    for a, b in ((x, dense), (dense, x)):
        with pytest.raises(ValueError, match="over x"):
            kernels._out_rows("layernorm", b, a, 4, 8, a.stride(0))
    assert kernels._out_rows("layernorm", x, x, 4, 8, 16)[1] == 16
    assert kernels._out_rows("layernorm", buf[:, 8:], x, 4, 8, 16)[1] == 16
    assert kernels._out_rows("layernorm", dense[:1], x[:1], 1, 8, 16)[1] == 8
