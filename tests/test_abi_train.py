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
            "pdb_rotary_desc": "RotaryDesc"}


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
    d = _norm(cols=0)
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_OK
    d.mean = 16
    assert lib.pdb_layernorm_fwd(C.byref(d), None) == _lib.PDB_ERR_SHAPE
    d = _norm_bwd()
    d.dbeta = None
    assert lib.pdb_layernorm_bwd(C.byref(d), None) == _lib.PDB_ERR_ARG
    d = _norm_bwd()
    need = lib.pdb_layernorm_bwd_workspace_size(C.byref(d))
    assert need == 2 * 2 * 8 * 4  # two rows: two partial rows of each gradient
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
