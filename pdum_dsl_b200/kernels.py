"""Device-tensor entry points over the C ABI (the zero-copy fast path).

Each function takes CUDA tensors, fills a descriptor of ``include/pdb.h`` and
launches on the current torch stream.  Nothing here computes on the host and
nothing falls back: a CPU tensor, a dtype the library does not build, or a
missing ``libpdb_sm100.so`` raises.
"""

from __future__ import annotations

import contextlib
import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from ._lib import FlashBwdDesc, FlashDesc, LayerNormDesc, RowSoftmaxDesc, check, load

_DTYPES = {torch.float32: _lib.PDB_F32, torch.bfloat16: _lib.PDB_BF16}


def _stream(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if not t.is_cuda:
            raise ValueError("pdum_dsl_b200 kernels take CUDA tensors (no host fallback)")


def _rows2d(x: torch.Tensor) -> torch.Tensor:
    if x.dim() < 1 or x.stride(-1) != 1:
        x = x.contiguous()
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    if x2.dim() == 2 and x2.shape[0] > 0 and x2.stride(-1) != 1:
        x2 = x2.contiguous()
    return x2


_HERE = contextlib.nullcontext()


def _on_device_of(t: torch.Tensor):
    """The library launches on the current device: make it the tensor's where it is another."""
    return _HERE if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _raw_stream(t: torch.Tensor) -> int:
    """The current torch stream of the tensor's device, without a stream object in between."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _param_dtype(what: str, x: torch.Tensor, cols: int, gamma, beta) -> torch.dtype:
    """The one dtype of the given per-column vectors (float32, or x's)."""
    ptype = None
    for nm, t in (("gamma", gamma), ("beta", beta)):
        if t is None:
            continue
        if (t.dtype != torch.float32 and t.dtype != x.dtype) or t.numel() != cols or t.device != x.device:
            raise ValueError(f"{what}: {nm} must be a CUDA f32 vector of length {cols} (or of x's dtype)")
        if ptype is not None and ptype != t.dtype:
            raise ValueError(f"{what}: gamma and beta must share one dtype")
        ptype = t.dtype
    return ptype or torch.float32


def _out_rows(what: str, out: torch.Tensor, x: torch.Tensor, R: int, C_: int, xs: int) -> tuple[torch.Tensor, int]:
    """out for the row kernels, and its row stride; x's rows lie xs apart."""
    if out.dtype != x.dtype or out.device != x.device or out.numel() != x.numel():
        raise ValueError(f"{what}: out must have x's size, dtype and device")
    y, ys = out, C_
    if not out.is_contiguous():
        y = out.view(R, C_)
        if C_ > 1 and y.stride(-1) != 1:
            raise ValueError(f"{what}: out must have unit stride along its last dim")
        ys = y.stride(0)
    if R > 1 and ys != xs and y.data_ptr() == x.data_ptr():
        raise ValueError(f"{what}: out over x must have x's row stride")
    return y, ys


def _own_rows(x: torch.Tensor) -> torch.Tensor:
    """x as 2-D rows that do not overlap (an expanded gradient is laid out first)."""
    x2 = _rows2d(x)
    return x2.contiguous() if x2.shape[0] > 1 and x2.stride(0) < x2.shape[1] else x2


def _rows(x: torch.Tensor, as_2d=_own_rows) -> tuple[torch.Tensor, int, int, int]:
    """(x, rows, cols, row stride) for the row kernels; a contiguous x as it is (a view is as dear as an allocation)."""
    if x.is_contiguous() and x.dim():
        C_ = x.shape[-1]
        return x, x.numel() // C_ if C_ else math.prod(x.shape[:-1]), C_, C_
    x2 = as_2d(x)
    R, C_ = x2.shape
    return x2, R, C_, x2.stride(0)


def row_softmax(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax over the last dim of an f32 CUDA tensor (row-normalization)."""
    _need_cuda(x)
    if x.dtype != torch.float32:
        raise TypeError("row_softmax: float32 only")
    x2 = _rows2d(x)
    y = torch.empty_like(x2) if out is None else out.view(x2.shape)
    d = RowSoftmaxDesc(x2.data_ptr(), y.data_ptr(), x2.shape[0], x2.shape[1], x2.stride(0) if x2.shape[0] else
                       x2.shape[1], y.stride(0) if y.shape[0] else y.shape[1])
    check(load().pdb_rowsoftmax_f32(C.byref(d), _stream(x)), "pdb_rowsoftmax_f32")
    return y.view(x.shape)


def layernorm(x: torch.Tensor, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None,
              eps: float = 1e-5, out: torch.Tensor | None = None, return_stats: bool = False):
    """Two-pass layernorm over the last dim (row-statistics), f32 or bf16 (sums and statistics in f32).

    gamma / beta are f32 vectors, or of x's dtype.  ``out`` may be x, and shares no memory with it otherwise.
    ``return_stats`` returns
    (y, mean, rstd), the rows' float32 statistics that ``layernorm_backward`` reads."""
    _need_cuda(x)
    if x.dtype not in _DTYPES:
        raise TypeError("layernorm: float32 or bfloat16")
    plain = x.dtype == torch.float32 and not return_stats  # and f32 parameters
    x2, R, C_, xs = _rows(x, _rows2d if plain else _own_rows)
    ptype = _param_dtype("layernorm", x, C_, gamma, beta)
    g = gamma.contiguous() if gamma is not None else None
    b = beta.contiguous() if beta is not None else None
    at_g, at_b = g.data_ptr() if g is not None else None, b.data_ptr() if b is not None else None
    y, ys = (torch.empty_like(x2), C_) if out is None else _out_rows("layernorm", out, x2, R, C_, xs)
    if plain:
        d = LayerNormDesc(x2.data_ptr(), at_g, at_b, y.data_ptr(), R, C_, xs if R else C_, ys if R else C_, float(eps))
        with _on_device_of(x):
            check(load().pdb_layernorm_f32(C.byref(d), _stream(x)), "pdb_layernorm_f32")
        return y.view(x.shape)
    mean = rstd = at_m = at_r = None
    if return_stats:
        mean = x.new_empty(R if x.dim() == 2 else x.shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
        at_m, at_r = mean.data_ptr(), rstd.data_ptr()
    d = _lib.LayerNormFwdDesc(x2.data_ptr(), at_g, at_b, y.data_ptr(), at_m, at_r, R, C_, xs, ys, eps,
                              _DTYPES[x.dtype], _DTYPES[ptype])
    with _on_device_of(x):
        check(load().pdb_layernorm_fwd(C.byref(d), _raw_stream(x)), "pdb_layernorm_fwd")
    if y.shape != x.shape:
        y = y.view(x.shape)
    return (y, mean, rstd) if return_stats else y


def layernorm_backward(dout: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       gamma: torch.Tensor | None = None, *, weight_grads: bool = True):
    """(dx, dgamma, dbeta) of layernorm from the forward's statistics.

    dgamma / dbeta are vectors of gamma's dtype (float32 without gamma), summed in
    float32 in a fixed order; None without ``weight_grads``."""
    _need_cuda(dout, x, mean, rstd)
    dt = x.dtype
    if dt not in _DTYPES or dout.dtype != dt:
        raise TypeError("layernorm_backward: dout and x must both be float32 or bfloat16")
    if dout.shape != x.shape:
        raise ValueError(f"layernorm_backward: dout {tuple(dout.shape)} does not match x {tuple(x.shape)}")
    x2, R, C_, xs = _rows(x)
    do2, _, _, dos = _rows(dout)
    dev, f32 = x.device, torch.float32
    for t in (mean, rstd):
        if t.dtype != f32 or t.numel() != R or t.device != dev:
            raise ValueError(f"layernorm_backward: mean and rstd must be the forward's float32 statistics of {R} rows")
    if dout.device != dev:
        raise ValueError("layernorm_backward: tensors on different devices")
    ptype = _param_dtype("layernorm_backward", x, C_, gamma, None)
    g = gamma.contiguous() if gamma is not None else None
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = torch.empty_like(x2)
    dgamma = dbeta = at_g = at_b = None
    if weight_grads:
        dgamma = x.new_empty(C_, dtype=ptype)
        dbeta = torch.empty_like(dgamma)
        at_g, at_b = dgamma.data_ptr(), dbeta.data_ptr()
    d = _lib.LayerNormBwdDesc(do2.data_ptr(), x2.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                              g.data_ptr() if g is not None else None, dx.data_ptr(), at_g, at_b, None, 0, R, C_,
                              dos, xs, C_, _DTYPES[dt], _DTYPES[ptype])
    lib = load()
    with _on_device_of(x):
        if weight_grads:
            nbytes = lib.pdb_layernorm_bwd_workspace_size(C.byref(d))
            ws = x.new_empty(nbytes + 16, dtype=torch.uint8)
            d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
        check(lib.pdb_layernorm_bwd(C.byref(d), _raw_stream(x)), "pdb_layernorm_bwd")
    return dx if x2 is x else dx.view(x.shape), dgamma, dbeta


def _as4d(t: torch.Tensor, name: str) -> torch.Tensor:
    n = t.dim()
    if n == 2:
        t = t[None, None]
    elif n == 3:
        t = t[None]
    elif n != 4:
        raise ValueError(f"{name}: expected (T, D), (H, T, D) or (B, H, T, D), got {tuple(t.shape)}")
    if t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _result_like(t: torch.Tensor) -> torch.Tensor:
    """A tensor for t's result, its features together.  empty_like keeps t's order of dims, and where two of them have
    stride 1 (overlapping windows) it may put the features further apart."""
    y = torch.empty_like(t)
    return y if y.stride(-1) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format)


def _s3(t: torch.Tensor):
    return _lib.I64x3(t.stride(0), t.stride(1), t.stride(2))


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None,
                    causal: bool = False, q_start: int = 0, out: torch.Tensor | None = None,
                    return_lse: bool = False, return_artifacts: bool = False, key_intervals=None,
                    sm_margin: int = 0):
    """softmax(scale * q k^T [causal: s <= t + q_start]) v.

    q (B, Hq, T, D), k/v (B, Hkv, S, D|Dv) with Hq a multiple of Hkv (GQA);
    2-D and 3-D inputs drop the leading dims.  bf16 runs the tcgen05 kernel
    (D, Dv multiples of 8 up to 256); f32 runs the IEEE CUDA-core kernel (any D, Dv <= 256).  Returns o, or
    (o, lse) / (o, m, den) with the per-row float32 statistics.
    ``key_intervals`` (a ``recognize.KeyIntervals`` of T rows) is a general
    closed mask: row t sees keys lo[t] <= s < hi[t] (``causal`` must be False).
    ``sm_margin`` SMs are left free by the persistent bf16 grid (for a collective
    that runs alongside, e.g. the all-gather of the previous slab's output)."""
    _need_cuda(q, k, v)
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"flash_attention: q/k/v must share dtype float32 or bfloat16, got {q.dtype}/{k.dtype}/{v.dtype}")
    shape_in = q.shape
    q4, k4, v4 = _as4d(q, "q"), _as4d(k, "k"), _as4d(v, "v")
    B, H, T, D = q4.shape
    Bk, HKV, S, Dk = k4.shape
    if Bk != B or Dk != D or v4.shape[:3] != (B, HKV, S):
        raise ValueError(f"flash_attention: incompatible q {tuple(q4.shape)} k {tuple(k4.shape)} v {tuple(v4.shape)}")
    DV = v4.shape[3]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    o = torch.empty((B, H, T, DV), dtype=q.dtype, device=q.device) if out is None else _as4d(out, "out")
    stats = {}
    want = ("lse",) if return_lse else ()
    want += ("m", "den") if return_artifacts else ()
    for nm in want:
        stats[nm] = torch.empty((B, H, T), dtype=torch.float32, device=q.device)
    d = FlashDesc()
    d.q, d.k, d.v, d.o = q4.data_ptr(), k4.data_ptr(), v4.data_ptr(), o.data_ptr()
    d.lse = stats["lse"].data_ptr() if "lse" in stats else None
    d.m = stats["m"].data_ptr() if "m" in stats else None
    d.den = stats["den"].data_ptr() if "den" in stats else None
    d.batch, d.heads_q, d.heads_kv, d.seqlen_q, d.seqlen_k, d.head_dim, d.head_dim_v = B, H, HKV, T, S, D, DV
    d.q_stride, d.k_stride, d.v_stride, d.o_stride = _s3(q4), _s3(k4), _s3(v4), _s3(o)
    d.q_start, d.scale, d.causal, d.dtype = int(q_start), float(scale), int(bool(causal)), _DTYPES[q.dtype]
    d.sm_margin = int(sm_margin)
    keep = None
    if key_intervals is not None:
        if causal:
            raise ValueError("flash_attention: key_intervals replace the causal flag")
        if len(key_intervals.lo) != T:
            raise ValueError(f"flash_attention: key_intervals has {len(key_intervals.lo)} rows, q has {T}")
        keep = torch.from_numpy(np.stack([key_intervals.lo, key_intervals.hi])).to(q.device)
        d.key_lo, d.key_hi = keep[0].data_ptr(), keep[1].data_ptr()
        d.mask_monotone = int(key_intervals.monotone)
    check(load().pdb_flash_fwd(C.byref(d), _stream(q)), "pdb_flash_fwd")
    del keep  # the launch is stream-ordered before any reuse of this memory by the caching allocator
    o_ret = o.view(*shape_in[:-1], DV) if out is None else out
    lead = shape_in[:-1]
    if return_artifacts:
        extra = (stats["lse"].view(lead),) if return_lse else ()
        return (o_ret, *extra, stats["m"].view(lead), stats["den"].view(lead))
    if return_lse:
        return o_ret, stats["lse"].view(lead)
    return o_ret


def flash_attention_backward(q, k, v, o, dout, lse=None, *, scale=None, causal=False, q_start=0):
    """(dq, dk, dv) of flash_attention; ``lse`` None recomputes it."""
    _need_cuda(q, k, v, o, dout)
    if q.dtype not in _DTYPES:
        raise TypeError("flash_attention_backward: float32 or bfloat16")
    shape_q, shape_k, shape_v = q.shape, k.shape, v.shape
    q4, k4, v4, o4, do4 = (_as4d(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (dout, "dout")))
    B, H, T, D = q4.shape
    _, HKV, S, _ = k4.shape
    DV = v4.shape[3]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    dq, dk, dv = torch.empty_like(q4), torch.empty_like(k4), torch.empty_like(v4)
    d = FlashBwdDesc()
    d.q, d.k, d.v, d.o, d.dout = q4.data_ptr(), k4.data_ptr(), v4.data_ptr(), o4.data_ptr(), do4.data_ptr()
    lse_c = lse.contiguous().view(B, H, T) if lse is not None else None
    d.lse = lse_c.data_ptr() if lse_c is not None else None
    d.dq, d.dk, d.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    d.batch, d.heads_q, d.heads_kv, d.seqlen_q, d.seqlen_k, d.head_dim, d.head_dim_v = B, H, HKV, T, S, D, DV
    d.q_stride, d.k_stride, d.v_stride, d.o_stride, d.do_stride = _s3(q4), _s3(k4), _s3(v4), _s3(o4), _s3(do4)
    d.dq_stride, d.dk_stride, d.dv_stride = _s3(dq), _s3(dk), _s3(dv)
    d.q_start, d.scale, d.causal, d.dtype = int(q_start), float(scale), int(bool(causal)), _DTYPES[q.dtype]
    lib = load()
    nbytes = lib.pdb_flash_bwd_workspace_size(C.byref(d))
    ws = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=q.device)
    d.workspace, d.workspace_bytes = ws.data_ptr(), int(nbytes)
    check(lib.pdb_flash_bwd(C.byref(d), _stream(q)), "pdb_flash_bwd")
    return dq.view(shape_q), dk.view(shape_k), dv.view(shape_v)


def rotary(q: torch.Tensor, k: torch.Tensor | None = None, *, inv_freq, positions: torch.Tensor | None = None,
           start: int = 0, interleaved: bool = False, amplitude: float = 1.0, inverse: bool = False, out=None):
    """Rotary positions on the heads that flash_attention reads: q (B, H, T, D), and k (B, Hkv, T, D) in the same
    launch; 2-D and 3-D inputs drop the leading dims, as there.  float32 or bfloat16 (turned in float32).

    Pair j of a head's first 2 * len(inv_freq) features turns by position * inv_freq[j] radians and is multiplied
    by ``amplitude``; the pairs are (j, j + len(inv_freq)), or (2j, 2j + 1) when ``interleaved``; later features
    pass through.  ``inv_freq`` is a host sequence of up to 128 numbers (see ``rotary_frequencies``).
    ``positions`` is an integer CUDA tensor (T,) or (B, T) (either may be broadcast), else row t has position
    start + t.  ``inverse`` turns backwards: the gradient of the forward turn.  ``out`` (a tensor, or a pair with k)
    may be the inputs themselves, and shares no memory otherwise.  Returns the turned q, or (q, k)."""
    ts = (q,) if k is None else (q, k)
    _need_cuda(*ts)
    dt = q.dtype
    if dt not in _DTYPES or (k is not None and k.dtype != dt):
        raise TypeError("rotary: q and k must both be float32 or bfloat16")
    x0 = _as4d(q, "q")
    x1 = x0 if k is None else _as4d(k, "k")
    B, H, T, D = x0.shape
    Bk, Hk, Tk, Dk = x1.shape
    if k is not None and (Bk != B or Tk != T or Dk != D or k.device != q.device):
        raise ValueError(f"rotary: incompatible q {tuple(q.shape)} and k {tuple(k.shape)}")
    freq = np.ascontiguousarray(inv_freq, dtype=np.float64)
    n = len(freq) if freq.ndim == 1 else -1
    if n < 0 or n > _lib.ROTARY_MAX_PAIRS or 2 * n > D:
        raise ValueError(f"rotary: inv_freq must be a vector of at most {_lib.ROTARY_MAX_PAIRS} pairs within the head's {D} features")
    if out is None:
        y0 = _result_like(x0)
        y1 = y0 if k is None else _result_like(x1)
    else:
        outs = (out,) if k is None else tuple(out)
        if len(outs) != len(ts):
            raise ValueError("rotary: out must be one tensor for each input")
        for o, t in zip(outs, ts):
            if o.shape != t.shape or o.dtype != dt or o.device != t.device:
                raise ValueError("rotary: out must have the inputs' shape, dtype and device")
            if (o.stride(-1) != 1 and not o.is_contiguous()) or any(m > 1 and st == 0 for m, st in zip(o.shape, o.stride())):
                raise ValueError("rotary: out must have unit stride along the features and no broadcast dim")
        y0, y1 = _as4d(outs[0], "out"), _as4d(outs[-1], "out")
    at_p, ps = 0, (0, 0)
    if positions is not None:
        if positions.device != q.device or positions.dtype not in (torch.int64, torch.int32):
            raise TypeError("rotary: positions must be an integer tensor on q's device")
        if positions.dim() not in (1, 2):
            raise ValueError("rotary: positions must be (T,) or (B, T)")
        p = positions if positions.dtype == torch.int64 else positions.to(torch.int64)
        if p.shape != (B, T):
            p = p.expand(B, T)
        at_p, ps = p.data_ptr(), p.stride()
    # one packed record: a third of the time of setting the descriptor's fields one by one
    d = _lib.RotaryDesc.from_buffer_copy(_lib.ROTARY_PACK.pack(
        x0.data_ptr(), x1.data_ptr(), y0.data_ptr(), y1.data_ptr(), H, 0 if k is None else Hk,
        *x0.stride()[:3], *x1.stride()[:3], *y0.stride()[:3], *y1.stride()[:3], at_p, *ps, start, B, T, D, 2 * n,
        amplitude, freq.tobytes(), bool(interleaved), bool(inverse), _DTYPES[dt], 0))
    with _on_device_of(q):
        check(load().pdb_rotary(C.byref(d), _raw_stream(q)), "pdb_rotary")
    if out is not None:
        return outs[0] if k is None else outs
    if x0 is not q:
        y0 = y0.view(q.shape)
    if k is None:
        return y0
    return y0, y1 if x1 is k else y1.view(k.shape)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       context: int = 0, fast: float = 32.0, slow: float = 1.0) -> tuple[np.ndarray, float]:
    """(inv_freq, amplitude) for ``rotary``: base^(-2j / rotary_dim), scaled for contexts ``factor`` times as long as
    the ``context`` that a model was trained on.

    scaling "none"; "linear": every angle divided by factor (position interpolation); "ntk": the base grown to
    base * factor^(rotary_dim / (rotary_dim - 2)), which divides the slowest pair's angle by factor and leaves the
    fastest; "by_parts" (YaRN, Peng et al. 2023): pairs that make at least ``fast`` turns over the context keep their
    frequency, those with at most ``slow`` are divided by factor, a ramp between, and amplitude 0.1 ln(factor) + 1."""
    if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > 2 * _lib.ROTARY_MAX_PAIRS:
        raise ValueError(f"rotary_frequencies: rotary_dim must be even and at most {2 * _lib.ROTARY_MAX_PAIRS}")
    if not base > 0 or not factor > 0:
        raise ValueError("rotary_frequencies: base and factor must be positive")
    j2 = np.arange(0, rotary_dim, 2, dtype=np.float64)
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("rotary_frequencies: ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-j2 / max(rotary_dim, 1))
    if scaling in ("none", "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling != "by_parts":
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if context <= 0 or not fast > slow:
        raise ValueError("rotary_frequencies: by_parts needs the trained context and fast > slow")
    keep = np.clip((context * freq / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
    return freq * keep + freq / factor * (1.0 - keep), (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)


def check_device_errors() -> None:
    """Synchronise the current stream and raise if a bounded device wait expired."""
    s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    check(load().pdb_check_error(s), "pdb_check_error")


def _ew_program(ops, out_shape):
    """ops: list of (name, operand) with operand None (unary), a float, or a CUDA
    float32 tensor broadcastable to out_shape (batch, m, n)."""
    if len(ops) > _lib.MAX_EW_OPS:
        raise ValueError(f"at most {_lib.MAX_EW_OPS} epilogue steps")
    arr = (_lib.EwOp * _lib.MAX_EW_OPS)()
    keep = []
    for i, (name, operand, swap) in enumerate(ops):
        o = arr[i]
        o.op = _lib.EW_OPS[name]
        o.swap = int(bool(swap))
        if operand is None:
            o.operand = 0
        elif isinstance(operand, (int, float)):
            o.operand, o.value = 1, float(operand)
        else:
            t = operand.float().expand(out_shape)
            keep.append(t)
            o.operand, o.ptr = 2, t.data_ptr()
            o.stride = _lib.I64x3(t.stride(0), t.stride(1), t.stride(2))
    return arr, keep


def contract(a: torch.Tensor, b: torch.Tensor, *, epilogue=(), alpha: float = 1.0,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """c[b, m, n] = epilogue(alpha * sum_k a[b, m, k] * b[b, n, k]).

    a (batch, m, k), b (batch, n, k): f32 (IEEE path, f32 out) or bf16 with k
    contiguous (tcgen05 path, bf16 out).  ``epilogue`` is a sequence of
    (op, operand, swap) steps with operand None (unary), a float, or a CUDA
    tensor broadcastable to (batch, m, n)."""
    _need_cuda(a, b)
    if a.dtype not in _DTYPES or b.dtype != a.dtype:
        raise TypeError("contract: a and b must both be float32 or bfloat16")
    Bt, M, K = a.shape
    Bb, N, Kb = b.shape
    if Bb != Bt or Kb != K:
        raise ValueError(f"contract: incompatible a {tuple(a.shape)} b {tuple(b.shape)}")
    if a.dtype == torch.bfloat16:
        a = a if a.stride(2) == 1 else a.contiguous()
        b = b if b.stride(2) == 1 else b.contiguous()
    c = torch.empty((Bt, M, N), dtype=a.dtype, device=a.device) if out is None else out
    d = _lib.ContractDesc()
    d.a, d.b, d.c = a.data_ptr(), b.data_ptr(), c.data_ptr()
    d.batch, d.m, d.n, d.k = Bt, M, N, K
    d.a_stride, d.b_stride, d.c_stride = _s3(a), _s3(b), _s3(c)
    d.alpha, d.dtype = float(alpha), _DTYPES[a.dtype]
    ops, keep = _ew_program(list(epilogue), (Bt, M, N))
    d.ops, d.n_ops = ops, len(epilogue)
    check(load().pdb_contract(C.byref(d), _stream(a)), "pdb_contract")
    del keep
    return c


def pointwise(x: torch.Tensor, program, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = program(x) elementwise over an f32 (batch, m, n) CUDA tensor (map-chain)."""
    _need_cuda(x)
    if x.dtype != torch.float32 or x.dim() != 3:
        raise TypeError("pointwise: a 3-D float32 tensor")
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device) if out is None else out
    d = _lib.PointwiseDesc()
    d.x, d.y = x.data_ptr(), y.data_ptr()
    d.batch, d.m, d.n = x.shape
    d.x_stride, d.y_stride = _s3(x), _s3(y)
    ops, keep = _ew_program(list(program), tuple(x.shape))
    d.ops, d.n_ops = ops, len(program)
    check(load().pdb_pointwise_f32(C.byref(d), _stream(x)), "pdb_pointwise_f32")
    del keep
    return y


def _head_operand(t: torch.Tensor) -> torch.Tensor:
    """A 2-D matrix as the products take it: 16-byte aligned rows with unit stride, laid out anew otherwise."""
    R, W = t.shape
    ok = t.data_ptr() % 16 == 0 and (W <= 1 or t.stride(1) == 1) and (
        R <= 1 or (t.stride(0) >= W and t.stride(0) * t.element_size() % 16 == 0))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _head_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _head_args(what: str, x, weight, target):
    _need_cuda(x, weight, target)
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise TypeError(f"{what}: x and weight must both be bfloat16 or float32, got {x.dtype} / {weight.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or target.shape != x.shape[:-1]:
        raise ValueError(f"{what}: incompatible x {tuple(x.shape)}, weight {tuple(weight.shape)} and target {tuple(target.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"{what}: target must be int64")
    if weight.device != x.device or target.device != x.device:
        raise ValueError(f"{what}: tensors on different devices")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    t = target if target.dim() == 1 else target.reshape(-1)
    return _head_operand(x2), _head_operand(weight), t.contiguous()


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         return_lse: bool = False):
    """The cross entropy of a linear head, per token, without storing its logits.

    x (..., width) and weight (vocab, width) bf16 (tcgen05 products) or f32 (IEEE), rows of whole 16 bytes (width a
    multiple of 8, or of 4); target (...) int64.  Returns the float32
    loss logsumexp_v(x . weight[v]) - x . weight[target], 0 where the target is ``ignore_index`` and NaN where it is
    another index outside the vocabulary; with ``return_lse`` (loss, lse), which the backward takes."""
    x2, w, t = _head_args("linear_cross_entropy", x, weight, target)
    N, W = x2.shape
    loss = x.new_empty(x.shape[:-1], dtype=torch.float32)
    lse = torch.empty_like(loss)
    d = _lib.LinearCeFwdDesc(x2.data_ptr(), w.data_ptr(), t.data_ptr(), loss.data_ptr(), lse.data_ptr(), None, 0,
                             N, w.shape[0], W, _head_stride(x2), _head_stride(w), int(ignore_index), _DTYPES[x.dtype], 0)
    lib = load()
    with _on_device_of(x):
        ws = x.new_empty(lib.pdb_linear_ce_fwd_workspace_size(C.byref(d)) + 16, dtype=torch.uint8)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.pdb_linear_ce_fwd(C.byref(d), _raw_stream(x)), "pdb_linear_ce_fwd")
    return (loss, lse) if return_lse else loss


def linear_cross_entropy_backward(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, dloss: torch.Tensor,
                                  lse: torch.Tensor | None = None, *, ignore_index: int = -100, need_dx: bool = True,
                                  need_dweight: bool = True):
    """(dx, dweight) of linear_cross_entropy, of x's dtype, from the per-token float32 gradient of the loss.

    ``dloss`` broadcasts to target's shape (for a mean over n tokens: a tensor holding 1 / n); ``lse`` None recomputes
    it.  A gradient that is not needed is None."""
    x2, w, t = _head_args("linear_cross_entropy_backward", x, weight, target)
    if not dloss.is_cuda or dloss.dtype != torch.float32 or dloss.device != x.device:
        raise TypeError("linear_cross_entropy_backward: dloss must be a float32 tensor on x's device")
    if not (need_dx or need_dweight):
        return None, None
    N, W = x2.shape
    V = w.shape[0]
    if lse is None:
        _, lse = linear_cross_entropy(x, weight, target, ignore_index=ignore_index, return_lse=True)
    elif lse.dtype != torch.float32 or lse.shape != target.shape or lse.device != x.device:
        raise ValueError("linear_cross_entropy_backward: lse must be the forward's float32 logsumexp")
    lse = lse.reshape(-1).contiguous()
    if dloss.numel() == 1:
        g, gs = dloss, 0
    else:
        g, gs = dloss.expand(target.shape).reshape(-1).contiguous(), 1
    dx = x.new_empty((N, W)) if need_dx else None
    dw = x.new_empty((V, W)) if need_dweight else None
    d = _lib.LinearCeBwdDesc(x2.data_ptr(), w.data_ptr(), t.data_ptr(), lse.data_ptr(), g.data_ptr(),
                             dx.data_ptr() if need_dx else None, dw.data_ptr() if need_dweight else None, None, 0,
                             N, V, W, _head_stride(x2), _head_stride(w), W, W, gs, int(ignore_index), _DTYPES[x.dtype], 0)
    lib = load()
    with _on_device_of(x):
        ws = x.new_empty(lib.pdb_linear_ce_bwd_workspace_size(C.byref(d)) + 16, dtype=torch.uint8)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.pdb_linear_ce_bwd(C.byref(d), _raw_stream(x)), "pdb_linear_ce_bwd")
    return dx.view(x.shape) if need_dx else None, dw
