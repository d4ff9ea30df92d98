"""The 8-bit floating-point layer for torch tensors on the GPU: quantisation, the norm that quantises, products
with a scale per block, routing and the layer of experts.

Quantised tensors are pairs: codes of dtype ``torch.float8_e4m3fn`` and fp32 scales, one per block of 128
consecutive elements of a row (activations: ``scale[m, k // 128]``) or of 128 x 128 elements (weights:
``scale[n // 128, k // 128]``).  The activation scales that these functions allocate are stored by column (a
[blocks, rows] tensor, transposed): that is how the products read them fastest.  Any strides are accepted.

Like ``gemm``, every function is asynchronous on ``stream`` (default torch's current one; results that it allocates
belong to that stream) and takes the tensors to write as optional arguments.  It raises RuntimeError for arguments that
do not fit together or are not on a GPU.
"""
from __future__ import annotations

import struct

import torch

from . import BFLOAT16, FLOAT16, FLOAT32, FP8_BLOCK, TV_E_SHAPE, check
from .matmul import _empty, _launch

_F8 = torch.float8_e4m3fn
_FLOATS = {torch.bfloat16: BFLOAT16, torch.float16: FLOAT16, torch.float32: FLOAT32}
_TORCH = {v: k for k, v in _FLOATS.items()}
_SCORING = {"softmax": 0, "sigmoid": 1}


def _fail(msg: str):
    raise RuntimeError(msg)


def _float(t: torch.Tensor, name: str) -> int:
    dt = _FLOATS.get(t.dtype)
    if dt is None:
        _fail(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    return dt


# A small call is bound by this host code, and every attribute of a tensor is a call into torch: the checks read each
# once and build their messages only when one fails.

def _row(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device) -> int:
    """Row stride of a tensor that must have this type, shape and device and contiguous rows."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        _fail(f"{name} must be {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    if t.is_contiguous():
        return shape[1]
    return _rows(t, name)


def _rows(t: torch.Tensor, name: str) -> int:
    s0, s1 = t.stride()
    if s1 != 1 and t.shape[1] > 1:
        _fail(f"{name} must have contiguous rows, got strides {(s0, s1)}")
    return s0


def _any(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device) -> tuple:
    """Strides of a tensor that must have this type, shape and device."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        _fail(f"{name} must be {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.stride()


def _dense(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device) -> int:
    """Address of a contiguous tensor that must have this type, shape and device."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        _fail(f"{name} must be {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")
    return t.data_ptr()


def _out(out, out_dtype, shape: tuple, device, stream) -> tuple:
    """The result tensor, its type and its row stride."""
    if out is None:
        out_dtype = BFLOAT16 if out_dtype is None else out_dtype
        if out_dtype not in _TORCH:
            _fail(f"out_dtype must be BFLOAT16, FLOAT16 or FLOAT32, got {out_dtype}")
        return _empty(shape, _TORCH[out_dtype], device, stream), out_dtype, shape[1]
    dt = _float(out, "out")
    return out, dt, _row(out, "out", out.dtype if out_dtype is None else _TORCH.get(out_dtype), shape, device)


def _scale_out(scale, shape: tuple, device, stream) -> tuple:
    """Activation scales, stored by column where they are made here, and their strides."""
    if scale is None:
        return _empty((shape[1], shape[0]), torch.float32, device, stream).t(), (1, shape[0])
    return scale, _any(scale, "scale", torch.float32, shape, device)


def _codes_out(q, shape: tuple, device, stream) -> tuple:
    if q is None:
        return _empty(shape, _F8, device, stream), shape[1]
    return q, _row(q, "q", _F8, shape, device)


def _call(name: str, args: bytes, device, stream) -> None:
    index = device.index
    if index is None:
        _fail(f"the tensors must be on a GPU, got {device}")
    rc = _launch(name, args, index, stream)
    if rc:
        check(rc)


_pack_quantize = struct.Struct("2i2qPqPqP2q").pack


def quantize_fp8(x: torch.Tensor, block_rows: int = 1, q: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                 stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of ``x`` [M, K] in blocks of ``block_rows`` x 128 (1: activations, 128: weights)."""
    if x.dim() != 2:
        _fail(f"x must have 2 dimensions, got {x.dim()}")
    dt, shape, dev = _float(x, "x"), x.shape, x.device
    m, k = shape
    if block_rows == 1:
        scale, ss = _scale_out(scale, (m, (k + 127) // 128), dev, stream)
    elif block_rows == FP8_BLOCK:
        grid = ((m + 127) // 128, (k + 127) // 128)
        if scale is None:
            scale = _empty(grid, torch.float32, dev, stream)
        ss = _any(scale, "scale", torch.float32, grid, dev)
    else:
        _fail(f"block_rows must be 1 or {FP8_BLOCK}, got {block_rows}")
    q, sq = _codes_out(q, shape, dev, stream)
    _call("tv_hip_quantize_fp8", _pack_quantize(dt, block_rows, m, k, x.data_ptr(), k if x.is_contiguous() else _rows(x, "x"),
                                                q.data_ptr(), sq, scale.data_ptr(), *ss), dev, stream)
    return q, scale


_pack_norm = struct.Struct("2i2qfiPqPqPPqP2qPqPq").pack


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                 q: torch.Tensor | None = None, scale: torch.Tensor | None = None, residual_out: torch.Tensor | None = None,
                 normed: torch.Tensor | bool | None = None, stream=None):
    """Root-mean-square norm of ``x + residual`` times ``weight``, quantised in blocks of 128: (q, scale, residual_out,
    normed).

    ``residual_out`` (allocated where ``residual`` is given; None without one) receives ``x + residual`` in x's type and
    may be ``x`` or ``residual`` itself; ``normed`` (a tensor, or True to allocate one; None without) the normalised
    rows in x's type, which a router reads.  ``weight`` has x's type or float32."""
    if x.dim() != 2:
        _fail(f"x must have 2 dimensions, got {x.dim()}")
    dt, shape, dev, dtype = _float(x, "x"), x.shape, x.device, x.dtype
    t, h = shape
    dw = weight.dtype
    if (dw is not dtype and dw is not torch.float32) or weight.shape != (h,) or weight.device != dev:
        _fail(f"weight must be {dtype} or torch.float32 {[h]} on {dev}, got {dw} {list(weight.shape)} on {weight.device}")
    if not weight.is_contiguous():
        _fail("weight must be contiguous")
    pr = sr = po = so = pn = sn = 0
    if residual is not None:
        pr, sr = residual.data_ptr(), _row(residual, "residual", dtype, shape, dev)
        if residual_out is None:
            residual_out = _empty(shape, dtype, dev, stream)
    if residual_out is not None:
        po, so = residual_out.data_ptr(), _row(residual_out, "residual_out", dtype, shape, dev)
    if normed is True:
        normed = _empty(shape, dtype, dev, stream)
    elif normed is False:
        normed = None
    if normed is not None:
        pn, sn = normed.data_ptr(), _row(normed, "normed", dtype, shape, dev)
    q, sq = _codes_out(q, shape, dev, stream)
    scale, ss = _scale_out(scale, (t, (h + 127) // 128), dev, stream)
    _call("tv_hip_rms_norm_fp8",
          _pack_norm(dt, _FLOATS[dw], t, h, eps, 0, x.data_ptr(), h if x.is_contiguous() else _rows(x, "x"), pr, sr,
                     weight.data_ptr(), q.data_ptr(), sq, scale.data_ptr(), *ss, po, so, pn, sn), dev, stream)
    return q, scale, residual_out, normed


_pack_gemm = struct.Struct("2i3qPqP2qPqP2qPq").pack


def gemm_fp8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out: torch.Tensor | None = None,
             out_dtype: int | None = None, stream=None) -> torch.Tensor:
    """``a @ w.T`` of codes ``a`` [M, K] (scales [M, K / 128]) and ``w`` [N, K] (scales [N / 128, K / 128]).

    ``out_dtype``: BFLOAT16 (default), FLOAT16 or FLOAT32."""
    sa, sw = a.shape, w.shape
    if len(sa) != 2 or len(sw) != 2 or sa[1] != sw[1]:
        _fail(f"a and w must be [M, K] and [N, K], got {list(sa)} and {list(sw)}")
    (m, k), n, dev = sa, sw[0], a.device
    ra, rw = _row(a, "a", _F8, sa, dev), _row(w, "w", _F8, sw, dev)
    kb = (k + 127) // 128
    ss = _any(a_scale, "a_scale", torch.float32, (m, kb), dev)
    ws = _any(w_scale, "w_scale", torch.float32, ((n + 127) // 128, kb), dev)
    out, dt, so = _out(out, out_dtype, (m, n), dev, stream)
    _call("tv_hip_gemm_fp8", _pack_gemm(dt, 0, m, n, k, a.data_ptr(), ra, a_scale.data_ptr(), *ss, w.data_ptr(), rw,
                                        w_scale.data_ptr(), *ws, out.data_ptr(), so), dev, stream)
    return out


_pack_route = struct.Struct("2iq6ifiPq3P").pack


def route(logits: torch.Tensor, k: int, scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          topk_groups: int = 1, group_top: int = 1, renormalize: bool = True, scale: float = 1.0,
          weights: torch.Tensor | None = None, ids: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` experts of each token and their weights, from ``logits`` [T, E]: (weights [T, k], ids [T, k] int32).

    Scores are ``softmax`` or ``sigmoid`` of the logits; the choice is by score + ``bias`` [E] (float32), the weights are
    the scores, divided by their sum (``renormalize``) and multiplied by ``scale``.  ``groups`` > 1: only the
    ``topk_groups`` groups of experts with the largest sum of their best ``group_top`` (1 or 2) values take part.
    Ties go to the lowest index.  An expert with a logit or bias of -inf or NaN is never chosen; slots that no
    expert fills have id -1 and weight 0."""
    if logits.dim() != 2:
        _fail(f"logits must have 2 dimensions, got {logits.dim()}")
    dt, (t, e), dev = _float(logits, "logits"), logits.shape, logits.device
    if scoring not in _SCORING:
        _fail(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if not 1 <= k <= e:
        check(TV_E_SHAPE)
    pb = 0 if bias is None else _dense(bias, "bias", torch.float32, (e,), dev)
    if weights is None:
        weights = _empty((t, k), torch.float32, dev, stream)
    if ids is None:
        ids = _empty((t, k), torch.int32, dev, stream)
    pw, pi = _dense(weights, "weights", torch.float32, (t, k), dev), _dense(ids, "ids", torch.int32, (t, k), dev)
    _call("tv_hip_route",
          _pack_route(dt, _SCORING[scoring], t, e, k, groups, topk_groups, group_top, bool(renormalize), scale, 0,
                      logits.data_ptr(), e if logits.is_contiguous() else _rows(logits, "logits"), pb, pw, pi), dev, stream)
    return weights, ids


_pack_experts = struct.Struct("2i3q2iPqP2qP3qPP2qPPPPq").pack


def experts_fp8(a: torch.Tensor, a_scale: torch.Tensor, w1: torch.Tensor, w1_scale: torch.Tensor, w2: torch.Tensor,
                w2_scale: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None,
                out_dtype: int | None = None, stream=None) -> torch.Tensor:
    """A layer of experts on quantised rows ``a`` [T, H]: for each token the sum over its slots of
    ``weights * (silu(x @ w1[e, 0].T) * (x @ w1[e, 1].T)) @ w2[e].T``, the inner rows quantised in blocks of 128.

    ``w1`` [E, 2, I, H] (gate, up) with scales [E, 2, I / 128, H / 128], ``w2`` [E, H, I] with scales [E, H / 128, I / 128];
    ``weights`` and ``ids`` [T, k] as ``route`` returns them (an id outside [0, E) is no expert)."""
    sa, s1, si = a.shape, w1.shape, ids.shape
    if len(sa) != 2 or len(s1) != 4 or w2.dim() != 3 or len(si) != 2:
        _fail("a, w1, w2 and ids must have 2, 4, 3 and 2 dimensions")
    (t, h), (e, _, i, _), k, dev = sa, s1, si[1], a.device
    hb, ib = (h + 127) // 128, (i + 127) // 128
    ra = _row(a, "a", _F8, sa, dev)
    t1, t2 = _any(w1, "w1", _F8, (e, 2, i, h), dev), _any(w2, "w2", _F8, (e, h, i), dev)
    if (t1[3] != 1 and h > 1) or (t2[2] != 1 and i > 1):
        _fail("w1 and w2 must have contiguous rows")
    ss = _any(a_scale, "a_scale", torch.float32, (t, hb), dev)
    p1 = _dense(w1_scale, "w1_scale", torch.float32, (e, 2, ib, hb), dev)
    p2 = _dense(w2_scale, "w2_scale", torch.float32, (e, hb, ib), dev)
    pw, pi = _dense(weights, "weights", torch.float32, (t, k), dev), _dense(ids, "ids", torch.int32, (t, k), dev)
    out, dt, so = _out(out, out_dtype, (t, h), dev, stream)
    _call("tv_hip_experts_fp8",
          _pack_experts(dt, 0, t, h, i, e, k, a.data_ptr(), ra, a_scale.data_ptr(), *ss, w1.data_ptr(), *t1[:3], p1,
                        w2.data_ptr(), *t2[:2], p2, pw, pi, out.data_ptr(), so), dev, stream)
    return out
