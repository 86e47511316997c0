"""Orthogonalised updates: `newton_schulz` for a list of matrices (`neosr_newton_schulz`)."""

from __future__ import annotations

import contextlib
import ctypes as C
import math

import torch

from neosr_amd import _C
from neosr_amd.hip.attention import refuse_tangents

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_DTYPES = {torch.float32: _C.DT_F32, torch.bfloat16: _C.DT_BF16}


def coefficient_table(steps: int, coefficients):
    """the (a, b, c) of every step as a C float array: one triple for all steps or one for each"""
    steps = int(steps)
    if not 1 <= steps <= 64:
        raise _C.NeosrAmdError(f"newton_schulz: {steps} steps (1 to 64)")
    rows = list(coefficients)
    if rows and not isinstance(rows[0], (tuple, list)):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 or not all(math.isfinite(float(x)) for x in r) for r in rows):
        raise _C.NeosrAmdError("newton_schulz: coefficients must be one finite (a, b, c) or one for each step")
    return (C.c_float * (3 * steps))(*[float(x) for r in rows for x in r])


def too_large(rows: int, cols: int) -> bool:
    """what one matrix may have: sides to 32768, 2^29 elements once they are padded to multiples of 32"""
    return max(rows, cols) > 32768 or (rows + 31) // 32 * 32 * ((cols + 31) // 32 * 32) > 1 << 29


def ns_item(t, out, name: str = "matrix"):
    """`neosr_ns_item` of a (..., rows, cols) tensor and where its result goes (same shape)"""
    rows, cols = t.shape[-2:]
    x, y = (v.unsqueeze(0) if v.dim() == 2 else v.flatten(0, -3) for v in (t, out))
    if x.shape[0] > 65536 or too_large(rows, cols):
        raise _C.NeosrAmdError(f"newton_schulz: {name} {tuple(t.shape)} is too large (sides to 32768, 2^29 elements, 65536 matrices)")
    return _C.NsItem(in_=x.data_ptr(), out=y.data_ptr(), in_sb=x.stride(0), in_sr=x.stride(1), out_sb=y.stride(0),
                     out_sr=y.stride(1), count=x.shape[0], rows=rows, cols=cols), x, y


def newton_schulz(matrices, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """Newton-Schulz iterates of matrices towards their orthogonal polar factor, as the `muon` optimizer applies them:
    X = G / (|G|_F + eps), then `steps` times X <- (a I + b A + c A A) X with A = X X^T (the mirrored form for tall ones).

    `matrices`: a tensor (..., rows, cols) — leading dimensions are a batch — or a list of such tensors of any shapes, float32
    or bfloat16 (one type per call), strided rows allowed.  A list advances together, one launch per product and step for all
    of it.  `coefficients`: (a, b, c), or one triple for each step.  Returns new dense tensors of the same shapes and type; fp32
    matrices are computed fp32-faithfully, bf16 ones with products good to 2^-16 and one rounding at the end.  Any finite matrix is
    normalised, whatever its size; a zero matrix gives 0 (NaN with eps = 0).  Not differentiable (an optimizer's operator)."""
    single = isinstance(matrices, torch.Tensor)
    mats = [matrices] if single else list(matrices)
    table = coefficient_table(steps, coefficients)
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise _C.NeosrAmdError(f"newton_schulz: eps must be finite and not negative (got {eps})")
    if not mats:
        return []
    for t in mats:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise _C.NeosrAmdError(f"neosr_amd: matrices must live on a HIP device (got {getattr(t, 'device', type(t))})")
        if t.dtype not in _DTYPES or t.dtype != mats[0].dtype or t.device != mats[0].device:
            raise _C.NeosrAmdError(f"newton_schulz: matrices must be all float32 or all bfloat16 on one device (got {t.dtype} on "
                                   f"{t.device})")
        if t.dim() < 2:
            raise _C.NeosrAmdError(f"newton_schulz: {tuple(t.shape)} is no matrix")
        if t.requires_grad and torch.is_grad_enabled():
            raise _C.NeosrAmdError("newton_schulz is not differentiable: pass detached tensors")
    refuse_tangents("newton_schulz", *mats)
    lib = _C.load()
    dev = mats[0].device
    with contextlib.nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev):
        outs = [torch.empty(t.shape, device=dev, dtype=t.dtype) for t in mats]
        items, keep = [], []
        for t, o in zip(mats, outs):
            if t.numel():
                it, x, _y = ns_item(t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous(), o)
                items.append(it)
                keep.append(x)          # (a copy made for the call lives until its launches are enqueued)
        if items:
            arr = (_C.NsItem * len(items))(*items)
            nbytes = lib.neosr_newton_schulz_workspace_bytes(arr, len(items), _DTYPES[mats[0].dtype])
            if nbytes < 0:
                _C.check(1, "neosr_newton_schulz_workspace_bytes")
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            _C.check(lib.neosr_newton_schulz(arr, len(items), _DTYPES[mats[0].dtype], int(steps), table, eps, ws.data_ptr(), nbytes,
                                             _C.stream_ptr()), "neosr_newton_schulz")
    return outs[0] if single else outs
