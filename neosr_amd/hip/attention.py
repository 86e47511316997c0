"""Attention over whole token sequences and the rotary positions that go with it.

The window forms (`hip/transformer.py`: `window_attention`, `flash_window_attention`) follow the reference's generators: fixed
windows, a relative-position bias table, fp32.  These two stand beside them for transformers whose tokens attend a whole
picture, a padded batch of pictures, another picture's tokens, or frames in order:

    q, k = axial_rope(q, k, positions, sections)           # (B, N, H, D) views of a fused projection, no copies
    y = attention(q, k, v, key_mask=mask)                   # (B, N, H, D)

Both are differentiable, take float32 (the framework's storage type; fp32-faithful products) or bfloat16 tensors, run on the
current stream and may be captured into a HIP graph.  torch is used for allocation and the autograd graph only.
"""

from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd import forward_ad

from neosr_amd import _C

_DTYPES = {torch.float32: _C.DT_F32, torch.bfloat16: _C.DT_BF16}
_POS_KINDS = {torch.float32: _C.POS_F32, torch.int32: _C.POS_I32, torch.int64: _C.POS_I64}


def _on(device):
    """The library launches on the current device: switch to the tensors' one if it is another (free otherwise)."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _tensor(t, name: str, dims: int, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _C.NeosrAmdError(f"neosr_amd: {name} must live on a HIP device (got {getattr(t, 'device', type(t))})")
    if t.dim() != dims:
        raise _C.NeosrAmdError(f"neosr_amd: {name} must have {dims} dimensions (got {tuple(t.shape)})")
    if like is not None and t.device != like.device:
        raise _C.NeosrAmdError(f"neosr_amd: {name} is on {t.device}, not on {like.device}")
    return t


def _heads(t, name: str, like=None):
    """a (B, L, heads, D) operand: any strides, unit channel stride (else one copy)"""
    t = _tensor(t, name, 4, like)
    if t.dtype not in _DTYPES:
        raise _C.NeosrAmdError(f"neosr_amd: {name} must be float32 or bfloat16 (got {t.dtype})")
    if like is not None and t.dtype != like.dtype:
        raise _C.NeosrAmdError(f"neosr_amd: {name} is {t.dtype}, not {like.dtype}")
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def refuse_tangents(name: str, *tensors):
    """Forward-mode derivatives: a dual tensor looks like any other (requires_grad is False, its pointer is readable), so a call
    would drop its tangent.  Outside a `dual_level` there are none, and the look at the level is all that a call pays."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _C.NeosrAmdError(f"{name} has no forward-mode derivative: pass tensors without a tangent")


def _ptr(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


def _attention_desc(q, k, v, out, rest, lse, key_mask, scale, causal):
    B, Lq, H, D = q.shape
    d = _C.AttentionDesc(q=_ptr(q), k=_ptr(k), v=_ptr(v), out=_ptr(out), out_rest=_ptr(rest), lse=_ptr(lse),
                         key_mask=_ptr(key_mask),
                         B=B, Lq=Lq, Lk=k.shape[1], H=H, Hk=k.shape[2], D=D, dtype=_DTYPES[q.dtype], causal=int(causal),
                         scale=scale)
    d.q_sb, d.q_sl, d.q_sh = q.stride()[:3]
    d.k_sb, d.k_sl, d.k_sh = k.stride()[:3]
    d.v_sb, d.v_sl, d.v_sh = v.stride()[:3]
    if key_mask is not None:
        d.mask_sb, d.mask_sl = key_mask.stride()
    return d


def _workspace(d, nbytes: int, like):
    if nbytes < 0:
        _C.check(1, "neosr_attention_workspace_bytes")
    if nbytes == 0:
        return None
    ws = torch.empty(nbytes, device=like.device, dtype=torch.uint8)
    d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _dense(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(q, k, v, scale, causal, key_mask, keep):
    lib = _C.load()
    with _on(q.device):
        out = _dense(q)
        lse = torch.empty(q.shape[0] * q.shape[1] * q.shape[2], device=q.device, dtype=torch.float32) if keep else None
        # bf16: what the rounding of `out` left, for the backward's rowsum(dout * out)
        rest = _dense(q) if keep and q.dtype == torch.bfloat16 else None
        d = _attention_desc(q, k, v, out, rest, lse, key_mask, scale, causal)
        ws = _workspace(d, lib.neosr_attention_fwd_workspace_bytes(d), q)  # noqa: F841  (alive until the launch)
        _C.check(lib.neosr_attention_fwd(d, _C.stream_ptr()), "neosr_attention_fwd")
    return out, rest, lse


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_mask):
        out, rest, lse = _forward(q, k, v, scale, causal, key_mask, True)
        ctx.save_for_backward(q, k, v, out, rest, lse, key_mask)
        ctx.meta = (scale, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        lib = _C.load()
        q, k, v, out, rest, lse, key_mask = ctx.saved_tensors
        scale, causal = ctx.meta
        g = _heads(g, "grad", q)
        with _on(q.device):
            d = _attention_desc(q, k, v, out, rest, lse, key_mask, scale, causal)
            dq, dk, dv = _dense(q), _dense(k), _dense(v)
            d.dout, d.dq, d.dk, d.dv = _ptr(g), _ptr(dq), _ptr(dk), _ptr(dv)
            d.do_sb, d.do_sl, d.do_sh = g.stride()[:3]
            ws = _workspace(d, lib.neosr_attention_bwd_workspace_bytes(d), q)  # noqa: F841
            _C.check(lib.neosr_attention_bwd(d, _C.stream_ptr()), "neosr_attention_bwd")
        return dq, dk, dv, None, None, None


def attention(q, k, v, *, scale: float | None = None, causal: bool = False, key_mask=None):
    """softmax(scale * q k^T) v.

    q (B, Lq, H, D); k, v (B, Lk, Hk, D) with H a multiple of Hk (query head h reads key head h // (H // Hk)); D from 1 to
    128; any lengths, also 0; any strides (views of a fused projection are read in place).  `scale`: positive (1e-30 to 1e30),
    default D ** -0.5.  `key_mask` (B, Lk) bool: False = the key is not there (its k and v may hold anything, NaN included;
    its gradients are 0).  `causal`: query i sees keys j <= i + Lk - Lq.  A query without a key gives 0.
    Values: any finite number, and infinities as the formula takes them (an infinite v makes its channel infinite, a score of
    minus infinity hides its key, one of plus infinity gives NaN), with three limits.  A row's sums over its keys are formed before
    they are divided, so |v| times the number of keys has to stay below 3.4e38.  0 times infinity or NaN is NaN: what k and v hold
    behind the causal limit must be finite (mask such keys).  And scaled scores are float32, to 2^-24 of their size: their probabilities and
    gradients are off by as much relative (6 % at 1e6), and from 1e9 on the result is not defined.
    bfloat16: the probabilities are rounded to bfloat16 before their product with v, and so are they and the score gradients in the
    backward pass of more than 1024 keys and rows (shorter ones keep twice the bits): 2.3e-3 of the result's norm, of which its own
    rounding is 1.7e-3.  Maxima, sums and accumulators are float32.
    Returns (B, Lq, H, D), dense, in q's type.  First reverse-mode derivatives only.  Bit-reproducible; how sums are split depends on
    the sizes only."""
    q = _heads(q, "q")
    k, v = _heads(k, "k", q), _heads(v, "v", q)
    B, Lq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise _C.NeosrAmdError(f"attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if k.shape[2] == 0 or H == 0 or H % k.shape[2]:
        raise _C.NeosrAmdError(f"attention: {H} query heads are no multiple of {k.shape[2]} key heads")
    if not 1 <= D <= 128:
        raise _C.NeosrAmdError(f"attention: head size {D} (1 to 128)")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise _C.NeosrAmdError(f"attention: scale must be positive, 1e-30 to 1e30 (got {scale})")
    if key_mask is not None:
        key_mask = _tensor(key_mask, "key_mask", 2, q)
        if key_mask.dtype != torch.bool or key_mask.shape != (B, k.shape[1]):
            raise _C.NeosrAmdError(f"attention: key_mask must be bool of shape {(B, k.shape[1])} "
                                   f"(got {key_mask.dtype} {tuple(key_mask.shape)})")
    refuse_tangents("attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return Attention.apply(q, k, v, scale, bool(causal), key_mask)
    return _forward(q, k, v, scale, bool(causal), key_mask, False)[0]


def _rope_call(q, k, positions, sections, theta, interleaved, inverse):
    lib = _C.load()
    B, N, H, D = q.shape
    with _on(q.device):
        qo, ko = _dense(q), None if k is None else _dense(k)
        if q.numel() == 0:
            return qo, ko
        d = _C.RopeDesc(q=_ptr(q), q_out=_ptr(qo), positions=_ptr(positions), theta=theta, B=B, N=N, H=H, D=D,
                        naxes=len(sections), dtype=_DTYPES[q.dtype], pos_kind=_POS_KINDS[positions.dtype],
                        interleaved=int(interleaved), inverse=int(inverse))
        d.q_sb, d.q_sn, d.q_sh = q.stride()[:3]
        if k is not None:
            d.k, d.k_out, d.Hk = _ptr(k), _ptr(ko), k.shape[2]
            d.k_sb, d.k_sn, d.k_sh = k.stride()[:3]
        d.pos_sb, d.pos_sn, d.pos_sa = (0, *positions.stride()) if positions.dim() == 2 else positions.stride()
        for i, s in enumerate(sections):
            d.sections[i] = s
        _C.check(lib.neosr_axial_rope(d, _C.stream_ptr()), "neosr_axial_rope")
    return qo, ko


class AxialRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, theta, interleaved):
        ctx.save_for_backward(positions)
        ctx.meta = (sections, theta, interleaved)
        qo, ko = _rope_call(q, k, positions, sections, theta, interleaved, False)
        return qo if k is None else (qo, ko)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk=None):
        (positions,) = ctx.saved_tensors
        gq = _heads(gq, "grad")
        gk = None if gk is None else _heads(gk, "grad", gq)
        return (*_rope_call(gq, gk, positions, *ctx.meta, True), None, None, None, None)


def axial_rope(q, k, positions, sections, *, theta: float = 10000.0, interleaved: bool = False):
    """Rotary positions with one section of the head for each axis: channels come as `sections` = (time, height, width, ...)
    (even sizes, up to four, together at most D; what is left over passes through), and pair j of section a turns by
    positions[..., a] * theta ** (-2 j / sections[a]).  A section's pairs are its channels (j, j + size / 2), or
    (2 j, 2 j + 1) with `interleaved`.

    q (B, N, H, D) and k (B, N, Hk, D) or None, any strides, D up to 256; positions (N, axes) or (B, N, axes), float32 /
    int32 / int64, any size: angles are formed in 64 bits and off by 2^-52 of their own size.  Returns dense (q, k) — q alone
    when k is None — in q's type; the gradient is the turn by the negative angle (none for the positions; reverse mode only)."""
    q = _heads(q, "q")
    if k is not None:
        k = _heads(k, "k", q)
        if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or k.shape[2] == 0:
            raise _C.NeosrAmdError(f"axial_rope: k {tuple(k.shape)} does not fit q {tuple(q.shape)}")
    B, N, H, D = q.shape
    if H == 0 or not 1 <= D <= 256:
        raise _C.NeosrAmdError(f"axial_rope: {H} heads of size {D} (size 1 to 256)")
    sections = tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= 4 or any(s < 0 or s % 2 for s in sections) or sum(sections) > D:
        raise _C.NeosrAmdError(f"axial_rope: sections {sections} must be one to four even sizes, together at most {D}")
    theta = float(theta)
    if not (theta > 1.0 and math.isfinite(theta)):
        raise _C.NeosrAmdError(f"axial_rope: theta must be above 1 (got {theta})")
    if not isinstance(positions, torch.Tensor) or positions.dim() not in (2, 3):
        raise _C.NeosrAmdError("axial_rope: positions must be a (N, axes) or (B, N, axes) tensor")
    _tensor(positions, "positions", positions.dim(), q)
    if positions.dtype not in _POS_KINDS:
        raise _C.NeosrAmdError(f"axial_rope: positions must be float32, int32 or int64 (got {positions.dtype})")
    want = (N, len(sections)) if positions.dim() == 2 else (B, N, len(sections))
    if tuple(positions.shape) != want:
        raise _C.NeosrAmdError(f"axial_rope: positions {tuple(positions.shape)}, expected {want}")
    refuse_tangents("axial_rope", q, k, positions)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return AxialRope.apply(q, k, positions.detach(), sections, theta, bool(interleaved))
    qo, ko = _rope_call(q, k, positions, sections, theta, bool(interleaved), False)
    return qo if k is None else (qo, ko)
