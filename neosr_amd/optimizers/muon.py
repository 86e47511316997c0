"""`muon`: orthogonalised momentum for the weight matrices of a network, AdamW for the rest, on flat HBM arenas.

`optim_g.type = "muon"` (or `optim_d`).  A parameter is a matrix when it has 2 or 4 dimensions and, as (out, everything else),
no side below `min_side` (and no more than `newton_schulz` takes: 2^29 elements): Linear weights and convolution kernels; bias
tables, norms, biases, position embeddings and the 3-channel ends of a network take the AdamW update in the same step.  The
orthogonalised update is scaled by rms * sqrt(max(rows, cols)), i.e. to an RMS of about `rms` per element — that of an AdamW
update — so ONE learning rate, its schedule and warm-up, and one weight decay serve both kinds.  Clip, gradient scale and EMA are
fused as in the other optimizers; a step cannot be captured into a HIP graph.  `state[p] = {exp_avg, exp_avg_sq}` are views into
flat arenas and round-trip through `.state` files.
"""

from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from neosr_amd import _C
from neosr_amd.hip.nets import arena_layout, flat_grad_of, pack_grads
from neosr_amd.optimizers.extra import _check_basic, _FlatOptimizer
from neosr_amd.optimizers.orthogonal import COEFFICIENTS, coefficient_table, too_large

CHUNK = 4096


class muon(_FlatOptimizer):
    ARENAS = ("exp_avg", "exp_avg_sq")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, momentum=0.95, nesterov=True, ns_steps=5,
                 ns_coefficients=COEFFICIENTS, rms=0.2, min_side=16, **kwargs):  # noqa: ARG002
        _check_basic(lr, eps, betas)
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"Invalid momentum: {momentum}")
        if not rms > 0.0:
            raise ValueError(f"Invalid rms: {rms}")
        if min_side < 1:
            raise ValueError(f"Invalid min_side: {min_side}")
        coefficient_table(ns_steps, ns_coefficients)   # (raises on bad steps / coefficients)
        self._init_common(params, {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay, "momentum": momentum,
                                   "nesterov": nesterov, "ns_steps": ns_steps, "ns_coefficients": ns_coefficients, "rms": rms,
                                   "min_side": min_side})

    @staticmethod
    def matrix_shape(p, min_side: int):
        """(rows, cols) of a parameter that gets orthogonalised updates, else None"""
        if p.dim() not in (2, 4) or p.numel() == 0:
            return None
        rows = p.shape[0]
        cols = p.numel() // rows
        return (rows, cols) if min_side <= min(rows, cols) and not too_large(rows, cols) else None

    def _plan(self, st, group, params):
        """chunk table (device), matrices [(offset, rows, cols)] of a group: laid out once, kept with its state"""
        key = (group["rms"], group["min_side"])
        if st.get("plan_key") != key or st.get("plan_params") is not params:
            mats, chunks = [], ([], [])
            for p, off in zip(params, arena_layout(params)[0]):
                shape = self.matrix_shape(p, group["min_side"])
                scale = group["rms"] * math.sqrt(max(shape)) if shape else 0.0
                bits = struct.unpack("<i", struct.pack("<f", scale))[0]
                if shape:
                    mats.append((off, *shape))
                chunks[0 if shape else 1].extend(((off + s) // 4, min(CHUNK, p.numel() - s), int(shape is not None), bits)
                                                 for s in range(0, p.numel(), CHUNK))
            st["mats"], st["nmatrix"] = mats, len(chunks[0])
            st["chunks"] = torch.tensor(chunks[0] + chunks[1], dtype=torch.int32).to(params[0].device)
            st["plan_key"], st["plan_params"] = key, params
        return st["mats"], st["chunks"], st["nmatrix"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = 0.0
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _C.load()
        for gi, group in enumerate(self.param_groups):
            pflat, params = self._group_arena(group)
            if pflat is None:
                raise _C.NeosrAmdError("neosr_amd.muon needs the parameter group in one flat arena "
                                       "(call flatten_parameters_ before building it)")
            _C.require_device(pflat, "parameter arena")
            if torch.cuda.is_current_stream_capturing():
                raise _C.NeosrAmdError("muon: a step cannot be captured into a graph (learning rate and bias corrections are numbers "
                                       "of the call, which a replay would repeat)")
            gflat = flat_grad_of(params)
            if gflat is None:
                gflat = pack_grads(params)
            total = pflat.numel()
            st = self._ensure_state(gi, params, total)
            mats, chunks, nmatrix = self._plan(st, group, params)
            t = group.get("step", 0) + 1
            if self._norm_ws is None or self._norm_ws.device != pflat.device:
                self._norm_ws = torch.zeros(4200, device=pflat.device, dtype=torch.float32)
            b1, b2 = group["betas"]
            d = _C.MuonDesc(param=pflat.data_ptr(), grad=gflat.data_ptr(), exp_avg=st["exp_avg"].data_ptr(),
                            exp_avg_sq=st["exp_avg_sq"].data_ptr(), norm_ws=self._norm_ws.data_ptr(), chunks=chunks.data_ptr(),
                            n=total, nchunks=chunks.shape[0], nmatrix=nmatrix, nitems=len(mats), ns_steps=group["ns_steps"],
                            nesterov=int(group["nesterov"]), lr=group["lr"], momentum=group["momentum"], beta1=b1, beta2=b2,
                            eps=group["eps"], weight_decay=group["weight_decay"], bias_correction1=1.0 - b1**t,
                            bias_correction2_sqrt=math.sqrt(1.0 - b2**t), ns_eps=1e-7, max_norm=self._pending_clip,
                            grad_scale=self._grad_scale)
            if mats:
                update = torch.empty(total, device=pflat.device, dtype=torch.float32)
                base = update.data_ptr()
                items = (_C.NsItem * len(mats))(*[
                    _C.NsItem(in_=base + 4 * off, out=base + 4 * off, in_sr=c, out_sr=c, count=1, rows=r, cols=c)
                    for off, r, c in mats])
                nbytes = lib.neosr_newton_schulz_workspace_bytes(items, len(mats), _C.DT_F32)
                if nbytes < 0:
                    _C.check(1, "neosr_newton_schulz_workspace_bytes")
                ws = torch.empty(nbytes, device=pflat.device, dtype=torch.uint8)
                table = coefficient_table(group["ns_steps"], group["ns_coefficients"])
                d.update, d.workspace, d.workspace_bytes = base, ws.data_ptr(), nbytes
                d.items, d.coefficients = items, C.cast(table, C.POINTER(C.c_float))
            if self._ema is not None and len(self.param_groups) == 1:
                ema_arena, decay, first = self._ema
                if ema_arena.numel() != total:
                    raise _C.NeosrAmdError("EMA arena size does not match the parameter arena")
                d.ema = ema_arena.data_ptr()
                d.ema_decay = -1.0 if first else decay
            _C.check(lib.neosr_muon_step(C.byref(d), _C.stream_ptr()), "neosr_muon_step")
            group["step"] = t                      # (a refused call is no step)
            _C.params_changed()
            if self._pending_clip > 0:
                self.last_grad_norm = self._norm_ws[0]
        self._pending_clip = 0.0
        self._ema = None
        return loss
