"""Whole-sequence attention and axial rotary positions (`neosr_amd.hip.attention`) against their definitions in 64 bits.

Tolerances are element-wise bounds worked out from the arithmetic, before the first run:

* a product of n terms accumulated in fp32 is off by at most (n + 8) 2^-24 of the sum of the terms' sizes (the +8: the six-term
  operand split and the scaling), so the scaled scores by e_s = (D + 8) 2^-24 scale |q| |k|, their base-2 exponents by another
  2^-24 |s log2 e| and 2 units of the exponential: a probability (numerator and row sum) by 2 e relative, e = e_s + 2^-23 |s| + 2^-22;
* bf16: P and dS are rounded once (2^-8 of the value, finfo(bf16).eps / 2) before the second product, outputs once more.
"""

from __future__ import annotations

import math

import pytest
import torch

from neosr_amd import _C

EPS = 2.0 ** -24
U = {torch.float32: EPS, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}
DEV = "cuda"


def _ops():
    from neosr_amd.hip.attention import attention, axial_rope

    return attention, axial_rope


# ------------------------------------------------------------------------------------------------- attention


def _reference(q, k, v, dout, scale, causal, key_mask):
    """values and element-wise error bounds of (out, dq, dk, dv), all 64-bit, heads expanded to the query's"""
    dt = q.dtype
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = H // Hk
    u = U[dt] if dt != torch.float32 else 0.0          # operand rounding of P, dS
    uo = U[dt]                                         # output rounding

    def hf(x):
        return x.double().permute(0, 2, 1, 3)

    ok = torch.ones(B, 1, Lq, Lk, dtype=torch.bool, device=q.device)
    if causal:
        ok &= torch.arange(Lk, device=q.device)[None] <= torch.arange(Lq, device=q.device)[:, None] + (Lk - Lq)
    if key_mask is not None:
        ok &= key_mask[:, None, None, :]
        gone = ~key_mask[:, :, None, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    Q, K, V = hf(q), hf(k).repeat_interleave(G, 1), hf(v).repeat_interleave(G, 1)
    Kt, Vt = K.transpose(2, 3).contiguous(), V.transpose(2, 3).contiguous()
    S = Q @ Kt * scale
    es = (D + 8) * EPS * (Q.abs() @ Kt.abs()) * scale + 2 ** -23 * S.abs() + 2 ** -22
    es = es.masked_fill(~ok, 0.0)
    S = S.masked_fill(~ok, -math.inf)
    P = torch.softmax(S, -1).nan_to_num(0.0) if Lk else S
    ep = P * (es + (P * es).sum(-1, keepdim=True) + 2 * (Lk + 8) * EPS)     # the probability's own error
    O = P @ V
    eO = (ep + u * P) @ V.abs() + (Lk + 8) * EPS * (P @ V.abs()) + uo * O.abs()
    res, bound = [O], [eO]
    if dout is not None:
        dO = hf(dout)
        dP = dO @ Vt
        edP = (D + 8) * EPS * (dO.abs() @ Vt.abs())
        delta = (dO * O).sum(-1, keepdim=True)
        edelta = (dO.abs() * eO).sum(-1, keepdim=True) + (D + 8) * EPS * (dO.abs() * O.abs()).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        edS = ep * (dP - delta).abs() + P * (edP + edelta) + 4 * EPS * P * (dP.abs() + delta.abs()) + u * dS.abs()
        Pt, dSt, ePt, edSt = (x.transpose(2, 3).contiguous() for x in (P, dS, ep + u * P, edS))
        dQ, dK, dV = dS @ K * scale, dSt @ Q * scale, Pt @ dO
        eQ = (edS @ K.abs() + (Lk + 8) * EPS * (dS.abs() @ K.abs())) * scale
        eK = (edSt @ Q.abs() + (Lq * G + 8) * EPS * (dSt.abs() @ Q.abs())) * scale
        eV = ePt @ dO.abs() + (Lq * G + 8) * EPS * (Pt @ dO.abs())
        fold = lambda x: x.reshape(B, Hk, G, Lk, D).sum(2)  # noqa: E731
        dK, dV, eK, eV = fold(dK), fold(dV), fold(eK), fold(eV)
        res += [dQ, dK, dV]
        bound += [eQ + uo * dQ.abs(), eK + uo * dK.abs(), eV + uo * dV.abs()]
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    return [back(x) for x in res], [back(x) for x in bound]


def _check(got, want, bound):
    for name, g, w, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert g.shape == w.shape and g.is_contiguous()
        assert torch.isfinite(g).all(), name
        over = (g.double() - w).abs() - (b + 1e-30)
        assert over.numel() == 0 or float(over.max()) <= 0, \
            f"{name}: off by {float((g.double() - w).abs().max()):.3e}, {float(over.max()):.3e} beyond its bound"


def _inputs(dt, B, Lq, Lk, H, Hk, D, seed=0, layout="fused"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)  # noqa: E731
    if layout == "fused" and Lq == Lk:
        x = rn(B, Lq, H + 2 * Hk, D)
        q, k, v = x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:]
    elif layout == "heads_first":
        q, k, v = (rn(B, n, L, D).transpose(1, 2) for n, L in ((H, Lq), (Hk, Lk), (Hk, Lk)))
    else:
        q, k, v = rn(B, Lq, H, D), rn(B, Lk, Hk, D), rn(B, Lk, Hk, D)
    return q, k, v, rn(B, Lq, H, D)


def _run(q, k, v, dout, **kw):
    attention, _ = _ops()
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(q, k, v, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


CASES = [
    # B, Lq, Lk, H, Hk, D, causal
    (1, 1, 1, 1, 1, 1, False), (2, 1, 5, 2, 1, 7, False), (1, 2, 2, 3, 3, 8, True), (2, 31, 33, 2, 2, 30, False),
    (1, 64, 64, 6, 6, 30, False), (2, 65, 63, 4, 2, 32, True), (1, 63, 65, 4, 2, 33, True), (1, 127, 300, 3, 1, 50, False),
    (2, 130, 130, 2, 1, 64, True), (1, 96, 200, 4, 1, 96, False), (1, 33, 129, 2, 2, 127, False), (2, 70, 70, 4, 4, 128, True),
    (1, 200, 3, 6, 2, 16, True), (1, 5, 1000, 8, 2, 64, False), (1, 700, 9, 2, 2, 60, False), (3, 1, 2050, 6, 6, 30, False),
    (1, 2050, 40, 1, 1, 24, True), (1, 3, 777, 4, 1, 128, True), (40, 130, 140, 8, 8, 30, False), (16, 300, 70, 16, 4, 64, False),
    (8, 260, 130, 16, 16, 40, True), (6, 260, 140, 24, 12, 128, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_attention_and_gradients(case, dt):
    B, Lq, Lk, H, Hk, D, causal = case
    q, k, v, dout = _inputs(dt, B, Lq, Lk, H, Hk, D, seed=Lq * 7 + Lk)
    got = _run(q, k, v, dout, causal=causal)
    _check(got, *_reference(q, k, v, dout, D ** -0.5, causal, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["plain", "fused", "heads_first"])
@pytest.mark.parametrize("D", [30, 31, 64])
def test_attention_layouts_and_scale(layout, D, dt):
    q, k, v, dout = _inputs(dt, 2, 90, 90, 6, 2, D, seed=3, layout=layout)
    dout = dout.transpose(1, 2).contiguous().transpose(1, 2)            # strided gradient too
    got = _run(q, k, v, dout, scale=0.31)
    _check(got, *_reference(q, k, v, dout, 0.31, False, None))


MASKS = ["all", "none", "one_empty_sample", "single_key", "holes", "ragged", "first_tile_empty"]


def _mask(kind, B, Lk, g):
    m = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)
    if kind == "all":
        m[:] = True
    elif kind == "one_empty_sample":
        m[1:] = True
    elif kind == "single_key":
        m[torch.arange(B), torch.randint(0, Lk, (B,), generator=g, device=DEV)] = True
    elif kind == "holes":
        m = torch.rand(B, Lk, generator=g, device=DEV) < 0.4
    elif kind == "ragged":
        m = torch.arange(Lk, device=DEV)[None] < torch.randint(1, Lk + 1, (B, 1), generator=g, device=DEV)
    elif kind == "first_tile_empty":
        m[:, 64:] = True
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", MASKS)
def test_masked_keys_hold_anything(kind, causal, dt):
    """rows without a key give 0 and no gradient; what masked keys hold (NaN, infinities, the lowest value) is never used"""
    B, Lq, Lk, H, Hk, D = 3, 75, 130, 4, 2, 30
    g = torch.Generator(device=DEV).manual_seed(MASKS.index(kind))
    q, k, v, dout = _inputs(dt, B, Lq, Lk, H, Hk, D, seed=11)
    m = _mask(kind, B, Lk, g)
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min], device=DEV).to(dt)
    junk = junk[torch.arange(Lk, device=DEV) % 4][None, :, None, None].expand_as(k)
    k, v = torch.where(m[:, :, None, None], k, junk), torch.where(m[:, :, None, None], v, junk)
    got = _run(q, k, v, dout, causal=causal, key_mask=m)
    want, bound = _reference(q, k, v, dout, D ** -0.5, causal, m)
    _check(got, want, bound)
    assert (got[2][~m] == 0).all() and (got[3][~m] == 0).all()
    if kind == "none":
        assert all((x == 0).all() for x in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_mask_with_split_keys_and_strided_mask(dt):
    """few rows over many keys (the keys are split and joined), splits that are empty, a mask that is a strided view"""
    B, Lq, Lk, H, Hk, D = 2, 4, 1500, 2, 1, 48
    q, k, v, dout = _inputs(dt, B, Lq, Lk, H, Hk, D, seed=5)
    m = torch.zeros(Lk, B, dtype=torch.bool, device=DEV)
    m[700:760, 0] = True
    m[::3, 1] = True
    got = _run(q, k, v, dout, key_mask=m.t())
    _check(got, *_reference(q, k, v, dout, D ** -0.5, False, m.t()))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(0, 4, 4, 2, 1, 8), (2, 0, 4, 2, 1, 8), (2, 4, 0, 2, 1, 8)])
def test_lengths_of_zero(shape, dt):
    q, k, v, dout = _inputs(dt, *shape, layout="plain")
    out, dq, dk, dv = _run(q, k, v, dout)
    for t in (out, dq, dk, dv):
        assert t.numel() == 0 or (t == 0).all()
    assert out.shape == q.shape and dk.shape == k.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [3, 300])
def test_rows_without_a_key_pass_no_gradient_whatever_dout_holds(Lq, dt):
    q, k, v, dout = _inputs(dt, 2, Lq, 40, 4, 2, 24, seed=8)
    m = torch.ones(2, 40, dtype=torch.bool, device=DEV)
    m[1] = False
    dout[1] = math.nan
    got = _run(q, k, v, dout, key_mask=m)
    _check([x[:1] for x in got], *[[y[:1] for y in z] for z in _reference(q, k, v, dout.nan_to_num(0.0), 24 ** -0.5, False, m)])
    assert all((x[1] == 0).all() for x in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_broadcast_and_misaligned_operands(dt):
    """keys shared by the batch and by the heads (stride 0), channel slices that start at an odd element, a gradient of one
    number expanded over the output"""
    g = torch.Generator(device=DEV).manual_seed(31)
    q = torch.randn(2, 70, 4, 33, generator=g, device=DEV).to(dt)[..., 1:]
    k = torch.randn(1, 90, 1, 35, generator=g, device=DEV).to(dt)[..., 3:].expand(2, 90, 2, 32)
    v = torch.randn(1, 90, 2, 32, generator=g, device=DEV).to(dt).expand(2, 90, 2, 32)
    dout = torch.full((1,), 0.37, device=DEV).to(dt).expand(2, 70, 4, 32)
    _check(_run(q, k, v, dout), *_reference(q, k, v, dout, 32 ** -0.5, False, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [5, 200])
def test_offsets_beyond_32_bits(Lq, dt):
    """rows 2^24 elements apart: the last of 200 keys lies 3.3 * 10^9 elements into its buffer"""
    attention, axial_rope = _ops()
    step, L, D = 1 << 24, 200, 16
    store = torch.empty(step * L, device=DEV, dtype=dt)
    g = torch.Generator(device=DEV).manual_seed(2)
    far = store.as_strided((1, L, 3, D), (step * L, step, D, 1))
    near = torch.randn(1, L, 3, D, generator=g, device=DEV).to(dt)
    far.copy_(near)
    q = torch.randn(1, Lq, 1, D, generator=g, device=DEV).to(dt)
    dout = torch.randn(1, Lq, 1, D, generator=g, device=DEV).to(dt)
    a = _run(q, far[:, :, :1], far[:, :, 1:2], dout)
    b = _run(q, near[:, :, :1], near[:, :, 1:2], dout)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    pos = torch.arange(L, device=DEV)[:, None]
    assert torch.equal(axial_rope(far, None, pos, (16,)), axial_rope(near, None, pos, (16,)))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    attention, axial_rope = _ops()
    q, k, v, dout = _inputs(torch.float32, 1, 8, 8, 1, 1, 8, layout="plain")
    q.requires_grad_(True)
    for out in (attention(q, k, v), axial_rope(q, None, torch.zeros(8, 1, device=DEV), (8,))):
        (g,) = torch.autograd.grad(out, q, dout.clone().requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.gpu
def test_two_streams_at_once():
    """calls on two streams side by side, each with its own workspace"""
    a = _inputs(torch.bfloat16, 2, 500, 900, 4, 2, 64, seed=41)
    b = _inputs(torch.float32, 2, 400, 700, 4, 2, 30, seed=42)
    want = [_run(*a), _run(*b)]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                got[i].append(_run(*x))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(x, y) for r in runs for x, y in zip(w, r))


@pytest.mark.gpu
def test_large_scores_keep_the_row_maximum():
    """scores of several hundred: the running maximum, not the exponent's range, carries the softmax"""
    q, k, v, dout = _inputs(torch.float32, 1, 70, 200, 2, 2, 32, seed=9, layout="plain")
    q, k = q * 6, k * 6
    got = _run(q, k, v, dout)
    _check(got, *_reference(q, k, v, dout, 32 ** -0.5, False, None))


@pytest.mark.gpu
def test_gradient_against_differences():
    attention, _ = _ops()
    q, k, v, dout = _inputs(torch.float32, 1, 37, 45, 2, 1, 24, seed=13, layout="plain")
    grads = _run(q, k, v, dout, causal=True)[1:]
    g = torch.Generator(device=DEV).manual_seed(1)
    for i, x in enumerate((q, k, v)):
        dirn = torch.randn(x.shape, generator=g, device=DEV)
        h = 2.0 ** -6
        args = [[q, k, v], [q, k, v]]
        args[0][i], args[1][i] = x + h * dirn, x - h * dirn
        f = [(attention(*a, causal=True).double() * dout.double()).sum() for a in args]
        num, ana = float((f[0] - f[1]) / (2 * h)), float((grads[i].double() * dirn.double()).sum())
        # truncation h^2 / 6 of a third derivative of size ~|grad| |dirn|, rounding 2^-24 |f| sqrt(n) / h
        scale = float(grads[i].double().norm() * dirn.double().norm())
        assert abs(num - ana) <= 2e-3 * scale, (i, num, ana, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_bits_repeat_and_other_stream(dt):
    q, k, v, dout = _inputs(dt, 2, 300, 1000, 4, 2, 40, seed=21)
    a = _run(q, k, v, dout)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = _run(q, k, v, dout)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_rope_attention_gradient_in_a_graph(dt):
    """the operators as they are used together — turn, attend, both gradients — captured once and replayed on new inputs"""
    attention, axial_rope = _ops()
    B, grid, H, Hk, D = 2, (9, 13), 4, 2, 32
    N = grid[0] * grid[1]
    x, dout = torch.empty(B, N, H + 2 * Hk, D, device=DEV, dtype=dt), torch.empty(B, N, H, D, device=DEV, dtype=dt)
    pos = torch.stack(torch.meshgrid(*[torch.arange(n, device=DEV) for n in grid], indexing="ij"), -1).reshape(N, 2)
    mask = torch.arange(N, device=DEV)[None] < torch.tensor([[N], [N - 40]], device=DEV)
    x.requires_grad_(True)

    def step():
        q, k, v = x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:]
        q, k = axial_rope(q, k, pos, (16, 16))
        out = attention(q, k, v, key_mask=mask)
        return out.detach(), torch.autograd.grad(out, x, dout)[0]

    def load(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            dout.copy_(torch.randn(dout.shape, generator=g, device=DEV))

    load(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        load(seed)
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in captured]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), seed


# ------------------------------------------------------------------------------------------------- axial_rope


def _rope_reference(x, positions, sections, theta, interleaved, sign):
    y, size, base = x.double().clone(), torch.zeros_like(x, dtype=torch.float64), 0
    pos = positions if positions.dim() == 3 else positions[None]
    size += x.double().abs() * 0
    for a, sec in enumerate(sections):
        for j in range(sec // 2):
            i0, i1 = (base + 2 * j, base + 2 * j + 1) if interleaved else (base + j, base + j + sec // 2)
            ang = pos[:, :, a].double() * theta ** (-2.0 * j / sec)
            c, s = ang.cos()[:, :, None], sign * ang.sin()[:, :, None]
            u, v = x[..., i0].double(), x[..., i1].double()
            y[..., i0], y[..., i1] = u * c - v * s, u * s + v * c
            size[..., i0] = size[..., i1] = u.abs() + v.abs()
        base += sec
    return y, size


def _rope_check(got, x, *args):
    """table entries are within 1.25 * 2^-23 (2 units of sincospi below 1, the reduced angle's rounding at 1/8 turn), the two
    products and their sum within 2 * 2^-24: 2.5 * 2^-23 of |x| + |y|, and the output's rounding.  64-bit angles of positions to
    10^6 are good to 1e-9."""
    want, size = _rope_reference(x, *args)
    bound = 2.5 * 2 ** -23 * size + (U[x.dtype] * want.abs() if x.dtype != torch.float32 else 0) + 2e-9 * size
    over = ((got.double() - want).abs() - bound).max()
    assert float(over) <= 0, float(over)
    assert got.is_contiguous() and got.shape == x.shape


ROPE = [
    # B, N, H, Hk, D, sections, positions
    (1, 1, 1, 1, 2, (2,), "int"), (2, 37, 6, 6, 30, (14, 14), "float"), (1, 64, 8, 2, 64, (16, 24, 24), "int"),
    (3, 50, 4, 1, 33, (10, 2, 12, 8), "batch"), (2, 9, 3, 3, 128, (64, 64), "far"), (1, 17, 2, 1, 256, (128, 128), "float"),
    (2, 1500, 2, 1, 31, (16, 14), "far"), (1, 40, 64, 64, 255, (0, 254), "int"), (2, 21, 5, 2, 20, (4, 6), "negative"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "x".join(map(str, c[:5])) + "_" + c[6])
def test_axial_rope_and_gradients(case, interleaved, dt):
    _, axial_rope = _ops()
    B, N, H, Hk, D, sections, kind = case
    g = torch.Generator(device=DEV).manual_seed(N)
    qk = torch.randn(B, N, H + Hk, D, generator=g, device=DEV).to(dt)
    q, k = qk[:, :, :H].detach().requires_grad_(True), qk[:, :, H:].detach().requires_grad_(True)
    A = len(sections)
    pos = {"int": lambda: torch.randint(0, 300, (N, A), generator=g, device=DEV),
           "float": lambda: torch.rand(N, A, generator=g, device=DEV) * 100,
           "batch": lambda: torch.randint(0, 300, (B, N, A), generator=g, device=DEV, dtype=torch.int32),
           "far": lambda: torch.randint(900_000, 1_000_000, (A, N), generator=g, device=DEV).t(),
           "negative": lambda: torch.rand(B, N, A, generator=g, device=DEV) * 50 - 25}[kind]()
    qo, ko = axial_rope(q, k, pos, sections, interleaved=interleaved)
    dq, dk = (torch.randn(t.shape, generator=g, device=DEV).to(dt) for t in (q, k))
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for got, x, sign in ((qo, q, 1.0), (ko, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        _rope_check(got.detach(), x.detach(), pos, sections, 10000.0, interleaved, sign)
    if D > sum(sections):
        assert torch.equal(qo[..., sum(sections):], q[..., sum(sections):])
    only = axial_rope(q.detach(), None, pos, sections, interleaved=interleaved)
    assert torch.equal(only, qo)


@pytest.mark.gpu
def test_axial_rope_layouts_theta_and_empty():
    _, axial_rope = _ops()
    x = torch.randn(2, 4, 50, 30, device=DEV).transpose(1, 2)          # heads first
    pos = torch.arange(50, device=DEV)[:, None].expand(50, 2)
    _rope_check(axial_rope(x, None, pos, (14, 14), theta=100.0), x, pos, (14, 14), 100.0, False, 1.0)
    y = torch.randn(2, 50, 30, 4, device=DEV).transpose(2, 3)          # channels are not the last in memory
    _rope_check(axial_rope(y, None, pos, (14, 16), interleaved=True), y, pos, (14, 16), 10000.0, True, 1.0)
    q, k = axial_rope(torch.empty(0, 5, 2, 8, device=DEV), torch.empty(0, 5, 1, 8, device=DEV), torch.zeros(5, 1, device=DEV), (8,))
    assert q.shape == (0, 5, 2, 8) and k.shape == (0, 5, 1, 8)


# ------------------------------------------------------------------------------------------------- refusals


def _desc(**kw):
    d = _C.AttentionDesc(q=16, k=16, v=16, out=16, lse=16, B=1, Lq=4, Lk=4, H=2, Hk=1, D=8, dtype=_C.DT_F32, scale=1.0,
                         dout=16, dq=16, dk=16, dv=16)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("bad", [dict(D=0), dict(D=129), dict(H=3, Hk=2), dict(Hk=0), dict(dtype=7), dict(scale=0.0),
                                 dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-38), dict(scale=3e38), dict(out_rest=24), dict(q=None), dict(k=None),
                                 dict(out=None), dict(out=20), dict(q=18), dict(B=-1), dict(Lk=2 ** 30)])
def test_c_entry_refuses(bad):
    """refused on the host, before anything is launched"""
    lib = _C.load()
    assert lib.neosr_attention_fwd(_desc(**bad), None) != 0
    assert lib.neosr_attention_fwd_workspace_bytes(_desc(**bad)) == -1
    assert lib.neosr_attention_bwd(_desc(**bad), None) != 0
    assert lib.neosr_last_error()


def test_descriptor_sizes_match_c_layout(tmp_path):
    import ctypes as C
    import subprocess

    from tests.conftest import ROOT

    names = {"neosr_attention_desc": _C.AttentionDesc, "neosr_rope_desc": _C.RopeDesc, "neosr_ns_item": _C.NsItem,
             "neosr_muon_desc": _C.MuonDesc}
    src = tmp_path / "probe.c"
    src.write_text('#include "neosr_amd.h"\n#include <stdio.h>\nint main(){' +
                   "".join(f'printf("%zu\\n",sizeof({n}));' for n in names) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    sizes = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split()
    assert [C.sizeof(t) for t in names.values()] == [int(v) for v in sizes]


def test_c_entry_refuses_missing_workspace():
    lib = _C.load()
    d = _desc(Lk=4096)
    assert lib.neosr_attention_fwd_workspace_bytes(d) > 0
    assert lib.neosr_attention_fwd(d, None) != 0 and b"workspace" in lib.neosr_last_error()
    assert lib.neosr_attention_bwd_workspace_bytes(d) > 0
    assert lib.neosr_attention_bwd(d, None) != 0 and b"workspace" in lib.neosr_last_error()


@pytest.mark.parametrize("bad", [dict(D=257), dict(D=0), dict(naxes=0), dict(naxes=5), dict(sections=(3, 4)), dict(sections=(8, 8)),
                                 dict(theta=1.0), dict(theta=math.nan), dict(dtype=3), dict(pos_kind=3), dict(k=16), dict(q=None),
                                 dict(positions=None), dict(H=0)])
def test_c_rope_refuses(bad):
    d = _C.RopeDesc(q=16, q_out=16, positions=16, theta=100.0, B=1, N=4, H=1, D=8, naxes=2)
    d.sections[0] = d.sections[1] = 4
    for n, x in bad.items():
        if n == "sections":
            d.sections[0], d.sections[1] = x
        else:
            setattr(d, n, x)
    lib = _C.load()
    assert lib.neosr_axial_rope(d, None) != 0 and lib.neosr_last_error()


def test_cpu_tensors_are_refused():
    attention, axial_rope = _ops()
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(_C.NeosrAmdError):
        attention(x, x, x)
    with pytest.raises(_C.NeosrAmdError):
        axial_rope(x, x, torch.zeros(4, 1), (8,))


@pytest.mark.gpu
def test_python_refusals():
    attention, axial_rope = _ops()
    x = torch.zeros(2, 4, 2, 8, device=DEV)
    bad = [lambda: attention(x.half(), x.half(), x.half()), lambda: attention(x, x.bfloat16(), x),
           lambda: attention(x, x[:, :, :, :4], x), lambda: attention(x, x[:1], x[:1]), lambda: attention(x, x, x[:, :3]),
           lambda: attention(torch.zeros(2, 4, 3, 8, device=DEV), x, x), lambda: attention(x, x, x, scale=0.0),
           lambda: attention(x, x, x, scale=math.nan), lambda: attention(x, x, x, key_mask=torch.ones(2, 4, device=DEV)),
           lambda: attention(x, x, x, key_mask=torch.ones(2, 5, device=DEV, dtype=torch.bool)), lambda: attention(x[0], x, x),
           lambda: attention(*(torch.zeros(1, 2, 1, 129, device=DEV),) * 3), lambda: attention(x, x.cpu(), x),
           lambda: axial_rope(x, x, torch.zeros(4, 2, device=DEV), (4,)), lambda: axial_rope(x, x, torch.zeros(4, 1, device=DEV), (3,)),
           lambda: axial_rope(x, x, torch.zeros(4, 2, device=DEV), (8, 2)), lambda: axial_rope(x, x, torch.zeros(4, 1), (4,)),
           lambda: axial_rope(x, x, torch.zeros(4, 1, device=DEV, dtype=torch.float64), (4,)),
           lambda: axial_rope(x, x[:, :3], torch.zeros(4, 1, device=DEV), (4,)), lambda: axial_rope(x, x, torch.zeros(3, 1, device=DEV), (4,)),
           lambda: axial_rope(x, x, torch.zeros(4, 1, device=DEV), (4,), theta=0.5)]
    for i, f in enumerate(bad):
        with pytest.raises(_C.NeosrAmdError):
            f()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------------------------------------- forward mode


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """a dual tensor has requires_grad = False and a readable pointer: without the refusal its tangent would be dropped"""
    import torch.autograd.forward_ad as fwd

    attention, axial_rope = _ops()
    q, k, v, dout = _inputs(torch.float32, 1, 8, 8, 2, 1, 8, layout="plain")
    pos = torch.zeros(8, 1, device=DEV)
    with fwd.dual_level():
        for i in range(3):
            args = [q, k, v]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(_C.NeosrAmdError):
                attention(*args)
        for args in ((fwd.make_dual(q, q), k, pos), (q, fwd.make_dual(k, k), pos), (q, k, fwd.make_dual(pos, pos)),
                     (fwd.make_dual(q, q), None, pos)):
            with pytest.raises(_C.NeosrAmdError):
                axial_rope(*args, (8,))
        inside = attention(q, k, v), axial_rope(q, None, pos, (8,))        # operands without a tangent are calls as any other
        grads = _run(q, k, v, dout)
    assert torch.equal(inside[0], attention(q, k, v)) and torch.equal(inside[1], axial_rope(q, None, pos, (8,)))
    assert all(torch.equal(a, b) for a, b in zip(grads, _run(q, k, v, dout)))


# ------------------------------------------------------------------------------------------------- infinities, fp32's largest values


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", [(1, 5, 90, 2, 1, 30), (8, 150, 200, 4, 4, 30), (8, 150, 200, 4, 4, 64), (8, 150, 200, 4, 4, 100),
                                  (1, 2, 70, 1, 1, 128)], ids=lambda c: "x".join(map(str, c)))
def test_infinite_values(case, dt):
    """a value that is infinite makes its channel of every row that sees the key infinite (a probability above 0 times infinity),
    values of both signs make it NaN, and the other channels and samples are as they were"""
    attention, _ = _ops()
    B, Lq, Lk, H, Hk, D = case
    q, k, v, _ = _inputs(dt, *case, seed=51, layout="plain")
    want = attention(q, k, v)
    w = v.clone()
    w[0, 3, 0, 1] = math.inf
    w[0, Lk - 1, 0, 4] = -math.inf
    w[0, 65, 0, 7], w[0, 2, 0, 7] = math.inf, -math.inf
    got = attention(q, k, w)
    rows = got[0, :, :H // Hk]
    assert (rows[..., 1] == math.inf).all() and (rows[..., 4] == -math.inf).all() and torch.isnan(rows[..., 7]).all()
    keep = torch.ones(B, H, D, dtype=torch.bool, device=DEV)
    keep[0, :H // Hk, [1, 4, 7]] = False
    keep = keep[:, None].expand(B, Lq, H, D)
    assert torch.equal(got[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", [(2, 5, 90, 2, 1, 30), (8, 150, 200, 4, 4, 30), (8, 150, 200, 4, 4, 64)], ids=lambda c: "x".join(map(str, c)))
def test_a_score_of_minus_infinity_hides_its_key(case, dt):
    """the same bits as with the key masked: its probability is exactly 0, everywhere"""
    attention, _ = _ops()
    q, k, v, _ = _inputs(dt, *case, seed=52, layout="plain")
    q[..., 0] = q[..., 0].abs() + 0.5
    m = torch.ones(case[0], case[2], dtype=torch.bool, device=DEV)
    m[:, 66] = m[1, 3] = False
    want = attention(q, k, v, key_mask=m)
    k = k.clone()
    k[..., 0] = torch.where(m[:, :, None], k[..., 0], -math.inf)
    assert torch.equal(attention(q, k, v), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [5, 150])
def test_largest_finite_values(size):
    """fp32 numbers that round to an infinity in bf16 (3.39e38 to 3.403e38) keep all their bits: as the one value of a row, and as
    queries and keys whose scores are ordinary"""
    attention, _ = _ops()
    top = torch.finfo(torch.float32).max
    q, k, v, _ = _inputs(torch.float32, 8, size, 200, 4, 4, 30, seed=53, layout="plain")
    m = torch.zeros(8, 200, dtype=torch.bool, device=DEV)
    m[torch.arange(8), torch.arange(8) * 25] = True
    v[..., 2], v[..., 9], v[..., 11] = top, -top, 3.3965e38
    out = attention(q, k, v, key_mask=m)
    # The one probability is 2^(fma(s, c, -round(s c))) = 1 + d, |d| <= ln 2 * 2^-24 |s c| <= 2^-22 (|s c| < 6), in the row sum as in
    # the product: out = v (1 + d)(1 + e1) / ((1 + d)(1 + e2)) up to the two roundings of the division's reciprocal and product:
    # 4 * 2^-24.  At the top of the range that is an infinity (taken here as 2^128, the number it was rounded from or beyond).
    one = (v * m[:, :, None, None]).double().sum(1, keepdim=True).expand_as(out)
    got = torch.where(out.isinf(), out.sign().double() * 2.0 ** 128, out.double())
    assert ((got - one).abs() <= 4 * EPS * one.abs()).all()
    g = torch.Generator(device=DEV).manual_seed(54)
    v = torch.randn(8, 200, 4, 30, generator=g, device=DEV)
    for L in ((size, 200), (200, size)):                                   # large queries, large keys
        big, low = (torch.randn(8, n, 4, 30, generator=g, device=DEV) for n in L)
        sign = big[..., 3] < 0
        big = big * 0.0
        big[..., 3] = torch.where(sign, -3.3965e38, top)
        low = low * 2.0 ** -27
        args = (big, low, v) if L[1] == 200 else (low, big, v)
        _check([attention(*args, scale=1e-30)], *_reference(*args, None, 1e-30, False, None))


# ------------------------------------------------------------------------------------------------- bf16: size of the errors


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(2, 500, 16, 8, 4, 40, False), (4, 400, 5, 4, 2, 64, False), (2, 1000, 1000, 4, 2, 30, True),
                                  (4, 4, 4096, 8, 4, 64, False), (2, 3, 2100, 4, 4, 128, False), (8, 16, 3000, 4, 4, 30, True),
                                  (2, 1024, 1500, 3, 3, 64, False), (2, 1300, 1024, 4, 4, 128, False)],
                         ids=lambda c: "x".join(map(str, c)))
def test_bf16_gradients_are_off_by_their_rounding_alone(case):
    """Up to 1024 keys or rows.  A bf16 rounding is uniform over a step of 2^-7 of the power of two below the value: a variance of
    2^-14 / 12 of that power's square, and over values spread evenly in their logarithm (mean square 3 / (2 ln 2) of the power's)
    1.53e-3 of their norm; 1.66e-3 over a normal distribution.  A rounding of the summands as well (one piece of P or dS) gives
    sqrt(2) times that, 2.2e-3 to 2.4e-3, and so does a delta from the rounded output over few keys.  The bound lies between; the
    output's own, whose P is rounded, at sqrt(2) times it."""
    B, Lq, Lk, H, Hk, D, causal = case
    q, k, v, dout = _inputs(torch.bfloat16, B, Lq, Lk, H, Hk, D, seed=61)
    got = _run(q, k, v, dout, causal=causal)
    want, _ = _reference(q, k, v, dout, D ** -0.5, causal, None)
    err = [float((g.double() - w).norm() / w.norm()) for g, w in zip(got, want)]
    assert err[0] < 2.7e-3 and max(err[1:]) < 1.9e-3, err


# ------------------------------------------------------------------------------------------------- which kernels a call runs

# B, Lq, Lk, H, Hk, D -> (tiles packed, key splits) of the forward and dQ, row splits of dK and dV
LAYOUTS = {
    # padded batches: packed tiles, split keys; head sizes with and without padding channels, and an odd one
    (8, 333, 577, 4, 4, 50): (True, 5, 3), (8, 333, 577, 4, 4, 64): (True, 5, 3), (8, 333, 577, 4, 4, 30): (True, 5, 3),
    (8, 333, 577, 4, 4, 32): (True, 5, 3), (8, 333, 577, 4, 4, 100): (True, 5, 3), (8, 333, 577, 4, 4, 128): (True, 5, 3),
    (8, 333, 577, 4, 4, 31): (True, 5, 3),
    # more than 1024 rows and keys: single waves; packed, split; packed, one split
    (1, 1100, 1100, 1, 1, 30): (False, 9, 9), (1, 1090, 1300, 1, 1, 64): (False, 7, 9), (1, 1030, 1100, 1, 1, 128): (False, 9, 6),
    (2, 1100, 1100, 4, 2, 30): (True, 6, 12), (2, 1100, 1100, 8, 2, 64): (True, 4, 14), (2, 1100, 1100, 16, 4, 128): (True, 2, 8),
    (16, 1030, 1100, 4, 4, 30): (True, 1, 1), (16, 1100, 1030, 4, 4, 60): (True, 1, 1), (9, 1100, 1040, 8, 8, 128): (True, 1, 1),
    (4, 1100, 1200, 4, 2, 40): (True, 4, 7),
}


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", LAYOUTS, ids=lambda c: "x".join(map(str, c)))
def test_calls_take_the_layout_that_they_are_meant_to_test(case, dt):
    """from the sizes of the workspaces: another rule for layouts must not silently leave kernels without their tests"""
    B, Lq, Lk, H, Hk, D = case
    packed, nk, nr = LAYOUTS[case]
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    np_, dp = (3 if dt == torch.float32 else 1), 32 if D <= 32 else 64 if D <= 64 else 128
    rows = 32 if np_ == 3 and D > 32 else 64
    image = lambda L: up(B * Hk * -(-L // rows) * 2 * np_ * rows * dp * 2)  # noqa: E731
    kv = image(Lk) + up(B * -(-Lk // rows) * 8) if packed else 0
    part = up(nk * B * H * Lq * 4) + up(nk * B * H * Lq * D * 4) if nk > 1 else 0
    d = _desc(B=B, Lq=Lq, Lk=Lk, H=H, Hk=Hk, D=D, dtype=_C.DT_F32 if np_ == 3 else _C.DT_BF16)
    lib = _C.load()
    assert lib.neosr_attention_fwd_workspace_bytes(d) == part + kv
    back = up(B * H * Lq * 4) + (up(nk * B * H * Lq * D * 4) if nk > 1 else 0) + (up(nr * 2 * B * Hk * Lk * D * 4) if nr > 1 else 0)
    assert lib.neosr_attention_bwd_workspace_bytes(d) == back + kv + image(Lq * (H // Hk))


PADDED = [c for c in LAYOUTS if c[1] == 333]


def _with_junk(k, v, m, dt):
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min], device=DEV).to(dt)
    junk = junk[torch.arange(k.shape[1], device=DEV) % 4][None, :, None, None].expand_as(k)
    return torch.where(m[:, :, None, None], k, junk), torch.where(m[:, :, None, None], v, junk)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind,causal", [(k, False) for k in MASKS] + [("ragged", True), ("holes", True), ("one_empty_sample", True)])
@pytest.mark.parametrize("case", PADDED, ids=lambda c: f"D{c[5]}")
def test_masks_through_packed_tiles(case, kind, causal, dt):
    """padded batches of the size that training has: truth words, masked keys in the packed tiles (and in the column of ones behind
    V's channels that sums an fp32 row), tiles skipped between two copies in flight, empty samples and splits"""
    B, Lq, Lk, H, Hk, D = case
    q, k, v, dout = _inputs(dt, *case, seed=71)
    m = _mask(kind, B, Lk, torch.Generator(device=DEV).manual_seed(72))
    k, v = _with_junk(k, v, m, dt)
    got = _run(q, k, v, dout, causal=causal, key_mask=m)
    _check(got, *_reference(q, k, v, dout, D ** -0.5, causal, m))
    assert (got[2][~m] == 0).all() and (got[3][~m] == 0).all()
    none = ~m.any(1)
    assert all((x[none] == 0).all() for x in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", [c for c in LAYOUTS if c[1] > 1024 and c[2] > 1024], ids=lambda c: "x".join(map(str, c)))
def test_long_calls(case, causal, dt):
    """more than 1024 rows and keys: the bf16 backward's one-piece kernels at every width, single waves and packed tiles, split and
    whole, ends inside tiles, a triangle that starts before the first row (fewer keys than rows) or behind it"""
    B, Lq, Lk, H, Hk, D = case
    q, k, v, dout = _inputs(dt, *case, seed=73)
    _check(_run(q, k, v, dout, causal=causal), *_reference(q, k, v, dout, D ** -0.5, causal, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["ragged", "holes", "single_key", "first_tile_empty"])
@pytest.mark.parametrize("case", [(4, 1100, 1200, 4, 2, 40), (2, 1100, 1100, 16, 4, 128)], ids=lambda c: "x".join(map(str, c)))
def test_masks_in_long_calls(case, kind, dt):
    q, k, v, dout = _inputs(dt, *case, seed=74)
    m = _mask(kind, case[0], case[2], torch.Generator(device=DEV).manual_seed(75))
    k, v = _with_junk(k, v, m, dt)
    _check(_run(q, k, v, dout, causal=True, key_mask=m), *_reference(q, k, v, dout, case[5] ** -0.5, True, m))
