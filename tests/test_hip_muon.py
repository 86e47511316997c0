"""`newton_schulz` and the `muon` optimizer against their definitions in 64 bits.

Tolerance of `newton_schulz` (relative, Frobenius), worked out before the first run: a step rounds its fp32-faithful products,
polynomial and stored pieces by about 2 units of 2^-24 of (a + |b| + c) |X|, and a later step amplifies an error by at most
L = max(a, |p'|) = a (p(x) = a x + b x^3 + c x^5 on [0, 1.25], a = 3.4445).  The sum over `steps` is
2 * 2^-24 * (a + |b| + c) * (a^steps - 1) / (a - 1): 2.4e-4 for five steps.  Products short of one bf16 piece (2^-16) would miss
it by two orders of magnitude.  bf16 outputs add half a step, 2^-8."""

from __future__ import annotations

import math

import pytest
import torch

from neosr_amd import _C
from tests.conftest import rel_err

DEV = "cuda"
ABC = (3.4445, -4.7750, 2.0315)


def _tol(steps, coefs=ABC):
    a, b, c = coefs
    return 2 * 2.0 ** -24 * (a + abs(b) + abs(c)) * (a ** steps - 1) / (a - 1)


def _exact(g, steps=5, coefs=ABC, eps=1e-7):
    rows = [coefs] * steps if not isinstance(coefs[0], tuple) else coefs
    x = g.detach().double().cpu()
    x = x / (x.norm() + eps)
    for a, b, c in rows:
        if x.shape[0] <= x.shape[1]:
            m = x @ x.t()
            x = a * x + (b * m + c * m @ m) @ x
        else:
            m = x.t() @ x
            x = a * x + x @ (b * m + c * m @ m)
    return x


def _mats(shapes, dt=torch.float32, seed=0, scale=1e-3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for s in shapes:
        r = max(1, min(s[-2:]) // 4)
        m = torch.matmul(torch.randn(*s[:-1], r, generator=g, device=DEV), torch.randn(*s[:-2], r, s[-1], generator=g, device=DEV))
        out.append((scale * (m / math.sqrt(r) + 0.2 * torch.randn(*s, generator=g, device=DEV))).to(dt))
    return out


def _compare(mats, outs, steps=5, coefs=ABC, eps=1e-7):
    for m, o in zip(mats, outs):
        assert o.shape == m.shape and o.dtype == m.dtype and o.is_contiguous()
        for x, y in zip(m.reshape(-1, *m.shape[-2:]), o.reshape(-1, *m.shape[-2:])):
            want = _exact(x, steps, coefs, eps)
            tol = _tol(steps) + (2 ** -8 if m.dtype == torch.bfloat16 else 0)
            assert rel_err(y, want) <= tol, (tuple(m.shape), rel_err(y, want), tol)


SHAPES = [(1, 1), (1, 50), (50, 1), (3, 576), (27, 180), (32, 32), (33, 31), (64, 64), (65, 200), (180, 180), (540, 180), (180, 360),
          (64, 1620), (128, 127), (513, 640), (700, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_newton_schulz_single(shape, dt):
    from neosr_amd.optimizers import newton_schulz

    (m,) = _mats([shape], dt, seed=shape[0] + shape[1])
    _compare([m], [newton_schulz(m)])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_newton_schulz_list_of_many_shapes(dt):
    """more shapes than one batch of classes holds (32), more items than one launch (40), batches, repeats, empty ones"""
    from neosr_amd.optimizers import newton_schulz

    shapes = [(5 + 3 * i, 40 + i) for i in range(36)] + [(3, 20, 30), (2, 2, 17, 9), (0, 4, 4), (5, 40), (20, 30)] * 3
    mats = _mats(shapes, dt, seed=1)
    outs = newton_schulz(mats)
    assert len(outs) == len(mats)
    _compare([m for m in mats if m.numel()], [o for o, m in zip(outs, mats) if m.numel()])
    alone = newton_schulz(mats[40])
    assert torch.equal(alone, outs[40])      # what else is in the list does not matter
    assert newton_schulz([]) == []


@pytest.mark.gpu
def test_newton_schulz_steps_coefficients_layouts():
    from neosr_amd.optimizers import newton_schulz

    (m,) = _mats([(60, 90)], seed=2)
    for steps in (1, 2, 6):
        _compare([m], [newton_schulz(m, steps=steps)], steps)
    table = [(1.5, -0.5, 0.0)] * 2 + [ABC]
    assert rel_err(newton_schulz(m, steps=3, coefficients=table), _exact(m, 3, table)) <= _tol(3)
    wide = torch.randn(60, 200, device=DEV)[:, 5:95]                     # row stride 200, 4-byte aligned
    _compare([wide], [newton_schulz(wide)])
    flipped = torch.randn(90, 60, device=DEV).t()                        # column-major
    _compare([flipped], [newton_schulz(flipped)])


@pytest.mark.gpu
def test_newton_schulz_extremes():
    """a zero matrix stays 0; sizes whose squares leave fp32's range are normalised; NaN stays in its own matrix"""
    from neosr_amd.optimizers import newton_schulz

    (m,) = _mats([(3, 40, 70)], seed=3)
    m[0] = 0.0
    m[2, 3, 4] = math.nan
    out = newton_schulz(m)
    assert (out[0] == 0).all() and torch.isnan(out[2]).all()
    _compare([m[1]], [out[1]])
    for s in (1e25, 1e-25):
        (x,) = _mats([(40, 70)], seed=4, scale=s)
        _compare([x], [newton_schulz(x, eps=0.0)], eps=0.0)


@pytest.mark.gpu
def test_newton_schulz_graph_and_bits():
    from neosr_amd.optimizers import newton_schulz

    mats = _mats([(4, 90, 60), (33, 500)], seed=5)
    first = newton_schulz(mats)
    assert all(torch.equal(a, b) for a, b in zip(first, newton_schulz(mats)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = newton_schulz(mats)
    for seed in (6, 7, 8):
        for m, n in zip(mats, _mats([(4, 90, 60), (33, 500)], seed=seed)):
            m.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        assert all(torch.equal(a, b) for a, b in zip(got, newton_schulz(mats))), seed


@pytest.mark.gpu
def test_newton_schulz_offsets_beyond_32_bits():
    from neosr_amd.optimizers import newton_schulz

    (m,) = _mats([(130, 40)], seed=9)
    far = torch.empty((1 << 24) * 130, device=DEV).as_strided((130, 40), (1 << 24, 1))
    far.copy_(m)
    assert torch.equal(newton_schulz(far), newton_schulz(m))


@pytest.mark.gpu
def test_newton_schulz_wide_tiles():
    """enough large matrices for the 128-wide tiles (512 of them in a launch), in both orientations, next to a small one"""
    from neosr_amd.optimizers import newton_schulz

    mats = _mats([(8, 1100, 1030), (4, 600, 2100), (4, 2100, 600), (50, 70)], seed=12)
    outs = newton_schulz(mats)
    _compare([m[:1] if m.dim() == 3 else m for m in mats], [o[:1] if o.dim() == 3 else o for o in outs])
    low = [m.bfloat16() for m in mats]
    _compare([m[-1:] if m.dim() == 3 else m for m in low], [o[-1:] if o.dim() == 3 else o for o in newton_schulz(low)])


@pytest.mark.gpu
def test_newton_schulz_refusals():
    from neosr_amd.optimizers import newton_schulz

    m = torch.zeros(4, 5, device=DEV)
    for bad in (lambda: newton_schulz(m.cpu()), lambda: newton_schulz(m.half()), lambda: newton_schulz([m, m.bfloat16()]),
                lambda: newton_schulz(m[0]), lambda: newton_schulz(m, steps=0), lambda: newton_schulz(m, steps=65),
                lambda: newton_schulz(m, eps=-1.0), lambda: newton_schulz(m, coefficients=(1.0, 2.0)),
                lambda: newton_schulz(m, steps=2, coefficients=[ABC]), lambda: newton_schulz(m, coefficients=(1.0, math.nan, 0.0)),
                lambda: newton_schulz(m.clone().requires_grad_(True)), lambda: newton_schulz(torch.zeros(1, 32769, device=DEV))):
        with pytest.raises(_C.NeosrAmdError):
            bad()


def test_newton_schulz_c_entry_refuses():
    """on the host, before anything is launched"""
    import ctypes as C

    lib = _C.load()
    coef = (C.c_float * 15)(*[1.0] * 15)

    def item(**kw):
        it = _C.NsItem(in_=16, out=16, in_sr=5, out_sr=5, count=1, rows=4, cols=5)
        for k, v in kw.items():
            setattr(it, k, v)
        return (_C.NsItem * 1)(it)

    good = item()
    need = lib.neosr_newton_schulz_workspace_bytes(good, 1, _C.DT_F32)
    assert need > 0 and lib.neosr_newton_schulz_workspace_bytes(good, 0, _C.DT_F32) == 0
    for bad in (dict(rows=0), dict(cols=0), dict(rows=32769), dict(count=0), dict(in_=None), dict(out=18)):
        assert lib.neosr_newton_schulz_workspace_bytes(item(**bad), 1, _C.DT_F32) == -1, bad
        assert lib.neosr_newton_schulz(item(**bad), 1, _C.DT_F32, 5, coef, 1e-7, 16, 1 << 30, None) != 0, bad
    for args in ((good, 1, 5, 5, coef, 1e-7, 16, need), (good, 1, 0, 0, coef, 1e-7, 16, need), (good, 1, 0, 5, None, 1e-7, 16, need),
                 (good, 1, 0, 5, coef, -1.0, 16, need), (good, 1, 0, 5, coef, 1e-7, None, need), (good, 1, 0, 5, coef, 1e-7, 16, need - 1),
                 (good, 1, 0, 5, coef, 1e-7, 24, need), (None, 1, 0, 5, coef, 1e-7, 16, need)):
        assert lib.neosr_newton_schulz(*args, None) != 0 and lib.neosr_last_error()
    assert lib.neosr_muon_step(C.byref(_C.MuonDesc()), None) != 0
    d = _C.MuonDesc(param=16, grad=16, exp_avg=16, exp_avg_sq=16, update=16, chunks=16, n=20, nchunks=1, nmatrix=1, nitems=1, ns_steps=5,
                    items=good, coefficients=C.cast(coef, C.POINTER(C.c_float)), workspace=16, workspace_bytes=need - 1)
    assert lib.neosr_muon_step(C.byref(d), None) != 0 and b"workspace" in lib.neosr_last_error()
    for bad in (dict(ns_steps=0), dict(nmatrix=2), dict(nitems=0), dict(update=None), dict(chunks=None)):
        e = _C.MuonDesc.from_buffer_copy(d)
        e.workspace_bytes = need
        for k, v in bad.items():
            setattr(e, k, v)
        assert lib.neosr_muon_step(C.byref(e), None) != 0, bad


# ------------------------------------------------------------------------------------------------- muon


def _arena_params(init):
    from neosr_amd.hip.nets import arena_layout

    offs, total = arena_layout(init)
    arena = torch.zeros(total, device=DEV)
    ps = []
    for t, off in zip(init, offs):
        arena[off: off + t.numel()].copy_(t.reshape(-1))
        ps.append(torch.nn.Parameter(arena[off: off + t.numel()].view(t.shape)))
    return ps, arena


PARAM_SHAPES = [(60, 33, 3, 3), (60,), (120, 60), (120,), (61, 120), (225, 6), (3, 60, 3, 3), (1, 50, 60), (17, 7)]


class _Oracle:
    """the documented update in 64 bits on the CPU"""

    def __init__(self, init, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, momentum=0.95, nesterov=True, rms=0.2, min_side=16):
        self.p = [t.double().cpu() for t in init]
        self.m = [torch.zeros_like(t) for t in self.p]
        self.v = [torch.zeros_like(t) for t in self.p]
        self.hp = (lr, betas, eps, weight_decay, momentum, nesterov, rms, min_side)
        self.t = 0

    def step(self, grads, max_norm=0.0, grad_scale=1.0):
        lr, (b1, b2), eps, wd, mu, nesterov, rms, min_side = self.hp
        self.t += 1
        g = [x.double().cpu() * grad_scale for x in grads]
        if max_norm:
            norm = torch.sqrt(sum((x * x).sum() for x in g))
            g = [x * min(1.0, float(max_norm / (norm + 1e-6))) for x in g]
        for i, x in enumerate(g):
            p = self.p[i]
            rows, cols = p.shape[0], p.numel() // p.shape[0]
            if p.dim() in (2, 4) and min(rows, cols) >= min_side:
                self.m[i] = mu * self.m[i] + (1 - mu) * x
                u = (1 - mu) * x + mu * self.m[i] if nesterov else self.m[i]
                u = _exact(u.reshape(rows, cols)).reshape(p.shape)
                self.p[i] = p * (1 - lr * wd) - lr * rms * math.sqrt(max(rows, cols)) * u
            else:
                self.m[i] = b1 * self.m[i] + (1 - b1) * x
                self.v[i] = b2 * self.v[i] + (1 - b2) * x * x
                mh, vh = self.m[i] / (1 - b1 ** self.t), self.v[i] / (1 - b2 ** self.t)
                self.p[i] = p * (1 - lr * wd) - lr * mh / (vh.sqrt() + eps)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, {"nesterov": False, "momentum": 0.8, "weight_decay": 0.0}, {"min_side": 64, "rms": 0.5}],
                         ids=["default", "heavy_ball", "min_side"])
def test_muon_steps(kw):
    """weights after 4 steps, with clipping, a gradient scale and the EMA shadow; a saved and reloaded state continues.
    The update of a step is off by `_tol(5)` relative, of size lr rms sqrt(max side) per unit norm: against weights of norm |p|
    4 steps of lr 1e-2 stay below 4 * 2.4e-4 |update|; the updates are compared themselves."""
    from neosr_amd.optimizers import muon

    g = torch.Generator().manual_seed(0)
    init = [torch.randn(*s, generator=g) * 0.05 for s in PARAM_SHAPES]
    ps, arena = _arena_params(init)
    ema = torch.zeros_like(arena)
    opt, ref = muon(ps, lr=1e-2, **kw), _Oracle(init, 1e-2, **kw)
    shadow = None
    for step in range(4):
        grads = [torch.randn(*s, generator=g) for s in PARAM_SHAPES]
        for p, x in zip(ps, grads):
            p.grad = x.to(DEV)
        if step == 2:                                    # resume in the middle
            state = opt.state_dict()
            opt = muon(ps, lr=1e-2, **kw)
            opt.load_state_dict(state)
        opt.set_grad_scale(0.5)
        if step != 1:
            opt.set_clip(1.0)
        opt.set_ema(ema, 0.9, step == 0)
        before = [p.detach().clone() for p in ps]
        opt.step()
        ref_before = [x.clone() for x in ref.p]
        ref.step(grads, 1.0 if step != 1 else 0.0, 0.5)
        for p, q, b, rb, s in zip(ps, ref.p, before, ref_before, PARAM_SHAPES):
            assert rel_err(p.detach() - b, q - rb) < (step + 1) * _tol(5) + 2 ** -18, (step, s)
        shadow = arena.clone() if shadow is None else shadow + (arena - shadow) * (1.0 - 0.9)
        assert rel_err(ema, shadow) < 1e-6
    assert set(opt.state[ps[0]]) == {"exp_avg", "exp_avg_sq"} and opt.param_groups[0]["step"] == 4


@pytest.mark.gpu
def test_muon_trains_a_swinir_through_the_model():
    """`optim_g.type = "muon"` through the options: one step moves every parameter by the documented update"""
    from neosr_amd.models import build_model
    from neosr_amd.utils.options import set_global_opt

    opt = {"name": "muon", "model_type": "image", "scale": 2, "manual_seed": 7, "is_train": True, "dist": False, "rank": 0,
           "world_size": 1, "num_gpu": 1, "datasets": {"train": {"type": "paired", "patch_size": 16, "batch_size": 2}}, "path": {},
           "network_g": {"type": "swinir_small"},
           "train": {"ema": 0.9, "grad_clip": True, "optim_g": {"type": "muon", "lr": 1e-3, "weight_decay": 0.0},
                     "pixel_opt": {"type": "L1Loss", "loss_weight": 1.0}}, "logger": {"total_iter": 10}}
    set_global_opt(opt)
    torch.manual_seed(7)
    model = build_model(opt)
    params = dict(model.net_g.named_parameters())
    before = {k: v.detach().clone() for k, v in params.items()}
    model.feed_data({"lq": torch.rand(2, 3, 16, 16), "gt": torch.rand(2, 3, 32, 32)})
    model.optimize_parameters(1)
    torch.cuda.synchronize()
    from neosr_amd.optimizers import muon

    assert isinstance(model.optimizer_g, muon)
    lr, n = model.optimizer_g.param_groups[0]["lr"], 0
    for k, p in params.items():
        if not p.requires_grad:
            continue
        step = (before[k] - p.detach()).double()
        assert torch.isfinite(step).all()
        shape = muon.matrix_shape(p, 16)
        if shape is None:
            assert float(step.abs().max()) <= lr * 1.01, k           # first AdamW step: lr * sign
        else:
            n += 1
            m = (before[k] - p.detach()).reshape(shape).double()
            sv = torch.linalg.svdvals(m) / (lr * 0.2 * math.sqrt(max(shape)))
            assert float(sv.max()) < 1.25, k                         # the iterates' singular values end in [0, 1.21]
    assert n >= 8


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(40,), (3, 7)], [(64, 48)], [(33, 32, 1, 1), (128,)]], ids=["no_matrix", "only_matrices", "1x1"])
def test_muon_groups(shapes):
    """groups without a matrix, of matrices alone, and two groups in one optimizer"""
    from neosr_amd.optimizers import muon

    g = torch.Generator().manual_seed(3)
    init = [[torch.randn(*s, generator=g) * 0.1 for s in shapes] for _ in range(2)]
    ps = [_arena_params(x)[0] for x in init]
    opt = muon([{"params": ps[0]}, {"params": ps[1], "lr": 3e-3}], lr=1e-2)
    refs = [_Oracle(init[0], 1e-2), _Oracle(init[1], 3e-3)]
    for _ in range(2):
        for group, ref in zip(ps, refs):
            grads = [torch.randn(*p.shape, generator=g) for p in group]
            for p, x in zip(group, grads):
                p.grad = x.to(DEV)
            ref.step(grads)
        opt.step()
    for group, ref in zip(ps, refs):
        for p, q in zip(group, ref.p):
            assert rel_err(p, q) < 1e-5


def test_muon_arguments():
    from neosr_amd.optimizers import muon

    p = [torch.nn.Parameter(torch.zeros(20, 20))]
    for bad in (dict(momentum=1.0), dict(rms=0.0), dict(min_side=0), dict(betas=(1.0, 0.9)), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            muon(p, **bad)
    with pytest.raises(_C.NeosrAmdError):
        muon(p, ns_steps=0)
    shape = lambda *s: muon.matrix_shape(torch.zeros(*s), 16)  # noqa: E731
    assert shape(64, 32, 3, 3) == (64, 288) and shape(225, 6) is None and shape(64) is None and shape(1, 64, 180) is None
    p[0].grad = torch.zeros(20, 20)
    with pytest.raises(_C.NeosrAmdError):     # a CPU parameter is an error, not a slow path
        muon(p).step()


@pytest.mark.gpu
def test_a_training_step_of_an_attention_block():
    """the operators together, as a trained block uses them: fused projection, rotary positions over a 9 x 11 picture, attention with
    shared key heads over a padded batch, projection, L2 loss, backward, one muon step — against the same block in 64 bits.
    The gradients' tolerance: fp32 chains of at most 120 terms through five products, 5 * 128 * 2^-24 of their norms; the updated
    weights': the update's own 2.4e-4."""
    import torch.nn.functional as F

    from neosr_amd.hip.attention import attention, axial_rope
    from neosr_amd.hip.transformer import linear
    from neosr_amd.optimizers import muon

    B, grid, C, H, Hk, D = 2, (9, 11), 60, 6, 2, 10
    N, g = grid[0] * grid[1], torch.Generator().manual_seed(4)
    init = [torch.randn(D * (H + 2 * Hk), C, generator=g) / math.sqrt(C), torch.randn(D * (H + 2 * Hk), generator=g) * 0.1,
            torch.randn(C, H * D, generator=g) / math.sqrt(C), torch.randn(C, generator=g) * 0.1]
    x, target = torch.randn(B, N, C, generator=g), torch.randn(B, N, C, generator=g)
    pos = torch.stack(torch.meshgrid(*[torch.arange(n) for n in grid], indexing="ij"), -1).reshape(N, 2)
    mask = torch.arange(N)[None] < torch.tensor([[N], [N - 30]])

    ps, _ = _arena_params(init)
    opt = muon(ps, lr=1e-2)
    qkv = linear(x.to(DEV), ps[0], ps[1]).view(B, N, H + 2 * Hk, D)
    q, k = axial_rope(qkv[:, :, :H], qkv[:, :, H:H + Hk], pos.to(DEV), (4, 6), theta=100.0)
    y = attention(q, k, qkv[:, :, H + Hk:], key_mask=mask.to(DEV))
    out = linear(y.reshape(B, N, H * D), ps[2], ps[3])
    (out - target.to(DEV)).square().sum().backward()

    w = [t.double().requires_grad_(True) for t in init]
    z = F.linear(x.double(), w[0], w[1]).view(B, N, H + 2 * Hk, D)

    def turn(t):
        parts, base = [], 0
        for axis, sec in enumerate((4, 6)):
            j = torch.arange(sec // 2, dtype=torch.float64)
            ang = (pos[:, axis].double()[:, None] * 100.0 ** (-2 * j / sec))[None, :, None]
            a, b = t[..., base:base + sec // 2], t[..., base + sec // 2:base + sec]
            parts += [a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()]
            base += sec
        return torch.cat([*parts, t[..., base:]], -1)

    q, k = turn(z[:, :, :H]), turn(z[:, :, H:H + Hk]).repeat_interleave(H // Hk, 2)
    v = z[:, :, H + Hk:].repeat_interleave(H // Hk, 2)
    s = (q.permute(0, 2, 1, 3) @ k.permute(0, 2, 3, 1)) / math.sqrt(D)
    p = s.masked_fill(~mask[:, None, None], -math.inf).softmax(-1)
    o = (p @ v.permute(0, 2, 1, 3)).permute(0, 2, 1, 3).reshape(B, N, H * D)
    (F.linear(o, w[2], w[3]) - target.double()).square().sum().backward()
    for a, b in zip(ps, w):
        assert rel_err(a.grad, b.grad) < 5 * 128 * 2.0 ** -24
    ref = _Oracle(init, 1e-2)
    ref.step([t.grad for t in w])
    opt.step()
    for a, i, b in zip(ps, init, ref.p):
        if a.dim() == 2:
            assert rel_err(a.detach().cpu() - i, b - i.double()) < 1e-3     # a first step's sign-like AdamW update: matrices only


@pytest.mark.gpu
def test_newton_schulz_refuses_forward_mode():
    import torch.autograd.forward_ad as fwd

    from neosr_amd.optimizers import newton_schulz

    (m,) = _mats([(20, 30)], seed=1)
    with fwd.dual_level():
        dual = fwd.make_dual(m, m)
        for bad in (dual, [m, dual]):
            with pytest.raises(_C.NeosrAmdError):
                newton_schulz(bad)
        inside = newton_schulz(m)
    assert torch.equal(inside, newton_schulz(m))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_newton_schulz_norms_outside_fp32(dt):
    """finite matrices whose norm passes fp32's largest number (50 x 70 of 1e37: 6e38), and ones whose norm has no fp32 reciprocal
    (sizes around 1e-39, made on the CPU: torch's device products flush them).  The values themselves are exact whatever their
    size, so the tolerance is the usual one."""
    from neosr_amd.optimizers import newton_schulz

    big = _mats([(50, 70), (2, 70, 50)], dt, seed=21, scale=1e37)
    assert all(torch.isfinite(m).all() and float(m.double().norm()) > 3.5e38 for m in big)
    _compare(big, newton_schulz(big))
    g = torch.Generator().manual_seed(22)
    tiny = torch.randint(-2, 3, (50, 4), generator=g).to(dt) * 2.0 ** -133
    assert 0 < float(tiny.double().norm()) < 2.0 ** -128
    want = _exact(tiny, eps=0.0)
    assert rel_err(newton_schulz(tiny.to(DEV), eps=0.0), want) <= _tol(5) + (2 ** -8 if dt == torch.bfloat16 else 0)
    only = torch.zeros(40, 60, device=DEV, dtype=dt)
    only[3, 5] = torch.finfo(dt).max
    _compare([only], newton_schulz([only]))


def test_muon_leaves_matrices_beyond_newton_schulz_to_adamw():
    """2^29 elements with sides padded to 32 is what one matrix may have: above it a parameter takes the other update"""
    from neosr_amd.optimizers import muon

    shape = lambda *s: muon.matrix_shape(torch.empty(*s, device="meta"), 16)  # noqa: E731
    assert shape(32768, 16384) == (32768, 16384) and shape(16384, 32768) == (16384, 32768)
    assert shape(32768, 16385) is None and shape(23200, 23200) is None and shape(32769, 16) is None
    assert shape(23168, 23168) == (23168, 23168)                            # 724 * 32: the largest square one


@pytest.mark.gpu
def test_a_refused_muon_step_is_no_step():
    """a step that raises has changed nothing: neither weights nor the count that the bias corrections go by"""
    from neosr_amd.optimizers import muon

    g = torch.Generator().manual_seed(5)
    init = [torch.randn(*s, generator=g) for s in [(20, 30), (7,)]]
    ps, arena = _arena_params(init)
    opt = muon(ps, lr=1e-2)
    for p in ps:
        p.grad = torch.ones_like(p)
    before = arena.clone()
    opt.set_ema(torch.zeros(3, device=DEV), 0.9, True)                      # a shadow of another network
    with pytest.raises(_C.NeosrAmdError):
        opt.step()
    assert torch.equal(arena, before) and opt.param_groups[0].get("step", 0) == 0
    opt.set_ema(torch.zeros_like(arena), 0.9, True)
    opt.step()
    assert opt.param_groups[0]["step"] == 1 and not torch.equal(arena, before)


@pytest.mark.gpu
def test_muon_through_the_model_moves_every_weight_by_the_oracles_step():
    """the first step of a swinir through the options, against the documented update of the gradients that it had, in 64 bits.
    Matrices: the update's own 2.4e-4, and the weights' rounding, half a step of 2^-23 of |p| against a step of norm |s|: twice that.
    The others' first AdamW step is lr g / (|g| + eps / 0.0316) up to 2^-18 of it (fp32 quotients, moments and corrections), the
    weights' rounding, and what fp32 makes of beta2: 0.999 is off by up to 2^-25, so 1 - beta2 by 3e-5 of it and the root of the second
    moment by 1.5e-5 (the corrections divide by the exact one).  Every parameter that has a gradient moves."""
    from neosr_amd.models import build_model
    from neosr_amd.optimizers import muon
    from neosr_amd.utils.options import set_global_opt

    opt = {"name": "muon", "model_type": "image", "scale": 2, "manual_seed": 7, "is_train": True, "dist": False, "rank": 0,
           "world_size": 1, "num_gpu": 1, "datasets": {"train": {"type": "paired", "patch_size": 16, "batch_size": 2}}, "path": {},
           "network_g": {"type": "swinir_small"},
           "train": {"grad_clip": True, "optim_g": {"type": "muon", "lr": 1e-3, "weight_decay": 0.0},
                     "pixel_opt": {"type": "L1Loss", "loss_weight": 1.0}}, "logger": {"total_iter": 10}}
    set_global_opt(opt)
    torch.manual_seed(8)
    model = build_model(opt)
    params = {k: p for k, p in model.net_g.named_parameters() if p.requires_grad}
    before = {k: p.detach().clone() for k, p in params.items()}
    taken, step = {}, model.optimizer_g.step

    def watched(*a, **kw):
        taken.update({k: p.grad.detach().clone() for k, p in params.items()})
        return step(*a, **kw)

    model.optimizer_g.step = watched
    model.feed_data({"lq": torch.rand(2, 3, 16, 16), "gt": torch.rand(2, 3, 32, 32)})
    model.optimize_parameters(1)
    torch.cuda.synchronize()
    lr = model.optimizer_g.param_groups[0]["lr"]
    ref = _Oracle([before[k] for k in params], lr, weight_decay=0.0)
    ref.step([taken[k] for k in params], 1.0)
    kinds = {True: 0, False: 0}
    for (k, p), q in zip(params.items(), ref.p):
        got, want = (p.detach() - before[k]).double().cpu(), q - before[k].double().cpu()
        assert float(taken[k].abs().max()) > 0 and float(want.norm()) > 0, k
        matrix = muon.matrix_shape(p, 16) is not None
        kinds[matrix] += 1
        rounding = 2 * 2.0 ** -24 * float(before[k].double().norm()) / float(want.norm())
        assert rel_err(got, want) <= (_tol(5) if matrix else 2.0 ** -18 + 2.0 ** -25 / 1e-3 / 2) + rounding, (k, rel_err(got, want), rounding)
    assert kinds[True] >= 8 and kinds[False] >= 8


@pytest.mark.gpu
def test_a_captured_muon_step_is_refused():
    """its learning rate and bias corrections are numbers of the call: every replay would take those of the captured step"""
    from neosr_amd.optimizers import muon

    g = torch.Generator().manual_seed(6)
    init = [torch.randn(*s, generator=g) for s in [(20, 30), (7,)]]
    ps, arena = _arena_params(init)
    opt = muon(ps, lr=1e-2)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    held, x, graph = arena.clone(), torch.zeros(4, device=DEV), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(_C.NeosrAmdError, match="captured"):
            opt.step()
        x.add_(1)
    for n in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(arena, held) and (x == n).all() and opt.param_groups[0]["step"] == 1
