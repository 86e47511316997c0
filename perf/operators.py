"""Measured cases of the operators that train and serve image transformers with attention over whole pictures:

* attention  - softmax(q k^T * scale) v over tokens, with its gradients (`neosr_amd.hip.attention.attention`)
* axial_rope - rotary positions with one section of the head for each axis (`neosr_amd.hip.attention.axial_rope`)
* newton_schulz - orthogonalised updates of weight matrices (`neosr_amd.optimizers.newton_schulz`)

`run` with `own = False` is the plain form in elementary torch operations (32 bits inside, one rounding at the end), with
`own = True` the framework's calls.  `exact` evaluates the same definitions in 64 bits, one head / one matrix at a time.
"""

from __future__ import annotations

import math

import torch

own = False

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------- cases


def _attn(name, dtype, B, Lq, Lk, H, Hk, D, causal=False, ragged=False, train=False):
    return {"name": name, "op": "attention", "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "D": D,
            "causal": causal, "ragged": ragged, "train": train}


def _rope(name, dtype, B, grid, H, Hk, D, sections, interleaved=False, train=False):
    return {"name": name, "op": "axial_rope", "dtype": dtype, "B": B, "grid": "x".join(map(str, grid)), "H": H, "Hk": Hk,
            "D": D, "sections": ",".join(map(str, sections)), "interleaved": interleaved, "train": train}


def _ns(name, dtype, shapes, steps=5):
    return {"name": name, "op": "newton_schulz", "dtype": dtype, "shapes": ";".join(f"{n}*{r}x{c}" for n, r, c in shapes),
            "steps": steps}


def listed():
    return [
        # one learned query per picture pools a 64 x 64 token grid (heads of swinir_medium: 6 x 30): a single-token call
        _attn("attn_pool_fp32", "fp32", 8, 1, 4096, 6, 6, 30),
        # validation of one 128 x 128 LR picture, every token sees every token, swinir_medium's heads
        _attn("attn_picture_fp32", "fp32", 1, 16384, 16384, 6, 6, 30),
        # the training step's 64 x 64 patches, swinir_medium's heads, forward and gradients
        _attn("attn_patch_train_fp32", "fp32", 2, 4096, 4096, 6, 6, 30, train=True),
        # a batch of pictures of unequal size, padded to the longest, one of them empty; odd lengths, a reference picture
        # as keys (Lq != Lk), odd head size
        _attn("attn_ragged_train_fp32", "fp32", 8, 333, 577, 4, 4, 50, ragged=True, train=True),
        # shared key / value heads in bf16, forward and gradients
        _attn("attn_shared_train_bf16", "bf16", 4, 4096, 4096, 8, 2, 64, train=True),
        # frames attended in order (causal), wide heads, a length that ends inside a tile
        _attn("attn_causal_train_bf16", "bf16", 2, 2047, 2047, 16, 4, 128, causal=True, train=True),
        # one 16 x 16 window's tokens: the smallest call, where latency counts
        _rope("rope_window_fp32", "fp32", 1, (16, 16), 6, 6, 30, (14, 14)),
        # eight 64 x 64 patches in training: forward and gradients; two of the 30 channels carry no position
        _rope("rope_patch_train_fp32", "fp32", 8, (64, 64), 6, 6, 30, (14, 14), train=True),
        # a 16-frame clip with time, height and width sections, shared key heads
        _rope("rope_clip_train_bf16", "bf16", 1, (16, 64, 64), 8, 2, 64, (16, 24, 24), interleaved=True, train=True),
        # one projection matrix: latency
        _ns("ns_single_fp32", "fp32", [(1, 180, 180)]),
        # every matrix of swinir_medium (36 blocks of qkv / proj / fc1 / fc2 and the convolutions, flattened)
        _ns("ns_swinir_medium_fp32", "fp32", [(36, 540, 180), (36, 180, 180), (36, 360, 180), (36, 180, 360), (7, 180, 1620),
                                              (1, 64, 1620), (2, 256, 576), (1, 3, 576), (1, 180, 27)]),
        # large matrices held in bf16
        _ns("ns_large_bf16", "bf16", [(1, 2048, 2048), (1, 1024, 4096), (1, 2304, 1024)]),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16"])
    op = rng.choice(["attention", "attention", "axial_rope", "newton_schulz"])
    if op == "attention":
        D = _log_int(rng, 8, 128)
        Hk = rng.choice([1, 2, 3, 4, 6, 8])
        H = Hk * rng.choice([1, 1, 1, 2, 4])
        train = rng.random() < 0.6
        Lq = 1 if rng.random() < 0.15 and not train else _log_int(rng, 1, 8192)
        Lk = Lq if rng.random() < 0.5 and Lq > 1 else _log_int(rng, 16, 8192)
        B = _log_int(rng, 1, 16)
        cap = 2.5e8 if train else 5e8     # score elements: at most the work of the largest listed cases
        while B > 1 and B * H * Lq * Lk > cap:
            B -= 1
        while H * Lq * Lk > cap:
            Lq, Lk = max(1, Lq * 2 // 3), max(16, Lk * 2 // 3)
        return {"op": op, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "D": D,
                "causal": rng.random() < 0.3, "ragged": rng.random() < 0.3, "train": train}
    if op == "axial_rope":
        axes = rng.choice([2, 2, 3])
        sections = [2 * rng.randint(2, 20) for _ in range(axes)]
        D = sum(sections) + rng.choice([0, 0, 2, 5])
        grid = [_log_int(rng, 2, 16)] * (axes == 3) + [_log_int(rng, 4, 96), _log_int(rng, 4, 96)]
        Hk = rng.choice([1, 2, 4, 6])
        H = Hk * rng.choice([1, 1, 2, 4])
        B = _log_int(rng, 1, 16)
        cap = 6e7
        while B > 1 and B * math.prod(grid) * (H + Hk) * D > cap:
            B -= 1
        while math.prod(grid) * (H + Hk) * D > cap:
            grid[-1], grid[-2] = max(4, grid[-1] * 2 // 3), max(4, grid[-2] * 2 // 3)
        return {"op": op, "dtype": dtype, "B": B, "grid": "x".join(map(str, grid)), "H": H, "Hk": Hk, "D": D,
                "sections": ",".join(map(str, sections)), "interleaved": rng.random() < 0.5, "train": rng.random() < 0.6}
    shapes, left = [], 1.5e10
    for _ in range(rng.randint(1, 5)):
        r, c = _log_int(rng, 3, 1536), _log_int(rng, 16, 2304)
        n = _log_int(rng, 1, 24)
        cost = min(r, c) ** 2 * max(r, c)
        n = min(n, int(left // cost))
        if n >= 1:
            shapes.append((n, r, c))
            left -= n * cost
    return {"op": op, "dtype": dtype, "shapes": ";".join(f"{n}*{r}x{c}" for n, r, c in shapes or [(1, 48, 432)]),
            "steps": rng.choice([5, 5, 5, 3, 6])}


# ------------------------------------------------------------------------------------------------- inputs


def _ns_shapes(case):
    out = []
    for part in case["shapes"].split(";"):
        n, rc = part.split("*")
        r, c = rc.split("x")
        out.append((int(n), int(r), int(c)))
    return out


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "attention":
        B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
        # projections as a fused Linear leaves them: heads side by side in one buffer when the lengths agree
        if Lq == Lk:
            qkv = randn(B, Lq, H + 2 * Hk, D).to(dt)
            q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        else:
            q = randn(B, Lq, H, D).to(dt)
            kv = randn(B, Lk, 2 * Hk, D).to(dt)
            k, v = kv[:, :, :Hk], kv[:, :, Hk:]
        mask = None
        if case["ragged"]:
            lengths = torch.randint(max(1, Lk // 3), Lk + 1, (B,), generator=g, device="cuda")
            lengths[0] = Lk
            if B > 1:
                lengths[B - 1] = 0                     # a picture of the batch without a token
            mask = torch.arange(Lk, device="cuda")[None, :] < lengths[:, None]
            # what lies behind a picture's last token was never written
            k.masked_fill_(~mask[:, :, None, None], float("nan"))
            v.masked_fill_(~mask[:, :, None, None], float("nan"))
        dout = randn(B, Lq, H, D).to(dt) if case["train"] else None
        return {"q": q, "k": k, "v": v, "mask": mask, "dout": dout}
    if case["op"] == "axial_rope":
        grid = [int(x) for x in case["grid"].split("x")]
        B, H, Hk, D = (case[k] for k in ("B", "H", "Hk", "D"))
        N = math.prod(grid)
        axes = torch.meshgrid(*[torch.arange(n, device="cuda", dtype=torch.float32) for n in grid], indexing="ij")
        # a crop's place in its picture: a seeded offset for each axis
        off = torch.randint(0, 500, (len(grid),), generator=g, device="cuda").float()
        positions = torch.stack([a.reshape(-1) for a in axes], dim=1) + off
        qk = randn(B, N, H + Hk, D).to(dt)
        q, k = qk[:, :, :H], qk[:, :, H:]
        dq, dk = (randn(B, N, H, D).to(dt), randn(B, N, Hk, D).to(dt)) if case["train"] else (None, None)
        return {"q": q, "k": k, "positions": positions, "dq": dq, "dk": dk}
    mats = []   # one stack for each kind of layer
    for n, r, c in _ns_shapes(case):
        rank = max(1, min(r, c) // 4)   # momentum of a gradient: a few strong directions over noise
        m = torch.bmm(randn(n, r, rank), randn(n, rank, c)) / math.sqrt(rank) + 0.2 * randn(n, r, c)
        mats.append((1e-3 * m).to(dt))
    return {"mats": mats}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = dict(case)
    if case["op"] == "axial_rope":
        state["sections"] = tuple(int(s) for s in case["sections"].split(","))
    if case.get("train"):
        for k in ("q", "k", "v"):
            if k in state:
                state[k] = state[k].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------- one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    c = s["case"]
    if c["op"] == "attention":
        from neosr_amd.hip.attention import attention

        out = attention(s["q"], s["k"], s["v"], causal=c["causal"], key_mask=s["mask"])
        if not c["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    if c["op"] == "axial_rope":
        from neosr_amd.hip.attention import axial_rope

        q, k = axial_rope(s["q"], s["k"], s["positions"], s["sections"], interleaved=c["interleaved"])
        if not c["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    from neosr_amd.optimizers import newton_schulz

    return newton_schulz(s["mats"], steps=c["steps"], coefficients=NS_COEFFICIENTS, eps=NS_EPS)


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    if c["op"] == "attention":
        return _attention_plain(s, c)
    if c["op"] == "axial_rope":
        return _rope_plain(s, c)
    return [_newton_schulz_plain(m, c["steps"]) for m in s["mats"]]


def _allowed(Lq, Lk, causal, mask, device):
    """(B or 1, 1, 1, Lq or 1, Lk) truth values, or None: the last query sees the last key"""
    ok = None
    if causal:
        i = torch.arange(Lq, device=device)[:, None]
        j = torch.arange(Lk, device=device)[None, :]
        ok = (j <= i + (Lk - Lq))[None, None, None]
    if mask is not None:
        m = mask[:, None, None, None, :]
        ok = m if ok is None else ok & m
    return ok


def _attention_plain(s, c):
    B, Lq, Lk, H, Hk, D = (c[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
    G, dt, scale = H // Hk, s["q"].dtype, D ** -0.5
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hk, G, Lq, D)
    k = s["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    if s["mask"] is not None:
        gone = ~s["mask"][:, None, None, :, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    ok = _allowed(Lq, Lk, c["causal"], s["mask"], q.device)
    if ok is not None:
        p = p.masked_fill(~ok, float("-inf"))
    m = p.amax(-1, keepdim=True)
    m = m.masked_fill(m == float("-inf"), 0.0)
    p = torch.exp(p - m)
    z = p.sum(-1, keepdim=True)
    p = p / torch.where(z == 0, torch.ones_like(z), z)
    o = torch.matmul(p, v.contiguous())

    def heads_last(x, n):   # (B, Hk, G, L, D) -> (B, L, n, D)
        return x.reshape(B, n, x.shape[-2], D).permute(0, 2, 1, 3).to(dt).contiguous()

    if not c["train"]:
        return heads_last(o, H)
    do = s["dout"].float().permute(0, 2, 1, 3).reshape(B, Hk, G, Lq, D)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do).sum(2)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k.contiguous())
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).sum(2)
    return heads_last(o, H), heads_last(dq, H), heads_last(dk, Hk), heads_last(dv, Hk)


def _rope_tables(positions, sections, D, interleaved):
    """cos, sin (N, pairs) in 64 bits and the two channels of each pair"""
    angles, first, second, base = [], [], [], 0
    for a, sec in enumerate(sections):
        half = sec // 2
        freq = 10000.0 ** (-torch.arange(half, device=positions.device, dtype=torch.float64) * 2 / sec)
        angles.append(positions[:, a].double()[:, None] * freq)
        j = torch.arange(half, device=positions.device)
        first.append(base + (2 * j if interleaved else j))
        second.append(base + (2 * j + 1 if interleaved else j + half))
        base += sec
    ang = torch.cat(angles, 1)
    return ang.cos(), ang.sin(), torch.cat(first), torch.cat(second)


def _rope_plain(s, c):
    cos, sin, i0, i1 = _rope_tables(s["positions"], s["sections"], c["D"], c["interleaved"])
    cos, sin = cos.float()[None, :, None, :], sin.float()[None, :, None, :]

    def rotate(x, sign):
        y = x.float().clone()
        a, b = x[..., i0].float(), x[..., i1].float()
        y[..., i0] = a * cos - sign * b * sin
        y[..., i1] = sign * a * sin + b * cos
        return y.to(x.dtype)

    out = (rotate(s["q"], 1.0), rotate(s["k"], 1.0))
    if c["train"]:
        out += (rotate(s["dq"], -1.0), rotate(s["dk"], -1.0))
    return out


def _newton_schulz_plain(mat, steps):
    a, b, c = NS_COEFFICIENTS
    x = mat.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / (x.double().square().sum((1, 2), keepdim=True).sqrt().float() + NS_EPS)
    for _ in range(steps):
        g = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * g + c * torch.bmm(g, g), x)
    return (x.transpose(1, 2) if tall else x).to(mat.dtype).contiguous()


# ------------------------------------------------------------------------------------------------- work


def work(case):
    el = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
        pairs = Lq * Lk
        if case["causal"]:
            pairs = sum(min(Lk, max(0, i + 1 + Lk - Lq)) for i in range(Lq))
        qo, kv = B * Lq * H * D, B * Lk * Hk * D
        flops = 4.0 * B * H * pairs * D
        nbytes = el * (2 * qo + 2 * kv)
        if case["train"]:
            flops *= 3.5              # the scores again, dP, dV, dK, dQ
            nbytes += el * (2 * qo + 2 * kv)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "axial_rope":
        N = math.prod(int(x) for x in case["grid"].split("x"))
        n = case["B"] * N * (case["H"] + case["Hk"]) * case["D"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * n * el, "flops": passes * 3.0 * n}
    nbytes = flops = 0
    for n, r, c in _ns_shapes(case):
        lo, hi = min(r, c), max(r, c)
        nbytes += 2 * n * r * c * el
        flops += n * case["steps"] * (3.0 * lo * lo * hi + 1.0 * lo ** 3)   # symmetric products count one triangle
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------- 64-bit definition


@torch.no_grad()
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        return _attention_exact(s, case)
    if case["op"] == "axial_rope":
        return _rope_exact(s, case)
    return [torch.stack([_newton_schulz_exact(m.double(), case["steps"]) for m in stack]) for stack in s["mats"]]


def _attention_exact(s, c):
    B, Lq, Lk, H, Hk, D = (c[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
    G, dev = H // Hk, s["q"].device
    out = torch.zeros(B, Lq, H, D, device=dev, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Lk, Hk, D, device=dev, dtype=torch.float64) for _ in range(2))
    rows = torch.arange(Lq, device=dev)[:, None] + (Lk - Lq)
    for b in range(B):
        keys = torch.arange(Lk, device=dev)
        if s["mask"] is not None:
            keys = keys[s["mask"][b]]              # only the keys that are there
        if keys.numel() == 0:
            continue
        for h in range(H):
            k, v = s["k"][b, keys, h // G].double(), s["v"][b, keys, h // G].double()
            q = s["q"][b, :, h].double()
            e = (q @ k.t()) / math.sqrt(D)
            if c["causal"]:
                e[keys[None, :] > rows] = float("-inf")
            p = torch.softmax(e, dim=1).nan_to_num(0.0)   # (a row without a key: nothing)
            o = p @ v
            out[b, :, h] = o
            if c["train"]:
                do = s["dout"][b, :, h].double()
                de = p * (do @ v.t() - (p * (do @ v.t())).sum(1, keepdim=True)) / math.sqrt(D)
                dq[b, :, h] = de @ k
                dk[b, keys, h // G] += de.t() @ q
                dv[b, keys, h // G] += p.t() @ do
    return (out, dq, dk, dv) if c["train"] else out


def _rope_exact(s, c):
    sections = [int(x) for x in c["sections"].split(",")]

    def turn(x, direction):
        y = x.double().clone()
        base = 0
        for axis, sec in enumerate(sections):
            for j in range(sec // 2):
                lo, hi = (base + 2 * j, base + 2 * j + 1) if c["interleaved"] else (base + j, base + j + sec // 2)
                phase = direction * s["positions"][:, axis].double() * 10000.0 ** (-2.0 * j / sec)
                z = torch.complex(x[..., lo].double(), x[..., hi].double()) * torch.polar(torch.ones_like(phase), phase)[None, :, None]
                y[..., lo], y[..., hi] = z.real, z.imag
            base += sec
        return y

    out = (turn(s["q"], 1.0), turn(s["k"], 1.0))
    if c["train"]:
        out += (turn(s["dq"], -1.0), turn(s["dk"], -1.0))
    return out


def _newton_schulz_exact(g, steps):
    a, b, c = NS_COEFFICIENTS
    y = g / (torch.linalg.matrix_norm(g) + NS_EPS)
    for _ in range(steps):
        if y.shape[0] <= y.shape[1]:
            m = y @ y.t()
            y = a * y + b * (m @ y) + c * (m @ (m @ y))
        else:
            m = y.t() @ y
            y = a * y + b * (y @ m) + c * ((y @ m) @ m)
    return y
