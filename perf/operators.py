"""Workloads of the framework's token-path operators: layer norm, rotary positions, block-sparse attention.

Each case is one call a program makes beside the KV cache.  ``run`` computes it
in elementary torch operations, or, where ``own`` is set, through the
framework's entry points (``pyramidkv.norm``, ``pyramidkv.rope``,
``pyramidkv.sparse``).  Sizes come from the DiT of this repository (1536
channels, 12 heads of 128, blocks of 3 latent frames of 30 x 52 tokens, K/V of
3 to 21 frames per head) or are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FRAME = 30 * 52           # tokens of a latent frame


def listed():
    return [
        # one embedding row (a time embedding, a pooled text token): latency
        dict(name="norm_row", op="norm", rows=1, cols=1536, groups=0, plus=0, dtype="bf16",
             wtype="fp32", train=0),
        # a block of 3 frames before its QKV projection, modulated per frame: 1 + scale, shift
        dict(name="norm_block", op="norm", rows=3 * FRAME, cols=1536, groups=3, plus=1,
             dtype="bf16", wtype="bf16", train=0),
        # training step over 8 videos' blocks, modulation of each video, fp32 modulation
        dict(name="norm_train", op="norm", rows=8 * 3 * FRAME, cols=1536, groups=8, plus=1,
             dtype="bf16", wtype="fp32", train=1),
        # odd sizes in fp32, a plain affine norm, training
        dict(name="norm_odd", op="norm", rows=777, cols=1111, groups=1, plus=0, dtype="fp32",
             wtype="fp32", train=1),
        # one decoded token far into a sequence, fewer key heads than query heads
        dict(name="rotary_token", op="rotary", tokens=1, heads=12, kheads=4, dim=128, pairs=64,
             axes=1, layout="half", scaling="linear", span=1_000_000, dtype="bf16", train=0),
        # the query and key block of 3 frames by (t, y, x)
        dict(name="rotary_block", op="rotary", tokens=3 * FRAME, heads=12, kheads=12, dim=128,
             pairs=64, axes=3, layout="interleaved", scaling="none", span=120, dtype="bf16",
             train=0),
        # a long training sequence, part of the head rotated, frequencies scaled for its length
        dict(name="rotary_train", op="rotary", tokens=65_521, heads=12, kheads=12, dim=128,
             pairs=32, axes=1, layout="half", scaling="yarn", span=65_521, dtype="fp16", train=1),
        # one query row per head over a long cache whose block means the program keeps
        dict(name="sparse_token", op="sparse", chunks=1, heads=12, rows=1, dim=128, top=16,
             block=64, group=128, lo=21 * FRAME, hi=21 * FRAME, unit=1, lens_seed=0, kept=1),
        # one frame's queries, ragged lengths, smaller heads and coarser blocks
        dict(name="sparse_frame", op="sparse", chunks=1, heads=7, rows=1001, dim=64, top=8,
             block=128, group=64, lo=0, hi=9001, unit=1, lens_seed=4, kept=0),
        # a layer step: 3 chunks of a frame, K/V of 3 to 21 frames per head
        dict(name="sparse_block", op="sparse", chunks=3, heads=12, rows=FRAME, dim=128, top=32,
             block=64, group=128, lo=3, hi=21, unit=FRAME, lens_seed=1, kept=0),
        # the layer step of 4 videos at once
        dict(name="sparse_batch", op="sparse", chunks=12, heads=12, rows=FRAME, dim=128, top=32,
             block=64, group=128, lo=3, hi=21, unit=FRAME, lens_seed=2, kept=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "sparse"])
    if op == "norm":
        cols = _log(rng, 64, 8192)
        groups = rng.choice([0, 1, 1, 2, 3, 8])
        rows = _log(rng, 1, min(8 * 3 * FRAME, 8 * 3 * FRAME * 1536 // cols))
        rows = max(1, groups) * max(1, rows // max(1, groups))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            rows = max(1, groups) * max(1, rows // (2 * max(1, groups)))
        return dict(op=op, rows=rows, cols=cols, groups=groups, plus=int(rng.random() < 0.5),
                    dtype=dtype, wtype=rng.choice([dtype, "fp32"]), train=int(rng.random() < 0.6))
    if op == "rotary":
        heads = rng.randint(1, 24)
        dim = 2 * rng.randint(16, 96) if rng.random() < 0.4 else rng.choice([64, 128, 256])
        pairs = dim // 2 if rng.random() < 0.5 else rng.randint(1, dim // 2)
        axes = rng.choice([1, 1, 2, 3])
        tokens = _log(rng, 1, max(1, 65_521 * 12 * 128 // (heads * dim)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            tokens = max(1, tokens // 2)
        return dict(op=op, tokens=tokens, heads=heads, kheads=rng.randint(1, heads), dim=dim,
                    pairs=pairs, axes=axes, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    span=_log(rng, 64, 1_000_000), dtype=dtype, train=int(rng.random() < 0.5))
    few = rng.random() < 0.4
    chunks, heads = (_log(rng, 1, 8), rng.randint(1, 16)) if few else (rng.randint(1, 4),
                                                                      rng.randint(1, 12))
    rows = rng.randint(1, 16) if few else _log(rng, 65, 2000)
    hi = min(_log(rng, 500, 40_000), 2_600_000 // (chunks * heads))
    block = rng.choice([64, 64, 128])
    return dict(op=op, chunks=chunks, heads=heads, rows=rows, dim=rng.choice([64, 128, 128]),
                top=_log(rng, 1, 2048 // block), block=block,
                group=rng.choice([64, 100, 128, 128]), lo=rng.choice([0, 1, hi // 4]), hi=hi,
                unit=1, lens_seed=rng.randrange(1 << 30), kept=int(rng.random() < 0.5))


# ---- inputs -----------------------------------------------------------------------------
def _lens(case):
    r = random.Random(case["lens_seed"])
    return [r.randint(case["lo"], case["hi"]) * case["unit"]
            for _ in range(case["chunks"] * case["heads"])]


def _frequencies(case):
    """(inv_freq float64 [pairs], axis of each pair, factor of the rotated part) on the host."""
    P, A = case["pairs"], case["axes"]
    axis = [min(A - 1, p * A // P) for p in range(P)]
    inv, base, factor = [], 10000.0, 4.0
    for a in range(A):
        n = axis.count(a)
        b = base * factor ** (n / max(1, n - 1)) if case["scaling"] == "ntk" else base
        inv += [b ** (-i / n) for i in range(n)]
    if case["scaling"] == "linear":
        inv = [f / factor for f in inv]
    scale = 1.0
    if case["scaling"] == "yarn":
        scale = 0.1 * math.log(factor) + 1.0
        length = 8192.0
        ramp = [min(1.0, max(0.0, (length * f / (2 * math.pi) - 1.0) / 31.0)) for f in inv]
        inv = [f * r + f / factor * (1.0 - r) for f, r in zip(inv, ramp)]
    return inv, axis, scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    s = dict(case)
    if case["op"] == "norm":
        dt, wt = DTYPES[case["dtype"]], DTYPES[case["wtype"]]
        N, C, G = case["rows"], case["cols"], case["groups"]
        # a residual stream: channels of different spread and offset
        s["x"] = (normal(N, C) * torch.exp(0.5 * normal(C)) + 0.5 * normal(C)).to(dt)
        shape = (G, C) if G > 1 else (C,)
        s["w"] = s["b"] = None
        if G:
            s["w"] = ((0.2 if case["plus"] else 1.0) * normal(*shape)).to(wt)
            s["b"] = (0.3 * normal(*shape)).to(wt)
        s["eps"] = 1e-6
        s["dy"] = normal(N, C).to(dt) if case["train"] else None
        for n in ("x", "w", "b"):
            if case["train"] and s[n] is not None:
                s[n].requires_grad_(True)
    elif case["op"] == "rotary":
        dt = DTYPES[case["dtype"]]
        T, H, HK, D, A = (case[n] for n in ("tokens", "heads", "kheads", "dim", "axes"))
        s["q"], s["k"] = normal(T, H, D).to(dt), normal(T, HK, D).to(dt)
        inv, axis, s["scale"] = _frequencies(case)
        s["inv_freq"] = torch.tensor(inv, dtype=torch.float64, device=DEVICE)
        s["axis"] = torch.tensor(axis, dtype=torch.int32, device=DEVICE)
        if A == 3:      # tokens of latent frames in (t, y, x) order, from some frame on
            t0 = int(torch.randint(0, case["span"], (1,), generator=g, device=DEVICE))
            i = torch.arange(T, device=DEVICE)
            s["pos"] = torch.stack([t0 + i // FRAME, i % FRAME // 52, i % 52], dim=1)
        else:
            s["pos"] = torch.randint(0, case["span"], (T, A), generator=g, device=DEVICE)
        if case["train"]:
            s["dq"], s["dk"] = normal(T, H, D).to(dt), normal(T, HK, D).to(dt)
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
    else:
        C, H, R, D = (case[n] for n in ("chunks", "heads", "rows", "dim"))
        lens = _lens(case)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        rows = max(1, cu[-1])
        # neighbouring tokens resemble one another, so blocks of keys have means that differ
        place = torch.arange(rows, device=DEVICE) // 48
        drift = 0.7 * normal(rows // 48 + 1, D)
        s["k"] = (normal(rows, D) + drift[place]).to(torch.bfloat16)
        s["v"] = normal(rows, D).to(torch.bfloat16)
        away = torch.arange(C * R, device=DEVICE) // 64
        s["q"] = (normal(C * R, H, D) + 0.7 * normal(C * R // 64 + 1, H, D)[away]).to(torch.bfloat16)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
        s["softmax_scale"] = D ** -0.5
        s["longest"] = max(lens)
        s["means"] = _means(s) if case["kept"] else None
    return s


# ---- the operators ------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _norm, "rotary": _rotary, "sparse": _sparse}[state["op"]](state)


def _own(s):
    import os
    import sys
    pkg = os.path.join(os.getcwd(), "pyramid-forcing_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    if s["op"] == "norm":
        from pyramidkv.norm import layer_norm
        y = layer_norm(s["x"], s["w"], s["b"], eps=s["eps"], one_plus=bool(s["plus"]))
        if not s["train"]:
            return {"y": y}
        leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
        grads = torch.autograd.grad(y, leaves, s["dy"])
        return {"y": y.detach(), "dx": grads[0], "dw": grads[1:2], "db": grads[2:3]}
    if s["op"] == "rotary":
        from pyramidkv.rope import rotary_apply
        q, k = rotary_apply((s["q"], s["k"]), s["pos"], s["inv_freq"], s["axis"],
                            layout=s["layout"], scale=s["scale"])
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    from pyramidkv.sparse import sparse_attention
    out, blocks = sparse_attention(s["q"], s["k"], s["v"], s["cu"], s["chunks"], s["rows"],
                                   s["top"], query_block=s["group"], block=s["block"],
                                   softmax_scale=s["softmax_scale"], means=s["means"])
    return {"out": out, "blocks": blocks}


def _norm(s):
    x = s["x"].float()
    N, C = x.shape
    mu = x.mean(dim=1, keepdim=True)
    d = x - mu
    rstd = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + s["eps"])
    xh = d * rstd
    if s["w"] is None:
        w, b = torch.ones(1, 1, device=x.device), torch.zeros(1, 1, device=x.device)
    else:
        w, b = s["w"].float().view(-1, 1, C) + float(s["plus"]), s["b"].float().view(-1, 1, C)
    G = w.shape[0]
    y = (xh.view(G, N // G, C) * w + b).view(N, C).to(s["x"].dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gr = (dy.view(G, N // G, C) * w).view(N, C)
    dx = rstd * (gr - gr.mean(dim=1, keepdim=True) - xh * (gr * xh).mean(dim=1, keepdim=True))
    out = {"y": y, "dx": dx.to(s["x"].dtype), "dw": (), "db": ()}
    if s["w"] is not None:
        out["dw"] = ((dy * xh).view(G, N // G, C).sum(dim=1).view(s["w"].shape).to(s["w"].dtype),)
        out["db"] = (dy.view(G, N // G, C).sum(dim=1).view(s["b"].shape).to(s["b"].dtype),)
    return out


def _turn(x, cos, sin, layout, scale):
    """The first 2P dims of x's heads turned by the angles of cos, sin [tokens, 1, P]."""
    P = cos.shape[-1]
    head, rest = x[..., :2 * P].float(), x[..., 2 * P:]
    if layout == "half":
        a, b = head[..., :P], head[..., P:]
    else:
        a, b = head[..., 0::2], head[..., 1::2]
    re, im = scale * (a * cos - b * sin), scale * (a * sin + b * cos)
    turned = torch.cat([re, im], -1) if layout == "half" else torch.stack([re, im], -1).flatten(-2)
    return torch.cat([turned.to(x.dtype), rest], dim=-1)


def _rotary(s):
    angle = s["pos"].double()[:, s["axis"].long()] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = {n: _turn(s[n], cos, sin, s["layout"], s["scale"]) for n in ("q", "k")}
    if s["train"]:
        out["dq"] = _turn(s["dq"], cos, -sin, s["layout"], s["scale"])
        out["dk"] = _turn(s["dk"], cos, -sin, s["layout"], s["scale"])
    return out


def _means(s):
    """fp32 means of the blocks of keys; block j of segment i at row cu[i] // block + i + j,
    zeros in rows between."""
    cu, B = s["cu"].long(), s["block"]
    n, D = cu.numel() - 1, s["dim"]
    slots = s["k"].shape[0] // B + n
    row = torch.arange(s["k"].shape[0], device=cu.device)
    seg = torch.searchsorted(cu, row, right=True) - 1
    live = seg < n
    seg = seg.clamp(max=n - 1)
    slot = torch.where(live, cu[seg] // B + seg + (row - cu[seg]) // B, slots)
    total = torch.zeros(slots + 1, D, dtype=torch.float64, device=cu.device)
    total.index_add_(0, slot, s["k"].double())
    count = torch.zeros(slots + 1, dtype=torch.float64, device=cu.device)
    count.index_add_(0, slot, torch.ones_like(row, dtype=torch.float64))
    return (total / count.clamp(min=1)[:, None]).float()[:slots]


def _sparse(s):
    C, H, R, D, B, top, gr = (s[n] for n in ("chunks", "heads", "rows", "dim", "block", "top",
                                             "group"))
    S, G = C * H, -(-R // gr)
    cu = s["cu"].long()
    n = cu[1:] - cu[:-1]                                         # keys of each segment
    means = s["means"] if s["means"] is not None else _means(s)
    # queries [segment, group, row of the group, D], zeros behind a chunk's last row
    q = s["q"].view(C, R, H, D).transpose(1, 2)
    pad = torch.zeros(C, H, G * gr - R, D, dtype=q.dtype, device=q.device)
    q = torch.cat([q, pad], dim=2).reshape(S, G, gr, D)
    # scores in 64 bits: which block comes last is a matter of a border
    nb = max(1, -(-s["longest"] // B))
    j = torch.arange(nb, device=cu.device)
    base = cu[:-1] // B + torch.arange(S, device=cu.device)
    there = j < (n[:, None] + B - 1) // B                        # [S, nb]
    table = means[(base[:, None] + j).clamp(max=means.shape[0] - 1)].double()
    score = q.double().sum(dim=2) @ table.transpose(1, 2)        # [S, G, nb]
    score = score.masked_fill(~there[:, None], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    kept = torch.gather(there[:, None].expand(S, G, nb), 2, order)
    order = torch.where(kept, order, nb).sort(dim=-1).values
    kept = order < nb
    blocks = torch.full((S, G, top), -1, dtype=torch.int32, device=cu.device)
    blocks[..., :order.shape[-1]] = torch.where(kept, order, -1).int()
    # attention over the kept blocks' keys
    key = order[..., None] * B + torch.arange(B, device=cu.device)     # [S, G, top, B]
    live = (kept[..., None] & (key < n[:, None, None, None])).flatten(2)
    row = torch.where(live, cu[:-1, None, None] + key.flatten(2), 0)
    sc = q.float() @ s["k"][row].float().transpose(2, 3) * s["softmax_scale"]
    sc = sc.masked_fill(~live[:, :, None], -math.inf)
    m = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(m), m, 0.0))
    total = p.sum(dim=-1, keepdim=True)
    out = p @ s["v"][row].float() / torch.where(total > 0, total, 1.0)
    out = out.view(C, H, G * gr, D)[:, :, :R].transpose(1, 2).reshape(C * R, H, D)
    return {"out": out.to(torch.bfloat16), "blocks": blocks}


# ---- work and exact values ------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        e, w = (2 if case[t] != "fp32" else 4 for t in ("dtype", "wtype"))
        x, p = case["rows"] * case["cols"], case["groups"] * case["cols"]
        if case["train"]:
            return {"bytes": 4 * x * e + 4 * p * w, "flops": 20 * x}
        return {"bytes": 2 * x * e + 2 * p * w, "flops": 8 * x}
    if case["op"] == "rotary":
        e = 2 if case["dtype"] != "fp32" else 4
        x = case["tokens"] * (case["heads"] + case["kheads"]) * case["dim"]
        turned = x // case["dim"] * case["pairs"]
        ways = 2 if case["train"] else 1
        return {"bytes": ways * (2 * x * e) + case["tokens"] * case["axes"] * 8,
                "flops": ways * 8 * turned}
    C, H, R, D, B = (case[n] for n in ("chunks", "heads", "rows", "dim", "block"))
    G = -(-R // case["group"])
    seen = moved = scored = keys = 0
    for n in _lens(case):
        used = min(n, case["top"] * B)
        seen += used * R
        moved += min(n, G * used)
        scored += G * -(-n // B)
        keys += n
    table = 4 * D * (keys // B + C * H)
    first = table + 2 * D * moved if case["kept"] else 2 * D * keys
    return {"bytes": 4 * C * R * H * D + first + 2 * D * moved + 4 * C * H * G * case["top"],
            "flops": 4 * seen * D + 2 * scored * D}


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in s.items()}
    if case["op"] == "norm":
        x = s["x"].double()
        G = max(1, case["groups"])
        out = {"y": torch.empty_like(x)}
        if case["train"]:
            out |= {"dx": torch.empty_like(x), "dw": (), "db": ()}
            if s["w"] is not None:
                out["dw"] = (torch.empty_like(s["w"], dtype=torch.float64),)
                out["db"] = (torch.empty_like(s["b"], dtype=torch.float64),)
        for i, part in enumerate(x.chunk(G)):
            here = slice(i * part.shape[0], (i + 1) * part.shape[0])
            w, b = (None, None) if s["w"] is None else (s[n].double().view(G, -1)[i] for n in "wb")
            w = 1.0 if w is None else w + case["plus"]
            var, mu = torch.var_mean(part, dim=1, keepdim=True, correction=0)
            xh = (part - mu) / torch.sqrt(var + s["eps"])
            out["y"][here] = xh * w + (0.0 if b is None else b)
            if case["train"]:
                dy = s["dy"][here].double()
                dxh = dy * w
                inner = dxh - (dxh.sum(1, keepdim=True) + xh * (dxh * xh).sum(1, keepdim=True)) / x.shape[1]
                out["dx"][here] = inner / torch.sqrt(var + s["eps"])
                if b is not None:
                    out["dw"][0].view(G, -1)[i] = (dy * xh).sum(0)
                    out["db"][0].view(G, -1)[i] = dy.sum(0)
        return out
    if case["op"] == "rotary":
        ang = torch.stack([s["pos"][:, a].double() * f
                           for a, f in zip(s["axis"].tolist(), s["inv_freq"].tolist())], dim=1)
        unit = torch.polar(torch.full_like(ang, s["scale"]), ang)[:, None]
        out, P = {}, case["pairs"]
        for n in ("q", "k", "dq", "dk")[:4 if case["train"] else 2]:
            x = s[n].double()
            head = x[..., :2 * P]
            z = head.unflatten(-1, (2, P)).transpose(-1, -2) if case["layout"] == "half" else \
                head.unflatten(-1, (P, 2))
            z = torch.view_as_complex(z.contiguous()) * (unit.conj() if n[0] == "d" else unit)
            z = torch.view_as_real(z)
            x[..., :2 * P] = (z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2)
            out[n] = x
        return out
    C, H, R, D, B, gr = (case[n] for n in ("chunks", "heads", "rows", "dim", "block", "group"))
    G = -(-R // gr)        # rows of one group share their blocks
    cu = s["cu"].tolist()
    out = torch.zeros(C * R, H, D, dtype=torch.float64, device=DEVICE)
    blocks = torch.full((C * H, G, case["top"]), -1, dtype=torch.int32, device=DEVICE)
    for i in range(C * H):
        n, c, h = cu[i + 1] - cu[i], i // H, i % H
        if n == 0:
            continue
        k, v = (s[t][cu[i]:cu[i + 1]].double() for t in ("k", "v"))
        nb = -(-n // B)
        fill = torch.zeros(nb * B - n, D, dtype=torch.float64, device=DEVICE)
        each = torch.tensor([min(B, n - b * B) for b in range(nb)], device=DEVICE).double()
        mean = (torch.cat([k, fill]).view(nb, B, D).sum(1) / each[:, None]).float().double()
        for g in range(G):
            here = slice(c * R + g * gr, c * R + min(R, (g + 1) * gr))
            q = s["q"][here, h].double()
            value = mean @ q.sum(0)
            best = torch.argsort(value, descending=True, stable=True)[:case["top"]].sort().values
            blocks[i, g, :best.numel()] = best.int()
            row = (best[:, None] * B + torch.arange(B, device=DEVICE)).flatten()
            row = row if int(best[-1]) < nb - 1 else row[row < n]
            p = torch.softmax(q @ k[row].T * s["softmax_scale"], dim=-1)
            out[here, h] = p @ v[row]
    return {"out": out, "blocks": blocks}
