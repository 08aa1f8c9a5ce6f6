"""Measured cases of the training-side operators: group norm with an activation
(channels last), embedding lookup with scaling and its gradient, and the global
gradient norm with clipping.

``run`` computes an operator either in its plain form (elementary torch
operations in 32 bits, rounded once) or, where ``own`` is true, through the
framework's public entry points.  ``exact`` gives the same outputs in 64 bits.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5          # group norm
_CLIP_EPS = 1e-6     # added to the norm before the division, as torch.nn.utils does

_HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_mods = None


def _own():
    global _mods
    if _mods is None:
        pkg = os.path.join(_HERE, "bev-kernels_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import grad_clip
        import group_norm_act
        import scaled_embedding
        _mods = (group_norm_act, scaled_embedding, grad_clip)
    return _mods


# ----------------------------------------------------------------- the cases
# Training cases of the group norm use a smooth activation: the gradient of a
# ReLU jumps where its argument is within rounding of zero, so two correct
# 32-bit computations disagree there by the whole value.

def _gn(name, n, c, h, w, g, dtype, pdtype, act, train):
    return {"name": name, "op": "gn", "n": n, "c": c, "h": h, "w": w, "g": g, "dtype": dtype,
            "pdtype": pdtype, "act": act, "train": train}


def _emb(name, v, d, n, ids, dtype, gdtype, grad, padding, scale):
    return {"name": name, "op": "emb", "v": v, "d": d, "n": n, "ids": ids, "dtype": dtype,
            "gdtype": gdtype, "grad": grad, "padding": padding, "scale": scale}


def _clip(name, tensors, total, dtype, odtype, packed, clip, norm):
    return {"name": name, "op": "clip", "tensors": tensors, "total": total, "dtype": dtype,
            "odtype": odtype, "packed": packed, "clip": clip, "norm": norm}


def listed():
    return [
        # the norm behind the smallest deformable layer (1 x 64 x 32 x 32) at inference
        _gn("gn small infer f32", 1, 64, 32, 32, 32, "f32", "f32", "relu", False),
        # behind the stage-4 deformable layer, six cameras, at inference
        _gn("gn stage4 infer f16", 6, 512, 29, 50, 32, "f16", "f16", "relu", False),
        # behind the stage-3 deformable layer, six cameras, mixed-precision training step
        _gn("gn stage3 train bf16", 6, 256, 58, 100, 32, "bf16", "f32", "silu", True),
        # odd image and channel counts: a head on a cropped map, fp16 training
        _gn("gn odd train f16", 3, 120, 37, 53, 5, "f16", "f16", "none", True),
        # the 200 x 200 bird's-eye-view map in fp32 training
        _gn("gn bev train f32", 1, 256, 200, 200, 32, "f32", "f32", "silu", True),
        # the finest feature level of two samples x six cameras, training
        _gn("gn level0 train bf16", 12, 256, 116, 200, 32, "bf16", "f32", "silu", True),
        # object queries looked up once a frame
        _emb("emb queries infer f32", 900, 256, 900, "arange", "f32", "f32", "none", False, 1.0),
        # learned column positions of a 200 x 200 map: every row is used 200 times
        _emb("emb positions train f32", 200, 128, 40000, "grid", "f32", "f32", "dense", False, 1.0),
        # tokens of a vocabulary, frequent ids far ahead of the rest, dense gradient
        _emb("emb tokens train bf16", 50021, 1024, 16384, "zipf", "bf16", "bf16", "dense", True, 32.0),
        # a long batch whose gradient is added to the fp32 main gradient
        _emb("emb tokens add bf16", 64000, 2048, 65536, "zipf", "bf16", "f32", "add", True, 45.0),
        # a head's gradients, within the limit: the norm is taken and nothing is scaled
        _clip("clip head f32", 40, 1_300_000, "f32", "same", False, False, "2"),
        # a whole network's bf16 gradients clipped into the fp32 main gradients of the optimizer
        _clip("clip network bf16", 330, 68_000_000, "bf16", "f32", True, True, "2"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gn", "emb", "clip"))
    if op == "gn":
        most = 12 * 256 * 116 * 200
        g, cpg = rng.choice(((32, 8), (32, 16), (32, 4), (32, 2), (1, 96), (8, 5), (5, 24), (48, 1),
                             (16, 64), (4, 48), (3, 7), (2, 32), (32, 32)))
        h, w = _log(rng, 1, 230), _log(rng, 1, 230)
        # 64 values a group at least: the gradient of a group of two or three
        # is a difference of nearly equal numbers, in 32 bits mostly rounding
        h = max(h, -(-64 // (cpg * w)))
        n = _log(rng, 1, 12)
        if n * g * cpg * h * w > most:
            n = 1
        dtype = rng.choice(("f32", "f16", "bf16"))
        train = rng.random() < 0.6
        return {"op": "gn", "n": n, "c": g * cpg, "h": h, "w": w, "g": g, "dtype": dtype,
                "pdtype": rng.choice(("f32", dtype)),
                "act": rng.choice(("none", "silu") if train else ("none", "relu", "silu")),
                "train": train}
    if op == "emb":
        n, v = _log(rng, 1, 65536), _log(rng, 2, 64000)
        d = rng.choice((_log(rng, 8, 2048), 8 * _log(rng, 1, 256)))
        dtype = rng.choice(("f32", "f16", "bf16"))
        if dtype == "f32":
            d = min(d, 1024)
        grad = rng.choice(("none", "dense", "add"))
        return {"op": "emb", "v": v, "d": d, "n": n, "ids": rng.choice(("grid", "zipf", "zipf")),
                "dtype": dtype, "gdtype": dtype if grad != "add" else "f32", "grad": grad,
                "padding": rng.random() < 0.5, "scale": round(math.sqrt(d), 3)}
    tensors = _log(rng, 1, 330)
    total = max(tensors, _log(rng, 2000, 68_000_000))
    dtype = rng.choice(("f32", "f16", "bf16"))
    clip = rng.random() < 0.6
    if dtype == "f32":
        total = min(total, 50_000_000)
    return {"op": "clip", "tensors": tensors, "total": total, "dtype": dtype,
            "odtype": rng.choice(("f32", dtype)) if clip else "same", "packed": rng.random() < 0.5,
            "clip": clip, "norm": rng.choice(("2", "2", "inf"))}


def _sizes(case):
    """Element counts of the case's tensors: a network's mix of vectors and
    matrices, adding up to the total."""
    r = random.Random("%d of %d" % (case["total"], case["tensors"]))
    share = [math.exp(r.uniform(0, 9)) for _ in range(case["tensors"])]
    room = case["total"] - case["tensors"]
    sizes = [1 + int(room * s / sum(share)) for s in share]
    sizes[0] += case["total"] - sum(sizes)
    return sizes


# ---------------------------------------------------------------- the inputs
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _views(sizes, dtype, packed):
    """One buffer and its tensors: back to back (bucket views) or each at the
    512-byte boundary that an allocation of its own has."""
    step = 1 if packed else 512 // dtype.itemsize
    at, end = [], 0
    for s in sizes:
        at.append(end)
        end += -(-s // step) * step
    flat = torch.zeros(end, dtype=dtype, device="cuda")
    return flat, [flat[a:a + s] for a, s in zip(at, sizes)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "gn":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]
        # channels of their own spread and offset, as a convolution gives them
        x = _rand(g, n, h, w, c) * (0.5 + torch.rand(c, generator=g, device="cuda")) + _rand(g, c)
        s["x"] = x.to(_DT[case["dtype"]]).permute(0, 3, 1, 2)
        s["weight"] = (1 + 0.2 * _rand(g, c)).to(_DT[case["pdtype"]])
        s["bias"] = (0.2 * _rand(g, c)).to(_DT[case["pdtype"]])
        if case["train"]:
            s["gy"] = _rand(g, n, h, w, c).to(_DT[case["dtype"]]).permute(0, 3, 1, 2)
    elif case["op"] == "emb":
        v, d, n = case["v"], case["d"], case["n"]
        s["table"] = (_rand(g, v, d) * d ** -0.5).to(_DT[case["dtype"]])
        if case["ids"] == "zipf":
            u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
            ids = (u * math.log(v + 1)).exp().long() - 1
            s["ids"] = ids.clamp_(0, v - 1)
        else:  # positions along a map's axis, or each id once
            s["ids"] = torch.arange(n, device="cuda") % v
        if case["grad"] != "none":
            s["gy"] = _rand(g, n, d).to(_DT[case["dtype"]])
        if case["grad"] == "add":
            s["main"] = _rand(g, v, d).to(_DT[case["gdtype"]])
    else:
        sizes, dt = _sizes(case), _DT[case["dtype"]]
        s["flat"], s["grads"] = _views(sizes, dt, case["packed"])
        s["flat"].normal_(generator=g)
        s["flat"] *= 0.01
        norm = 0.01 * math.sqrt(case["total"]) if case["norm"] == "2" else 0.05
        s["max_norm"] = 0.3 * norm if case["clip"] else 1000.0 * norm
        if case["odtype"] != "same":
            s["out_flat"], s["out"] = _views(sizes, _DT[case["odtype"]], True)
    return s


# ------------------------------------------------------------------- a pass
def run(s):
    op = s["case"]["op"]
    if op == "gn":
        return _run_gn(s, s["case"])
    if op == "emb":
        return _run_emb(s, s["case"])
    return _run_clip(s, s["case"])


def _run_gn(s, case):
    x, weight, bias, groups, act = s["x"], s["weight"], s["bias"], case["g"], case["act"]
    if own:
        gna = _own()[0]
        if not case["train"]:
            return gna.group_norm_act(x, groups, weight, bias, _EPS, act)
        y, mean, rstd = gna.group_norm_act_forward(x, groups, weight, bias, eps=_EPS, act=act)
        return (y, mean, rstd) + tuple(
            gna.group_norm_act_backward(s["gy"], x, mean, rstd, groups, weight, bias, act=act))
    n, c, h, w = x.shape
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups).float()  # noqa: E731
    back = lambda t: t.to(x.dtype).reshape(n, h, w, c).permute(0, 3, 1, 2)  # noqa: E731
    gamma, beta = (t.float().view(groups, c // groups) for t in (weight, bias))
    xf = rows(x)
    mean = xf.mean((1, 3), keepdim=True)
    centred = xf - mean
    rstd = (centred.square().mean((1, 3), keepdim=True) + _EPS).rsqrt()
    xhat = centred * rstd
    z = xhat * gamma + beta
    if act == "silu":
        sig = 1 / (1 + (-z).exp())
        y = z * sig
    else:
        y = z.clamp_min(0) if act == "relu" else z
    if not case["train"]:
        return back(y)
    dz = rows(s["gy"])
    if act == "silu":
        dz = dz * (sig * (1 + z * (1 - sig)))
    dgamma, dbeta = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    dxhat = dz * gamma
    dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True)
                 - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
    return (back(y), mean.view(n, groups), rstd.view(n, groups), back(dx),
            dgamma.view(c).to(weight.dtype), dbeta.view(c).to(bias.dtype))


def _run_emb(s, case):
    table, ids, scale = s["table"], s["ids"], case["scale"]
    pad = 0 if case["padding"] else None
    if own:
        emb = _own()[1]
        y = emb.scaled_embedding_forward(table, ids, scale)
        if case["grad"] == "none":
            return y
        return y, emb.scaled_embedding_backward(s["gy"], ids, case["v"], scale, padding_idx=pad,
                                                grad_weight=s.get("main"))
    y = (table[ids].float() * scale).to(table.dtype)
    if case["grad"] == "none":
        return y
    rows = s["gy"].float() * scale
    if case["padding"]:
        rows = rows * (ids != 0).unsqueeze(1)
    if case["grad"] == "add":
        return y, s["main"].index_add_(0, ids, rows)
    total = torch.zeros(case["v"], case["d"], device=ids.device).index_add_(0, ids, rows)
    return y, total.to(_DT[case["gdtype"]])


def _run_clip(s, case):
    grads, out = s["grads"], s.get("out")
    kind = float(case["norm"])
    flat = s["flat"] if out is None else s["out_flat"]
    if own:
        return _own()[2].clip_grads(grads, s["max_norm"], norm_type=kind, out=out), flat
    g32 = [g.float() for g in grads]
    if kind == 2.0:
        norm = torch.stack([t.sum() for t in torch._foreach_mul(g32, g32)]).sum().sqrt()
    else:
        norm = torch.stack([t.max() for t in torch._foreach_abs(g32)]).max()
    coef = (s["max_norm"] / (norm + _CLIP_EPS)).clamp(max=1.0)
    torch._foreach_copy_(grads if out is None else out, torch._foreach_mul(g32, coef))
    return norm, flat


# ---------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gn":
        n, c, h, w, g = case["n"], case["c"], case["h"], case["w"], case["g"]
        grad = case["train"]
        x = s["x"].double().contiguous().requires_grad_(grad)
        gamma = s["weight"].double().requires_grad_(grad)
        beta = s["bias"].double().requires_grad_(grad)
        var, mean = torch.var_mean(x.view(n, g, -1), -1, correction=0)
        sd = (var + _EPS).sqrt()
        each = lambda t: t.repeat_interleave(c // g, 1).view(n, c, 1, 1)  # noqa: E731
        y = (x - each(mean)) / each(sd) * gamma.view(c, 1, 1) + beta.view(c, 1, 1)
        if case["act"] == "relu":
            y = torch.relu(y)
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        if not grad:
            return y
        gx, gg, gb = torch.autograd.grad(y, (x, gamma, beta), s["gy"].double())
        return y.detach(), mean.detach(), (1 / sd).detach(), gx, gg, gb
    if case["op"] == "emb":
        ids, v = s["ids"], case["v"]
        y = torch.nn.functional.embedding(ids, s["table"].double()) * case["scale"]
        if case["grad"] == "none":
            return y
        counted = torch.ones_like(ids, dtype=torch.float64)
        if case["padding"]:
            counted[ids == 0] = 0
        total = s["main"].double() if case["grad"] == "add" else torch.zeros(
            v, case["d"], dtype=torch.float64, device="cuda")
        total.index_put_((ids,), s["gy"].double() * (case["scale"] * counted[:, None]), accumulate=True)
        return y, total
    g = torch.cat([t.double() for t in s["grads"]])
    norm = torch.linalg.vector_norm(g, float(case["norm"]))
    coef = min(1.0, s["max_norm"] / (norm.item() + _CLIP_EPS))
    return norm, (s["flat"].double() if case["odtype"] == "same" else g) * coef


# ------------------------------------------------ what a pass cannot do without
def _distinct(case):
    """Rows of the table that the ids reach (expected, for random ids)."""
    if case["ids"] != "zipf":
        return min(case["n"], case["v"])
    k = torch.arange(case["v"], dtype=torch.float64)
    p = torch.log1p(1 / (k + 1)) / math.log(case["v"] + 1)
    return float((1 - (1 - p) ** case["n"]).sum())


def work(case):
    if case["op"] == "gn":
        each = case["n"] * case["c"] * case["h"] * case["w"]
        size, rows = _SIZE[case["dtype"]], case["c"] * _SIZE[case["pdtype"]]
        stats = 2 * 4 * case["n"] * case["g"]
        if not case["train"]:
            return {"bytes": 2 * each * size + 2 * rows, "flops": 8.0 * each}
        return {"bytes": 4 * each * size + 4 * rows + stats, "flops": 30.0 * each}
    if case["op"] == "emb":
        size, gsize = _SIZE[case["dtype"]], _SIZE[case["gdtype"]]
        each, rows = case["n"] * case["d"], _distinct(case) * case["d"]
        total = 8 * case["n"] + (rows + each) * size
        if case["grad"] == "none":
            return {"bytes": total, "flops": each}
        total += each * size + (2 * rows if case["grad"] == "add" else case["v"] * case["d"]) * gsize
        return {"bytes": total, "flops": 3.0 * each}
    size = _SIZE[case["dtype"]]
    if case["odtype"] == "same":  # nothing changes
        return {"bytes": case["total"] * size, "flops": 2.0 * case["total"]}
    return {"bytes": case["total"] * (size + _SIZE[case["odtype"]]), "flops": 3.0 * case["total"]}
