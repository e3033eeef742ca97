"""Measured cases of the serialised-cloud attention operators.

``norm_rotate``        norms of queries and keys for each head, then the rotation by position
``window_attention``   attention along the serialised order of each cloud of a ragged batch, with a
                       sliding window, first rows that stay visible (sinks) and a learned relative
                       position bias by buckets; forward, training step, single new rows

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the calls of
``mps_pointops.attention``.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_BLOCK = 512  # query rows that the plain form scores at once


# ----------------------------------------------------------------------------- cases

def listed() -> list[dict]:
    return [
        # One new row for each of 64 running streams: latency of the norms and the rotation.
        {"name": "rotate-step", "op": "rotate", "mode": "forward", "dtype": "bf16", "rows": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 1, "interleaved": False},
        # Training on 32 clouds of 8192 points (the Chamfer step's batch), grid coordinates on 3 axes.
        {"name": "rotate-train", "op": "rotate", "mode": "training", "dtype": "bf16",
         "rows": 262144, "heads": 8, "kv_heads": 8, "dim": 64, "rot": 48, "axes": 3,
         "interleaved": False},
        # Odd row count, shared key heads, part of the head rotated, neighbouring pairs, 32 bits.
        {"name": "rotate-odd", "op": "rotate", "mode": "training", "dtype": "f32", "rows": 50021,
         "heads": 6, "kv_heads": 2, "dim": 48, "rot": 24, "axes": 1, "interleaved": True},
        # One small cloud through a biased layer: latency of a forward call.
        {"name": "cloud-small", "op": "attend", "mode": "forward", "dtype": "bf16", "clouds": 1,
         "points": 1024, "new": 0, "ragged": False, "heads": 4, "kv_heads": 4, "dim": 32,
         "left": 128, "right": 127, "sinks": 0, "causal": False, "bias": "grid", "reach": 15},
        # Inference on 8 clouds of 4096 points, 1024 neighbours along the order, 4 summary rows.
        {"name": "clouds-forward", "op": "attend", "mode": "forward", "dtype": "bf16", "clouds": 8,
         "points": 4096, "new": 0, "ragged": False, "heads": 8, "kv_heads": 8, "dim": 64,
         "left": 512, "right": 511, "sinks": 4, "causal": False, "bias": "none", "reach": 0},
        # Ragged clouds with narrow heads and a position table, 16-bit floats of the other kind.
        {"name": "clouds-ragged", "op": "attend", "mode": "forward", "dtype": "f16", "clouds": 13,
         "points": 5003, "new": 0, "ragged": True, "heads": 6, "kv_heads": 6, "dim": 16,
         "left": 300, "right": 300, "sinks": 0, "causal": False, "bias": "grid", "reach": 31},
        # A chunk of 512 new rows for each of 4 streams over what is cached.
        {"name": "chunk", "op": "attend", "mode": "forward", "dtype": "bf16", "clouds": 4,
         "points": 16384, "new": 512, "ragged": True, "heads": 16, "kv_heads": 4, "dim": 128,
         "left": 4095, "right": 0, "sinks": 16, "causal": True, "bias": "none", "reach": 0},
        # Training step of a biased layer on 8 clouds of 8192 points.
        {"name": "clouds-train", "op": "attend", "mode": "training", "dtype": "bf16", "clouds": 8,
         "points": 8192, "new": 0, "ragged": False, "heads": 8, "kv_heads": 8, "dim": 64,
         "left": 512, "right": 511, "sinks": 4, "causal": False, "bias": "grid", "reach": 31},
        # Training step of a causal layer with shared key heads on ragged sequences.
        {"name": "causal-train", "op": "attend", "mode": "training", "dtype": "bf16", "clouds": 5,
         "points": 4099, "new": 0, "ragged": True, "heads": 16, "kv_heads": 4, "dim": 128,
         "left": 1023, "right": 0, "sinks": 8, "causal": True, "bias": "none", "reach": 0},
        # Training step in 32 bits, ragged, biased.
        {"name": "full-precision-train", "op": "attend", "mode": "training", "dtype": "f32",
         "clouds": 3, "points": 4096, "new": 0, "ragged": True, "heads": 4, "kv_heads": 4,
         "dim": 32, "left": 256, "right": 255, "sinks": 2, "causal": False, "bias": "grid",
         "reach": 15},
        # Single new rows of 32 short streams, logarithmic buckets along the order.
        {"name": "step-biased", "op": "attend", "mode": "forward", "dtype": "bf16", "clouds": 32,
         "points": 2047, "new": 1, "ragged": True, "heads": 8, "kv_heads": 8, "dim": 64,
         "left": -1, "right": 0, "sinks": 0, "causal": True, "bias": "log", "reach": 128},
        # Single new rows of 64 long streams with shared key heads: the caches are read once.
        {"name": "step-long", "op": "attend", "mode": "forward", "dtype": "bf16", "clouds": 64,
         "points": 8192, "new": 1, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "left": -1, "right": 0, "sinks": 0, "causal": True, "bias": "none", "reach": 0},
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    if rng.random() < 0.25:
        kv = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([16, 24, 32, 48, 64, 96, 128])
        rot = rng.choice([dim, dim, 8 * rng.randint(1, dim // 8)])
        rows = min(_spread(rng, 1, 262144), 262144 * 512 // (kv * 4 * dim))
        return {"op": "rotate", "mode": rng.choice(["forward", "training"]), "dtype": dtype,
                "rows": rows, "heads": kv * rng.choice([1, 1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rot": rot, "axes": rng.choice([1, 2, 3]), "interleaved": rng.random() < 0.3}
    step = rng.random() < 0.3
    kv = rng.choice([1, 2, 4, 8])
    case = {"op": "attend", "mode": "forward", "dtype": dtype, "kv_heads": kv,
            "heads": kv * rng.choice([1, 1, 2, 4]),
            "dim": rng.choice([16, 24, 32, 64, 64, 80, 128]), "ragged": rng.random() < 0.7}
    if step:
        case.update(clouds=_spread(rng, 1, 64), points=_spread(rng, 16, 8192),
                    new=rng.choice([1, 1, 1, 2, 5, _spread(rng, 8, 512)]), causal=True, right=0,
                    left=rng.choice([-1, -1, _spread(rng, 16, 4096)]))
    else:
        causal = rng.random() < 0.4
        span = _spread(rng, 16, 1024)
        case.update(clouds=_spread(rng, 1, 16), points=_spread(rng, 33, 8192), new=0,
                    causal=causal, left=span, right=0 if causal else span - rng.randint(0, 1),
                    mode=rng.choice(["forward", "training", "training"]))
        if dtype == "f32":
            case["points"] = min(case["points"], 4096)
            case["clouds"] = min(case["clouds"], 3)
        rows = max(1, 8 * 8192 * 8 * 64 // (case["heads"] * case["dim"]))
        case["clouds"] = max(1, min(case["clouds"], rows // case["points"]))
    case["sinks"] = 0 if case["left"] < 0 else rng.choice([0, 1, 4, 16])
    case["bias"] = rng.choice(["none", "grid", "log"] if case["causal"] else ["none", "grid"])
    case["reach"] = {"none": 0, "grid": rng.choice([7, 15, 31]), "log": 128}[case["bias"]]
    return case


# ----------------------------------------------------------------------------- inputs

def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Query rows and key rows of each cloud, from the case alone."""
    rng = random.Random(1000003 * case["clouds"] + case["points"])
    keys = [rng.randint(max(1, case["points"] // 2), case["points"]) if case["ragged"]
            else case["points"] for _ in range(case["clouds"])]
    return ([min(case["new"], n) for n in keys] if case["new"] else list(keys)), keys


def _ends(lengths: list[int]) -> torch.Tensor:
    return torch.tensor(np.cumsum(lengths), dtype=torch.int64, device="cuda")


def _curve_cloud(n: int, g: torch.Generator) -> torch.Tensor:
    """Grid coordinates (n, 3) of points near a sphere's surface, ordered along the Z curve."""
    xyz = torch.randn(n, 3, device="cuda", generator=g)
    xyz = xyz / xyz.norm(dim=1, keepdim=True).clamp_min(1e-6)
    xyz = xyz + 0.01 * torch.randn(n, 3, device="cuda", generator=g)
    cells = max(8.0, math.sqrt(n))
    grid = ((xyz + 1.2) * (cells / 2.4)).clamp(0, 1023).to(torch.int64)
    code = torch.zeros(n, dtype=torch.int64, device="cuda")
    for bit in range(10):
        for axis in range(3):
            code |= ((grid[:, axis] >> bit) & 1) << (3 * bit + axis)
    return grid[code.argsort()].to(torch.int32)


def _log_map(buckets: int, reach: int) -> torch.Tensor:
    """Bucket of each distance key - query in [-reach, reach], causal: keys ahead share bucket 0,
    distances back are exact up to half of the buckets, then logarithmic up to `reach`."""
    exact = buckets // 2
    out = []
    for d in range(-reach, reach + 1):
        back = max(-d, 0)
        if back < exact:
            out.append(back)
        else:
            out.append(min(buckets - 1, exact + int(math.log(back / exact)
                                                    / math.log(reach / exact) * (buckets - exact))))
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dt=dtype):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)

    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] == "rotate":
        n, A, P = case["rows"], case["axes"], case["rot"] // 2
        # q and k are views of one projection's output, as a layer has them.
        packed = normal(n, H + K, D, scale=1.5)
        state["q"], state["k"] = packed[:, :H], packed[:, H:]
        state["q_weight"] = 1 + 0.2 * normal(D, dt=torch.float32)
        state["k_weight"] = 1 + 0.2 * normal(D, dt=torch.float32)
        top = 1024 if A > 1 else 8192
        state["position"] = torch.randint(0, top, (n, A), device="cuda", generator=g,
                                          dtype=torch.int32)
        freqs = torch.zeros(A, P, device="cuda")
        for p in range(P):
            freqs[p % A, p] = (100.0 if A > 1 else 10000.0) ** (-(p // A) / max(1, P // A))
        state["freqs"] = freqs
        if case["mode"] == "training":
            state["grad_q"], state["grad_k"] = normal(n, H, D), normal(n, K, D)
        return state

    rows, keys = _lengths(case)
    nq, nk = sum(rows), sum(keys)
    if case["new"]:
        state["q"], state["k"], state["v"] = normal(nq, H, D), normal(nk, K, D), normal(nk, K, D)
    else:  # views of one projection's output
        packed = normal(nq, H + 2 * K, D)
        state["q"], state["k"], state["v"] = packed.split([H, K, K], dim=1)
    state["lengths"] = (rows, keys)
    state["offset"], state["key_offset"] = _ends(rows), _ends(keys)
    if case["bias"] == "grid":
        pos = torch.cat([_curve_cloud(n, g) for n in keys])
        state["table"] = normal(3, 2 * case["reach"] + 1, H, scale=0.5, dt=torch.float32)
        state["buckets"] = None
    elif case["bias"] == "log":
        pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in keys])[:, None]
        state["table"] = normal(1, 32, H, scale=0.5, dt=torch.float32)
        state["buckets"] = _log_map(32, case["reach"])
    if case["bias"] != "none":
        ends = np.cumsum(keys)
        pick = np.concatenate([np.arange(e - r, e) for e, r in zip(ends, rows)])
        state["key_position"] = pos.contiguous()
        state["position"] = pos[torch.from_numpy(pick).cuda()].contiguous()
    if case["mode"] == "training":
        state["grad"] = normal(nq, H, D)
    if own:
        # The layout of the ragged batch: made once for a batch, kept for all of its layers.
        state["segments"] = _package().Segments(state["offset"], state["key_offset"])
    return state


# ----------------------------------------------------------------------------- the framework's calls

def _package():
    path = str(Path(__file__).resolve().parent.parent / "mps-pointops_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mps_pointops import attention

    return attention


def _leaf(x: torch.Tensor) -> torch.Tensor:
    return x.detach().requires_grad_()


def _own_rotate(s: dict):
    case, attention = s["case"], _package()
    args = dict(eps=1e-6, interleaved=case["interleaved"])
    if case["mode"] == "forward":
        return attention.norm_rotate(s["q"], s["k"], s["position"], s["freqs"],
                                     q_weight=s["q_weight"], k_weight=s["k_weight"], **args)
    q, k, wq, wk = (_leaf(s[n]) for n in ("q", "k", "q_weight", "k_weight"))
    yq, yk = attention.norm_rotate(q, k, s["position"], s["freqs"], q_weight=wq, k_weight=wk,
                                   **args)
    grads = torch.autograd.grad((yq, yk), (q, k, wq, wk), (s["grad_q"], s["grad_k"]))
    return (yq.detach(), yk.detach(), *grads)


def _own_attend(s: dict):
    case, attention = s["case"], _package()
    args = dict(window=(case["left"], case["right"]), sinks=case["sinks"], causal=case["causal"])
    if case["bias"] != "none":
        args.update(position=s["position"], key_position=s["key_position"], buckets=s["buckets"])
    if case["mode"] == "forward":
        if case["bias"] != "none":
            args["bias_table"] = s["table"]
        return attention.window_attention(s["q"], s["k"], s["v"], s["segments"], **args)
    leaves = [_leaf(s[n]) for n in ("q", "k", "v")]
    if case["bias"] != "none":
        leaves.append(_leaf(s["table"]))
        args["bias_table"] = leaves[3]
    out = attention.window_attention(*leaves[:3], s["segments"], **args)
    return (out.detach(), *torch.autograd.grad(out, leaves, s["grad"]))


# ----------------------------------------------------------------------------- plain forms

def _pairs_of(x: torch.Tensor, rot: int, interleaved: bool):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _turn(x, cos, sin, rot, interleaved):
    u, v = _pairs_of(x, rot, interleaved)
    a, b = u * cos - v * sin, u * sin + v * cos
    out = x.clone()
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = a, b
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = a, b
    return out


def _plain_rotate(s: dict):
    case = s["case"]
    rot, il = case["rot"], case["interleaved"]
    theta = (s["position"].float()[:, :, None] * s["freqs"][None]).sum(1)[:, None, :]
    cos, sin = torch.cos(theta), torch.sin(theta)
    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        outs.append(_turn(x * r * w, cos, sin, rot, il).to(s[name].dtype))
        if case["mode"] == "training":
            gy = _turn(s["grad_" + name].float(), cos, -sin, rot, il)
            weights.append((gy * (x * r)).sum((0, 1)))
            h = gy * w
            grads.append((r * h - x * (r ** 3) * (h * x).mean(-1, keepdim=True)).to(s[name].dtype))
    return (*outs, *grads, *weights)


def _blocks(case: dict, rows: list[int], keys: list[int]):
    """(first query row, end, position of the first, first key row, keys used) for each block of
    query rows: the keys used are the sinks and the block's window, local to the cloud."""
    q0 = k0 = 0
    for nq, nk in zip(rows, keys):
        for a in range(0, nq, _BLOCK):
            b = min(nq, a + _BLOCK)
            first, last = a + nk - nq, b - 1 + nk - nq
            lo = 0 if case["left"] < 0 else min(max(0, first - case["left"]), nk)
            right = 0 if case["causal"] else case["right"]
            hi = nk if right < 0 else max(lo, min(nk, last + right + 1))
            head = min(case["sinks"], lo)
            use = torch.cat([torch.arange(head, device="cuda"),
                             torch.arange(lo, hi, device="cuda")])
            yield q0 + a, q0 + b, first, k0, use
        q0, k0 = q0 + nq, k0 + nk


def _visible(case: dict, first: int, rows: int, use: torch.Tensor) -> torch.Tensor:
    p = torch.arange(first, first + rows, device="cuda")[:, None]
    j = use[None, :]
    seen = torch.ones(rows, use.numel(), dtype=torch.bool, device="cuda")
    if case["left"] >= 0:
        seen &= j >= p - case["left"]
    if case["right"] >= 0:
        seen &= j <= p + case["right"]
    seen |= j < case["sinks"]
    if case["causal"]:
        seen &= j <= p
    return seen


def _bucket_index(s: dict, a: int, b: int, kr: torch.Tensor) -> torch.Tensor:
    """(axes, rows, keys) bucket numbers."""
    reach = s["case"]["reach"]
    d = (s["key_position"][kr][None, :, :] - s["position"][a:b][:, None, :]).clamp(-reach, reach)
    d = (d + reach).long().permute(2, 0, 1)
    return d if s["buckets"] is None else s["buckets"].long()[d]


def _plain_attend(s: dict):
    case = s["case"]
    H, G, D = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    scale = 1.0 / math.sqrt(D)
    train, biased = case["mode"] == "training", case["bias"] != "none"
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    if train:
        dq = torch.empty(q.shape, dtype=torch.float32, device="cuda")
        dk = torch.zeros(k.shape, dtype=torch.float32, device="cuda")
        dv = torch.zeros(v.shape, dtype=torch.float32, device="cuda")
        dt = torch.zeros_like(s["table"]) if biased else None
    for a, b, first, k0, use in _blocks(case, *s["lengths"]):
        kr = k0 + use
        qf = q[a:b].float().transpose(0, 1)                                  # (H, rows, D)
        kf = k[kr].float().transpose(0, 1).repeat_interleave(G, 0)           # (H, keys, D)
        vf = v[kr].float().transpose(0, 1).repeat_interleave(G, 0)
        score = (qf @ kf.transpose(1, 2)) * scale
        if biased:
            idx = _bucket_index(s, a, b, kr)
            for axis in range(idx.shape[0]):
                score = score + s["table"][axis][idx[axis]].permute(2, 0, 1)
        seen = _visible(case, first, b - a, use)
        score = torch.where(seen, score, float("-inf"))
        top = score.amax(-1, keepdim=True) if use.numel() else score.new_zeros(H, b - a, 1)
        top = torch.where(top == float("-inf"), 0.0, top)
        p = torch.exp(score - top)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o = p @ vf
        out[a:b] = o.transpose(0, 1).to(out.dtype)
        if train:
            go = s["grad"][a:b].float().transpose(0, 1)
            dp = go @ vf.transpose(1, 2)
            ds = p * (dp - (go * o).sum(-1, keepdim=True))
            dq[a:b] = ((ds @ kf) * scale).transpose(0, 1)
            shared = (case["kv_heads"], G, use.numel(), D)
            dk[kr] += ((ds.transpose(1, 2) @ qf) * scale).view(shared).sum(1).transpose(0, 1)
            dv[kr] += (p.transpose(1, 2) @ go).view(shared).sum(1).transpose(0, 1)
            if biased:
                flat = ds.reshape(H, -1)
                names = torch.arange(s["table"].shape[1], device="cuda")
                for axis in range(idx.shape[0]):
                    hot = (idx[axis].reshape(-1, 1) == names).float()
                    dt[axis] += (flat @ hot).transpose(0, 1)
    if not train:
        return out
    grads = (out, dq.to(q.dtype), dk.to(q.dtype), dv.to(q.dtype))
    return (*grads, dt) if biased else grads


def run(state: dict):
    if state["case"]["op"] == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    return _own_attend(state) if own else _plain_attend(state)


# ----------------------------------------------------------------------------- work

def _visible_counts(case: dict, nq: int, nk: int) -> np.ndarray:
    """Visible keys of each query row of one cloud."""
    p = np.arange(nq) + nk - nq
    right = 0 if case["causal"] else case["right"]
    top = np.full(nq, nk) if right < 0 else np.clip(p + right + 1, 0, nk)
    low = np.zeros(nq, dtype=np.int64) if case["left"] < 0 else np.clip(p - case["left"], 0, nk)
    low = np.minimum(low, top)
    head = np.minimum(case["sinks"], low)
    if case["causal"]:
        head = np.minimum(head, np.clip(p + 1, 0, nk))
    return top - low + head


def work(case: dict) -> dict:
    H, K, D, size = case["heads"], case["kv_heads"], case["dim"], _SIZE[case["dtype"]]
    if case["op"] == "rotate":
        n = case["rows"]
        moved = n * (H + K) * D * size
        passes = 2 if case["mode"] == "forward" else 5  # training reads q and k once
        return {"bytes": passes * moved + 4 * n * case["axes"],
                "flops": n * (H + K) * D * (8 if case["mode"] == "forward" else 24)}
    rows, keys = _lengths(case)
    pairs, read = 0, 0
    for nq, nk in zip(rows, keys):
        seen = _visible_counts(case, nq, nk)
        pairs += int(seen.sum())
        read += int(seen.max()) if nq == 1 else nk
    nq = sum(rows)
    total = (2 * nq * H + 2 * read * K) * D * size
    if case["mode"] == "training":
        total += (2 * nq * H + 2 * read * K) * D * size  # grad in, dq, dk, dv
    if case["bias"] != "none":
        total += 4 * (3 if case["bias"] == "grid" else 1) * (nq + read)
    per = 4 if case["mode"] == "forward" else 12
    return {"bytes": total, "flops": per * D * H * pairs}


# ----------------------------------------------------------------------------- 64 bits

def _exact_rotate(s: dict):
    case = s["case"]
    rot, n = case["rot"], case["rows"]
    theta = s["position"].double() @ s["freqs"].double()
    turn = torch.polar(torch.ones_like(theta), theta)[:, None, :]
    leaves, outs = [], []
    for name in ("q", "k"):
        x = s[name].double().clone().requires_grad_()
        w = s[name + "_weight"].double().clone().requires_grad_()
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + 1e-6) * w
        head = y[..., :rot]
        if case["interleaved"]:
            z = torch.view_as_complex(head.reshape(n, -1, rot // 2, 2).contiguous()) * turn
            head = torch.view_as_real(z).reshape(n, -1, rot)
        else:
            z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
            head = torch.cat([z.real, z.imag], -1)
        outs.append(torch.cat([head, y[..., rot:]], -1))
        leaves.append((x, w))
    if case["mode"] == "forward":
        return tuple(o.detach() for o in outs)
    (q, wq), (k, wk) = leaves
    grads = torch.autograd.grad(outs, (q, k, wq, wk),
                                (s["grad_q"].double(), s["grad_k"].double()))
    return (*(o.detach() for o in outs), *grads)


def _exact_attend(s: dict):
    """Cloud by cloud, head by head, blocks of rows against all of the cloud's keys up to the last
    that the block can see, gradients by differentiation."""
    case = s["case"]
    H, G, D = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    train, biased = case["mode"] == "training", case["bias"] != "none"
    whole = [s[n].double().contiguous() for n in ("q", "k", "v")]
    if biased:
        whole.append(s["table"].double())
    result = torch.zeros(whole[0].shape, dtype=torch.float64, device="cuda")
    sums = [torch.zeros_like(x) for x in whole]
    row0 = key0 = 0
    for nq, nk in zip(*s["lengths"]):
        for start in range(0, nq, 1024):
            stop = min(nq, start + 1024)
            lo, hi = 0, nk
            if case["left"] >= 0:
                lo = min(max(start + nk - nq - case["left"], 0), nk)
            if case["causal"] or case["right"] >= 0:
                hi = min(nk, max(stop + nk - nq + (0 if case["causal"] else case["right"]), 0))
            j = torch.tensor(sorted(set(range(lo, hi)) | set(range(min(case["sinks"], nk)))),
                             dtype=torch.int64, device="cuda")
            p = torch.arange(start, stop, device="cuda") + (nk - nq)
            gap = j[None, :] - p[:, None]
            inside = torch.ones_like(gap, dtype=torch.bool)
            if case["left"] >= 0:
                inside = inside & (gap >= -case["left"])
            if case["right"] >= 0:
                inside = inside & (gap <= case["right"])
            inside = inside | (j < case["sinks"])[None, :]
            if case["causal"]:
                inside = inside & (gap <= 0)
            rows = slice(row0 + start, row0 + stop)
            if biased:
                step = s["key_position"][key0 + j].long()[None] - s["position"][rows].long()[:, None]
                step = torch.clamp(step, -case["reach"], case["reach"]) + case["reach"]
                if s["buckets"] is not None:
                    step = s["buckets"].long()[step]
            for h in range(H):
                parts = [whole[0][rows, h], whole[1][key0 + j, h // G], whole[2][key0 + j, h // G]]
                if biased:
                    parts.append(whole[3][:, :, h])
                parts = [x.clone().requires_grad_(train) for x in parts]
                x = parts[0] @ parts[1].T / math.sqrt(D)
                if biased:
                    for axis in range(step.shape[-1]):
                        x = x + parts[3][axis][step[..., axis]]
                x = x.masked_fill(~inside, -1e300)
                prob = torch.softmax(x, -1) * inside
                o = prob @ parts[2]
                result[rows, h] = o.detach()
                if train:
                    got = torch.autograd.grad(o, parts, s["grad"][rows, h].double())
                    sums[0][rows, h] = got[0]
                    sums[1][key0 + j, h // G] += got[1]
                    sums[2][key0 + j, h // G] += got[2]
                    if biased:
                        sums[3][:, :, h] += got[3]
        row0, key0 = row0 + nq, key0 + nk
    return (result, *sums) if train else result


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(state)
    pairs = work(case)["flops"] / case["dim"]
    if pairs > (7e9 if case["mode"] == "training" else 2e10):
        return None
    return _exact_attend(state)
