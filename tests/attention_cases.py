"""Definitions in 64 bits of the attention of serialised clouds, for its tests.

``attention`` returns each result with an elementwise bound of what rounding may
do to it.  With u the unit roundoff of the element type (2^-24, 2^-11, 2^-8), to
first order:
  out   the stored value and, for 16-bit types, each weight round: u (|o| + sum P |v|);
  dv    as out: u (|dv| + sum P |do|);
  D     formed from the stored out: e_i = sum_d |do| u (|o| + sum P |v|); where the
        table's gradient is wanted, in float32 from the pairs themselves (allowed here:
        u replaced by 2^-15);
  dq    sum_j (u |dS| + P e_i) |k| scale + u |dq|; dk likewise over i;
  dT    sum over the pairs of a bucket of P e_i.
Float32 arithmetic adds to every score (64-term sums of exact products, the
exponent's argument, the exponential) at most eps_s below, absolutely, hence to
every weight 2 eps_s relatively, and to every product sum n 2^-23 of the sum of
magnitudes.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(lq, lk, left, right, sinks, causal):
    p = torch.arange(lq)[:, None] + lk - lq
    j = torch.arange(lk)[None, :]
    seen = torch.ones(lq, lk, dtype=torch.bool)
    if left >= 0:
        seen &= j >= p - left
    if right >= 0:
        seen &= j <= p + right
    seen |= j < sinks
    if causal:
        seen &= j <= p
    return seen


def bucket_index(qpos, kpos, reach, mapping):
    d = (kpos[None].long() - qpos[:, None].long()).clamp(-reach, reach) + reach
    return d if mapping is None else mapping.long()[d]


def attention(q, k, v, lens, key_lens, *, left=-1, right=-1, sinks=0, causal=False, scale=None,
              table=None, qpos=None, kpos=None, mapping=None, grad=None):
    """{name: (value, bound)} in float64 on the CPU; names out, lse and, with
    ``grad``, dq, dk, dv, dtable."""
    dtype = q.dtype
    u = UNIT[dtype]
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    H, K, D = q.shape[1], k.shape[1], q.shape[2]
    G = H // K
    scale = 1 / math.sqrt(D) if scale is None else scale
    uw = u if dtype != torch.float32 else 2.0 ** -22
    ud = 2.0 ** -15 if table is not None else uw   # precision of D
    out, out_b = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((H, q.shape[0]), -math.inf, dtype=torch.float64)
    lse_b = torch.zeros_like(lse)
    res = {}
    if table is not None:
        table = table.detach().cpu().double()
        qpos, kpos = qpos.cpu(), kpos.cpu()
        qpos = qpos[:, None] if qpos.ndim == 1 else qpos
        kpos = kpos[:, None] if kpos.ndim == 1 else kpos
        mapping = None if mapping is None else mapping.cpu()
        reach = (table.shape[1] if mapping is None else len(mapping)) // 2
    if grad is not None:
        grad = grad.detach().cpu().double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dq_b, dk_b, dv_b = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        if table is not None:
            dt, dt_b = torch.zeros_like(table), torch.zeros_like(table)
    q0 = k0 = 0
    for lq, lk in zip(lens, key_lens):
        seen = visible(lq, lk, left, right, sinks, causal)
        if table is not None and lq and lk:
            idx = bucket_index(qpos[q0:q0 + lq], kpos[k0:k0 + lk], reach, mapping)
        for h in range(H):
            if not lq or not lk:
                continue
            a, b, c = q[q0:q0 + lq, h], k[k0:k0 + lk, h // G], v[k0:k0 + lk, h // G]
            s = (a @ b.T) * scale
            mag = (a.abs() @ b.abs().T) * abs(scale)
            if table is not None:
                for ax in range(table.shape[0]):
                    bias = table[ax, :, h][idx[..., ax]]
                    s = s + bias
                    mag = mag + bias.abs().nan_to_num(0.0, 0.0, 0.0)
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True)
            top = top.masked_fill(top == -math.inf, 0.0)
            w = torch.exp(s - top)
            tot = w.sum(1, keepdim=True)
            p = torch.where(tot == 0, 0.0, w / tot)
            fin = mag.masked_fill(~seen, 0.0)
            eps = float(fin.max()) * (D + 8) * 2.0 ** -23 + 2.0 ** -20 if fin.numel() else 0.0
            pv = p @ c.abs()
            o = torch.where(seen[..., None], p[..., None] * c[None], 0.0).sum(1) \
                if not torch.isfinite(c).all() else p @ c
            ob = u * o.abs() + (uw + 2 * eps) * pv
            out[q0:q0 + lq, h], out_b[q0:q0 + lq, h] = o, ob
            row = torch.where(tot[:, 0] == 0, -math.inf, top[:, 0] + torch.log(tot[:, 0]))
            lse[h, q0:q0 + lq] = row
            lse_b[h, q0:q0 + lq] = 2 * eps + 2.0 ** -21 * row.abs().nan_to_num(0, 0, 0)
            if grad is None:
                continue
            g = grad[q0:q0 + lq, h]
            dp = g @ c.T
            delta = (g * o).sum(1, keepdim=True)
            e = (g.abs() * ((u if table is None else ud) * o.abs() + (ud + 2 * eps) * pv)) \
                .sum(1, keepdim=True)
            ds = torch.where(seen, p * (dp - delta), 0.0)
            n32 = (max(lq, lk) + D) * 2.0 ** -23
            dpm = g.abs() @ c.abs().T
            err32 = p * (e + D * 2.0 ** -23 * dpm + 2 * eps * ((dp - delta).abs() + dpm)) \
                + n32 * ds.abs()
            err = uw * ds.abs() + err32
            dq[q0:q0 + lq, h] = scale * (ds @ b)
            dq_b[q0:q0 + lq, h] = abs(scale) * (err @ b.abs()) + u * (scale * (ds @ b)).abs()
            dk[k0:k0 + lk, h // G] += scale * (ds.T @ a)
            dk_b[k0:k0 + lk, h // G] += abs(scale) * (err.T @ a.abs())
            dv[k0:k0 + lk, h // G] += p.T @ g
            dv_b[k0:k0 + lk, h // G] += (uw + 2 * eps + n32) * (p.T @ g.abs())
            if table is not None:
                for ax in range(table.shape[0]):
                    flat = idx[..., ax].reshape(-1)
                    dt[ax, :, h].index_add_(0, flat, ds.reshape(-1))
                    dt_b[ax, :, h].index_add_(0, flat, err32.reshape(-1))
        q0, k0 = q0 + lq, k0 + lk
    res["out"], res["lse"] = (out, out_b), (lse, lse_b)
    if grad is not None:
        res["dq"] = (dq, dq_b)
        res["dk"] = (dk, dk_b + u * dk.abs())
        res["dv"] = (dv, dv_b + u * dv.abs())
        if table is not None:
            res["dtable"] = (dt, dt_b)
    return res


def check(got, want, name, floor=1e-30):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, name
    inf = ~torch.isfinite(value)
    assert torch.equal(got[inf].nan_to_num(7.0), value[inf].nan_to_num(7.0)), f"{name}: non-finite"
    over = (got - value)[~inf].abs() - 1.02 * bound[~inf] - floor
    assert not torch.isnan(over).any(), f"{name}: NaN"
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{name}: {float(over.max()):.3g} over its bound ({float(bound.max()):.3g})"
