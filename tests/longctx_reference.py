"""Packed causal attention from its definition in 64 bits, with the most
that a computation in bf16 operands and fp32 sums may be off, element by
element.

A rounding to bf16 moves a value by at most u = 2**-8 of it.  The kernels
round the weights P (forward, dV), their gradient dS (dQ, dK) and the
result; delta = dO.O is taken from the rounded output.  So, with A = P|V|:

    O        u (A + |O|)                         weights, result
    delta    e = |dO| . u (A + |O|)              through O
    dV       u (P'|dO| + |dV|)
    dQ       scale (u |dS||K| + (e P)|K|) + u |dQ|
    dK       scale (u |dS|'|Q| + (e P)'|Q|) + u |dK|
    dtable   sum over the bucket of e P, u |dtable| where it is bf16

``SLACK`` of the same sums without signs covers what fp32 leaves: scores
of size s (here below 2**5) are off by s 2**-24 sqrt(d) at most and move
a weight by that factor; second orders of u are 2**-8 of the bounds and
are covered by the factor SECOND.
"""

import math

import torch

U = torch.finfo(torch.bfloat16).eps / 2
SLACK = 2.0 ** -15
SECOND = 1.02


def bucket_by_count(n, side, far):
    """Bucket of distance n: below half of them itself, else half and the
    number of steps of the logarithm passed."""
    half = side // 2
    steps = side - half
    if n < half:
        return n
    if n >= far:
        return side - 1
    return half + sum(n ** steps * half ** t >= far ** t * half ** steps
                      for t in range(1, steps))


def attention(q, k, v, lengths, scale=None, table=None, far=128, do=None):
    """({name: value}, {name: bound}) in 64 bits."""
    q, k, v = (t.detach().double() for t in (q, k, v))
    do = torch.zeros_like(q) if do is None else do.detach().double()
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    val = {n: torch.zeros_like(t) for n, t in
           (("o", q), ("dq", q), ("dk", k), ("dv", k))}
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    narrow = False
    if table is not None:
        narrow = table.dtype == torch.bfloat16
        table = table.detach().double()
        val["dtable"] = torch.zeros_like(table)
        tol["dtable"] = torch.zeros_like(table)
        by = torch.tensor([bucket_by_count(n, table.shape[0], far)
                           for n in range(max(lengths, default=0))],
                          dtype=torch.long, device=q.device)
    first = 0
    for n in lengths:
        at = slice(first, first + n)
        first += n
        i = torch.arange(n, device=q.device)
        gap = i[:, None] - i
        for h in range(heads if n else 0):
            g = h // group
            qh, kh, vh, dh = q[at, h], k[at, g], v[at, g], do[at, h]
            s = qh @ kh.T * scale
            if table is not None:
                which = by[gap.clamp(min=0)]
                s = s + table[:, h][which]
            s = s.masked_fill(gap < 0, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
            total = p.sum(-1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1)
            o = p @ vh
            val["o"][at, h] = o
            off = U * (p @ vh.abs() + o.abs())
            tol["o"][at, h] = off + SLACK * (p @ vh.abs())
            ds = p * (dh @ vh.T - (dh * o).sum(-1, keepdim=True))
            size = p * (dh.abs() @ vh.abs().T
                        + (dh * o).abs().sum(-1, keepdim=True))
            e = p * (dh.abs() * off).sum(-1, keepdim=True) + SLACK * size
            val["dv"][at, g] += p.T @ dh
            tol["dv"][at, g] += (U + SLACK) * (p.T @ dh.abs())
            val["dq"][at, h] = ds @ kh * scale
            tol["dq"][at, h] = (U * ds.abs() + e) @ kh.abs() * scale
            val["dk"][at, g] += ds.T @ qh * scale
            tol["dk"][at, g] += (U * ds.abs() + e).T @ qh.abs() * scale
            if table is not None:
                last = table.shape[0] - 1
                for b in range(table.shape[0]):
                    there = (which == b) & (gap >= 0)
                    val["dtable"][b, h] += ds[there].sum()
                    tol["dtable"][b, h] += e[there].sum()
                # the last bucket comes as minus the sum of the others
                tol["dtable"][last, h] += e[(which < last)
                                            & (gap >= 0)].sum()
    for name in tol:
        rounds = U if name != "dtable" or narrow else 2.0 ** -24
        if name == "o":
            tol[name] = SECOND * tol[name]
        else:
            tol[name] = SECOND * (tol[name] + rounds * val[name].abs())
    return val, tol


def check(got, want, bound, what):
    got = got.detach().double()
    off = (got - want).abs()
    bad = ~(off <= bound + 1e-30)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, first at "
        f"{tuple(bad.nonzero()[0].tolist())}: got "
        f"{got[bad][0].item():.6g}, want {want[bad][0].item():.6g}, "
        f"bound {bound.expand_as(want)[bad][0].item():.3g}")
