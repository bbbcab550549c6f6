"""Float64 formulas of attention with a relative position bias, the per-head norm with rotation, and the router's
balance loss.  TEST INFRASTRUCTURE ONLY; none of them has a reference counterpart.

Every backward function is written from its formula and also returns the sum of the absolute values of the terms that
each result adds up, from which the tests derive how far rounded inputs may move it.
"""
from __future__ import annotations

import math

import torch


def bucket_of(rel: int, n_buckets: int, max_distance: int, bidirectional: bool) -> int:
    """Bucket of one relative position (key - query), by exact whole-number comparisons."""
    side = n_buckets // 2 if bidirectional else n_buckets
    d = abs(rel) if bidirectional else max(-rel, 0)
    near = side // 2
    k = d if d < near else near
    if side > 1 and d >= near:
        wide = side - near
        while k < side - 1 and d ** wide >= max_distance ** (k + 1 - near) * near ** (wide - (k + 1 - near)):
            k += 1
    return k + (side if bidirectional and rel > 0 else 0)


def bucket_matrix(S, n_buckets, max_distance, bidirectional):
    row = torch.tensor([bucket_of(r, n_buckets, max_distance, bidirectional) for r in range(-(S - 1), S)])
    at = torch.arange(S)
    return row[at[None, :] - at[:, None] + S - 1]


def relbias_forward(qkv, table, H, scale, max_distance, bidirectional, causal, lengths=None, keep=None, p=0.0):
    """(out [b, S, H, 64], lse [b, H, S], probabilities [b, H, S, S], |terms| of out) in float64; a bias at or below -1e8
    hides its pairs; a query without visible keys gives zeros and -inf.  ``keep``: bool [b, H, S, S] dropout decisions."""
    b, S = qkv.shape[:2]
    q, k, v = (t.transpose(1, 2) for t in qkv.double().view(b, S, 3, H, -1).unbind(2))
    t = table.double()
    t = torch.where(t <= -1e8, torch.full_like(t, -math.inf), t)
    s = q @ k.transpose(-1, -2) * scale + t[bucket_matrix(S, table.shape[0], max_distance, bidirectional)].permute(2, 0, 1)
    at = torch.arange(S)
    hidden = torch.zeros(b, 1, S, S, dtype=torch.bool)
    if causal:
        hidden = hidden | (at[None, :] > at[:, None])
    if lengths is not None:
        inside = at[None, :] < lengths[:, None]
        hidden = hidden | ~(inside[:, None, :, None] & inside[:, None, None, :])
    s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, -1)
    prob = torch.where(torch.isinf(lse)[..., None], torch.zeros_like(s), (s - lse[..., None]).exp())
    drop = prob if keep is None else prob * keep.double() / (1 - p)
    out, terms = drop @ v, drop @ v.abs()
    return out.transpose(1, 2), lse, prob, terms.transpose(1, 2)


def relbias_backward(qkv, table, out, dout, lse, H, scale, max_distance, bidirectional, causal, lengths=None, keep=None, p=0.0):
    """Gradients from forward's ``out`` and ``lse`` as given: dict name -> (gradient, sum of the |products| that it adds up,
    the same with every score gradient replaced by the sum of its own |terms|); dq / dk / dv [b, S, H, 64], dtable
    [n_buckets, H]."""
    b, S = qkv.shape[:2]
    _, own_lse, prob, _ = relbias_forward(qkv, table, H, scale, max_distance, bidirectional, causal, lengths)
    shift = torch.where(torch.isinf(own_lse), torch.zeros_like(own_lse), own_lse - lse.double())
    prob = prob * shift.exp()[..., None]                       # normalised by the given lse
    q, k, v = (t.transpose(1, 2) for t in qkv.double().view(b, S, 3, H, -1).unbind(2))
    do, o = (t.double().view(b, S, H, -1).transpose(1, 2) for t in (dout, out))
    delta = (do * o).sum(-1, keepdim=True)
    dp = do @ v.transpose(-1, -2)
    mult = torch.ones_like(prob) if keep is None else keep.double() / (1 - p)
    ds = prob * (dp * mult - delta)
    size = prob * ((do.abs() @ v.abs().transpose(-1, -2)) * mult + (do * o).abs().sum(-1, keepdim=True))
    bucket = bucket_matrix(S, table.shape[0], max_distance, bidirectional).reshape(-1)
    to = lambda x: torch.zeros(table.shape[0], H, dtype=torch.float64).index_add_(0, bucket, x.sum(0).reshape(H, -1).t().contiguous())  # noqa: E731
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    pm = prob * mult
    return {"dq": (back(ds @ k) * scale, back(ds.abs() @ k.abs()) * scale, back(size @ k.abs()) * scale),
            "dk": (back(ds.transpose(-1, -2) @ q) * scale, back(ds.abs().transpose(-1, -2) @ q.abs()) * scale,
                   back(size.transpose(-1, -2) @ q.abs()) * scale),
            "dv": (back(pm.transpose(-1, -2) @ do), *(back(pm.transpose(-1, -2) @ do.abs()),) * 2),
            "dtable": (to(ds), to(ds.abs()), to(size))}


def _pairs(rot, interleaved):
    lo = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    return lo, (lo + 1 if interleaved else lo + rot // 2)


def turn(x, angles, interleaved, back=False):
    """x [..., D] with its first 2 * angles.shape[-2] dimensions turned; angles [..., rot / 2, 2] broadcast against it."""
    lo, hi = _pairs(2 * angles.shape[-2], interleaved)
    c, s = angles[..., 0].double(), angles[..., 1].double() * (-1 if back else 1)
    y = x.clone()
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y


def qk_norm_forward(qkv, H, q_gain, k_gain, angles, interleaved, eps):
    """angles [b, S, rot / 2, 2] (the positions' rows) or None -> [b, S, 3, H, D] float64."""
    b, S = qkv.shape[:2]
    q, k, v = qkv.double().view(b, S, 3, H, -1).unbind(2)
    parts = []
    for x, g in ((q, q_gain), (k, k_gain)):
        n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1.0 if g is None else g.double())
        parts.append(n if angles is None else turn(n, angles[:, :, None], interleaved))
    return torch.stack(parts + [v], 2)


def qk_norm_backward(dout, qkv, H, q_gain, k_gain, angles, interleaved, eps):
    """(dqkv [b, S, 3, H, D], dq_gain, dk_gain, |terms| of the two gain gradients) in float64."""
    b, S = qkv.shape[:2]
    x, d = qkv.double().view(b, S, 3, H, -1), dout.double().view(b, S, 3, H, -1).clone()
    gains = []
    for t, g in ((0, q_gain), (1, k_gain)):
        dn = d[:, :, t] if angles is None else turn(d[:, :, t], angles[:, :, None], interleaved, back=True)
        r = 1 / torch.sqrt((x[:, :, t] ** 2).mean(-1, keepdim=True) + eps)
        u = x[:, :, t] * r
        gains.append(((dn * u).sum((0, 1, 2)), (dn * u).abs().sum((0, 1, 2))))
        w = dn * (1.0 if g is None else g.double())
        d[:, :, t] = r * (w - u * (w * u).mean(-1, keepdim=True))
    return d, gains[0][0], gains[1][0], gains[0][1], gains[1][1]


def balance(probs, index, slot, choices, coef, lengths=None, dgate=None):
    """(loss, counts, kept, prob_sum, dlogits) of one routing, row by row."""
    B, S, E = probs.shape
    p = probs.double()
    counts, kept = torch.zeros(B, E, dtype=torch.int32), torch.zeros(B, E, dtype=torch.int32)
    sums, loss, d = torch.zeros(B, E, dtype=torch.float64), 0.0, torch.zeros(B, S, E, dtype=torch.float64)
    ns = [S if lengths is None else min(max(int(n), 0), S) for n in (lengths if lengths is not None else range(B))]
    rows = sum(n > 0 for n in ns)
    for b, n in enumerate(ns):
        for s in range(n):
            for k in range(choices):
                e = int(index[b, s, k])
                counts[b, e] += 1
                kept[b, e] += int(slot[b, s, k] > 0)
        sums[b] = p[b, :n].sum(0)
        if n:
            w = coef * E * counts[b].double() / (rows * choices * n * n)
            loss = loss + (w * sums[b]).sum()
            d[b, :n] += p[b, :n] * (w - (p[b, :n] * w).sum(-1, keepdim=True))
        if dgate is not None:
            dp = torch.zeros(S, E, dtype=torch.float64).scatter_add_(1, index[b].long(), dgate[b].double() * (slot[b] > 0))
            d[b] += p[b] * (dp - (p[b] * dp).sum(-1, keepdim=True))
    return torch.as_tensor(loss, dtype=torch.float64), counts, kept, sums, d
