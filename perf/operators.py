"""The operators that a layer's training step takes from this library beside its GEMMs, as measured cases.

* attention with a learned relative position bias by buckets, forward and backward (bf16, packed projections);
* the norm of queries and keys per head with the position rotation, forward and backward (bf16 / float32);
* the router's balance loss with per-expert counts and its gradient (float32 / int32).

``run`` makes the library's calls where ``own`` is true and computes the same in elementary torch operations, in
float32, where it is false; ``exact`` is the definition in float64.
"""
import math
import random

import torch

own = False

HD = 64                                   # head dimension of the fused attention
NEG = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- the cases ------------------------------------------------------------------------------------------------

def _attn(name, way, b, S, H, causal=False, ragged=False, buckets=32, reach=128):
    return {"name": name, "op": "relbias", "way": way, "b": b, "S": S, "H": H, "causal": causal, "ragged": ragged,
            "buckets": buckets, "reach": reach}


def _norm(name, way, b, S, H, D, dtype, rot, interleaved=False, far=0):
    return {"name": name, "op": "qknorm", "way": way, "b": b, "S": S, "H": H, "D": D, "dtype": dtype, "rot": rot,
            "interleaved": interleaved, "far": far}


def _bal(name, B, S, E, choices, ragged=False, gate=False):
    return {"name": name, "op": "balance", "B": B, "S": S, "E": E, "choices": choices, "ragged": ragged, "gate": gate}


def listed():
    return [
        # a small language model's attention over a short context: every launch counts
        _attn("relbias_fwd_short", "fwd", 3, 128, 8),
        # the uneven shard of the bidirectional encoder that the benchmark trains: 12 samples of 512 tokens, 16 heads
        _attn("relbias_fwd_encoder", "fwd", 12, 512, 16),
        # one long document under the causal mask
        _attn("relbias_fwd_long_causal", "fwd", 1, 8192, 16, causal=True),
        # the encoder shard's backward pass with the table's gradient
        _attn("relbias_bwd_encoder", "bwd", 12, 512, 16),
        # a padded batch of odd length, 12 heads, a table of another size and reach
        _attn("relbias_bwd_ragged", "bwd", 6, 1001, 12, ragged=True, buckets=48, reach=300),
        # long causal training
        _attn("relbias_bwd_long_causal", "bwd", 2, 4096, 16, causal=True),
        # one new token for each of 48 running sequences, positions far into a table
        _norm("qknorm_fwd_one_token", "fwd", 48, 1, 16, 64, "bf16", 64, far=32768),
        # the encoder shard's packed projection
        _norm("qknorm_fwd_encoder", "fwd", 12, 512, 16, 64, "bf16", 64),
        # a long batch's backward pass with both gains' gradients
        _norm("qknorm_bwd_long", "bwd", 4, 8192, 16, 64, "bf16", 64),
        # float32 training of wider heads of which half is rotated, odd length, neighbouring pairs
        _norm("qknorm_bwd_odd", "bwd", 3, 333, 6, 128, "f32", 64, interleaved=True, far=4096),
        # the benchmark's routed layer: 16 rows of 512 tokens over 16 experts, loss, counts and gradient
        _bal("balance_layer", 16, 512, 16, 1),
        # a large padded batch over 64 experts, both choices counted, together with the gate's own gradient
        _bal("balance_large", 64, 2048, 64, 2, ragged=True, gate=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["relbias", "relbias", "qknorm", "balance"])
    if op == "relbias":
        way = rng.choice(["fwd", "bwd"])
        S = _log_int(rng, 9, 8192 if way == "fwd" else 4096)
        most = (1 << 30 if way == "fwd" else 1 << 29) // (S * S)
        H = rng.randint(1, max(1, min(16, most)))
        b = _log_int(rng, 1, max(1, min(24, most // H, 16384 // S)))
        buckets = 2 * rng.randint(4, 32)
        return {"op": op, "way": way, "b": b, "S": S, "H": H, "causal": rng.random() < 0.5, "ragged": rng.random() < 0.4,
                "buckets": buckets, "reach": _log_int(rng, buckets + 1, 512)}
    if op == "qknorm":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        D = rng.choice([32, 64, 64, 96, 128])
        H = rng.randint(1, 20)
        tokens = _log_int(rng, 1, (32768 * 1024) // (H * D) // (1 if dtype == "bf16" else 2))
        S = _log_int(rng, 1, min(8192, tokens))
        return {"op": op, "way": rng.choice(["fwd", "bwd"]), "b": max(1, min(256, tokens // S)), "S": S, "H": H, "D": D,
                "dtype": dtype, "rot": rng.choice([D, D // 2, 16]), "interleaved": rng.random() < 0.4,
                "far": rng.choice([0, 0, 20000])}
    S = _log_int(rng, 1, 8192)
    E = rng.randint(2, 64)
    B = _log_int(rng, 1, max(1, min(128, 131072 // S)))
    return {"op": op, "B": B, "S": S, "E": E, "choices": rng.choice([1, 2]), "ragged": rng.random() < 0.5,
            "gate": rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------------------------------------------

def _bucket_starts(half, reach):
    """starts[k]: the smallest distance of bucket k of one side.  The first half // 2 buckets hold one distance each,
    the others grow geometrically up to ``reach``: d >= exact * (reach / exact) ** (j / wide), in whole numbers."""
    exact_n = half // 2
    wide = half - exact_n
    return [*range(exact_n + 1),
            *(next(d for d in range(exact_n, reach + 1) if d ** wide >= reach ** j * exact_n ** (wide - j))
              for j in range(1, wide))]


def _row_lengths(case, n, S):
    """Lengths of a padded batch: the rows' fill grows evenly from a third to whole."""
    return [max(1, S - (2 * S // 3) * (n - 1 - i) // max(1, n - 1)) if n > 1 else max(1, 2 * S // 3) for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    st = dict(case)
    if case["op"] == "relbias":
        b, S, H = case["b"], case["S"], case["H"]
        half = case["buckets"] if case["causal"] else case["buckets"] // 2
        st["qkv"] = r(b, S, 3 * H * HD).bfloat16()
        st["table"] = r(case["buckets"], H)
        st["starts"] = torch.tensor(_bucket_starts(half, case["reach"]), device="cuda")
        st["scale"] = HD ** -0.5
        order = torch.randperm(b, generator=g, device="cuda")
        st["lengths"] = (torch.tensor(_row_lengths(case, b, S), dtype=torch.int32, device="cuda")[order].contiguous()
                         if case["ragged"] else None)
        st["out"] = torch.empty(b, S, H * HD, dtype=torch.bfloat16, device="cuda")
        st["lse"] = torch.empty(b, H, S, device="cuda")
        if case["way"] == "bwd":                       # what the forward pass has kept
            out, lse = _attention_forward(st)
            st["out"].copy_(out)
            st["lse"].copy_(lse)
            st["dout"] = r(b, S, H * HD).bfloat16()
            st["dqkv"] = torch.empty_like(st["qkv"])
            st["dtable"] = torch.empty_like(st["table"])
            st["delta"] = torch.empty(b, H, S, device="cuda")
    elif case["op"] == "qknorm":
        b, S, H, D, dt = case["b"], case["S"], case["H"], case["D"], DTYPES[case["dtype"]]
        st["qkv"] = (r(b, S, 3 * H * D) * 1.5).to(dt)
        st["q_gain"], st["k_gain"] = 1 + 0.2 * r(D), 1 + 0.2 * r(D)
        n_pos = case["far"] + S
        freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        angle = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * freq
        st["rotary"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        st["positions"] = None
        if case["far"]:
            first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")
            st["positions"] = (first + torch.arange(S, device="cuda")).to(torch.int32).contiguous()
        st["out"] = torch.empty_like(st["qkv"])
        if case["way"] == "bwd":
            st["dout"] = r(b, S, 3 * H * D).to(dt)
            st["dq_gain"], st["dk_gain"] = torch.empty_like(st["q_gain"]), torch.empty_like(st["k_gain"])
    else:
        B, S, E = case["B"], case["S"], case["E"]
        logits = r(B, S, E) + 0.5 * r(B, 1, E)         # some experts are liked better than others
        probs = torch.softmax(logits, -1)
        index = probs.topk(2, -1).indices
        gate = probs.gather(-1, index)
        seen = torch.nn.functional.one_hot(index, E).cumsum(1)          # [B, S, 2, E]: position among a choice's earlier ones
        place = seen.gather(-1, index[..., None])[..., 0]
        place[..., 1] += seen[:, -1, 0].gather(-1, index[..., 1])
        slots = max(2, 2 * S // E + 1)
        st["r"] = {"probs": probs.contiguous(), "index": index.int().contiguous(), "gate": gate.contiguous(),
                   "slot": torch.where(place < slots, place, 0).int().contiguous()}
        order = torch.randperm(B, generator=g, device="cuda")
        st["lengths"] = (torch.tensor(_row_lengths(case, B, S), dtype=torch.int32, device="cuda")[order].contiguous()
                         if case["ragged"] else None)
        st["dgate"] = r(B, S, 2) * 1e-3 if case["gate"] else None
        st["loss"] = torch.empty(1, device="cuda")
        st["counts"] = torch.empty(B, E, dtype=torch.int32, device="cuda")
        st["kept"] = torch.empty(B, E, dtype=torch.int32, device="cuda")
        st["prob_sum"] = torch.empty(B, E, device="cuda")
        st["dlogits"] = torch.empty(B, S, E, device="cuda")
    return st


# ---- plain forms ----------------------------------------------------------------------------------------------

COEF = 0.01                               # weight of the balance loss


def _relative(st):
    """Bucket of every relative position key - query from -(S - 1) to S - 1."""
    S, starts = st["S"], st["starts"]
    rel = torch.arange(-(S - 1), S, device="cuda")
    distance = (-rel).clamp(min=0) if st["causal"] else rel.abs()
    bucket = (distance[:, None] >= starts[1:]).sum(-1)
    return bucket if st["causal"] else bucket + (rel > 0) * starts.numel()


def _scores(st):
    b, S, H = st["b"], st["S"], st["H"]
    q, k, v = (t.transpose(1, 2) for t in st["qkv"].float().view(b, S, 3, H, HD).unbind(2))
    at = torch.arange(S, device="cuda")
    rel = at[None, :] - at[:, None]
    bias = st["table"].t()[:, _relative(st)][:, rel + S - 1]            # [H, S, S]
    s = q @ k.transpose(2, 3) * st["scale"] + bias
    if st["causal"]:
        s = s.masked_fill(rel > 0, NEG)
    if st["lengths"] is not None:
        inside = at[None, :] < st["lengths"][:, None]                   # [b, S]
        s = s.masked_fill(~(inside[:, None, :, None] & inside[:, None, None, :]), NEG)
    return q, k, v, s


def _attention_forward(st):
    b, S, H = st["b"], st["S"], st["H"]
    q, k, v, s = _scores(st)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == NEG, torch.zeros_like(m), m)
    p = (s - m).exp()
    del s
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.transpose(1, 2).reshape(b, S, H * HD).bfloat16(), (m + total.log())[..., 0]


def _attention_backward(st):
    b, S, H = st["b"], st["S"], st["H"]
    heads = lambda t: t.float().view(b, S, H, HD).transpose(1, 2)  # noqa: E731
    q, k, v, s = _scores(st)
    lse = st["lse"][..., None]
    p = torch.where(lse == NEG, torch.zeros_like(s), (s - lse).exp())
    del s
    do = heads(st["dout"])
    delta = (do * heads(st["out"])).sum(-1, keepdim=True)
    dv = p.transpose(2, 3) @ do
    ds = p * (do @ v.transpose(2, 3) - delta)
    del p
    dq, dk = ds @ k * st["scale"], ds.transpose(2, 3) @ q * st["scale"]
    # sums along the diagonals: rows flipped and shifted against each other by one column each
    wide = torch.nn.functional.pad(ds.sum(0).flip(1), (0, S)).view(H, -1)[:, :S * (2 * S - 1)]
    along = wide.view(H, S, 2 * S - 1).double().sum(1)                  # [H, 2 S - 1]
    dtable = (torch.nn.functional.one_hot(_relative(st), st["buckets"]).double().t() @ along.t()).float()
    dqkv = torch.stack([t.transpose(1, 2) for t in (dq, dk, dv)], 2).reshape(b, S, 3 * H * HD).bfloat16()
    return dqkv, dtable


def _rotate(st, x, sign):
    """x [b, S, H, D], the first ``rot`` dimensions turned by the position's angles (sign -1: back)."""
    rot, tab = st["rot"], st["rotary"]
    tab = tab[st["positions"].long()] if st["positions"] is not None else tab[:st["S"]]
    c, s = tab[..., None, :, 0], tab[..., None, :, 1] * sign
    x0, x1 = (x[..., 0:rot:2], x[..., 1:rot:2]) if st["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = (x0 * c - x1 * s, x0 * s + x1 * c)
    y = torch.stack(y, -1).flatten(-2) if st["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., rot:]], -1)


EPS = 1e-6


def _norm_forward(st):
    b, S, H, D = st["b"], st["S"], st["H"], st["D"]
    x = st["qkv"].view(b, S, 3, H, D)
    each = lambda t, gain: _rotate(st, t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain, 1)  # noqa: E731
    q, k = each(x[:, :, 0].float(), st["q_gain"]), each(x[:, :, 1].float(), st["k_gain"])
    return torch.stack([q.to(x.dtype), k.to(x.dtype), x[:, :, 2]], 2).view(b, S, 3 * H * D)


def _norm_backward(st):
    b, S, H, D = st["b"], st["S"], st["H"], st["D"]
    x, dy = st["qkv"].view(b, S, 3, H, D), st["dout"].view(b, S, 3, H, D)

    def each(t, d, gain):
        rs = (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
        unit, dn = t * rs, _rotate(st, d, -1)
        w = dn * gain
        return rs * (w - unit * (w * unit).mean(-1, keepdim=True)), (dn * unit).sum((0, 1, 2), dtype=torch.float64).float()

    dq, dgq = each(x[:, :, 0].float(), dy[:, :, 0].float(), st["q_gain"])
    dk, dgk = each(x[:, :, 1].float(), dy[:, :, 1].float(), st["k_gain"])
    return torch.stack([dq.to(x.dtype), dk.to(x.dtype), dy[:, :, 2]], 2).view(b, S, 3 * H * D), dgq, dgk


def _balance(st):
    B, S, E, k, r = st["B"], st["S"], st["E"], st["choices"], st["r"]
    n = st["lengths"].long() if st["lengths"] is not None else torch.full((B,), S, device="cuda")
    inside = torch.arange(S, device="cuda") < n[:, None]
    hit = torch.nn.functional.one_hot(r["index"][..., :k].long(), E) * inside[..., None, None]
    counts = hit.sum((1, 2))
    kept = (hit * (r["slot"][..., :k, None] > 0)).sum((1, 2))
    p = r["probs"] * inside[..., None]
    prob_sum = p.sum(1)
    per_row = COEF * E / (n > 0).sum().clamp(min=1) / (k * n.clamp(min=1).double() ** 2)
    loss = (per_row * (counts * prob_sum.double()).sum(-1)).sum().float().view(1)
    w = (per_row[:, None] * counts).float()[:, None, :]
    d = p * (w - (p * w).sum(-1, keepdim=True))
    if st["dgate"] is not None:
        dg = torch.where(r["slot"] > 0, st["dgate"], torch.zeros_like(st["dgate"]))
        onto = (torch.nn.functional.one_hot(r["index"].long(), E) * dg[..., None]).sum(2)
        d = d + r["probs"] * (onto - (r["probs"] * onto).sum(-1, keepdim=True))
    return loss, counts.int(), kept.int(), prob_sum, d


def run(st):
    op = st["op"]
    if own:
        from hap_amd import ops
        if op == "relbias":
            at = dict(max_distance=st["reach"], causal=st["causal"], lengths=st["lengths"])
            if st["way"] == "fwd":
                ops.attention_relbias_fwd(st["qkv"], st["table"], st["out"], st["lse"], st["b"], st["S"], st["H"],
                                          st["scale"], **at)
                return st["out"], st["lse"]
            ops.attention_relbias_bwd(st["qkv"], st["table"], st["out"], st["dout"], st["lse"], st["dqkv"], st["dtable"],
                                      st["delta"], st["b"], st["S"], st["H"], st["scale"], **at)
            return st["dqkv"], st["dtable"]
        if op == "qknorm":
            at = dict(q_gain=st["q_gain"], k_gain=st["k_gain"], rotary=st["rotary"], positions=st["positions"],
                      interleaved=st["interleaved"], eps=EPS)
            if st["way"] == "fwd":
                ops.qk_norm_rotary_fwd(st["qkv"], st["out"], st["b"], st["S"], st["H"], **at)
                return st["out"]
            ops.qk_norm_rotary_bwd(st["dout"], st["qkv"], st["out"], st["b"], st["S"], st["H"], dq_gain=st["dq_gain"],
                                   dk_gain=st["dk_gain"], **at)
            return st["out"], st["dq_gain"], st["dk_gain"]
        ops.balance_loss_fwd(st["r"], st["loss"], st["counts"], st["kept"], st["prob_sum"], choices=st["choices"],
                             coef=COEF, lengths=st["lengths"])
        ops.balance_loss_bwd(st["r"], st["counts"], st["dlogits"], choices=st["choices"], coef=COEF, dgate=st["dgate"],
                             lengths=st["lengths"])
        return st["loss"], st["counts"], st["kept"], st["prob_sum"], st["dlogits"]
    if op == "relbias":
        return _attention_forward(st) if st["way"] == "fwd" else _attention_backward(st)
    if op == "qknorm":
        return _norm_forward(st) if st["way"] == "fwd" else _norm_backward(st)
    return _balance(st)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    if case["op"] == "relbias":
        b, S, H = case["b"], case["S"], case["H"]
        lens = _row_lengths(case, b, S) if case["ragged"] else [S] * b
        pairs = H * sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        packed, head = 2 * 3 * H * HD, 2 * H * HD                       # bytes of a token
        table = 4 * case["buckets"] * H
        if case["way"] == "fwd":
            return {"bytes": sum(lens) * packed + b * S * (head + 4 * H) + table, "flops": 4 * HD * pairs}
        return {"bytes": sum(lens) * (packed + 2 * head + 4 * H) + b * S * packed + 2 * table, "flops": 10 * HD * pairs}
    if case["op"] == "qknorm":
        size = 2 if case["dtype"] == "bf16" else 4
        tokens, E = case["b"] * case["S"], case["H"] * case["D"]
        angles = 4 * case["rot"] * (min(tokens, case["far"] + case["S"]) if case["far"] else case["S"])
        if case["way"] == "fwd":
            return {"bytes": tokens * 6 * E * size + angles, "flops": tokens * 2 * E * 7}
        return {"bytes": tokens * 8 * E * size + angles, "flops": tokens * 2 * E * 13}
    B, S, E = case["B"], case["S"], case["E"]
    records = 4 * case["choices"] * 2 + (16 if case["gate"] else 0)
    return {"bytes": B * S * (2 * 4 * E + records) + 16 * B * E, "flops": B * S * E * 6}


# ---- the definitions in float64 ---------------------------------------------------------------------------------

def _bucket_of(case, distance):
    """Bucket of distances on one side from the logarithm, in float64; a distance on a border belongs to the farther bucket."""
    half = case["buckets"] if case["causal"] else case["buckets"] // 2
    near = half // 2
    far = near + torch.floor(torch.log(distance.clamp(min=1).double() / near) / math.log(case["reach"] / near) * (half - near)
                             + 1e-9).long()
    return torch.where(distance < near, distance, far.clamp(max=half - 1))


def _exact_attention(case, st):
    b, S, H = case["b"], case["S"], case["H"]
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None, :]
    bucket = _bucket_of(case, (i - j).clamp(min=0) if case["causal"] else (i - j).abs())
    if not case["causal"]:
        bucket = bucket + (j > i) * (case["buckets"] // 2)
    visible = (j <= i) if case["causal"] else torch.ones(S, S, dtype=torch.bool, device="cuda")
    table = st["table"].double()
    out = torch.zeros(b, S, H, HD, dtype=torch.float64, device="cuda")
    lse = torch.full((b, H, S), NEG, dtype=torch.float64, device="cuda")
    dqkv = torch.zeros(b, S, 3, H, HD, dtype=torch.float64, device="cuda")
    dtable = torch.zeros(case["buckets"], H, dtype=torch.float64, device="cuda")
    x = st["qkv"].view(b, S, 3, H, HD)
    for z in range(b):
        n = int(st["lengths"][z]) if st["lengths"] is not None else S
        for h in range(H):
            q, k, v = (x[z, :n, t, h].double() for t in range(3))
            s = (torch.mm(q, k.t().contiguous()) * st["scale"] + table[:, h][bucket[:n, :n]]).masked_fill(~visible[:n, :n], NEG)
            if case["way"] == "fwd":
                lse[z, h, :n] = torch.logsumexp(s, 1)
                out[z, :n, h] = torch.mm(torch.softmax(s, 1), v)
                continue
            p = torch.exp(s - st["lse"][z, h, :n, None].double())
            do = st["dout"].view(b, S, H, HD)[z, :n, h].double()
            o = st["out"].view(b, S, H, HD)[z, :n, h].double()
            ds = p * (torch.mm(do, v.t().contiguous()) - (do * o).sum(1)[:, None])
            dqkv[z, :n, 0, h] = torch.mm(ds, k) * st["scale"]
            dqkv[z, :n, 1, h] = torch.mm(ds.t().contiguous(), q) * st["scale"]
            dqkv[z, :n, 2, h] = torch.mm(p.t().contiguous(), do)
            dtable[:, h] += torch.bincount(bucket[:n, :n].reshape(-1), weights=ds.reshape(-1), minlength=case["buckets"])
    if case["way"] == "fwd":
        return out.view(b, S, H * HD), lse
    return dqkv.view(b, S, 3 * H * HD), dtable


def _exact_norm(case, st):
    b, S, H, D, rot = case["b"], case["S"], case["H"], case["D"], case["rot"]
    lo = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
    hi = lo + 1 if case["interleaved"] else lo + rot // 2
    pos = st["positions"].long() if st["positions"] is not None else torch.arange(S, device="cuda").expand(b, S)
    turn = torch.view_as_complex(st["rotary"].double())[pos][:, :, None, :]           # [b, S, 1, rot / 2]
    x = st["qkv"].double().view(b, S, 3, H, D)
    grads, res = [], torch.empty_like(x)
    for t, gain in ((0, st["q_gain"]), (1, st["k_gain"])):
        gain = gain.double()
        r = 1 / torch.sqrt((x[:, :, t] ** 2).mean(-1, keepdim=True) + EPS)
        u = x[:, :, t] * r
        if case["way"] == "fwd":
            y = u * gain
            z = torch.complex(y[..., lo], y[..., hi]) * turn
            y[..., lo], y[..., hi] = z.real, z.imag
            res[:, :, t] = y
        else:
            dy = st["dout"].double().view(b, S, 3, H, D)[:, :, t].clone()
            z = torch.complex(dy[..., lo], dy[..., hi]) * turn.conj()
            dy[..., lo], dy[..., hi] = z.real, z.imag
            grads.append((dy * u).sum((0, 1, 2)))
            du = dy * gain
            res[:, :, t] = r * du - u * r * (du * u).sum(-1, keepdim=True) / D
    res[:, :, 2] = (st["qkv"] if case["way"] == "fwd" else st["dout"]).double().view(b, S, 3, H, D)[:, :, 2]
    return res.view(b, S, 3 * H * D) if case["way"] == "fwd" else (res.view(b, S, 3 * H * D), *grads)


def _exact_balance(case, st):
    B, S, E, k, r = case["B"], case["S"], case["E"], case["choices"], st["r"]
    lengths = st["lengths"].tolist() if st["lengths"] is not None else [S] * B
    rows = sum(n > 0 for n in lengths)
    probs = r["probs"].double()
    counts = torch.zeros(B, E, dtype=torch.int32, device="cuda")
    kept, sums = torch.zeros_like(counts), torch.zeros(B, E, dtype=torch.float64, device="cuda")
    loss, d = torch.zeros(1, dtype=torch.float64, device="cuda"), torch.zeros(B, S, E, dtype=torch.float64, device="cuda")
    for z, n in enumerate(lengths):
        if st["dgate"] is not None:
            dp = torch.zeros(S, E, dtype=torch.float64, device="cuda")
            dp.scatter_add_(1, r["index"][z].long(), st["dgate"][z].double() * (r["slot"][z] > 0))
            d[z] += probs[z] * dp - probs[z] * (probs[z] * dp).sum(1, keepdim=True)
        if n == 0:
            continue
        chosen, slot = r["index"][z, :n, :k].reshape(-1).long(), r["slot"][z, :n, :k].reshape(-1)
        counts[z] = torch.bincount(chosen, minlength=E)
        kept[z] = torch.bincount(chosen[slot > 0], minlength=E)
        sums[z] = probs[z, :n].sum(0)
        w = COEF * E * counts[z].double() / (rows * k * n * n)
        loss += (w * sums[z]).sum()
        d[z, :n] += probs[z, :n] * w - probs[z, :n] * (probs[z, :n] @ w)[:, None]
    return loss, counts, kept, sums, d


def exact(case, seed):
    st = prepare(case, seed)
    return {"relbias": _exact_attention, "qknorm": _exact_norm, "balance": _exact_balance}[case["op"]](case, st)
