"""Balance loss, per-expert counts and the router's gradient on the GPU against the float64 formulas.

Tolerances: probability sums add up to n values in [0, 1] in float32, at most n * 2^-24 of the sum; the loss is a sum of
B * E such products, 16 more roundings; a gradient element is a handful of float32 operations on one token's values: 32 * 2^-24
of the sum of its |terms|."""
import pytest
import torch

from hap_amd import ops
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
E24 = 2.0 ** -24


def routing(cuda, seed, B, S, E, switch=False, capacity=None):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, S, E, generator=g) + torch.randn(1, 1, E, generator=g)
    gate = ops.switch_gate if switch else ops.top2_gate
    r = gate(logits.to(cuda), capacity or max(2, 2 * S // E))
    return r, torch.randn(B, S, 2, generator=g)


def outputs(cuda, B, S, E):
    nan = lambda *s: torch.full(s, float("nan"), device=cuda)  # noqa: E731
    whole = lambda: torch.full((B, E), -77, dtype=torch.int32, device=cuda)  # noqa: E731
    return nan(1), whole(), whole(), nan(B, E), nan(B, S, E)


CASES = [(1, 1, 2, 1, None, False), (2, 7, 4, 2, None, False), (3, 64, 5, 1, None, True), (4, 33, 16, 2, [33, 0, 1, 20], False), (2, 512, 64, 2, None, False),
         (1, 3000, 63, 2, [2999], False), (16, 512, 16, 1, None, False), (600, 5, 8, 2, None, False), (3, 900, 24, 1, [0, 0, 0], True), (1, 4097, 3, 2, None, False),
         (5, 300, 61, 2, [300, 299, -4, 1000, 1], False),
         # one block's work: several rows a wave, one token or few a load, tokens that do not fill a wave, empty rows
         (40, 6, 5, 2, [i % 7 for i in range(40)], False), (17, 64, 33, 2, None, False), (16, 63, 64, 1, None, True), (3, 300, 8, 2, [300, 257, 0], False),
         (1, 96, 63, 2, None, False), (7, 257, 2, 2, None, False), (48, 96, 4, 1, None, True), (2, 65, 3, 2, [65, 64], False)]


@pytest.mark.parametrize("B,S,E,choices,lengths,switch", CASES)
def test_loss_counts_and_gradient(cuda, B, S, E, choices, lengths, switch):
    r, dgate = routing(cuda, B + S + E, B, S, E, switch)
    loss, counts, kept, sums, d = outputs(cuda, B, S, E)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda)
    ops.balance_loss_fwd(r, loss, counts, kept, sums, choices=choices, coef=0.02, lengths=ln)
    cpu = {k: v.cpu() for k, v in r.items()}
    real = None if lengths is None else torch.tensor(lengths).clamp(0, S)
    wl, wc, wk, ws, wd = L.balance(cpu["probs"], cpu["index"], cpu["slot"], choices, 0.02, real)
    assert torch.equal(counts.cpu(), wc) and torch.equal(kept.cpu(), wk)
    assert ((sums.double().cpu() - ws).abs() <= S * E24 * ws).all()
    assert abs(loss.item() - wl.item()) <= (S + 16) * E24 * wl.item()
    ops.balance_loss_bwd(r, counts, d, choices=choices, coef=0.01, grad=2.0, lengths=ln)
    p = cpu["probs"].double()
    n = torch.full((B,), S) if real is None else real
    w = 0.02 * E * wc.double() / ((n > 0).sum().clamp(min=1) * choices * n.clamp(min=1)[:, None].double() ** 2)
    size = p * (w[:, None] + (p * w[:, None]).sum(-1, keepdim=True))
    assert ((d.double().cpu() - wd).abs() <= 32 * E24 * size + 1e-30).all()
    for b in range(B):
        assert (d[b, int(n[b]):] == 0).all()
    # with the gate's own gradient in the same pass
    _, _, _, _, both = L.balance(cpu["probs"], cpu["index"], cpu["slot"], choices, 0.02, real, dgate)
    ops.balance_loss_bwd(r, counts, d, choices=choices, coef=0.02, dgate=dgate.to(cuda), lengths=ln)
    dp = torch.zeros(B, S, E, dtype=torch.float64).scatter_add_(2, cpu["index"].long(), dgate.double().abs() * (cpu["slot"] > 0))
    size = size + p * (dp + (p * dp).sum(-1, keepdim=True))
    assert ((d.double().cpu() - both).abs() <= 32 * E24 * size + 1e-30).all()


def test_agrees_with_the_gate_backward_at_coefficient_zero(cuda):
    r, dgate = routing(cuda, 3, 4, 100, 16)
    loss, counts, kept, sums, d = outputs(cuda, 4, 100, 16)
    ops.balance_loss_fwd(r, loss, counts, kept, sums, coef=0.0)
    assert loss.item() == 0.0
    g = dgate.to(cuda)
    ops.balance_loss_bwd(r, counts, d, coef=0.0, dgate=g)
    want = torch.empty_like(d)
    ops.top2_gate_bwd(r, g, want)
    torch.testing.assert_close(d, want, rtol=1e-5, atol=1e-6)


def test_gradient_against_differences(cuda):
    """Counts do not move, so the loss is smooth in the logits: central differences along random directions.  The loss (about
    coef) carries 2^-24 * sqrt(B S) relative noise; over a step of 0.05 that is 1e-4 of the slope's scale."""
    B, S, E = 2, 200, 8
    g = torch.Generator().manual_seed(2)
    logits, step = torch.randn(B, S, E, generator=g), torch.randn(B, S, E, generator=g)
    r = ops.top2_gate(logits.to(cuda), 60)
    loss, counts, kept, sums, d = outputs(cuda, B, S, E)
    ops.balance_loss_fwd(r, loss, counts, kept, sums, coef=1.0)
    ops.balance_loss_bwd(r, counts, d, coef=1.0)
    vals = []
    for sign in (1, -1):
        moved = dict(r, probs=torch.softmax((logits + sign * 0.05 * step).to(cuda), -1).contiguous())
        ops.balance_loss_fwd(moved, loss, counts, kept, sums, coef=1.0)
        vals.append(loss.item())
    want = (d.double().cpu() * step.double()).sum().item()
    assert abs((vals[0] - vals[1]) / 0.1 - want) < 1e-2 * d.double().norm().item() * step.double().norm().item() ** 0.5


def test_an_expert_index_outside_the_range_counts_nowhere(cuda):
    r, _ = routing(cuda, 1, 1, 8, 4)
    r["index"][0, 3] = torch.tensor([-1, 4], dtype=torch.int32, device=cuda)
    loss, counts, kept, sums, _ = outputs(cuda, 1, 8, 4)
    ops.balance_loss_fwd(r, loss, counts, kept, sums, choices=2)
    assert counts.sum().item() == 14


def test_same_bits_every_time_and_in_a_replayed_graph(cuda):
    B, S, E = 3, 2000, 32
    r, dgate = routing(cuda, 8, B, S, E)
    loss, counts, kept, sums, d = outputs(cuda, B, S, E)
    ln, dg = torch.tensor([2000, 700, 1], dtype=torch.int32, device=cuda), dgate.to(cuda)

    def step():
        ops.balance_loss_fwd(r, loss, counts, kept, sums, lengths=ln)
        ops.balance_loss_bwd(r, counts, d, dgate=dg, lengths=ln)
    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (loss, counts, kept, sums, d)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert all(torch.equal(t, w) for t, w in zip((loss, counts, kept, sums, d), want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        for t in (loss, counts, kept, sums, d):
            t.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for t, w in zip((loss, counts, kept, sums, d), want)), i
        r["probs"].sum().item()


def test_refused_calls(cuda):
    r, dgate = routing(cuda, 1, 2, 8, 4)
    loss, counts, kept, sums, d = outputs(cuda, 2, 8, 4)
    f = lambda **kw: ops.balance_loss_fwd(**{**dict(r=r, loss=loss, counts=counts, kept=kept, prob_sum=sums), **kw})  # noqa: E731
    f()
    for kw, err in ((dict(counts=sums), TypeError), (dict(prob_sum=counts), TypeError), (dict(loss=sums), TypeError), (dict(kept=counts), ValueError),
                    (dict(choices=3), ops._lib.HapmiError), (dict(lengths=torch.zeros(2, device=cuda)), TypeError),
                    (dict(lengths=torch.zeros(3, dtype=torch.int32, device=cuda)), TypeError), (dict(r=dict(r, slot=r["slot"].long())), TypeError),
                    (dict(r=dict(r, index=r["index"][:1])), ops._lib.HapmiError)):
        with pytest.raises(err):
            f(**kw)
    with pytest.raises(ValueError):
        ops.balance_loss_bwd(r, counts, r["probs"])
    with pytest.raises(ops._lib.HapmiError):
        ops.balance_loss_bwd(r, counts, d, dgate=dgate[:, :4].to(cuda).contiguous())


@pytest.mark.parametrize("B,S,E,lengths", [(3, 100, 16, [60, 0, 100]), (2, 50, 5, [49, 1]), (4, 300, 64, [299, 7, 150, 300]), (5, 9, 33, [-3, 40, 8, 0, 9])])
@pytest.mark.parametrize("filler", [float("nan"), float("inf")])
def test_padding_may_hold_anything(cuda, B, S, E, lengths, filler):
    """Tokens that do not count: their probabilities are not finite, and no gate gradient reaches them (zero, or of a choice
    without a slot).  They get zeros, the others the bits that a clean padding gives."""
    r, dgate = routing(cuda, S, B, S, E)
    loss, counts, kept, sums, d = outputs(cuda, B, S, E)
    ln = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    pad = torch.arange(S, device=cuda)[None] >= ln[:, None]
    dirty = {k: v.clone() for k, v in r.items()}
    dirty["probs"][pad] = filler
    dirty["index"][pad] = -7
    dg = dgate.to(cuda)
    dg[pad] = 0.0
    dropped = dg.clone()
    dropped[pad] = filler
    dirty["slot"][pad] = 0
    clean = outputs(cuda, B, S, E)
    ops.balance_loss_fwd(r, *clean[:4], lengths=ln)
    ops.balance_loss_fwd(dirty, loss, counts, kept, sums, lengths=ln)
    assert torch.equal(loss, clean[0]) and torch.equal(counts, clean[1]) and torch.equal(kept, clean[2]) and torch.equal(sums, clean[3])
    for clean_gate, dirty_gate in ((None, None), (dg, dg), (dg, dropped)):
        want = clean[4]
        ops.balance_loss_bwd(r, counts, want, dgate=clean_gate, lengths=ln)
        d.fill_(float("nan"))
        ops.balance_loss_bwd(dirty, counts, d, dgate=dirty_gate, lengths=ln)
        assert (d[pad] == 0).all()
        assert torch.equal(d[~pad], want[~pad])


@pytest.mark.parametrize("B,S,E,choices,ragged", [(3000, 4, 8, 2, True), (1025, 40, 64, 2, True), (2049, 33, 33, 1, True), (1500, 3, 64, 1, False), (5000, 7, 2, 2, True)])
def test_more_rows_than_the_joining_block_has_threads(cuda, B, S, E, choices, ragged):
    """A row for every short sequence: the joining block walks the rows and their lengths in turns."""
    r, _ = routing(cuda, B, B, S, E)
    ln = torch.tensor([(i * 7) % (S + 2) - 1 for i in range(B)], dtype=torch.int32) if ragged else None
    n = ln.clamp(0, S).double() if ragged else torch.full((B,), float(S), dtype=torch.float64)
    loss, counts, kept, sums, d = outputs(cuda, B, S, E)
    up = None if ln is None else ln.to(cuda)
    ops.balance_loss_fwd(r, loss, counts, kept, sums, choices=choices, coef=0.02, lengths=up)
    ops.balance_loss_bwd(r, counts, d, choices=choices, coef=0.02, lengths=up)
    inside = torch.arange(S)[None] < n[:, None]
    p, index, slot = r["probs"].double().cpu(), r["index"].cpu().long()[..., :choices], r["slot"].cpu()[..., :choices]
    hit = torch.nn.functional.one_hot(index, E) * inside[:, :, None, None]
    wc, wk = hit.sum((1, 2)), (hit * (slot > 0)[..., None]).sum((1, 2))
    ws = (p * inside[..., None]).sum(1)
    w = 0.02 * E * wc.double() / ((n > 0).sum() * choices * n.clamp(min=1)[:, None] ** 2)
    want = (w * ws).sum().item()
    assert torch.equal(counts.cpu().long(), wc) and torch.equal(kept.cpu().long(), wk)
    assert ((sums.double().cpu() - ws).abs() <= S * E24 * ws).all()
    # a thread adds B E / 1024 products one after the other, the block 16 + 6 more, each product has 8 roundings and S of its sum
    assert abs(loss.item() - want) <= (S + 32 + B * E / 1024) * E24 * want
    g = torch.where(inside[..., None], w[:, None], torch.zeros(1, 1, 1, dtype=torch.float64))
    dot = (p * g).sum(-1, keepdim=True)
    assert ((d.double().cpu() - p * (g - dot)).abs() <= 32 * E24 * p * (g + dot) + 1e-30).all()
