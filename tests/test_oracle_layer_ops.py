"""The float64 formulas behind the GPU tests of the relative position bias, the per-head norm with rotation and the
balance loss: buckets against hand-worked values, gradients against autograd and against differences."""
import math

import pytest
import torch

from hap_amd import ops
from oracle import layer_ops as L


def test_buckets_at_hand_worked_distances():
    # 32 buckets over two sides, reach 128: 8 single distances, then borders at 8 * 16 ** (j / 8): 8, 11.3, 16, 22.6, 32, 45.3, 64, 90.5
    starts = ops.relative_bucket_starts(32, 128, True)
    assert starts == (0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)
    assert [L.bucket_of(r, 32, 128, True) for r in (0, -1, 1, -7, 7, -8, -11, -12, 15, 16, -90, -91, 5000)] == \
        [0, 1, 17, 7, 23, 8, 8, 9, 25, 26, 14, 15, 31]
    assert [L.bucket_of(r, 32, 128, False) for r in (3, 0, -1, -15, -16, -18, -19, -112, -113, -9999)] == [0, 0, 1, 15, 16, 16, 17, 30, 31, 31]


@pytest.mark.parametrize("n,reach,two", [(2, 9, False), (2, 1, True), (4, 2, True), (5, 17, False), (6, 4, True), (16, 9, True), (32, 128, True),
                                         (64, 1024, False), (128, 700, True), (3, 3, False), (64, 33, False)])
def test_bucket_starts_and_the_formula_agree(n, reach, two):
    side = n // 2 if two else n
    starts = ops.relative_bucket_starts(n, reach, two)
    assert len(starts) == side and starts[0] == 0
    for d in list(range(0, 200)) + [reach - 1, reach, reach + 1, 5 * reach]:
        want = max(k for k in range(side) if starts[k] <= d)
        assert L.bucket_of(-d, n, reach, two) == want
        if d:
            assert L.bucket_of(d, n, reach, two) == (want + side if two else 0)


@pytest.mark.parametrize("bad", [(1, 128, False), (7, 128, True), (0, 128, True), (32, 8, True), (32, 1 << 21, True), (130, 512, True),
                                 (64, 5000, False)])
def test_bucket_descriptions_that_are_refused(bad):
    with pytest.raises(ValueError, match="relative_bucket_starts"):
        ops.relative_bucket_starts(*bad)


def _inputs(seed, b=2, S=7, H=2, hd=4, n=8):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return r(b, S, 3 * H * hd), r(n, H), r(b, S, H * hd)


@pytest.mark.parametrize("causal,two,lens", [(False, True, None), (True, False, None), (True, True, [7, 0]), (False, False, [3, 5])])
def test_relative_bias_gradients(causal, two, lens):
    qkv, table, dout = _inputs(3)
    lengths = None if lens is None else torch.tensor(lens)
    args = (2, 0.5, 6, two, causal, lengths)
    g = torch.Generator().manual_seed(9)
    keep = torch.rand(2, 2, 7, 7, generator=g) > 0.3
    for kp in ({}, {"keep": keep, "p": 0.3}):
        x, t = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
        out, lse, _, _ = L.relbias_forward(x, t, *args, **kp)
        (out.reshape(2, 7, -1) * dout).sum().backward()
        got = L.relbias_backward(qkv, table, out.detach().reshape(2, 7, -1), dout, lse.detach(), *args, **kp)
        want = x.grad.view(2, 7, 3, 2, 4)
        for name, ref in (("dq", want[:, :, 0]), ("dk", want[:, :, 1]), ("dv", want[:, :, 2]), ("dtable", t.grad)):
            torch.testing.assert_close(got[name][0], ref, rtol=1e-10, atol=1e-12)
        step = 1e-5                                            # central differences of one table entry each
        f = lambda tt: (L.relbias_forward(qkv, tt, *args, **kp)[0].reshape(2, 7, -1) * dout).sum()  # noqa: E731
        for u, h in ((0, 0), (1, 1), (5, 0)):
            e = torch.zeros_like(table)
            e[u, h] = step
            diff = (f(table + e) - f(table - e)) / (2 * step)
            assert abs(diff - got["dtable"][0][u, h]) < 1e-7


@pytest.mark.parametrize("interleaved,rot", [(False, 8), (True, 8), (False, 4), (True, 2), (False, 0)])
def test_norm_and_rotation_gradients(interleaved, rot):
    b, S, H, D = 2, 3, 2, 8
    g = torch.Generator().manual_seed(rot)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    qkv, dout, qg, kg = r(b, S, 3 * H * D), r(b, S, 3 * H * D), r(D), r(D)
    angles = ops.rotary_table(S, rot).double()[None].expand(b, S, -1, 2) if rot else None
    x, a, c = qkv.clone().requires_grad_(True), qg.clone().requires_grad_(True), kg.clone().requires_grad_(True)
    (L.qk_norm_forward(x, H, a, c, angles, interleaved, 1e-6).reshape(b, S, -1) * dout).sum().backward()
    d, dq, dk, _, _ = L.qk_norm_backward(dout, qkv, H, qg, kg, angles, interleaved, 1e-6)
    torch.testing.assert_close(d.reshape(b, S, -1), x.grad, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(dq, a.grad, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(dk, c.grad, rtol=1e-10, atol=1e-12)


def test_rotation_keeps_pair_lengths_and_depends_on_distance_only():
    table = ops.rotary_table(70000, 16)
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(16, generator=g, dtype=torch.float64), torch.randn(16, generator=g, dtype=torch.float64)
    for inter in (False, True):
        dots = [torch.dot(L.turn(q, table[i], inter), L.turn(k, table[j], inter)) for i, j in ((5, 2), (1003, 1000), (69999, 69996))]
        assert max(dots) - min(dots) < 1e-5                   # the table is float32
        assert abs(L.turn(q, table[69999], inter).norm() - q.norm()) < 1e-5
    assert table.shape == (70000, 8, 2) and table.dtype == torch.float32
    assert abs(table[69999, 0, 1].item() - math.sin(69999.0)) < 1e-7


def test_balance_of_even_and_one_sided_routings():
    E, S = 4, 8
    even = torch.full((2, S, E), 1 / E)
    index = torch.stack([torch.arange(S) % E, (torch.arange(S) + 1) % E], -1).expand(2, S, 2)
    slot = torch.ones(2, S, 2, dtype=torch.int32)
    for k in (1, 2):
        loss, counts, kept, sums, _ = L.balance(even, index, slot, k, 0.01)
        assert abs(loss.item() - 0.01) < 1e-8 and (counts == k * S // E).all() and torch.equal(counts, kept)
    one = torch.zeros(1, S, E)
    one[..., 2] = 1
    loss, counts, kept, _, _ = L.balance(one, torch.full((1, S, 2), 2), torch.zeros(1, S, 2, dtype=torch.int32), 1, 0.01)
    assert abs(loss.item() - 0.01 * E) < 1e-12 and counts.tolist() == [[0, 0, S, 0]] and kept.sum() == 0


@pytest.mark.parametrize("choices,lens", [(1, None), (2, [5, 0, 6])])
def test_balance_gradient(choices, lens):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(3, 6, 5, generator=g, dtype=torch.float64)
    probs = torch.softmax(logits, -1)
    index = probs.topk(2, -1).indices
    slot = torch.randint(0, 2, (3, 6, 2), generator=g)
    dgate = torch.randn(3, 6, 2, generator=g, dtype=torch.float64)
    lengths = None if lens is None else torch.tensor(lens)
    x = logits.clone().requires_grad_(True)
    pr = torch.softmax(x, -1)
    loss, counts, _, _, d = L.balance(probs, index, slot, choices, 0.3, lengths, dgate)
    ns = torch.tensor(lens if lens else [6] * 3)
    total = 0.0
    for b, n in enumerate(ns.tolist()):
        if n:
            total = total + 0.3 * 5 / int((ns > 0).sum()) * (counts[b].double() / (choices * n) * pr[b, :n].mean(0)).sum()
    assert abs(total.item() - loss.item()) < 1e-12
    (total + (pr.gather(-1, index) * dgate * (slot > 0)).sum()).backward()
    torch.testing.assert_close(d, x.grad, rtol=1e-10, atol=1e-14)
