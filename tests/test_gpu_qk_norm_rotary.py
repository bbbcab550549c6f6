"""Per-head norm with rotation on the GPU against its float64 formula.

Tolerances: one rounding to the element type, u = eps / 2 of the value; in float32 before it, a mean of up to 256 squares
and some ten multiplications and additions of one head's values: below 64 * 2^-24 = 4e-6 of the largest value that enters, F =
1e-5.  Gain gradients are float32 sums of up to a few thousand terms a lane and tree sums above that: F of the sum of |terms|."""
import pytest
import torch

from hap_amd import ops
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
F = 1e-5
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def within(got, want, tol, what):
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got.double().cpu() - want).abs()[bad].max().item())


def make(seed, b, S, H, D, dtype, rot, far):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    qkv, dout = (r(b, S, 3 * H * D) * 1.5).to(dtype), r(b, S, 3 * H * D).to(dtype)
    table = ops.rotary_table(far + S, rot) if rot else None
    pos = (torch.randint(0, far + 1, (b, 1), generator=g) + torch.arange(S)).int() if far else None
    return qkv, dout, 1 + 0.3 * r(D), 1 + 0.3 * r(D), table, pos


def rows(table, pos, b, S):
    if table is None:
        return None
    return table[pos.long()] if pos is not None else table[:S][None].expand(b, S, -1, 2)


CASES = [  # b, S, H, D, dtype, rot, interleaved, far
    (2, 5, 3, 64, torch.bfloat16, 64, False, 0), (1, 1, 1, 64, torch.bfloat16, 64, True, 100000), (48, 1, 16, 64, torch.bfloat16, 64, False, 5000),
    (1, 333, 6, 128, torch.float32, 64, True, 4096), (2, 40, 5, 96, torch.bfloat16, 32, False, 0), (2, 40, 5, 96, torch.float32, 48, False, 10),
    (3, 17, 2, 8, torch.bfloat16, 8, True, 0), (3, 17, 2, 4, torch.float32, 0, False, 0), (2, 9, 3, 16, torch.bfloat16, 16, False, 0),
    (1, 130, 20, 32, torch.bfloat16, 16, True, 300), (1, 70, 2, 256, torch.bfloat16, 256, False, 0), (1, 70, 2, 256, torch.float32, 256, True, 0),
    (2, 33, 7, 40, torch.bfloat16, 16, False, 0), (2, 33, 7, 24, torch.bfloat16, 8, True, 0), (2, 31, 3, 12, torch.float32, 8, False, 5),
    (4, 200, 16, 64, torch.bfloat16, 0, False, 0), (2, 700, 16, 64, torch.float32, 64, False, 0)]


@pytest.mark.parametrize("b,S,H,D,dtype,rot,inter,far", CASES)
@pytest.mark.parametrize("gains", [True, False])
def test_forward_and_backward(cuda, b, S, H, D, dtype, rot, inter, far, gains):
    qkv, dout, qg, kg, table, pos = make(D + S, b, S, H, D, dtype, rot, far)
    if not gains:
        qg = kg = None
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    kw = dict(q_gain=up(qg), k_gain=up(kg), rotary=up(table), positions=up(pos), interleaved=inter, eps=1e-5)
    x, d = up(qkv), up(dout)
    out = torch.full_like(x, float("nan"))
    ops.qk_norm_rotary_fwd(x, out, b, S, H, **kw)
    ang = rows(table, pos, b, S)
    want = L.qk_norm_forward(qkv, H, qg, kg, ang, inter, 1e-5)
    big = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
    got = out.view(b, S, 3, H, D)
    within(got[:, :, :2], want[:, :, :2], (U[dtype] * want.abs() + F * big(want))[:, :, :2], "forward")
    assert torch.equal(got[:, :, 2], x.view(b, S, 3, H, D)[:, :, 2])
    same = x.clone()
    ops.qk_norm_rotary_fwd(same, same, b, S, H, **kw)          # in place: the same bits
    assert torch.equal(same, out)

    dx = torch.full_like(x, float("nan"))
    dqg, dkg = (torch.full((D,), float("nan"), device=cuda) for _ in range(2)) if gains else (None, None)
    ops.qk_norm_rotary_bwd(d, x, dx, b, S, H, dq_gain=dqg, dk_gain=dkg, **kw)
    wd, wq, wk, sq, sk = L.qk_norm_backward(dout, qkv, H, qg, kg, ang, inter, 1e-5)
    xs = qkv.double().view(b, S, 3, H, D)
    r = 1 / torch.sqrt((xs * xs).mean(-1, keepdim=True) + 1e-5)
    size = r * big(dout.double().view(b, S, 3, H, D)) * (2 if qg is None else 2 * max(qg.abs().max(), kg.abs().max()).item()) * (1 + big(xs * r))
    got = dx.view(b, S, 3, H, D)
    within(got[:, :, :2], wd[:, :, :2], (U[dtype] * wd.abs() + F * size)[:, :, :2], "dqkv")
    assert torch.equal(got[:, :, 2], d.view(b, S, 3, H, D)[:, :, 2])
    if gains:
        within(dqg, wq, F * sq, "dq_gain")
        within(dkg, wk, F * sk, "dk_gain")
    into = d.clone()
    aq, ak = (torch.full((D,), 4.0, device=cuda), torch.full((D,), -3.0, device=cuda)) if gains else (None, None)
    ops.qk_norm_rotary_bwd(into, x, into, b, S, H, dq_gain=aq, dk_gain=ak, accumulate=True, **kw)
    assert torch.equal(into, dx)
    if gains:
        assert torch.equal(aq, dqg + 4.0) and torch.equal(ak, dkg - 3.0)


def test_one_gain_only(cuda):
    qkv, dout, qg, kg, table, _ = make(1, 2, 30, 3, 64, torch.bfloat16, 64, 0)
    x, d, t = qkv.to(cuda), dout.to(cuda), table.to(cuda)
    full = [torch.empty(64, device=cuda) for _ in range(2)]
    dx = torch.empty_like(x)
    kw = dict(q_gain=qg.to(cuda), k_gain=kg.to(cuda), rotary=t)
    ops.qk_norm_rotary_bwd(d, x, dx, 2, 30, 3, dq_gain=full[0], dk_gain=full[1], **kw)
    only = torch.empty(64, device=cuda)
    ops.qk_norm_rotary_bwd(d, x, dx, 2, 30, 3, dk_gain=only, **kw)
    assert torch.equal(only, full[1])


def test_gradient_against_differences(cuda):
    """Directional central differences of sum(out * weight) in float32: the quotient's own rounding is 2^-24 * sqrt(terms) *
    |out| / step = 3e-3 for 1536 terms and a step of 1e-2, its curvature below 1e-3 relative."""
    b, S, H, D = 2, 8, 2, 32
    qkv, weight, qg, kg, table, _ = make(2, b, S, H, D, torch.float32, 32, 0)
    g = torch.Generator().manual_seed(5)
    x, w, t = qkv.to(cuda), weight.to(cuda), table.to(cuda)
    a, c = qg.to(cuda), kg.to(cuda)
    dirs = [torch.randn(*s.shape, generator=g).to(cuda) for s in (x, a, c)]
    out = torch.empty_like(x)

    def f(x_, a_, c_):
        ops.qk_norm_rotary_fwd(x_, out, b, S, H, q_gain=a_, k_gain=c_, rotary=t)
        return (out.double() * w.double()).sum().item()
    dx, dq, dk = torch.empty_like(x), torch.empty_like(a), torch.empty_like(c)
    ops.qk_norm_rotary_bwd(w, x, dx, b, S, H, q_gain=a, k_gain=c, dq_gain=dq, dk_gain=dk, rotary=t)
    h = 1e-2
    for base, grad, i in ((x, dx, 0), (a, dq, 1), (c, dk, 2)):
        args = [x, a, c]
        args[i] = base + h * dirs[i]
        hi = f(*args)
        args[i] = base - h * dirs[i]
        lo = f(*args)
        want = (grad.double() * dirs[i].double()).sum().item()
        assert abs((hi - lo) / (2 * h) - want) < 1e-2 * max(1.0, grad.double().norm().item()), i


def test_positions_outside_the_table_give_nan_and_nothing_else(cuda):
    qkv, dout, qg, kg, table, _ = make(1, 2, 6, 2, 64, torch.bfloat16, 64, 0)
    pos = torch.arange(6).repeat(2, 1).int()
    pos[0, 2], pos[1, 5] = -1, 6
    x, out = qkv.to(cuda), torch.empty_like(qkv, device=cuda)
    ops.qk_norm_rotary_fwd(x, out, 2, 6, 2, rotary=table.to(cuda), positions=pos.to(cuda))
    nan = torch.isnan(out.view(2, 6, 3, 2, 64))
    want = torch.zeros_like(nan)
    want[0, 2, :2] = want[1, 5, :2] = True
    assert torch.equal(nan, want)


def test_zero_rows_and_empty_batch(cuda):
    x = torch.zeros(1, 4, 3 * 64, dtype=torch.bfloat16, device=cuda)
    out = torch.full_like(x, 9)
    ops.qk_norm_rotary_fwd(x, out, 1, 4, 1, eps=1e-6)
    assert (out == 0).all()
    ops.qk_norm_rotary_fwd(x[:0], out[:0], 0, 4, 1)


def test_offsets_beyond_32_bits(cuda):
    b, S, H, D = 22, 65536, 8, 64
    assert b * S * 3 * H * D > 1 << 31
    x = torch.ones(b, S, 3 * H * D, dtype=torch.bfloat16, device=cuda)
    tail, dtail, qg, kg, table, _ = make(3, 1, S, H, D, torch.bfloat16, 64, 0)
    x[-1, -50:] = tail[0, -50:].to(cuda)
    t, a, c = table.to(cuda), qg.to(cuda), kg.to(cuda)
    ops.qk_norm_rotary_fwd(x, x, b, S, H, q_gain=a, k_gain=c, rotary=t)
    one = tail.to(cuda)
    ops.qk_norm_rotary_fwd(one, one, 1, S, H, q_gain=a, k_gain=c, rotary=t)
    assert torch.equal(x[-1, -50:], one[0, -50:]) and torch.equal(x[0], x[-2])


def test_same_bits_other_stream_and_replayed_graph(cuda):
    b, S, H, D = 3, 500, 4, 64
    qkv, dout, qg, kg, table, _ = make(4, b, S, H, D, torch.bfloat16, 64, 0)
    x, d, a, c, t = (v.to(cuda) for v in (qkv, dout, qg, kg, table))
    out, dx, dq, dk = torch.empty_like(x), torch.empty_like(x), torch.empty_like(a), torch.empty_like(c)

    def step():
        ops.qk_norm_rotary_fwd(x, out, b, S, H, q_gain=a, k_gain=c, rotary=t)
        ops.qk_norm_rotary_bwd(d, x, dx, b, S, H, q_gain=a, k_gain=c, dq_gain=dq, dk_gain=dk, rotary=t)
    step()
    torch.cuda.synchronize()
    want = [v.clone() for v in (out, dx, dq, dk)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert all(torch.equal(v, w) for v, w in zip((out, dx, dq, dk), want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        for v in (out, dx, dq, dk):
            v.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, w) for v, w in zip((out, dx, dq, dk), want)), i
        (x.float() @ x.float().transpose(1, 2)).sum().item()   # eager work in between


def test_refused_calls(cuda):
    x = torch.zeros(1, 4, 3 * 64, dtype=torch.bfloat16, device=cuda)
    out, t = torch.empty_like(x), ops.rotary_table(4, 64, device=cuda)
    f = lambda **kw: ops.qk_norm_rotary_fwd(**{**dict(qkv=x, out=out, b=1, S=4, H=1), **kw})  # noqa: E731
    f(rotary=t)
    for kw, err in ((dict(H=5), ValueError), (dict(S=3), ValueError), (dict(out=out.float()), TypeError), (dict(q_gain=torch.ones(63, device=cuda)), TypeError),
                    (dict(k_gain=torch.ones(64, device=cuda).half()), TypeError), (dict(rotary=t.double()), TypeError), (dict(rotary=t[:2]), ops._lib.HapmiError),
                    (dict(rotary=t, positions=torch.zeros(4, device=cuda)), TypeError), (dict(rotary=t, positions=torch.zeros(3, dtype=torch.int32, device=cuda)), TypeError),
                    (dict(qkv=x.half(), out=out.half()), TypeError), (dict(rotary=ops.rotary_table(4, 24, device=cuda)), ops._lib.HapmiError)):
        with pytest.raises(err):
            f(**kw)
    big = torch.zeros(2 * x.numel(), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError):                            # partly overlapping is neither in place nor apart
        f(qkv=big[:x.numel()].view_as(x), out=big[64:64 + x.numel()].view_as(x))
    with pytest.raises(ValueError):
        ops.qk_norm_rotary_bwd(out, x, x, 1, 4, 1)
    g = torch.empty(64, device=cuda)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary_bwd(out, x, torch.empty_like(x), 1, 4, 1, dq_gain=g, dk_gain=g)


@pytest.mark.parametrize("dtype,inter,H,D", [(torch.bfloat16, False, 2, 64), (torch.float32, True, 3, 32), (torch.bfloat16, True, 1, 24)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_backward_leaves_out_tokens_without_a_position(cuda, dtype, inter, H, D, accumulate):
    """A token whose position lies outside the table (padding marked with -1) has no gradient: zeros for its queries and keys,
    nothing in the gains' gradients, whatever its rows hold; its value rows are copied.  The others are the bits of the same
    call with that token's rows zero and its position valid (zero rows add nothing to the gains)."""
    b, S = 2, 37
    qkv, dout, qg, kg, table, _ = make(7, b, S, H, D, dtype, 16, 0)
    pos = torch.arange(S).repeat(b, 1).int()
    bad = torch.zeros(b, S, dtype=torch.bool)
    bad[0, 5] = bad[1, 30:] = True
    dirty, ddirty, gone = qkv.clone(), dout.clone(), pos.clone()
    dirty[bad], gone[bad] = float("nan"), -1
    gone[0, 5] = S
    ddirty.view(b, S, 3, H * D)[:, :, :2][bad] = float("inf")
    qkv[bad] = 0
    dout.view(b, S, 3, H * D)[:, :, :2][bad] = 0
    res = []
    for x, d, at in ((qkv, dout, pos), (dirty, ddirty, gone)):
        dx = torch.full_like(x, float("nan"), device=cuda)
        dq, dk = torch.full((D,), 2.0, device=cuda), torch.full((D,), -1.0, device=cuda)
        ops.qk_norm_rotary_bwd(d.to(cuda), x.to(cuda), dx, b, S, H, q_gain=qg.to(cuda), k_gain=kg.to(cuda), dq_gain=dq, dk_gain=dk, rotary=table.to(cuda),
                               positions=at.to(cuda), interleaved=inter, accumulate=accumulate)
        res.append((dx, dq, dk))
    (want, wq, wk), (got, dq, dk) = res
    assert torch.equal(got, want) and torch.equal(dq, wq) and torch.equal(dk, wk)
    assert (got.cpu().view(b, S, 3, H * D)[:, :, :2][bad] == 0).all()


@pytest.mark.parametrize("dtype,b,S,H,D,rot,inter", [(torch.bfloat16, 2, 4501, 12, 64, 64, False), (torch.float32, 1, 12001, 5, 64, 32, True),
                                                     (torch.bfloat16, 3, 9000, 5, 24, 16, True)])
def test_backward_over_more_rows_than_resident_blocks_hold(cuda, dtype, b, S, H, D, rot, inter):
    """768 blocks take all rows in turns: every lane adds the gain terms of two or more rows in its registers before the joining
    launch.  A gain's sum runs over up to 3 rows a lane, 128 groups a block and 768 blocks in 32 runs of 24: below 200 roundings."""
    lanes = 1
    while lanes < (D // (8 if dtype == torch.bfloat16 else 4) + 1) // 2:
        lanes *= 2
    assert b * S * H > 768 * (256 // lanes)
    qkv, dout, qg, kg, table, _ = make(11, b, S, H, D, dtype, rot, 0)
    x, d, t, a, c = (v.to(cuda) for v in (qkv, dout, table, qg, kg))
    dx, dq, dk = torch.full_like(x, float("nan")), torch.full_like(a, float("nan")), torch.full_like(c, float("nan"))
    ops.qk_norm_rotary_bwd(d, x, dx, b, S, H, q_gain=a, k_gain=c, dq_gain=dq, dk_gain=dk, rotary=t, interleaved=inter, eps=1e-5)
    wd, wq, wk, sq, sk = L.qk_norm_backward(dout, qkv, H, qg, kg, rows(table, None, b, S), inter, 1e-5)
    big = lambda v: v.abs().amax(-1, keepdim=True)  # noqa: E731
    xs = qkv.double().view(b, S, 3, H, D)
    r = 1 / torch.sqrt((xs * xs).mean(-1, keepdim=True) + 1e-5)
    size = r * big(dout.double().view(b, S, 3, H, D)) * 2 * max(qg.abs().max(), kg.abs().max()).item() * (1 + big(xs * r))
    got = dx.view(b, S, 3, H, D)
    within(got[:, :, :2], wd[:, :, :2], (U[dtype] * wd.abs() + F * size)[:, :, :2], "dqkv")
    assert torch.equal(got[:, :, 2], d.view(b, S, 3, H, D)[:, :, 2])
    # a term is off by 16 roundings of its own, the sum by 200 of the partial sums
    within(dq, wq, 216 * 2.0 ** -24 * sq, "dq_gain")
    within(dk, wk, 216 * 2.0 ** -24 * sk, "dk_gain")
    again = torch.full_like(a, 1.5)
    ops.qk_norm_rotary_bwd(d, x, dx, b, S, H, q_gain=a, k_gain=c, dq_gain=again, rotary=t, interleaved=inter, eps=1e-5, accumulate=True)
    assert torch.equal(again, dq + 1.5)
