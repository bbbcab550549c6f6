"""Attention with a learned relative position bias on the GPU against its float64 formula.

Tolerances.  A bf16 rounding is off by at most u = 2^-8 of the value.  Forward rounds every probability and the result:
u * (|out| + sum_j p_ij |v_j|).  Backward rounds every score gradient (dq, dk) or probability (dv) and the result:
u * (|g| + sum |ds| |k|); the table's gradient adds unrounded float32 score gradients.  In float32 a score of 64 products of
unit normals (sum of |products| below 10 after scaling) is off by 64 * 2^-24 * 10 = 4e-5 at most, its probability by twice
that relatively; with the exponential's and the sums' own roundings below 2e-5, F = 1e-4 of the sum of |terms| covers it."""
import math

import pytest
import torch

from hap_amd import ops
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
U, F = 2.0 ** -8, 1e-4
HD = 64
SCALE = 1.0 / math.sqrt(HD)


def within(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got - want).abs()[bad].max().item(), tol[bad].min().item() if torch.is_tensor(tol) else tol)


def make(seed, b, S, H, n, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return r(b, S, 3 * H * HD).bfloat16(), r(n, H) * spread, r(b, S, H * HD).bfloat16()


def run(cuda, qkv, table, dout, H, lengths=None, keep=None, p=0.0, dtable=None, **kw):
    """out, lse, dqkv, dtable of one forward and backward; every output starts as NaN."""
    b, S = qkv.shape[:2]
    nan = lambda dt, *s: torch.full(s, float("nan"), dtype=dt, device=cuda)  # noqa: E731
    x, t, d = qkv.to(cuda), table.to(cuda) if table.device.type == "cpu" else table, dout.to(cuda)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda)
    out, lse = nan(torch.bfloat16, b, S, H * HD), nan(torch.float32, b, H, S)
    kf = {} if keep is None else {"keep_rows": keep[0], "p": p}
    ops.attention_relbias_fwd(x, t, out, lse, b, S, H, SCALE, lengths=ln, **kf, **kw)
    dqkv, delta = nan(torch.bfloat16, b, S, 3 * H * HD), nan(torch.float32, b, H, S)
    acc = dtable is not None
    dtable = nan(torch.float32, *table.shape) if dtable is None else dtable
    kb = {} if keep is None else {"keep_rows": keep[0], "keep_cols": keep[1], "p": p}
    ops.attention_relbias_bwd(x, t, out, d, lse, dqkv, dtable, delta, b, S, H, SCALE, lengths=ln, accumulate=acc, **kb, **kw)
    return out, lse, dqkv, dtable


def compare(res, qkv, table, dout, H, max_distance, bidirectional, causal, lengths=None, masks=None, p=0.0):
    b, S = qkv.shape[:2]
    out, lse, dqkv, dtable = (t.cpu() for t in res)
    ln = None if lengths is None else torch.tensor(lengths)
    args = (H, SCALE, max_distance, bidirectional, causal, ln, masks, p)
    want, wlse, _, terms = L.relbias_forward(qkv, table, *args)
    within(out.view(b, S, H, HD), want, U * (want.abs() + terms) + F * terms, "out")
    none = torch.isinf(wlse)
    assert torch.equal(torch.isneginf(lse), none) and (out.view(b, S, H, HD)[none.transpose(1, 2)] == 0).all()
    within(lse[~none], wlse[~none], 1e-4 + 2 ** -23 * wlse[~none].abs(), "lse")
    ref = L.relbias_backward(qkv, table, out, dout, lse, *args)
    for i, name in enumerate(("dq", "dk", "dv")):
        g, rounded, size = ref[name]
        within(dqkv.view(b, S, 3, H, HD)[:, :, i], g, U * (g.abs() + rounded * (1 + U)) + F * size, name)
    g, _, size = ref["dtable"]
    within(dtable, g, F * size, "dtable")


CASES = [  # b, S, H, buckets, max_distance, bidirectional, causal
    (1, 50, 2, 2, 5, True, False),
    (1, 1, 1, 2, 2, False, False), (2, 2, 3, 4, 2, True, False), (1, 31, 2, 8, 20, True, False), (1, 32, 2, 32, 128, False, True),
    (2, 33, 1, 32, 128, True, False), (1, 63, 3, 6, 9, True, True), (1, 64, 2, 32, 128, True, False), (1, 65, 2, 5, 17, False, True),
    (2, 127, 2, 48, 300, True, False), (1, 128, 5, 32, 128, False, True), (1, 129, 1, 2, 2, False, True), (1, 200, 4, 32, 128, False, False),
    (2, 300, 2, 10, 9, True, False), (1, 257, 2, 128, 700, True, False), (1, 333, 3, 16, 40, True, True), (1, 700, 2, 4, 524288, False, True),
    (1, 513, 1, 64, 33, False, True), (3, 96, 16, 32, 128, True, False)]


@pytest.mark.parametrize("b,S,H,n,reach,two,causal", CASES)
def test_forward_and_backward(cuda, b, S, H, n, reach, two, causal):
    qkv, table, dout = make(S + n, b, S, H, n)
    res = run(cuda, qkv, table, dout, H, max_distance=reach, bidirectional=two, causal=causal)
    compare(res, qkv, table, dout, H, reach, two, causal)


@pytest.mark.parametrize("b,S,H,n,reach,two,causal", [
    (65, 40, 8, 32, 128, True, False), (65, 33, 8, 6, 9, False, True), (40, 150, 8, 32, 128, False, True), (33, 257, 6, 10, 40, True, False)])
def test_launches_that_fill_the_card(cuda, b, S, H, n, reach, two, causal):
    """More than two blocks a compute unit: dQ's other form."""
    qkv, table, dout = make(S + n, b, S, H, n)
    res = run(cuda, qkv, table, dout, H, max_distance=reach, bidirectional=two, causal=causal)
    compare(res, qkv, table, dout, H, reach, two, causal)


def test_padded_batch_that_fills_the_card(cuda):
    lengths = [(37 * i) % 151 for i in range(100)]
    qkv, table, dout = make(3, 100, 150, 8, 32)
    for z, n in enumerate(lengths):
        qkv[z, n:] = 0
        dout[z, n:] = 0
    for causal in (False, True):
        res = run(cuda, qkv, table, dout, 8, lengths=lengths, causal=causal)
        compare(res, qkv, table, dout, 8, 128, not causal, causal, lengths)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S,lengths", [(65, [65, 0, 1, 64]), (200, [129, 128, 33, 200]), (300, [0, 0, 0, 7]), (17, [17, -5, 900, 16])])
def test_padded_batches(cuda, S, lengths, causal):
    """Rows behind a sequence's end get zeros, whatever its padding holds (NaN here); lengths outside 0 .. S are clamped."""
    qkv, table, dout = make(S, 4, S, 2, 32)
    real = [min(max(n, 0), S) for n in lengths]
    for z, n in enumerate(real):
        qkv[z, n:] = 0
        dout[z, n:] = 0
    dirty, ddirty = qkv.clone(), dout.clone()
    for z, n in enumerate(real):
        dirty[z, n:] = float("nan")
        ddirty[z, n:] = float("inf")
    res = run(cuda, dirty, table, ddirty, 2, lengths=lengths, causal=causal)
    compare(res, qkv, table, dout, 2, 128, not causal, causal, real)
    for z, n in enumerate(real):
        assert (res[2][z, n:] == 0).all() and torch.isneginf(res[1][z, :, n:]).all()


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e30, -1e8])
def test_hidden_buckets(cuda, low):
    """A bias at the type's lowest value hides its pairs; a query left with nothing gets zeros and no gradient."""
    qkv, table, dout = make(5, 2, 150, 2, 32)
    table[0] = low                                             # nobody sees itself: causal query 0 sees nothing at all
    table[20, 1] = low
    for causal in (True, False):
        res = run(cuda, qkv, table, dout, 2, causal=causal)
        compare(res, qkv, table, dout, 2, 128, not causal, causal)
        assert (res[3][0] == 0).all()
        if causal:
            assert torch.isneginf(res[1][:, :, 0]).all() and (res[0][:, 0] == 0).all()
    table[:] = low
    res = run(cuda, qkv, table, dout, 2)
    assert (res[0] == 0).all() and (res[2] == 0).all() and (res[3] == 0).all() and torch.isneginf(res[1]).all()


def test_large_scores_do_not_overflow(cuda):
    """Scores of some hundreds and biases of 1e4: the running maximum keeps every exponential at or below 1.  The float32
    error of a score grows with its size: 64 * 2^-24 * 6400 from the products (40 * 40 * 4 of |q| |k| scale) and 2^-23 * 1e4
    from the bias add up to 0.03, so probabilities are compared at 10 % and results by their finiteness and norm."""
    qkv, table, dout = make(8, 1, 140, 2, 32)
    qkv = (qkv * 20).bfloat16()
    table = table * 3000
    out, lse, dqkv, dtable = run(cuda, qkv, table, dout, 2)
    want, wlse, _, _ = L.relbias_forward(qkv, table, 2, SCALE, 128, True, False)
    assert all(torch.isfinite(t).all() for t in (out, dqkv, dtable))
    within(lse, wlse, 0.03 + 2 ** -22 * wlse.abs(), "lse")
    assert ((out.double().cpu().view_as(want) - want).norm() / want.norm()).item() < 0.1


@pytest.mark.parametrize("low", [-1e4, -65504.0, -1e6, -9e7])
def test_low_biases_that_hide_nothing(cuda, low):
    """Every pair has the same very low bias: a softmax does not see it.  float32 scores of that size keep 2^-24 * |low| * log2 e
    of theirs apart at best, so all weights are compared with the even ones: results are averages of the values."""
    qkv, table, dout = make(9, 1, 150, 2, 32)
    qkv[..., :2 * 2 * HD] = 0                                  # queries and keys
    table[:] = low
    out, lse, dqkv, dtable = run(cuda, qkv, table, dout, 2)
    mean = qkv.double().view(1, 150, 3, 2, HD)[:, :, 2].mean(1, keepdim=True)
    size = qkv.double().view(1, 150, 3, 2, HD)[:, :, 2].abs().mean(1, keepdim=True)
    # weights: one rounding to bf16 each (2^-8, all the same way); the mean's own rounding
    assert ((out.double().cpu().view(1, 150, 2, HD) - mean).abs() <= 2 ** -8 * size + 2 ** -8 * mean.abs() + 1e-6).all()
    within(lse, torch.full((1, 2, 150), low + 5.0106353, dtype=torch.float64), 2 ** -22 * abs(low) + 1e-4, "lse")
    assert torch.isfinite(dqkv.float()).all() and torch.isfinite(dtable).all()


@pytest.mark.parametrize("S,causal", [(64, False), (129, True), (200, False), (33, True)])
def test_dropout_of_the_probabilities(cuda, S, causal):
    b, H, p, sid = 2, 2, 0.25, 3
    qkv, table, dout = make(S + 1, b, S, H, 32)
    row_len = (S + 7) // 8 * 8
    state = torch.tensor([77, 5], dtype=torch.int64, device=cuda)
    words = ops.attention_keep_words(b, S, H)
    kr, kc = (torch.empty(words, dtype=torch.int32, device=cuda) for _ in range(2))
    ops.attention_keep_bits(kr, kc, b, S, H, row_len, p, state, sid)
    masks = ops.dropout_mask(b * H * S * row_len, p, state, sid).view(b, H, S, row_len)[..., :S].bool().cpu()
    for lengths in (None, [S, S // 2]):
        if lengths:
            qkv[1, S // 2:] = 0
            dout[1, S // 2:] = 0
        res = run(cuda, qkv, table, dout, H, lengths=lengths, keep=(kr, kc), p=p, causal=causal)
        compare(res, qkv, table, dout, H, 128, not causal, causal, lengths, masks, p)


def test_columns_of_a_wider_table_and_accumulation(cuda):
    """A device's heads are columns of the whole table; a table that layers share gets the sum of their gradients; the
    neighbouring columns stay as they were."""
    qkv, _, dout = make(3, 2, 100, 3, 32)
    g = torch.Generator().manual_seed(0)
    whole = torch.randn(32, 10, generator=g)
    dev, grad = whole.to(cuda), torch.full((32, 10), 2.0, device=cuda)
    first = run(cuda, qkv, dev[:, 4:7], dout, 3)[3]
    res = run(cuda, qkv, dev[:, 4:7], dout, 3, dtable=grad[:, 4:7])
    compare((*res[:3], first), qkv, whole[:, 4:7], dout, 3, 128, True, False)
    assert torch.equal(grad[:, 4:7], first + 2.0)
    assert (grad[:, :4] == 2).all() and (grad[:, 7:] == 2).all()


def test_same_bits_every_time_and_nothing_written_beside_the_outputs(cuda):
    b, S, H = 2, 333, 3
    qkv, table, dout = make(1, b, S, H, 32)
    first = run(cuda, qkv, table, dout, H)
    for _ in range(3):
        assert all(torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y)
                   for x, y in zip(first, run(cuda, qkv, table, dout, H)))
    # outputs in the middle of larger buffers of a marker value
    mid = lambda n, dt: torch.full((n + 2048,), 7.0, dtype=dt, device=cuda)  # noqa: E731
    x, t, d = qkv.to(cuda), table.to(cuda), dout.to(cuda)
    sizes = dict(out=(b * S * H * HD, torch.bfloat16), lse=(b * H * S, torch.float32), dqkv=(b * S * 3 * H * HD, torch.bfloat16),
                 dtable=(32 * H, torch.float32), delta=(b * H * S, torch.float32),
                 ws=(ops.attention_relbias_workspace_elems(t, b, S, H), torch.float32))
    buf = {k: mid(*v) for k, v in sizes.items()}
    v = {k: buf[k][1024:1024 + sizes[k][0]] for k in buf}
    ops.attention_relbias_fwd(x, t, v["out"].view(b, S, -1), v["lse"], b, S, H, SCALE)
    ops.attention_relbias_bwd(x, t, v["out"].view(b, S, -1), d, v["lse"], v["dqkv"], v["dtable"].view(32, H), v["delta"], b, S, H, SCALE, workspace=v["ws"])
    assert torch.equal(v["dqkv"].view(b, S, -1), first[2]) and torch.equal(v["dtable"].view(32, H), first[3])
    for k, whole in buf.items():
        assert (whole[:1024] == 7).all() and (whole[1024 + sizes[k][0]:] == 7).all(), k


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 elements of qkv and dqkv; short sequences in a long padded batch keep the arithmetic small."""
    b, S, H, n = 11, 65552, 16, 70
    assert b * S * 3 * H * HD > 1 << 31
    qkv = torch.zeros(b, S, 3 * H * HD, dtype=torch.bfloat16, device=cuda)
    small, table, dsmall = make(2, 1, n, H, 32)
    qkv[-1, :n] = small[0].to(cuda)
    dout = torch.zeros(b, S, H * HD, dtype=torch.bfloat16, device=cuda)
    dout[-1, :n] = dsmall[0].to(cuda)
    lengths = torch.full((b,), n, dtype=torch.int32, device=cuda)
    out, lse = torch.full_like(dout, 3.0), torch.empty(b, H, S, device=cuda)
    t = table.to(cuda)
    ops.attention_relbias_fwd(qkv, t, out, lse, b, S, H, SCALE, lengths=lengths)
    dqkv, dtable = torch.full_like(qkv, 3.0), torch.empty_like(t)
    ops.attention_relbias_bwd(qkv, t, out, dout, lse, dqkv, dtable, torch.empty_like(lse), b, S, H, SCALE, lengths=lengths)
    # the other rows have zero inputs: uniform up to the bias, zero values, zero gradients
    assert not out[:-1].any() and not out[-1, n:].any() and not dqkv[:-1].any() and not dqkv[-1, n:].any()
    compare((out[-1:, :n], lse[-1:, :, :n], dqkv[-1:, :n], dtable), small, table, dsmall, H, 128, True, False)


def test_another_stream_and_a_replayed_graph(cuda):
    b, S, H = 2, 130, 2
    qkv, table, dout = make(6, b, S, H, 32)
    want = run(cuda, qkv, table, dout, H, causal=True)
    x, t, d = qkv.to(cuda), table.to(cuda), dout.to(cuda)
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    dqkv, dtable, delta = torch.empty_like(want[2]), torch.empty_like(want[3]), torch.empty_like(want[1])

    def step():
        ops.attention_relbias_fwd(x, t, out, lse, b, S, H, SCALE, causal=True)
        ops.attention_relbias_bwd(x, t, out, d, lse, dqkv, dtable, delta, b, S, H, SCALE, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert torch.equal(dqkv, want[2]) and torch.equal(dtable, want[3])
    graphs = []
    for _ in range(2):                                         # two graphs over the same buffers, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(6):
        for buf in (out, lse, dqkv, dtable, delta):
            buf.fill_(float("nan"))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip((out, dqkv, dtable), (want[0], want[2], want[3]))), i
        run(cuda, qkv, table * i, dout, H)                     # eager work of other values in between


def test_refused_calls(cuda):
    b, S, H = 1, 16, 2
    x = torch.zeros(b, S, 3 * H * HD, dtype=torch.bfloat16, device=cuda)
    out, lse = torch.empty(b, S, H * HD, dtype=torch.bfloat16, device=cuda), torch.empty(b, H, S, device=cuda)
    t = torch.zeros(32, H, device=cuda)
    f = lambda **kw: ops.attention_relbias_fwd(**{**dict(qkv=x, table=t, out=out, lse=lse, b=b, S=S, H=H, scale=SCALE), **kw})  # noqa: E731
    f()
    for kw, err in ((dict(table=torch.zeros(32, H + 1, device=cuda)), ValueError), (dict(table=t.half()), ValueError), (dict(table=t.t()), ValueError),
                    (dict(table=torch.zeros(31, H, device=cuda)), ValueError), (dict(max_distance=4), ValueError),
                    (dict(qkv=x.float()), TypeError), (dict(out=out.float()), TypeError), (dict(lengths=torch.zeros(b, device=cuda)), TypeError),
                    (dict(lengths=torch.zeros(b + 1, dtype=torch.int32, device=cuda)), TypeError), (dict(qkv=x[:, :8]), ops._lib.HapmiError),
                    (dict(out=x.view(-1)[:out.numel()].view_as(out)), ValueError), (dict(scale=-1.0), ops._lib.HapmiError),
                    (dict(table=t.cpu()), ops._lib.HapmiError)):
        with pytest.raises(err):
            f(**kw)
    dq, dt, dl = torch.empty_like(x), torch.empty_like(t), torch.empty_like(lse)
    g = lambda **kw: ops.attention_relbias_bwd(**{**dict(qkv=x, table=t, out=out, dout=out, lse=lse, dqkv=dq, dtable=dt, delta_ws=dl, b=b, S=S, H=H,  # noqa: E731
                                                         scale=SCALE), **kw})
    g()
    for kw, err in ((dict(dtable=dt[:16]), ValueError), (dict(workspace=torch.empty(3, device=cuda)), ops._lib.HapmiError), (dict(dqkv=x), ValueError),
                    (dict(delta_ws=lse), ValueError), (dict(keep_rows=torch.zeros(64, dtype=torch.int32, device=cuda)), ValueError)):
        with pytest.raises(err):
            g(**kw)


@pytest.mark.parametrize("b,S,H,causal", [(1, 640, 1, False), (1, 640, 1, True), (33, 257, 9, False), (33, 257, 9, True)])
def test_table_gradient_where_every_block_meets_its_neighbours_words(cuda, b, S, H, causal):
    """A window that reaches over (nearly) the whole sequence: every 32 x 32 block's diagonals go into it, each word is added to by
    one lane in one block and by another in the next one.  Few blocks and a launch that fills the card: both forms of dQ."""
    qkv, table, dout = make(S + b, b, S, H, 128 if not causal else 64)
    kw = dict(max_distance=1000, bidirectional=not causal, causal=causal)
    res = run(cuda, qkv, table, dout, H, **kw)
    want = L.relbias_backward(qkv, table, res[0].cpu(), dout, res[1].cpu(), H, SCALE, 1000, not causal, causal)["dtable"]
    within(res[3], want[0], F * want[2], "dtable")


def test_table_and_gradient_as_columns_of_one_buffer(cuda):
    """Tables and gradients of two groups of heads side by side in one buffer share no memory: the calls are taken, give the bits
    of buffers of their own and leave the other columns alone."""
    qkv, table, dout = make(4, 2, 90, 3, 32)
    want = run(cuda, qkv, table, dout, 3)
    buf = torch.full((32, 12), 7.0, device=cuda)
    buf[:, 2:5] = table.to(cuda)
    buf[:, 5:8] = 0.0
    res = run(cuda, qkv, buf[:, 2:5], dout, 3, dtable=buf[:, 5:8])
    assert all(torch.equal(a, b) for a, b in zip(res, want))
    assert (buf[:, :2] == 7).all() and (buf[:, 8:] == 7).all() and torch.equal(buf[:, 2:5], table.to(cuda))
    with pytest.raises(ValueError):
        run(cuda, qkv, buf[:, 2:5], dout, 3, dtable=buf[:, 4:7])


@pytest.mark.parametrize("exponent", [-62, 66])
def test_scales_near_the_ends_of_their_range(cuda, exponent):
    """Queries and keys of size 2^(-exponent / 2) under a scale of 2^exponent / 8 give ordinary scores; so does the bias that the
    window holds divided by it.  Powers of two leave every rounding where it is: the bits of the usual scale, but for dqkv's
    queries and keys, which carry the power."""
    qkv, table, dout = make(4, 1, 90, 2, 32)
    want = run(cuda, qkv, table, dout, 2)
    moved = qkv.view(1, 90, 3, 2, HD).clone()
    half = 2.0 ** (-exponent // 2)
    moved[:, :, :2] *= half
    x, t, d = moved.view_as(qkv).to(cuda), table.to(cuda), dout.to(cuda)
    out, lse, dx, dt = (torch.empty_like(w) for w in want)
    scale = SCALE * 2.0 ** exponent
    ops.attention_relbias_fwd(x, t, out, lse, 1, 90, 2, scale)
    ops.attention_relbias_bwd(x, t, out, d, lse, dx, dt, torch.empty_like(lse), 1, 90, 2, scale)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(dt, want[3])
    dx, dw = dx.view(1, 90, 3, 2, HD), want[2].view(1, 90, 3, 2, HD)
    assert torch.equal(dx[:, :, 2], dw[:, :, 2]) and torch.equal(dx[:, :, :2].float() * half, dw[:, :, :2].float())


@pytest.mark.parametrize("b,S,H,causal,lengths", [(6, 760, 8, False, None), (5, 900, 7, True, None), (7, 800, 8, False, [800, 1, 700, 333, 0, 799, 512]), (1, 1100, 3, False, None)])
def test_windows_that_fill_the_lds(cuda, b, S, H, causal, lengths):
    """Windows from 697 distances a side on leave room for one block of dQ's look-ahead form a compute unit: launches of more than 256
    blocks (padded: 384) take the other form, smaller ones keep it."""
    n, reach = (64, 950) if not causal else (32, 950)
    assert ops.relative_bucket_starts(n, reach, not causal)[-1] > 697
    qkv, table, dout = make(S, b, S, H, n)
    for z, k in enumerate(lengths or []):
        qkv[z, k:] = 0
        dout[z, k:] = 0
    res = run(cuda, qkv, table, dout, H, lengths=lengths, max_distance=reach, causal=causal)
    compare(res, qkv, table, dout, H, reach, not causal, causal, lengths)
