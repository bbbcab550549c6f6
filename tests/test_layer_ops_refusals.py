"""Calls that the entry points of the relative position bias, the per-head norm with rotation and the balance loss refuse
on the host, before any device is touched (the pointers below are never followed)."""
import ctypes

import pytest
import torch

from hap_amd._lib import BF16, F32, HapmiError, RelBias, _load
from hap_amd import ops

P = 0x10000                                                   # 16-byte aligned, never dereferenced
EINVAL, EALIGN, ELIMIT = -1, -2, -5


def bias(starts=(0, 1, 2, 4), n=None, two=0, ld=8, table=P):
    arr = (ctypes.c_int32 * len(starts))(*starts)
    r = RelBias()
    r.table, r.ld, r.n_buckets, r.bidirectional, r.starts_host = table, ld, n if n is not None else len(starts) * (2 if two else 1), two, ctypes.addressof(arr)
    r._keep = arr
    return r


def refused(rc, code, text):
    msg = _load().hapmi_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def rel_fwd(r=None, qkv=P, out=P, lse=P, b=2, S=16, H=4, scale=0.125, keep=None, p=0.0):
    r = bias() if r is None else r
    return _load().hapmi_attention_relbias_fwd(qkv, ctypes.byref(r), 0, None, out, lse, b, S, H, scale, keep, p, None)


def rel_bwd(r=None, b=2, S=16, H=4, ws=P, elems=1 << 30, ldd=8, kr=None, kc=None, dtable=P, dqkv=P):
    r = bias() if r is None else r
    return _load().hapmi_attention_relbias_bwd(P, ctypes.byref(r), 0, None, P, P, P, dqkv, dtable, ldd, 0, P, ws, elems, b, S, H, 0.125, kr, kc, 0.0, None)


def test_relative_bias_descriptions():
    refused(rel_fwd(bias(n=1)), EINVAL, "at least 2")
    refused(rel_fwd(bias(n=7, two=1)), EINVAL, "even")
    refused(rel_fwd(bias(starts=tuple(range(65)))), ELIMIT, "at most 64")
    refused(rel_fwd(bias(starts=(1, 2, 3, 4))), EINVAL, "distance 0")
    refused(rel_fwd(bias(starts=(0, 3, 2, 4))), EINVAL, "must not fall")
    refused(rel_fwd(bias(starts=(0, 1, 2, 1025))), ELIMIT, "1025")
    refused(rel_fwd(bias(ld=3)), EINVAL, "heads")
    refused(rel_fwd(bias(table=None)), EINVAL, "null pointer")
    r = bias()
    r.starts_host = None
    refused(rel_fwd(r), EINVAL, "null bias")
    assert _load().hapmi_attention_relbias_fwd(P, None, 0, None, P, P, 2, 16, 4, 0.125, None, 0.0, None) == EINVAL


@pytest.mark.parametrize("kw,code,text", [
    (dict(b=-1), EINVAL, "bad shape"), (dict(S=0), EINVAL, "bad shape"), (dict(H=0), EINVAL, "bad shape"),
    (dict(S=1 << 24), ELIMIT, "too long"), (dict(b=20000, H=4), ELIMIT, "65535"), (dict(b=1 << 62, H=4), ELIMIT, "65535"),
    (dict(scale=0.0), EINVAL, "positive"), (dict(scale=-1.0), EINVAL, "positive"), (dict(scale=float("nan")), EINVAL, "positive"),
    (dict(scale=float("inf")), EINVAL, "positive"), (dict(p=1.0, keep=P), EINVAL, "[0, 1)"), (dict(p=-0.1, keep=P), EINVAL, "[0, 1)"),
    (dict(qkv=None), EINVAL, "null"), (dict(out=None), EINVAL, "null"), (dict(lse=None), EINVAL, "null"),
    (dict(qkv=P + 8), EALIGN, "16-byte"), (dict(out=P + 2), EALIGN, "16-byte"), (dict(keep=P + 4), EALIGN, "keep words"),
    (dict(lse=P + 2), EALIGN, "aligned")])
def test_relative_bias_forward(kw, code, text):
    refused(rel_fwd(**kw), code, text)


def test_relative_bias_forward_of_an_empty_batch_does_nothing():
    assert rel_fwd(b=0) == 0


def test_relative_bias_backward():
    need = ctypes.c_int64()
    r = bias()
    assert _load().hapmi_attention_relbias_workspace_elems(ctypes.byref(r), 2, 300, 4, ctypes.byref(need)) == 0
    assert need.value > 0 and need.value % (2 * 4 * 3) == 0
    refused(rel_bwd(S=300, elems=need.value - 1), ELIMIT, "workspace")
    refused(rel_bwd(ws=None), EINVAL, "null")
    refused(rel_bwd(dtable=None), EINVAL, "null")
    refused(rel_bwd(b=0), EINVAL, "empty batch")
    refused(rel_bwd(ldd=3), EINVAL, "gradient rows")
    refused(rel_bwd(kr=P), EINVAL, "come together")
    refused(rel_bwd(kc=P), EINVAL, "come together")
    refused(rel_bwd(dqkv=P + 4), EALIGN, "16-byte")
    refused(_load().hapmi_attention_relbias_workspace_elems(ctypes.byref(r), 2, 300, 4, None), EINVAL, "null")


def qn_fwd(qkv=P, out=P, qg=P, kg=P, ang=P, n_pos=64, rot=64, inter=0, pos=None, b=2, S=16, H=4, D=64, eps=1e-6, dt=BF16):
    return _load().hapmi_qk_norm_rotary_fwd(qkv, out, qg, kg, ang, n_pos, rot, inter, pos, b, S, H, D, eps, dt, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(D=0), EINVAL, "bad"), (dict(D=60), EALIGN, "multiple of 8"), (dict(D=66, dt=F32), EALIGN, "multiple of 4"), (dict(D=264), ELIMIT, "256"),
    (dict(rot=72), EALIGN, "rot"), (dict(rot=24), EALIGN, "rot"), (dict(rot=12, inter=1), EALIGN, "rot"), (dict(rot=0), EINVAL, "come together"),
    (dict(ang=None), EINVAL, "come together"), (dict(n_pos=0, pos=P), EINVAL, "empty"), (dict(n_pos=15), EINVAL, "sequences of 16"),
    (dict(eps=-1.0), EINVAL, "bad"), (dict(eps=float("nan")), EINVAL, "bad"), (dict(dt=7), EINVAL, "bad"), (dict(S=0), EINVAL, "bad"),
    (dict(b=1 << 30, S=1 << 20, n_pos=1 << 21), ELIMIT, "2^40"), (dict(ang=P + 4), EALIGN, "16-byte"), (dict(pos=P + 2), EALIGN, "aligned"),
    (dict(qkv=P + 8), EALIGN, "16-byte"), (dict(out=P + 8), EALIGN, "16-byte"), (dict(qkv=None), EINVAL, "null"), (dict(out=None), EINVAL, "null")])
def test_norm_and_rotation_forward(kw, code, text):
    refused(qn_fwd(**kw), code, text)


def test_norm_and_rotation_backward():
    L = _load()
    need = ctypes.c_int64()
    assert L.hapmi_qk_norm_rotary_workspace_elems(64, ctypes.byref(need)) == 0 and need.value >= 2 * 64
    refused(L.hapmi_qk_norm_rotary_workspace_elems(257, ctypes.byref(need)), EINVAL, "bad")

    def bwd(dout=P, dqg=P, ws=P, elems=1 << 40, b=2):
        return L.hapmi_qk_norm_rotary_bwd(dout, P, P, P, P, dqg, None, 0, P, 64, 64, 0, None, b, 16, 4, 64, 1e-6, BF16, ws, elems, None)
    refused(bwd(elems=2 * 64 - 1), ELIMIT, "workspace")
    refused(bwd(ws=None), ELIMIT, "workspace")
    refused(bwd(dout=None), EINVAL, "null")
    refused(bwd(b=0), EINVAL, "empty batch")
    refused(bwd(dqg=P + 2), EALIGN, "aligned")
    assert qn_fwd(b=0) == 0


def test_balance_loss():
    L = _load()

    def fwd(probs=P, B=4, S=8192, E=8, choices=1, ws=P, elems=1 << 40, loss=P):
        return L.hapmi_balance_loss_fwd(probs, P, P, None, loss, P, P, P, B, S, E, 0.01, choices, ws, elems, None)

    def bwd(probs=P, index=P, dgate=None, B=4, E=8, choices=1, dlogits=P):
        return L.hapmi_balance_loss_bwd(probs, index, P, dgate, P, None, dlogits, B, 16, E, 0.01, choices, None)
    for call in (fwd, bwd):
        refused(call(E=65), ELIMIT, "64 experts")
        refused(call(E=0), EINVAL, "bad")
        refused(call(choices=3), EINVAL, "bad")
        refused(call(choices=0), EINVAL, "bad")
        refused(call(B=65536), ELIMIT, "65535 rows")
        refused(call(probs=P + 4), EALIGN, "16-byte")
        refused(call(probs=None), EINVAL, "null")
    refused(fwd(B=0), EINVAL, "empty batch")
    refused(fwd(S=1 << 24), ELIMIT, "tokens a row")
    refused(fwd(ws=None), ELIMIT, "workspace")
    refused(fwd(elems=10), ELIMIT, "workspace")
    refused(bwd(dgate=P, index=None), EINVAL, "null")
    refused(bwd(dlogits=P + 8), EALIGN, "16-byte")
    assert bwd(B=0) == 0
    need = ctypes.c_int64()
    assert L.hapmi_balance_workspace_elems(60000, 16, 8, ctypes.byref(need)) == 0 and need.value == 0     # whole rows: none needed
    refused(L.hapmi_balance_workspace_elems(4, 16, 8, None), EINVAL, "null")


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 4, 192, dtype=torch.bfloat16)
    with pytest.raises(HapmiError, match="GPU tensors only"):
        ops.qk_norm_rotary_fwd(t, t, 1, 4, 1)
    with pytest.raises(HapmiError, match="GPU tensors only"):
        ops.attention_relbias_fwd(t, torch.zeros(4, 1), t, t, 1, 4, 1, 0.125)
    with pytest.raises(ValueError):
        ops.rotary_table(0, 8)
    with pytest.raises(ValueError):
        ops.rotary_table(8, 7)


def test_bias_tables_whose_rows_overlap():
    """A table broadcast over its buckets, or one with rows closer than its heads, would be read beyond its memory."""
    whole = torch.zeros(8, 4)
    row = torch.zeros(1, 4)
    for odd in (row.expand(8, 4), torch.zeros(64).as_strided((8, 4), (3, 1)), torch.zeros(8, 8)[:, ::2], whole.double(), whole[:, :3], whole[0]):
        with pytest.raises(ValueError, match="table must be"):
            ops._relbias("x", odd, 4, 8, False, True)
    assert ops._relbias("x", torch.zeros(8, 6)[:, 1:5], 4, 8, False, True).ld == 6
    x = torch.zeros(1, 2, 3 * 4 * 64)
    for odd in (row.expand(8, 4), torch.zeros(8, 3), torch.zeros(8, 8)[:, ::2]):
        with pytest.raises(ValueError, match="dtable must be"):
            ops.attention_relbias_bwd(x, whole, x, x, x, x, odd, x, 1, 2, 4, 0.125, max_distance=8, causal=True)


EALIAS = -6


@pytest.mark.parametrize("shared", ["out/qkv", "lse/qkv", "lse/out", "out/table", "lse/lengths", "lse/keep", "out/qkv+8000"])
def test_bias_forward_outputs_apart(shared):
    """b 2, S 16, H 4: qkv 49152 bytes, out 16384, lse 512; an output that starts inside another operand is refused."""
    at = dict(qkv=1 << 20, out=2 << 20, lse=3 << 20, table=4 << 20, lengths=5 << 20, keep=6 << 20)
    name, other = shared.split("/")
    other, _, off = other.partition("+")
    at[name] = at[other] + int(off or 0) // 16 * 16
    r = bias(table=at["table"])
    rc = _load().hapmi_attention_relbias_fwd(at["qkv"], ctypes.byref(r), 0, at["lengths"], at["out"], at["lse"], 2, 16, 4, 0.125, at["keep"], 0.1, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("shared", ["dqkv/qkv", "dqkv/dout", "dtable/table", "dtable/dqkv", "delta/lse", "ws/delta", "ws/out", "dtable/ws", "delta/kc", "dqkv/lengths"])
def test_bias_backward_outputs_apart(shared):
    names = ("qkv", "out", "dout", "lse", "dqkv", "dtable", "delta", "ws", "table", "lengths", "kr", "kc")
    at = {n: (i + 1) << 20 for i, n in enumerate(names)}
    name, other = shared.split("/")
    at[name] = at[other]
    r = bias(table=at["table"])
    rc = _load().hapmi_attention_relbias_bwd(at["qkv"], ctypes.byref(r), 0, at["lengths"], at["out"], at["dout"], at["lse"], at["dqkv"], at["dtable"], 8, 0,
                                             at["delta"], at["ws"], 1 << 16, 2, 16, 4, 0.125, at["kr"], at["kc"], 0.1, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("shared", ["out/q", "out/k", "out/angles", "out/positions", "out/qkv+512"])
def test_norm_forward_outputs_apart(shared):
    at = {n: (i + 1) << 20 for i, n in enumerate(("qkv", "out", "q", "k", "angles", "positions"))}
    name, other = shared.split("/")
    other, _, off = other.partition("+")
    at[name] = at[other] + int(off or 0)
    rc = _load().hapmi_qk_norm_rotary_fwd(at["qkv"], at["out"], at["q"], at["k"], at["angles"], 64, 64, 0, at["positions"], 2, 16, 4, 64, 1e-6, BF16, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("shared", ["dqkv/qkv", "dq/dk", "dq/q", "dk/ws", "ws/dout", "dqkv/ws", "dqkv/dout+1024"])
def test_norm_backward_outputs_apart(shared):
    at = {n: (i + 1) << 20 for i, n in enumerate(("dout", "qkv", "dqkv", "q", "k", "dq", "dk", "angles", "positions", "ws"))}
    name, other = shared.split("/")
    other, _, off = other.partition("+")
    at[name] = at[other] + int(off or 0)
    rc = _load().hapmi_qk_norm_rotary_bwd(at["dout"], at["qkv"], at["dqkv"], at["q"], at["k"], at["dq"], at["dk"], 0, at["angles"], 64, 64, 0, at["positions"],
                                          2, 16, 4, 64, 1e-6, BF16, at["ws"], 1 << 24, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("shared", ["loss/counts", "counts/kept", "kept/index", "sums/probs", "loss/lengths", "ws/probs", "ws/slot"])
def test_balance_outputs_apart(shared):
    at = {n: (i + 1) << 20 for i, n in enumerate(("probs", "index", "slot", "lengths", "loss", "counts", "kept", "sums", "ws"))}
    name, other = shared.split("/")
    at[name] = at[other]
    rc = _load().hapmi_balance_loss_fwd(at["probs"], at["index"], at["slot"], at["lengths"], at["loss"], at["counts"], at["kept"], at["sums"], 2, 4096, 16, 0.01, 2,
                                        at["ws"], 1 << 20, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("other", ["probs", "index", "slot", "dgate", "counts", "lengths"])
def test_balance_gradient_apart(other):
    at = {n: (i + 1) << 20 for i, n in enumerate(("probs", "index", "slot", "dgate", "counts", "lengths"))}
    rc = _load().hapmi_balance_loss_bwd(at["probs"], at["index"], at["slot"], at["dgate"], at["counts"], at["lengths"], at[other], 2, 64, 16, 0.01, 2, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("off,ldd,ws", [(0, 8, None), (12, 8, None), (20, 8, None), (28, 8, None), (32, 8, None), (16, 12, None), (-92, 8, None), (16, 8, 20),
                                        (16, 8, 36)])
def test_table_gradients_among_the_tables_columns(off, ldd, ws):
    """A table of 4 heads in rows of 8 floats leaves its columns 4 .. 7 to others: a gradient (or scratch) that begins or ends in the
    table's own columns, or has rows of another length, is refused."""
    table = 8 << 20
    at = {n: (i + 1) << 20 for i, n in enumerate(("qkv", "out", "dout", "lse", "dqkv", "delta", "ws"))}
    r = bias(table=table)
    rc = _load().hapmi_attention_relbias_bwd(at["qkv"], ctypes.byref(r), 0, None, at["out"], at["dout"], at["lse"], at["dqkv"], table + off, ldd, 0,
                                             at["delta"], table + ws if ws else at["ws"], 1 << 16, 2, 16, 4, 0.125, None, None, 0.0, None)
    refused(rc, EALIAS, "shares memory")


@pytest.mark.parametrize("scale", [1e-38, 9e-21, 1.1e20, 3e38])
def test_scales_that_the_bias_window_cannot_hold(scale):
    """The bias is kept divided by the scale: a bias of 1e7 over 1e-38 is beyond float32, one of 1 over 3e38 below it."""
    refused(rel_fwd(scale=scale), ELIMIT, "1e-20")
    r = bias()
    rc = _load().hapmi_attention_relbias_bwd(P, ctypes.byref(r), 0, None, P, P, P, P, P, 8, 0, P, P, 1 << 30, 2, 16, 4, scale, None, None, 0.0, None)
    refused(rc, ELIMIT, "1e-20")


@pytest.mark.parametrize("B,S,E", [(4, 64, 16), (16, 512, 16), (64, 2048, 64), (1, 4097, 3), (600, 5, 8), (2, 1 << 20, 64)])
def test_scratch_of_the_balance_loss_is_what_the_library_asks_for(B, S, E):
    need = ops.balance_workspace_elems(B, S, E)

    def fwd(ws, elems):
        # an index that shares memory with the loss: what a call that passes the scratch check is refused for
        return _load().hapmi_balance_loss_fwd(P, 1 << 40, 2 << 40, None, 1 << 40, 3 << 40, 4 << 40, 5 << 40, B, S, E, 0.01, 2, ws, elems, None)
    if need:
        refused(fwd(6 << 40, need - 1), ELIMIT, "workspace")
        refused(fwd(None, need), ELIMIT, "workspace")
    refused(fwd(6 << 40 if need else None, need), EALIAS, "shares memory")
