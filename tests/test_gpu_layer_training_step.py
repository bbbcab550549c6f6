"""The relative position bias, the norm with rotation and the balance loss in one routed layer's training step, as a program
would call them next to the GEMMs, the residual LayerNorm, the gate and the expert gathers, against float64 autograd.

    qkv = x W_in^T;  q, k normalised and rotated;  a = attention with bias;  y = LN(a W_out^T + x)
    routing of y W_r, identity experts: z = sum over the kept choices of gate * y;  loss = <z, w> + balance loss

The tolerance is the library's parity bar for bf16 programs, 2e-2 of a gradient's norm: activations are rounded to bf16 some
ten times on the way, each by 2^-8 at most.  The routing's whole numbers are taken from the kernels on both sides."""
import math

import pytest
import torch

from hap_amd import ops
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu

B, S, H, E, C, BUCKETS, COEF = 2, 72, 2, 8, 24, 16, 0.5
D = H * 64


def parameters():
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"w_in": (r(3 * D, D) / math.sqrt(D)).bfloat16(), "w_out": (r(D, D) / math.sqrt(D)).bfloat16(), "w_r": (r(D, E) / math.sqrt(D)).bfloat16(),
            "q_gain": 1 + 0.2 * r(64), "k_gain": 1 + 0.2 * r(64), "table": 0.5 * r(BUCKETS, H), "x": r(B, S, D).bfloat16(),
            "w": r(B, S, D).bfloat16(), "lengths": torch.tensor([S, 41], dtype=torch.int32)}


class Step:
    """Static buffers and one forward + backward, as an executor would hold them."""

    def __init__(self, dev, causal):
        self.p = {k: v.to(dev) for k, v in parameters().items()}
        self.causal, self.angles = causal, ops.rotary_table(S, 64, device=dev)
        bf = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=dev)  # noqa: E731
        f32 = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.qkv, self.rot, self.att, self.proj, self.y, self.z = bf(B, S, 3 * D), bf(B, S, 3 * D), bf(B, S, D), bf(B, S, D), bf(B, S, D), bf(B, S, D)
        self.lse, self.delta, self.rstd, self.logits = f32(B, H, S), f32(B, H, S), f32(B * S), f32(B, S, E)
        self.r = dict(probs=f32(B, S, E), index=i32(B, S, 2), slot=i32(B, S, 2), gate=f32(B, S, 2), token_of_slot=i32(B, E, C))
        self.loss, self.counts, self.kept, self.sums = f32(1), i32(B, E), i32(B, E), f32(B, E)
        self.ein, self.dein = bf(E, B, C, D), bf(E, B, C, D)
        self.dgate, self.dlogits, self.dlogits_bf = f32(B, S, 2), f32(B, S, E), bf(B, S, E)
        self.dy, self.dsum, self.datt, self.drot, self.dqkv = bf(B, S, D), bf(B, S, D), bf(B, S, D), bf(B, S, 3 * D), bf(B, S, 3 * D)
        self.g = {"w_in": f32(3 * D, D), "w_out": f32(D, D), "w_r": f32(D, E), "q_gain": f32(64), "k_gain": f32(64), "table": f32(BUCKETS, H)}
        self.ws = torch.empty(1 << 20, device=dev)

    def run(self):
        p, g, M, at = self.p, self.g, B * S, dict(max_distance=24, causal=self.causal, lengths=self.p["lengths"])
        rot = dict(q_gain=p["q_gain"], k_gain=p["k_gain"], rotary=self.angles)
        ops.gemm(p["x"], p["w_in"], self.qkv, M, 3 * D, D, transB=True)
        ops.qk_norm_rotary_fwd(self.qkv, self.rot, B, S, H, **rot)
        ops.attention_relbias_fwd(self.rot, p["table"], self.att, self.lse, B, S, H, 0.125, **at)
        ops.gemm(self.att, p["w_out"], self.proj, M, D, D, transB=True)
        ops.add_layernorm_fwd(self.proj, p["x"], self.y, self.rstd)
        ops.gemm(self.y, p["w_r"], self.logits, M, E, D)
        ops.top2_gate_into(self.logits, C, self.r)
        ops.balance_loss_fwd(self.r, self.loss, self.counts, self.kept, self.sums, coef=COEF, lengths=p["lengths"], workspace=self.ws)
        ops.moe_dispatch(self.y, self.r, self.ein, E, C, 0, E)
        ops.moe_combine(self.ein, self.r, self.z, C, 0, E)
        # backward: dz = w
        ops.moe_combine_bwd(p["w"], self.ein, self.r, self.dein, self.dgate, E, C, 0, E)
        ops.moe_dispatch_bwd(self.dein, self.r, self.dy, C, 0, E, accumulate=False)
        ops.balance_loss_bwd(self.r, self.counts, self.dlogits, coef=COEF, dgate=self.dgate, lengths=p["lengths"])
        ops.cast(self.dlogits, self.dlogits_bf)
        ops.gemm(self.y, self.dlogits_bf, g["w_r"], D, E, M, transA=True, workspace=self.ws)
        ops.gemm(self.dlogits_bf, p["w_r"], self.dy, M, D, E, transB=True, accumulate=True)
        ops.layernorm_bwd(self.dy, self.y, self.rstd, None, self.dsum)
        ops.gemm(self.dsum, self.att, g["w_out"], D, D, M, transA=True, workspace=self.ws)
        ops.gemm(self.dsum, p["w_out"], self.datt, M, D, D)
        ops.attention_relbias_bwd(self.rot, p["table"], self.att, self.datt, self.lse, self.drot, g["table"], self.delta, B, S, H, 0.125, workspace=self.ws, **at)
        ops.qk_norm_rotary_bwd(self.drot, self.qkv, self.dqkv, B, S, H, dq_gain=g["q_gain"], dk_gain=g["k_gain"], workspace=self.ws, **rot)
        ops.gemm(self.dqkv, p["x"], g["w_in"], 3 * D, D, M, transA=True, workspace=self.ws)

    def results(self):
        return [t.clone() for t in (self.loss, self.counts, self.kept, self.sums, self.z, *self.g.values())]


def reference(step, causal):
    p = {k: (v.double() if v.is_floating_point() else v) for k, v in parameters().items()}
    names = ("w_in", "w_out", "w_r", "q_gain", "k_gain", "table")
    for k in names:
        p[k].requires_grad_(True)
    qkv = p["x"] @ p["w_in"].t()
    angles = ops.rotary_table(S, 64)[None].expand(B, S, -1, 2)
    rot = L.qk_norm_forward(qkv, H, p["q_gain"], p["k_gain"], angles, False, 1e-6).reshape(B, S, 3 * D)
    att = L.relbias_forward(rot, p["table"], H, 0.125, 24, not causal, causal, p["lengths"])[0].reshape(B, S, D)
    y = torch.nn.functional.layer_norm(att @ p["w_out"].t() + p["x"], (D,))
    probs = torch.softmax(y @ p["w_r"], -1)
    index, slot = step.r["index"].cpu().long(), step.r["slot"].cpu()
    gates = probs.gather(-1, index) * (slot > 0)
    z = gates.sum(-1, keepdim=True) * y
    _, counts, _, _, _ = L.balance(probs.detach(), index, slot, 2, COEF, p["lengths"])
    balance = sum(COEF * E / B * (counts[b].double() / (2 * n) * probs[b, :n].mean(0)).sum() for b, n in enumerate(p["lengths"].tolist()))
    (balance + (z * p["w"]).sum()).backward()
    return balance.item(), counts, z.detach(), {k: p[k].grad for k in names}


@pytest.mark.parametrize("causal", [False, True])
def test_one_layer_forward_and_backward(cuda, causal):
    step = Step(cuda, causal)
    step.run()
    torch.cuda.synchronize()
    balance, counts, z, grads = reference(step, causal)
    assert torch.equal(step.counts.cpu(), counts)
    assert (step.kept <= step.counts).all() and step.kept.sum().item() <= 2 * (S + 41)
    assert abs(step.loss.item() - balance) < 2e-2 * balance
    rel = lambda a, b: ((a.double().cpu() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(step.z, z) < 2e-2
    for k, want in grads.items():
        assert rel(step.g[k], want) < 2e-2, (k, rel(step.g[k], want))


def test_the_step_in_a_replayed_graph(cuda):
    step = Step(cuda, True)
    step.run()
    torch.cuda.synchronize()
    want = step.results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    for i in range(5):
        for t in (step.loss, step.sums, step.z, step.lse, step.att, step.dqkv, *step.g.values()):
            t.fill_(float("nan"))
        step.counts.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.results(), want)), i
        ops.fill_value(step.ws, float(i))                      # eager work in between, in the shared scratch too


def test_the_step_as_a_recorded_launch_list(cuda):
    """The library's launch lists replay the recorded calls without re-marshalling their arguments."""
    from hap_amd import _lib
    step = Step(cuda, False)
    _lib.start_recording()
    try:
        step.run()
        # scratch of the calls' own has to outlive the call
        ops.balance_loss_fwd(step.r, step.loss, step.counts, step.kept, step.sums, coef=COEF, lengths=step.p["lengths"])
        ops.attention_relbias_bwd(step.rot, step.p["table"], step.att, step.datt, step.lse, step.drot, step.g["table"], step.delta, B, S, H, 0.125,
                                  max_distance=24, lengths=step.p["lengths"])
    finally:
        calls = _lib.stop_recording()
    torch.cuda.synchronize()
    want = step.results()
    for i in range(3):
        for t in (step.loss, step.sums, step.z, *step.g.values()):
            t.fill_(float("nan"))
        junk = [torch.full((1 << 16,), float("nan"), device=cuda) for _ in range(8)]         # takes freed memory, if there is any
        _lib.replay(calls)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.results(), want)), i
        del junk


def test_the_documented_step_gives_the_gradients_of_its_own_forward(cuda):
    """The code block of the integration guide, run as it stands: the norm's backward has to find forward's input."""
    import os
    import re
    guide = open(os.path.join(os.path.dirname(__file__), "..", "INTEGRATION.md")).read()
    block = [b for b in re.findall(r"```python\n(.*?)```", guide, re.S) if "qk_norm_rotary_fwd" in b]
    assert len(block) == 1
    b, S_, H_, n = 2, 40, 2, [40, 23]
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    qkv, dout, table, qg, kg = r(b, S_, 3 * H_ * 64).bfloat16(), r(b, S_, H_ * 64).bfloat16(), r(32, H_), 1 + 0.2 * r(64), 1 + 0.2 * r(64)
    dout[1, 23:] = 0
    records = ops.top2_gate(r(b, S_, 4).to(cuda), 20)
    up = lambda t: t.to(cuda)  # noqa: E731
    f32 = lambda *s: torch.full(s, float("nan"), device=cuda)  # noqa: E731
    x = up(qkv)
    names = dict(ops=ops, b=b, S=S_, H=H_, dev=cuda, qkv=x, rot=torch.empty_like(x), dqkv=torch.empty_like(x), q_gain=up(qg), k_gain=up(kg),
                 table=up(table), out=torch.empty_like(up(dout)), dout=up(dout), lse=f32(b, H_, S_), delta=f32(b, H_, S_), dtable=f32(32, H_),
                 dq_gain=f32(64), dk_gain=f32(64), lengths=torch.tensor(n, dtype=torch.int32, device=cuda), records=records, loss=f32(1),
                 counts=torch.empty(b, 4, dtype=torch.int32, device=cuda), kept=torch.empty(b, 4, dtype=torch.int32, device=cuda),
                 prob_sum=f32(b, 4), dlogits=f32(b, S_, 4), dgate=up(r(b, S_, 2)))
    exec(block[0], names)
    torch.cuda.synchronize()
    p = {k: v.double().requires_grad_(True) for k, v in (("qkv", qkv), ("table", table), ("qg", qg), ("kg", kg))}
    angles = ops.rotary_table(S_, 64)[None].expand(b, S_, -1, 2)
    rot = L.qk_norm_forward(p["qkv"], H_, p["qg"], p["kg"], angles, False, 1e-6).reshape(b, S_, -1)
    att = L.relbias_forward(rot, p["table"], H_, 0.125, 128, True, False, torch.tensor(n))[0].reshape(b, S_, -1)
    (att * dout.double()).sum().backward()
    rel = lambda a, w: ((a.double().cpu() - w).norm() / w.norm()).item()  # noqa: E731
    for k, got in (("qkv", names["dqkv"]), ("table", names["dtable"]), ("qg", names["dq_gain"]), ("kg", names["dk_gain"])):
        assert rel(got, p[k].grad) < 2e-2, (k, rel(got, p[k].grad))
    _, counts, _, _, _ = L.balance(records["probs"].cpu(), records["index"].cpu(), records["slot"].cpu(), 2, 0.01)
    assert torch.equal(names["counts"].cpu(), counts)
