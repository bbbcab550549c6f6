"""Clipping and Adam of the driver's loop (worker.py:74-76) at full width, replayed on the CPU from the gradients that the GPU
computed, with the clipping norm summed in float64.

torch's own float32 norm is no yardstick at this size: its CPU sum over the 9e7 squared elements of this shard comes out 0.12 to
0.23 % low (printed below), and Adam's updates of elements whose gradient is near its epsilon follow."""
import pytest
import torch

import hap_amd
from hap_amd import driver


@pytest.mark.gpu
def test_clipping_and_adam_against_a_float64_norm(cuda):
    """Two layers of the BERT-large shard in bf16, four steps with clip_grad_norm_(0.5) and Adam lr 5e-4.

    The GPU's norm adds 64 squares a thread, 9e7 / 16384 / 256 = 22 chunks a thread and two trees of 16 + 6 in float32: the sum is good
    to (64 + 22 + 44) * 2^-24 = 8e-6, the norm and the coefficient to half of it, and so are m and sqrt(v) in it: with some 16 float32
    roundings on either side an update, at most 1.1 lr in size over the first steps, is good to 2 * 4e-6 + 32 * 2^-24 = 1e-5 of
    that: four steps 4 * 1.1 * 5e-4 * 1e-5 = 2.2e-8.  The master itself is rounded once a step on either side: 8 * 2^-24 of it."""
    import bench
    iters, clip, lr = 4, 0.5, 5e-4
    gm, x, y, meta = bench.build_workload("bert", layers_override=2)
    ex = hap_amd.compile_program(gm, [x, y], dtype="bf16", wire=hap_amd.SyntheticWire(seed=11), rank=0, world_size=len(meta["ratios"]))
    twins = {n: rec["master"].cpu().clone().requires_grad_(True) for n, rec in ex.params.items()}
    opt = torch.optim.Adam(list(twins.values()), lr=lr)
    torch.set_num_threads(16)
    norms = []

    def replay(it, executor):
        torch.cuda.synchronize()
        grads = {n: executor.params[n]["grad"].cpu().clone() for n in twins}
        norm = sum(g.double().pow(2).sum() for g in grads.values()).sqrt().item()
        norms.append((norm, torch.nn.utils.get_total_norm(list(grads.values())).item()))
        coef = min(1.0, clip / (norm + 1e-6))
        for n, g in grads.items():
            twins[n].grad = (g.double() * coef).float()
        opt.step()

    driver.train_loop(ex, x, y, batch_size=32, seqlen=512, run_iter=iters, log_iter=iters, avg_iter=2, lr=lr, clip_grad_norm=clip, report=lambda line: None,
                      after_backward=replay)
    torch.cuda.synchronize()
    print("\n  norms in float64 and by torch in float32 on the CPU:", norms)
    assert all(a > 100 * clip for a, _ in norms)               # clipping was at work in every step
    for n, rec in ex.params.items():
        got, want = rec["master"].cpu().double(), twins[n].detach().double()
        off = (got - want).abs() - (2.2e-8 + 8 * 2.0 ** -24 * want.abs())
        assert off.max() <= 0, (n, off.max().item(), (got - want).abs().max().item())
