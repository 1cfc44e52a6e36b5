"""Sampling by mass alone: rows whose border lies among some hundred to two thousand tokens of one step of the histogram, drawn again and again."""

import pytest
import torch

import test_sample_filters_gpu as filters

pytestmark = pytest.mark.gpu

IN_STEP = (150, 193, 200, 257, 300, 400, 511, 512, 513, 700, 1000, 1023, 1025, 1500, 1900, 2000)      # tokens beside the best one


def flat_rows(R, V, seed):
    """Row r has IN_STEP[r % 16] tokens within a hundredth of a step (1/64) of each other, the others 60 below them; and what asks for a mass of them."""
    g = filters.gen(seed)
    logits = torch.full((R, V), -60.0, device="cuda")
    for r in range(R):
        n = IN_STEP[r % len(IN_STEP)]
        at = torch.randperm(V, generator=g, device="cuda")[:n]
        logits[r, at] = 1.0 + torch.rand(n, generator=g, device="cuda") * (0.01 / 64)
    T = torch.full((R,), 1.0, device="cuda")
    seeds = torch.randint(0, 1 << 62, (R,), generator=g, device="cuda")
    index = torch.randint(0, 1000, (R,), generator=g, device="cuda", dtype=torch.int32)
    p = 0.03 + 0.94 * torch.rand(R, generator=g, device="cuda")
    return logits, T, seeds, index, p


@pytest.mark.parametrize("cluster", [0, 1, 2, 4, 8, 16])
def test_the_same_flat_rows_a_hundred_times(cluster, monkeypatch):
    """The first CTA narrows the step's tokens down by rounds; what one round leaves in shared memory is read by all warps before the next one writes it."""
    from pyre_b200.kernels import ops
    R, V = 256, 12000
    logits, T, seeds, index, p = flat_rows(R, V, 5)
    off = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, device="cuda")
    want = ops.sample(logits, T, seeds, index, top_p=p)
    filters.check(want, logits, T, seeds, index, off[0], p, off[1])
    monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", cluster)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(100):
        differ += (ops.sample(logits, T, seeds, index, top_p=p) != want).sum()
    assert int(differ) == 0
