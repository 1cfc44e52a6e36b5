"""Logits that are no numbers, in rows without filters: they count as -inf, in the kernels without filters as in the one with them."""

import pytest
import torch

import test_sample_filters_gpu as filters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 50, 700, 3000, 9000, 16384, 40000])
def test_a_nan_counts_as_minus_infinity(V):
    from pyre_b200.kernels import ops
    R = 18
    logits = torch.randn((R, V), generator=filters.gen(V), device="cuda") * 2
    nan = float("nan")
    logits[0:2, 0] = nan
    logits[2:4, :1024] = nan          # what any thread of a block sees first
    logits[4:6, ::4096] = nan         # where slices start
    logits[6:8, ::2] = nan
    logits[8:10] = nan                # nothing is left
    last = logits[10:12, -1:].clone()
    logits[10:12] = nan
    logits[10:12, -1:] = last         # one entry is left
    logits[12:14, :V // 2] = nan
    logits[12:14, V // 2:] = float("-inf")
    logits[14:16, 0] = nan
    logits[14:16, -1] = float("inf")
    T = torch.where(torch.arange(R, device="cuda") % 2 == 0, 0.0, 0.8)
    seeds, index = torch.arange(R, device="cuda") * 31, torch.arange(R, device="cuda", dtype=torch.int32)
    zero, one = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.ones(R, device="cuda")
    ids = ops.sample(logits, T, seeds, index)
    filters.check(ids, logits, T, seeds, index, zero, one, one * 0)
    assert torch.equal(ids, filters.call(logits, T, seeds, index, zero, one, one * 0))
    assert torch.equal(ids, ops.sample(torch.where(torch.isnan(logits), float("-inf"), logits), T, seeds, index))
    # all rows greedy: no temperature at all
    best = torch.where(torch.isnan(logits), float("-inf"), logits)
    first = (best == best.amax(dim=1, keepdim=True)).int().argmax(dim=1)
    assert torch.equal(ops.sample(logits).long(), first)


def test_an_infinite_temperature_and_masked_entries():
    """-inf times 0 is no number: such a token is not drawn, with either kernel."""
    from pyre_b200.kernels import ops
    for V in (700, 3000, 40000):
        R = 12
        logits = torch.randn((R, V), generator=filters.gen(V + 1), device="cuda")
        logits[:, :1024 if V > 1024 else V // 2] = float("-inf")
        logits[1::2, ::2] = float("-inf")
        T = torch.full((R,), float("inf"), device="cuda")
        seeds, index = torch.arange(R, device="cuda") * 17, torch.arange(R, device="cuda", dtype=torch.int32)
        ids = ops.sample(logits, T, seeds, index)
        off = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.ones(R, device="cuda"), torch.zeros(R, device="cuda")
        assert torch.equal(ids, filters.call(logits, T, seeds, index, *off))
        noise = torch.where(logits == float("-inf"), float("-inf"), filters.noise(seeds, index, V))
        for r in range(R):
            assert float(noise[r, int(ids[r])]) >= float(noise[r].max()) - 2.0 ** -18 * (1 + abs(float(noise[r].max())))
