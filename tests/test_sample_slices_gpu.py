"""Filtered sampling where a CTA's part of a row just fits into its share of an SM's shared memory, and where it just does not: the same tokens."""

import pytest
import torch

import test_sample_filters_gpu as filters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per_cta", [17600, 17696, 17700, 17704, 17708, 18500, 19700, 19712])
@pytest.mark.parametrize("cluster,R", [(1, 160), (2, 80), (4, 40), (16, 9)])
def test_slices_about_the_limit(per_cta, cluster, R, monkeypatch):
    from pyre_b200.kernels import ops
    V = per_cta * cluster
    logits = torch.randn((R, V), generator=filters.gen(per_cta), device="cuda") * 2
    rule = filters.rules(per_cta, R)
    monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", cluster)
    ids = filters.call(logits, *rule)
    filters.check(ids[:18], logits[:18], *(t[:18] for t in rule))
    monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", 0)
    assert torch.equal(filters.call(logits, *rule), ids)
