"""With 4-bit weights a request alone, beside a few and beside many: the products' variants and shares go by the number of rows."""

import numpy as np
import pytest
import torch

import helpers as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["B", "D"])
def test_alone_beside_a_few_and_beside_many(tmp_path, name):
    """Each run's logits are off those of the 4-bit weights' values by 4.6 % at most (two 8-bit and bf16 roundings a product: 2.3 % after three layers, twice
    that allowed, as where they are compared with the plain model), so two runs' by 9.2 % of each other, as long as their tokens are the same.  Where a token
    differs, the two candidates were as near each other as twice the largest difference between the two runs' logits."""
    from pyre_b200 import Engine, SamplingParams
    raw = H.TINY[name]
    H.make_model_dir(tmp_path / name, raw, seed=600, sharpen=1.0)
    prompts = [H.random_ids(raw["vocab_size"], 3 + (7 * i) % 29, seed=40 + i) for i in range(44)]
    params = SamplingParams(max_new_tokens=9, return_logits=True)
    kw = dict(weight_bits=4, page_size=H.PAGE_SIZE[name], max_cache_tokens=44 * 128, max_num_seqs=44, max_num_batched_tokens=256, prefill_chunk=64)
    eng = Engine(tmp_path / name, **kw)
    many = eng.generate(prompts, params)
    chosen = (0, 9, 21, 43)
    for group in (1, 4, 12, 20, 30):
        others = [eng.generate([prompts[(i + j) % 44] for j in range(group)], params)[0] for i in chosen]
        for i, o in zip(chosen, others):
            a, b = o.logits, many[i].logits
            same = [x == y for x, y in zip(o.token_ids, many[i].token_ids)]
            n = same.index(False) if False in same else len(same) - 1      # steps 0 .. n have the same tokens before them
            for k in range(n + 1):
                off = np.linalg.norm(a[k] - b[k]) / np.linalg.norm(b[k])
                assert off <= 0.092, (group, i, k, off)
            if False in same:
                t, u = o.token_ids[n], many[i].token_ids[n]
                assert a[n][t] - a[n][u] <= 2 * np.abs(a[n] - b[n]).max(), (group, i, n)


def test_a_request_without_filters_beside_one_with(monkeypatch):
    """The same logits: the request's token is its own, whichever kernel the batch takes."""
    from pyre_b200.sampling import Sampler, SamplingParams
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    for V in (600, 9000, 40000):
        logits = torch.randn((6, V), generator=g, device="cuda") * 2
        logits[2, :5] = float("nan")
        plain = [SamplingParams(temperature=1.2, seed=4), SamplingParams(), SamplingParams(temperature=0.7, seed=9)]
        filtered = [SamplingParams(temperature=1.0, seed=1, top_k=3), SamplingParams(temperature=1.5, seed=2, top_p=0.4, min_p=0.1), SamplingParams(top_k=2)]
        s = Sampler("cuda:0")
        for index in range(40):
            alone = s.sample(logits[:3].contiguous(), plain, [index] * 3)
            assert s.sample(logits, plain + filtered, [index] * 6)[:3] == alone
