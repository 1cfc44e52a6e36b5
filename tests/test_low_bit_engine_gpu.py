"""The engine with 4-bit weights, and with requests that draw from the likeliest tokens."""

import json
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import helpers as H
from plain import qwen2_plain

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def in_4_bits(w):
    """A matrix as its 4-bit form holds it: per 128 elements of a row, multiples of bf16(max / 7) within -8 .. 7."""
    N, K = w.shape
    G = -(-K // 128)
    g = torch.nn.functional.pad(w, (0, G * 128 - K)).view(N, G, 128)
    s = (g.abs().amax(dim=2, keepdim=True) / 7).to(torch.bfloat16).float()
    return (torch.round(g / torch.where(s > 0, s, 1.0)).clamp(-8, 7) * s).view(N, -1)[:, :K]


@pytest.fixture(scope="module")
def model_dirs(tmp_path_factory):
    out = {}
    for n, (name, raw) in enumerate(H.TINY.items()):
        d = tmp_path_factory.mktemp(f"low_{name}")
        # sharpen=1: scores of attention of moderate size (a score's error would multiply its weight's otherwise)
        H.make_model_dir(d, raw, seed=500 + n, sharpen=1.0)
        out[name] = d
    return out


@pytest.mark.parametrize("name", list(H.TINY))
def test_logits_are_those_of_the_4_bit_weights(model_dirs, name):
    """Against the plain implementation with the layers' matrices in 4 bits.  What is left is the 8-bit rows: a group's step is max / 127, so a
    row is off by max / 127 / sqrt(12) / rms = 0.65 % (max of 128 normal numbers: 2.8 rms), four times a layer, and each layer's bf16 roundings, 0.3 % all
    told: after three layers sqrt(3 (4 0.65^2 + 0.3^2)) = 2.3 %.  Twice that is allowed for rows with fewer elements and larger peaks."""
    from pyre_b200 import Engine, SamplingParams
    d, raw = model_dirs[name], H.TINY[name]
    weights = H.load_plain_weights(d, round_matrices_to_bf16=True)
    low = {k: in_4_bits(v) if v.dim() == 2 and ".layers." in k else v for k, v in weights.items()}
    eng = Engine(d, weight_bits=4, page_size=H.PAGE_SIZE[name], max_cache_tokens=1024, max_num_seqs=8, max_num_batched_tokens=64, prefill_chunk=24)
    prompts = [H.random_ids(raw["vocab_size"], n, seed=n) for n in (1, 7, 40, 63)]
    outs = eng.generate(prompts, SamplingParams(max_new_tokens=12, return_logits=True))
    off, other = [], []
    for p, o in zip(prompts, outs):
        ids = list(p) + o.token_ids
        with torch.inference_mode():
            want, plain = (qwen2_plain.forward(ids[:-1], w, raw).numpy()[len(p) - 1:] for w in (low, weights))
        off.append(np.linalg.norm(o.logits - want) / np.linalg.norm(want))
        other.append(np.linalg.norm(plain - want) / np.linalg.norm(want))
    assert max(off) <= 0.046, off
    assert np.mean(off) < np.mean(other), "the weights in 4 bits are nearer than those they were made from"
    assert eng.stepper.graph_replays > 0


def test_batched_and_alone_and_without_graphs(model_dirs):
    """Tokens of a request beside others are those of its logits alone, near ties aside; captured steps give what eager ones give."""
    from pyre_b200 import Engine, SamplingParams
    raw = H.TINY["B"]
    prompts = [H.random_ids(raw["vocab_size"], n, seed=n) for n in (5, 30, 71)]
    kw = dict(weight_bits=4, max_cache_tokens=1024, max_num_seqs=8, prefill_chunk=32)
    params = SamplingParams(max_new_tokens=10, return_logits=True)
    together = Engine(model_dirs["B"], **kw).generate(prompts, params)
    eager = Engine(model_dirs["B"], cuda_graphs=False, **kw).generate(prompts, params)
    for a, b in zip(together, eager):
        assert a.token_ids == b.token_ids
        # the same kernels on the same rows, in steps that are padded or not
        assert np.array_equal(a.logits, b.logits)


def test_drawing_from_the_likeliest(model_dirs):
    """Each request's tokens lie among its likeliest ones, are its own (not the batch's), and come again from the same seed."""
    from pyre_b200 import Engine, SamplingParams
    raw = H.TINY["B"]
    prompts = [H.random_ids(raw["vocab_size"], n, seed=n) for n in (4, 9, 17, 25)]
    params = [SamplingParams(temperature=1.5, seed=3, max_new_tokens=14, top_k=4, return_logits=True),
              SamplingParams(max_new_tokens=14, return_logits=True),
              SamplingParams(temperature=1.2, seed=4, max_new_tokens=14, return_logits=True),
              SamplingParams(temperature=2.0, seed=5, max_new_tokens=14, top_p=0.3, min_p=0.5, return_logits=True)]
    for kw in ({}, {"weight_bits": 4}, {"dtype": "float32"}):
        eng = Engine(model_dirs["B"], max_cache_tokens=1024, max_num_seqs=8, **kw)
        outs = eng.generate(prompts, params)
        again = eng.generate(prompts, params)
        assert [o.token_ids for o in outs] == [o.token_ids for o in again]
        for tok, row in zip(outs[0].token_ids, outs[0].logits):
            assert tok in np.argsort(-row, kind="stable")[:4]
        for tok, row in zip(outs[1].token_ids, outs[1].logits):
            assert tok == int(np.argmax(row))
        for tok, row in zip(outs[3].token_ids, outs[3].logits):
            assert np.exp((row[tok] - row.max()) / 2.0) >= 0.5 * (1 - 1e-5)
        # without filters in the batch the unfiltered request draws through the other kernels: the same tokens, as long as its logits are
        alone = eng.generate([prompts[1], prompts[2]], [params[1], params[2]])
        same = [np.array_equal(a, b) for a, b in zip(alone[1].logits, outs[2].logits)]
        n = same.index(False) if False in same else len(same)
        assert alone[1].token_ids[:n] == outs[2].token_ids[:n]


def test_command_line(model_dirs, tmp_path):
    out = tmp_path / "r.json"
    run = subprocess.run([sys.executable, "-m", "pyre_b200", "generate", "--model", str(model_dirs["B"]), "--prompt-ids", "5,17,3", "--max-new-tokens", "6",
                          "--temperature", "0.9", "--top-k", "5", "--top-p", "0.9", "--min-p", "0.01", "--weight-bits", "4", "--num-pages", "32", "--out", str(out)],
                         cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert len(json.loads(out.read_text())["outputs"][0]["token_ids"]) == 6
