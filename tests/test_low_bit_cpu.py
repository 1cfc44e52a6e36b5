"""4-bit weights and filtered sampling on the host: what the configuration, the model's data and the sampler make of them."""

import numpy as np
import pytest
import torch

import helpers as H


def test_engine_configuration():
    from pyre_b200.config import EngineConfig
    assert EngineConfig().weight_bits is None and EngineConfig(weight_bits=4).weight_bits == 4
    with pytest.raises(ValueError, match="weight_bits must be 4"):
        EngineConfig(weight_bits=8)
    with pytest.raises(ValueError, match="go with dtype bfloat16"):
        EngineConfig(dtype="float32", weight_bits=4)


def test_sampling_parameters():
    from pyre_b200.sampling import SamplingParams
    assert not SamplingParams(temperature=1.0).filters and not SamplingParams(top_k=5).filters
    assert all(SamplingParams(temperature=0.5, **kw).filters for kw in ({"top_k": 1}, {"top_p": 0.9}, {"min_p": 0.1}))
    for kw in ({"top_k": -1}, {"top_k": 1 << 31}, {"top_p": 0.0}, {"top_p": 1.1}, {"top_p": float("nan")}, {"min_p": -0.1}, {"min_p": 1.5}):
        with pytest.raises(ValueError, match=next(iter(kw))):
            SamplingParams(temperature=1.0, **kw)


def test_parts_with_weights_in_4_bits_keep_the_checkpoints_names():
    from pyre_b200.config import architecture_of, config_from_dict
    from pyre_b200.models.model import Model, tensor_table
    from pyre_b200.models.spec import with_weight_bits
    cfg = config_from_dict(H.TINY["B"])
    plain = architecture_of(cfg).build(cfg)
    low = with_weight_bits(plain, 4)
    assert with_weight_bits(plain, None) is plain
    assert tensor_table(low) == tensor_table(plain)
    model = Model(low, torch.bfloat16, "meta")
    for block in model.blocks:
        assert block.mixer.weight_bits == block.ffn.weight_bits == 4
        assert block._kw1 == block._kw2 == {"rows8_ok": True}
        assert not block.mixer.takes_scaled_rows and not block.ffn.interleaved
    assert {"gemm_w4", "rows8"} <= set(model.kernel_libraries())
    other = Model(plain, torch.bfloat16, "meta")
    assert not {"gemm_w4", "rows8"} & set(other.kernel_libraries())
    assert all("rows8_ok" not in b._kw1 for b in other.blocks)


def test_an_architecture_without_them_is_refused():
    import modovik_helpers
    from pyre_b200.config import architecture_of, config_from_dict
    from pyre_b200.models.spec import with_weight_bits
    from pyre_b200.kernels import ops
    from pyre_b200.parts.base import PartSpec, make_part
    raw = next(v for v in vars(modovik_helpers).values() if isinstance(v, dict) and v.get("architecture") == "Modovik")
    cfg = config_from_dict(raw)
    with pytest.raises(ValueError, match="in 4 bits"):
        spec = with_weight_bits(architecture_of(cfg).build(cfg), 4)
        [make_part("block", b, torch.bfloat16, "meta") for b in spec.blocks]
    attention = {"width": 64, "n_heads": 4, "n_kv_heads": 2, "head_dim": 16, "weight_bits": 4}
    make_part("mixer", PartSpec("attention", attention), torch.bfloat16, "meta")
    with pytest.raises(ops.UnsupportedSize, match="plain attention only"):
        make_part("mixer", PartSpec("attention", {**attention, "out_gate": True}), torch.bfloat16, "meta")
    with pytest.raises(ops.UnsupportedSize, match="weights of 3 bits"):
        make_part("mixer", PartSpec("attention", {**attention, "weight_bits": 3}), torch.bfloat16, "meta")


def test_the_sampler_sends_filters_only_where_a_row_has_one(monkeypatch):
    from pyre_b200.kernels import ops
    from pyre_b200.sampling import Sampler, SamplingParams
    seen = []

    def fake(logits, temperature=None, seeds=None, token_index=None, **kw):
        seen.append((temperature, kw))
        return torch.zeros(logits.shape[0], dtype=torch.int32)

    class Event:
        def record(self):
            pass

        def synchronize(self):
            pass

    monkeypatch.setattr(ops, "sample", fake)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **kw: real(*a, **kw))
    s = Sampler("cpu")
    logits = torch.zeros((3, 10))
    s.sample(logits, [SamplingParams(), SamplingParams(top_k=3), SamplingParams()], [0, 0, 0])
    assert seen[-1] == (None, {})
    s.sample(logits, [SamplingParams(), SamplingParams(temperature=1.0), SamplingParams()], [0, 0, 0])
    assert seen[-1][1] == {} and seen[-1][0].tolist() == [0.0, 1.0, 0.0]
    s.sample(logits, [SamplingParams(temperature=0.5, top_k=7, min_p=0.25), SamplingParams(), SamplingParams(temperature=1.0, top_p=0.5)], [0, 0, 0])
    temperature, kw = seen[-1]
    assert temperature.tolist() == [0.5, 0.0, 1.0]
    assert kw["top_k"].tolist() == [7, 0, 0] and kw["top_p"].tolist() == [1.0, 1.0, 0.5] and kw["min_p"].tolist() == [0.25, 0.0, 0.0]
    assert kw["top_k"].dtype == torch.int32 and kw["top_p"].dtype == kw["min_p"].dtype == torch.float32


def test_forms_are_checked_before_anything_is_launched():
    from pyre_b200.kernels import ops
    rows, scales = torch.zeros((3, 256), dtype=torch.int8), torch.zeros((2, 3))
    assert ops.Rows8(rows, scales, 200).shape == (3, 200)
    for bad in ((rows, scales, 300), (rows, scales, 128), (rows.float(), scales, 200), (rows, scales.t(), 200), (rows, scales.double(), 200), (rows, scales, 0)):
        with pytest.raises(ValueError):
            ops.Rows8(*bad)
    with pytest.raises(ValueError, match="CUDA"):
        ops.materialize(ops.Rows8(rows, scales, 200))
    packed, ws = torch.zeros((5, 128), dtype=torch.uint8), torch.zeros((2, 5), dtype=torch.bfloat16)
    for bad in ((packed, ws, 300), (packed, ws, 100), (packed.int(), ws, 200), (packed, ws.float(), 200), (packed, ws.t(), 200), (packed, ws, 200)):
        with pytest.raises(ValueError):      # the last one: on the CPU
            ops.Weight4(*bad)
    for f in (ops.quantize_rows8, ops.quantize_weight4):
        with pytest.raises(ValueError, match="CUDA"):
            f(torch.zeros((2, 64)))
    with pytest.raises(ValueError, match="CUDA"):
        ops.add_rmsnorm_rows8(torch.zeros((2, 64)), None, torch.ones(64), 1e-6)
