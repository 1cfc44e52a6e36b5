"""Which models take weights in 4 bits: all of a model's products, or a refusal."""

import pytest

from pyre_b200.models.spec import ModelSpec, with_weight_bits
from pyre_b200.parts.base import PartSpec


def spec(*blocks):
    return ModelSpec(vocab_size=64, width=32, embed=PartSpec("token_embedding", {"vocab": 64, "width": 32}), blocks=list(blocks), schedule=[],
                     final_norm=PartSpec("rms_norm", {"width": 32, "eps": 1e-6}), head=PartSpec("linear_head", {"vocab": 64, "width": 32}))


ATTENTION = PartSpec("attention", {"width": 32, "n_heads": 2, "n_kv_heads": 1, "head_dim": 16})
FFN = PartSpec("gated_mlp", {"width": 32, "intermediate": 64})


def test_every_mixer_and_feed_forward_takes_them():
    low = with_weight_bits(spec(PartSpec("prenorm", {"mixer": ATTENTION, "ffn": FFN}), PartSpec("output_norm", {"mixer": ATTENTION, "ffn": None})), 4)
    assert [b.params[r].params["weight_bits"] for b, r in zip([low.blocks[0], low.blocks[0], low.blocks[1]], ("mixer", "ffn", "mixer"))] == [4, 4, 4]
    assert low.blocks[1].params["ffn"] is None and "weight_bits" not in ATTENTION.params


@pytest.mark.parametrize("other", [PartSpec("own_arrangement", {"left": ATTENTION, "right": FFN}), PartSpec("own_arrangement", {"mixer": None, "ffn": None})])
def test_a_block_without_either_is_refused(other):
    with pytest.raises(ValueError, match="neither a mixer nor a feed-forward"):
        with_weight_bits(spec(PartSpec("prenorm", {"mixer": ATTENTION, "ffn": FFN}), other), 4)
    assert len(with_weight_bits(spec(other), None).blocks) == 1
