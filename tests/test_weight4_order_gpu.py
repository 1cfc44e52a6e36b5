"""A product and what has just written its 4-bit weight: only a weight that was waited for is read ahead of the kernels in front of it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def normal(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.fixture
def read_ahead(monkeypatch):
    """What each product was told about its weight."""
    from pyre_b200.kernels import ops
    seen, real = [], ops.lib.call

    def call(name, *args):
        if name == "pyre_w4_linear":
            seen.append(bool(args[10]))
        return real(name, *args)

    monkeypatch.setattr(ops.lib, "call", call)
    return seen


def test_which_weights_are_read_ahead(read_ahead):
    from pyre_b200.kernels import ops
    x, plain = ops.quantize_rows8(normal(1, 5, 512)), normal(2, 200, 512)

    def ahead(w):
        ops.linear(x, w)
        return read_ahead[-1]

    loaded = ops.linear_weight(plain, 4)
    assert loaded.settled and ahead(loaded)
    made = ops.quantize_weight4(plain)
    assert not made.settled and not ahead(made) and not ahead(made)      # a product before does not settle it
    given = ops.Weight4(made.packed.clone(), made.scales.clone(), 512)
    assert not ahead(given)
    assert given.settle() is given and ahead(given)
    for change in (lambda: given.packed.copy_(made.packed), lambda: given.scales.mul_(1)):
        change()
        assert not given.settled and not ahead(given) and not ahead(given)
        assert ahead(given.settle())
    with torch.inference_mode():      # of ordinary tensors: their versions count
        given.scales.mul_(1)
    assert not ahead(given)
    for name in ("packed", "scales"):      # other tensors in the same handle
        given.settle()
        setattr(given, name, getattr(given, name).clone())
        assert not ahead(given)
    other = ops.Weight4(given.packed, given.scales, 512)      # the same memory, with a handle of its own
    assert not ahead(other)
    with torch.inference_mode():
        assert not ahead(ops.quantize_weight4(plain).settle())


def test_parts_of_a_model_settle_theirs(read_ahead):
    from pyre_b200.parts.base import PartSpec, load_part, make_part
    part = make_part("ffn", PartSpec("gated_mlp", {"width": 256, "intermediate": 384, "weight_bits": 4}), torch.bfloat16, torch.device("cuda:0"))
    load_part(part, {f"{n}_proj.weight": normal(i, *s) for i, (n, s) in enumerate((("gate", (384, 256)), ("up", (384, 256)), ("down", (256, 384))))}, "")
    assert part.w_gate_up.settled and part.w_down.settled


@pytest.mark.parametrize("T", [1, 20, 50, 300])
@pytest.mark.parametrize("settled", [False, True])
def test_weights_written_just_before(T, settled):
    """A kernel writes the weight, another one that lets its successors start early comes between, then the product: eager, and captured with the
    writing kernel in the graph or in front of it."""
    from pyre_b200.kernels import ops
    N, K = 9000, 4096
    both = [ops.quantize_weight4(normal(3 + i, N, K)) for i in range(2)]
    rows = normal(7, T, K)
    torch.cuda.synchronize()
    want = []
    for w in both:
        want.append(ops.linear(ops.quantize_rows8(rows), w))
        torch.cuda.synchronize()
    w = ops.Weight4(both[0].packed.clone(), both[0].scales.clone(), K)
    if settled:
        w.settle()

    def write(i):
        w.packed.copy_(both[i].packed)
        w.scales.copy_(both[i].scales)

    got = []
    for i in range(30):
        write(i % 2)
        got.append(ops.linear(ops.quantize_rows8(rows), w))
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    if settled:
        w.settle()
    alone = torch.cuda.CUDAGraph()
    with torch.cuda.graph(alone):
        y = ops.linear(ops.quantize_rows8(rows), w)
    whole = torch.cuda.CUDAGraph()
    with torch.cuda.graph(whole):
        for i in range(2):
            write(i)
            x = ops.quantize_rows8(rows)
            z = ops.linear(x, w)
            z2 = ops.linear(x, w)
    for i in range(20):
        write(i % 2)
        alone.replay()
        assert torch.equal(y, want[i % 2])
        whole.replay()
        assert torch.equal(z, want[1]) and torch.equal(z2, want[1])
