"""Rows in 8 bits, 4-bit weights and their product against plain evaluations in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

GROUP = 128
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # a rounding's largest relative error


@pytest.fixture(autouse=True)
def _no_device_error():
    from pyre_b200.kernels import ops
    yield
    ops.check_device_errors("cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def grouped(y):
    """[T, K] -> [T, G, 128] in 64 bits, zeros beyond K."""
    T, K = y.shape
    G = -(-K // GROUP)
    return torch.nn.functional.pad(y.double(), (0, G * GROUP - K)).view(T, G, GROUP)


def values(r):
    T, K = r.shape
    return (r.rows.view(T, -1, GROUP).double() * r.scales.double().t()[:, :, None]).view(T, -1)[:, :K]


def check_rows8(r, y):
    """``r`` against the exact rows ``y`` (64 bits).  A scale is off by the roundings that led to it: the division, and 2^-20 relative for y
    itself (a norm's sums in 32 bits over thousands of terms, an activation's exponential; generous by a factor of four).  A value is
    off by at most half a scale, by 127 scales' errors, and by y's own error."""
    T, K = r.shape
    assert (T, K) == tuple(y.shape)
    g = grouped(y)
    most = g.abs().amax(dim=2)
    want = most / 127
    near = 2.0 ** -20
    assert ((r.scales.double().t() - want).abs() <= want * near).all()
    assert (r.rows.view(T, -1).int().abs() <= 127).all()
    off = (grouped(values(r)) - g).abs()
    assert (off <= want[:, :, None] * (0.5 + 2 * 127 * near)).all()
    # the largest element of a group takes the largest byte
    assert (r.rows.view(T, -1, GROUP).int().abs().amax(dim=2)[want > 0] == 127).all()
    assert (r.rows.view(T, -1)[:, K:] == 0).all()


@pytest.mark.parametrize("T,H", [(1, 64), (1, 3584), (3, 129), (5, 1001), (7, 130), (2, 4), (1, 1), (130, 896), (9, 8192), (2, 16640), (3, 9001)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm(T, H, dtype):
    from pyre_b200.kernels import ops
    x, d, w = normal(1, T, H), normal(2, T, H, dtype=dtype), 1 + 0.1 * normal(3, H)
    v = x.double() + d.double()
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * w.double()
    r = ops.add_rmsnorm_rows8(x, d, w, 1e-6, dtype=dtype)
    check_rows8(r, y)
    assert r.dtype == dtype and (x.double() - v).abs().max() <= 2.0 ** -24 * v.abs().max()
    back = ops.materialize(r)
    assert back.dtype == dtype
    assert ((back.double() - values(r)).abs() <= values(r).abs() * EPS[dtype] * 1.001 + 1e-37).all()


def test_norm_of_rows_partial_sums_and_a_stream_left_alone():
    from pyre_b200.kernels import ops
    T, H = 6, 1000
    x, w = normal(1, T, H), 1 + 0.1 * normal(3, H)
    parts = normal(2, 3, T, H)
    v = x.double() + parts.double().sum(0)
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-5) * w.double()
    kept = x.clone()
    rows = torch.tensor([5, 0, 5], dtype=torch.int32, device="cuda")
    r = ops.add_rmsnorm_rows8(x, ops.PartialSums(parts, torch.bfloat16), w, 1e-5, rows=rows)
    check_rows8(r, y[rows.long()])
    r = ops.add_rmsnorm_rows8(x, ops.PartialSums(parts, torch.bfloat16), w, 1e-5, update_x=False)
    check_rows8(r, y)
    assert torch.equal(x, kept)
    r = ops.add_rmsnorm_rows8(x, ops.PartialSums(parts, torch.bfloat16), w, 1e-5)
    check_rows8(r, y)
    assert (x.double() - v).abs().max() <= 4 * 2.0 ** -24 * (v.abs().max() + 4)
    v0 = kept.double()
    check_rows8(ops.add_rmsnorm_rows8(kept, None, w, 1e-5), v0 / torch.sqrt((v0 * v0).mean(dim=1, keepdim=True) + 1e-5) * w.double())
    empty = ops.add_rmsnorm_rows8(kept[:0], None, w, 1e-5)
    assert tuple(empty.shape) == (0, H) and ops.materialize(empty).shape == (0, H)


def test_rows_off_every_boundary():
    """Contiguous tensors that start off 16-byte boundaries take the same kernels by single elements."""
    from pyre_b200.kernels import ops
    T, H = 3, 256
    x = normal(1, T * H + 1)[1:].view(T, H)
    d = normal(2, T * H + 1, dtype=torch.bfloat16)[1:].view(T, H)
    w = normal(3, H + 1)[1:]
    v = x.double() + d.double()
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * w.double()
    check_rows8(ops.add_rmsnorm_rows8(x, d, w, 1e-6), y)
    check_rows8(ops.quantize_rows8(d), d.double())
    wide = normal(4, T, H + 5, dtype=torch.bfloat16)
    check_rows8(ops.quantize_rows8(wide[:, 3:H]), wide[:, 3:H].double())


def test_the_same_row_several_times_and_a_captured_norm():
    from pyre_b200.kernels import ops
    T, H = 6, 1100
    x, d, w = normal(11, T, H), normal(12, T, H, dtype=torch.bfloat16), 1 + 0.1 * normal(13, H)
    before = x.clone()
    rows = torch.tensor([5, 0, 5, 5, 2, 2, 1, 5, 3], dtype=torch.int32, device="cuda")
    v = (x.double() + d.double())[rows.long()]
    check_rows8(ops.add_rmsnorm_rows8(x, d, w, 1e-6, rows=rows), v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * w.double())
    assert torch.equal(x, before)      # rows may name one twice: nothing is added to the stream
    graphs = []
    for size in (T, 3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.add_rmsnorm_rows8(x[:size], d[:size], w, 1e-6)
            values_ = ops.materialize(r)
            gate = ops.gate_rows8(values_)
        graphs.append((g, size, r, values_, gate))
    v = before.double()
    for i in (0, 1, 0, 1):
        g, size, r, values_, gate = graphs[i]
        g.replay()
        v[:size] = (v[:size].float() + d[:size].float()).double()
        assert torch.equal(x.double(), v)
        y = v[:size]
        check_rows8(r, y / torch.sqrt((y * y).mean(dim=1, keepdim=True) + 1e-6) * w.double())
        a, u = values_.double().split(H // 2, dim=1)
        check_rows8(gate, a / (1 + torch.exp(-a)) * u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 128), (4, 200), (3, 77), (65, 1024)])
@pytest.mark.parametrize("kind,limit", [("silu", 0.0), ("relu", 0.0), ("clamped", 1.5)])
def test_gate(T, K, dtype, kind, limit):
    from pyre_b200.kernels import ops
    gu = normal(5, T, 2 * K, dtype=dtype) * 3
    g, u = gu.double().split(K, dim=1)
    if kind == "clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        y = g / (1 + torch.exp(-1.702 * g)) * u
    else:
        y = (g.clamp(min=0) if kind == "relu" else g / (1 + torch.exp(-g))) * u
    check_rows8(ops.gate_rows8(gu, kind, limit), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K", [(2500, 520), (1301, 1001), (9999, 77), (130, 9472)])
def test_many_groups_are_as_few(T, K, dtype):
    """Above some 10,000 groups a warp takes four at a time: the bytes and scales are those of the same rows a few at a time, NaN and zeros included."""
    from pyre_b200.kernels import ops
    gu = normal(9, T, 2 * K, dtype=dtype) * 3
    gu[3, 5], gu[4, 70], gu[5] = float("inf"), float("nan"), 0
    x = gu[:, :K]
    live = torch.ones(T, dtype=torch.bool, device="cuda")
    live[3:5] = False
    check = ops.quantize_rows8(x[8:].contiguous())
    check_rows8(check, x[8:].double())
    for form in (lambda v: ops.quantize_rows8(v[:, :K]), ops.gate_rows8, lambda v: ops.gate_rows8(v, "relu"), lambda v: ops.gate_rows8(v, "clamped", 1.5)):
        r = form(gu)
        for a in (0, T // 2, T - 9):
            few = form(gu[a:a + 9].contiguous())
            assert torch.equal(r.rows[a:a + 9], few.rows) and torch.equal(r.scales[:, a:a + 9].nan_to_num(-1), few.scales.nan_to_num(-1))
        assert (r.rows.view(T, -1)[:, K:] == 0).all()
        v, want = ops.materialize(r), values(r)
        off = (v.double() - want).abs()
        assert (off[live] <= want[live].abs() * EPS[dtype] * 1.01).all()      # one product in 32 bits and a rounding


def test_groups_of_zeros_and_of_what_is_no_number():
    from pyre_b200.kernels import ops
    x = normal(6, 4, 384)
    x[0, 128:256] = 0
    x[1, 5] = float("inf")
    x[2, 300] = float("nan")
    x[3, :128] = 1e-32      # below 2^-100: counts as zeros
    r = ops.quantize_rows8(x)
    s = r.scales.t()
    assert s[0, 1] == 0 and s[3, 0] == 0 and (r.rows[0, 128:256] == 0).all() and (r.rows[3, :128] == 0).all()
    bad = torch.isnan(s)
    assert bad[1, 0] and bad[2, 2] and int(bad.sum()) == 2
    assert torch.isnan(ops.materialize(r)[1, :128]).all()
    w = ops.quantize_weight4(normal(7, 24, 384))
    y = ops.linear(r, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(1, 128), (40, 384), (7, 77), (3, 1001), (130, 512)])
def test_weight(N, K, dtype):
    from pyre_b200.kernels import ops
    w = normal(8, N, K, dtype=dtype) * 0.05
    if K > 128:
        w[0, :128] = 0
    q = ops.quantize_weight4(w)
    g = grouped(w)
    want = (g.abs().amax(dim=2) / 7).to(torch.float32).to(torch.bfloat16).double()
    s = q.scales.double().t()
    # the division in 32 bits may fall to the other side of a bf16 border
    assert ((s - want).abs() <= want * 2.0 ** -7).all() and (s == want).double().mean() > 0.98
    v = q.values()
    assert v.dtype == torch.float32 and tuple(v.shape) == (N, K)
    # an element is off by half a scale, the largest one by what the scale's rounding cuts off (7 s 2^-8 < s / 32)
    assert ((grouped(v) - g).abs() <= s[:, :, None] * 0.5001 + 1e-30).all()
    # the documented bytes
    p = q.packed.view(N, -1, 4)
    e = torch.cat([p & 15, p >> 4], dim=2).view(N, -1, GROUP).int()
    e = torch.where(e > 7, e - 16, e)
    assert torch.equal((e.double() * s[:, :, None]).view(N, -1)[:, :K].float(), v) and (e.view(N, -1)[:, K:] == 0).all()


def weight(seed, N, K):
    """All of -8 .. 7 and scales of several sizes."""
    from pyre_b200.kernels import ops
    G = -(-K // GROUP)
    live = torch.arange(G * GROUP, device="cuda") < K
    w = (torch.randint(-8, 8, (N, G * GROUP), generator=gen(seed), device="cuda") * live).to(torch.int8)
    h = w.view(N, -1, 2, 4)
    packed = ((h[:, :, 0] & 15) | (h[:, :, 1] << 4)).view(torch.uint8).reshape(N, -1).contiguous()
    scales = (torch.rand((G, N), generator=gen(seed + 1), device="cuda") * 0.1 + 0.01).to(torch.bfloat16)
    return ops.Weight4(packed, scales, K), (w.view(N, G, GROUP).double() * scales.double().t()[:, :, None]).view(N, -1)


def rows8(seed, T, K):
    from pyre_b200.kernels import ops
    G = -(-K // GROUP)
    live = torch.arange(G * GROUP, device="cuda") < K
    q = (torch.randint(-127, 128, (T, G * GROUP), generator=gen(seed), device="cuda") * live).to(torch.int8)
    s = torch.rand((G, T), generator=gen(seed + 1), device="cuda") + 0.1
    return ops.Rows8(q, s, K), (q.view(T, G, GROUP).double() * s.double().t()[:, :, None]).view(T, -1)


def check_product(y, x, w, out_dtype):
    """Off by 32-bit roundings only: per group the integer's scaling (two products) and one addition, G additions in all, each at most 2^-24 of
    the sum of the groups' magnitudes so far; then the rounding to the output's type."""
    T, G = x.shape[0], x.shape[1] // GROUP
    want = x @ w.t()
    part = torch.einsum("tgk,ngk->tgn", x.view(T, G, GROUP), w.view(w.shape[0], G, GROUP)).abs().sum(dim=1)
    off = (y.double() - want).abs()
    assert y.dtype == out_dtype and tuple(y.shape) == tuple(want.shape)
    assert (off <= part * (G + 4) * 2.0 ** -24 + want.abs() * (EPS[out_dtype] * 1.01 if out_dtype == torch.bfloat16 else 0)).all()


SIZES = [(1, 1, 128), (1, 17, 1), (2, 16, 77), (1, 4608, 3584), (3, 130, 384), (8, 300, 1001), (9, 257, 640), (15, 100, 2176), (17, 48, 512), (31, 999, 256), (33, 640, 1152),
         (64, 129, 384), (65, 200, 896), (127, 384, 128), (128, 128, 1280), (129, 385, 640), (200, 1000, 1001), (300, 515, 2048), (8, 3584, 18944), (16, 64, 18944), (511, 260, 2176),
         (512, 300, 2176), (513, 129, 2048), (700, 515, 2047), (1000, 1, 2560), (640, 2000, 1920), (530, 3999, 4480), (2048, 1000, 3584),
         (256, 9500, 2048), (257, 9472, 2304), (300, 9001, 2050), (1290, 5000, 2048),
         (8, 130, 4224), (40, 130, 4224), (100, 200, 4200), (64, 500, 2700)]      # shares of K of several lengths, of none


@pytest.mark.parametrize("T,N,K", SIZES)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_product(T, N, K, out_dtype):
    from pyre_b200.kernels import ops
    w, wv = weight(11, N, K)
    x, xv = rows8(13, T, K)
    check_product(ops.linear(x, w, out_dtype=out_dtype), xv, wv, out_dtype)


def test_product_of_extremes_is_exact():
    """-8 times 127 over whole groups: the largest sums that the integers meet."""
    from pyre_b200.kernels import ops
    for T, K in ((1, 1024), (9, 1024), (40, 1024), (130, 1024), (600, 2048)):
        N = 48
        packed = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
        w = ops.Weight4(packed, torch.ones((K // GROUP, N), dtype=torch.bfloat16, device="cuda"), K)
        x = ops.Rows8(torch.full((T, K), 127, dtype=torch.int8, device="cuda"), torch.ones((K // GROUP, T), device="cuda"), K)
        assert (ops.linear(x, w, out_dtype=torch.float32) == -8 * 127 * K).all()
        x = ops.Rows8(torch.full((T, K), -127, dtype=torch.int8, device="cuda"), torch.ones((K // GROUP, T), device="cuda"), K)
        assert (ops.linear(x, w, out_dtype=torch.float32) == 8 * 127 * K).all()


@pytest.mark.parametrize("T", [1, 5, 40, 150])
def test_plain_activations_and_unrounded_results(T):
    from pyre_b200.kernels import ops
    N, K = 264, 700
    w, wv = weight(17, N, K)
    x = normal(19, T, K, dtype=torch.bfloat16)
    r = ops.quantize_rows8(x)
    xv = grouped(values(r)).view(T, -1)
    check_product(ops.linear(x, w), xv, wv, torch.bfloat16)
    parts = ops.linear(r, w, partials_ok=True)
    assert isinstance(parts, ops.PartialSums) and parts.dtype == torch.bfloat16
    check_product(parts.parts.sum(0), xv, wv, torch.float32)
    y = ops.materialize(parts)
    check_product(y, xv, wv, torch.bfloat16)
    # a plain weight of the same product takes rows in 8 bits too
    assert ops.linear(r, normal(21, N, 704, dtype=torch.bfloat16)[:, :700].contiguous()).shape == (T, N)


def test_scales_with_a_stride_and_rows_left_as_they_are():
    """Scales may be a slice of a longer table; what lies behind the last row of an output's memory stays."""
    from pyre_b200.kernels import ops
    N, K = 200, 640
    w, wv = weight(23, N, K)
    for T in (5, 70):
        x, xv = rows8(25, T + 3, K)
        part = ops.Rows8(x.rows[2:T + 2], x.scales[:, 2:T + 2], K)
        check_product(ops.linear(part, w, out_dtype=torch.float32), xv[2:T + 2], wv, torch.float32)
    empty = ops.linear(ops.Rows8(x.rows[:0], x.scales[:, :0], K), w)
    assert tuple(empty.shape) == (0, N)


@pytest.mark.parametrize("T,K", [(1, 1280), (12, 1280), (64, 1280), (160, 1280), (520, 2176)])
def test_another_stream_and_a_captured_replay(T, K):
    from pyre_b200.kernels import ops
    N = 384
    w, wv = weight(27, N, K)
    x, _ = rows8(29, T, K)
    want = ops.linear(x, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear(x, w, out_dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    # two captured products of different sizes, replayed in turn, then on new rows
    other, ov = weight(31, 72, K)
    graphs = []
    for weight_ in (w, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear(x, weight_, out_dtype=torch.float32)
        graphs.append((g, y))
    for seed in (33, 35):
        fresh, fv = rows8(seed, T, K)
        x.rows.copy_(fresh.rows)
        x.scales.copy_(fresh.scales)
        for g, _ in graphs:
            g.replay()
        check_product(graphs[0][1], fv, wv, torch.float32)
        check_product(graphs[1][1], fv, ov, torch.float32)


def test_weights_made_just_before_their_product():
    """A product asks for weights ahead of the kernels before it: one that follows its weight's own kernel finds them whole."""
    from pyre_b200.kernels import ops
    N, K = 4000, 2048
    plain = [normal(71 + i, N, K, dtype=torch.bfloat16) for i in range(4)]
    for T in (4, 90):
        x, _ = rows8(70, T, K)
        want = []
        for p in plain:
            w = ops.quantize_weight4(p)
            torch.cuda.synchronize()
            want.append(ops.linear(x, w))
        got = [ops.linear(x, ops.quantize_weight4(p)) for p in plain for _ in range(5)]
        assert all(torch.equal(y, want[i // 5]) for i, y in enumerate(got))
        # ... and weights that a plain copy has just put in their place
        both = [ops.quantize_weight4(p) for p in plain[:2]]
        w = ops.Weight4(both[0].packed.clone(), both[0].scales.clone(), K)
        got = []
        for i in range(10):
            w.packed.copy_(both[i % 2].packed)
            w.scales.copy_(both[i % 2].scales)
            got.append(ops.linear(x, w))
        assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


def test_two_streams_at_once():
    from pyre_b200.kernels import ops
    K = 2048
    cases = [(rows8(81, 6, K)[0], weight(82, 3000, K)[0]), (rows8(83, 200, K)[0], weight(84, 1500, K)[0])]
    want = [ops.linear(x, w) for x, w in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_offsets_beyond_32_bits():
    """Rows, weights and streams of more than 2^31 elements: the last ones against the same ones alone."""
    from pyre_b200.kernels import ops
    T, K, N = 70000, 31000, 24
    x = torch.empty((T, K), device="cuda")
    x.normal_(generator=gen(91))
    gain = 1 + 0.1 * normal(92, K)
    tail = x[-5:].clone()
    r, alone = ops.add_rmsnorm_rows8(x, None, gain, 1e-6), ops.add_rmsnorm_rows8(tail, None, gain, 1e-6)
    assert torch.equal(r.rows[-5:], alone.rows) and torch.equal(r.scales[:, -5:], alone.scales)
    r, alone = ops.quantize_rows8(x), ops.quantize_rows8(tail)
    assert torch.equal(r.rows[-5:], alone.rows) and torch.equal(r.scales[:, -5:], alone.scales)
    del x
    assert torch.equal(ops.materialize(r)[-5:], ops.materialize(alone))
    w, wv = weight(93, N, K)
    check_product(ops.linear(r, w, out_dtype=torch.float32)[-5:], grouped(values(alone)).view(5, -1), wv, torch.float32)
    del r
    G, N = -(-K // GROUP), 140000
    plain = torch.empty((N, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen(94))
    w, last = ops.quantize_weight4(plain), ops.quantize_weight4(plain[-40:].clone())
    del plain
    assert torch.equal(w.packed[-40:], last.packed) and torch.equal(w.scales[:, -40:], last.scales)
    assert torch.equal(w.values(torch.bfloat16)[-40:], last.values(torch.bfloat16))
    wv = grouped(last.values()).view(40, -1)
    for n in (2, 5):
        part = ops.Rows8(alone.rows[:n], alone.scales[:, :n], K)
        check_product(ops.linear(part, w, out_dtype=torch.float32)[:, -40:], grouped(values(alone)).view(5, -1)[:n], wv, torch.float32)
    many = ops.quantize_rows8(normal(95, 66, K))
    check_product(ops.linear(many, w, out_dtype=torch.float32)[:, -40:], grouped(values(many)).view(66, -1), wv, torch.float32)


def test_a_run_of_them_as_a_layer_uses_them():
    """Norm, product, gate, product, residual: what a feed-forward of a decode step launches, against the same steps in 64 bits on the
    values that the 8-bit rows stand for."""
    from pyre_b200.kernels import ops
    T, H, inter = 5, 512, 896
    x, delta, gain = normal(41, T, H), normal(42, T, H, dtype=torch.bfloat16), 1 + 0.1 * normal(43, H)
    w1, v1 = weight(45, 2 * inter, H)
    w2, v2 = weight(47, H, inter)
    r = ops.add_rmsnorm_rows8(x, delta, gain, 1e-6)
    gu = ops.linear(r, w1)
    check_product(gu, grouped(values(r)).view(T, -1), v1, torch.bfloat16)
    a = ops.gate_rows8(gu)
    g, u = gu.double().split(inter, dim=1)
    check_rows8(a, g / (1 + torch.exp(-g)) * u)
    y = ops.linear(a, w2, partials_ok=True)
    check_product(y.parts[0], grouped(values(a)).view(T, -1), v2, torch.float32)
    before = x.double()
    r2 = ops.add_rmsnorm_rows8(x, y, gain, 1e-6)
    v = before + y.parts[0].double()
    check_rows8(r2, v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * gain.double())


@pytest.mark.parametrize("T,N", [(3, 140), (50, 140), (600, 140), (300, 9480)])
def test_scales_of_any_size_and_features_of_zeros(T, N):
    """Scales across a feature's groups that differ by 2^20, features and tokens of zeros, features of the smallest and largest scales."""
    from pyre_b200.kernels import ops
    K = 2176
    G = K // GROUP
    w, _ = weight(61, N, K)
    scales = torch.exp2(torch.randint(-20, 1, (G, N), generator=gen(62), device="cuda").float()) * (1 + torch.rand((G, N), generator=gen(63), device="cuda"))
    scales[:, 5] = 0
    scales[3, :] = 0
    scales[:, 6] *= 2.0 ** -70
    scales[:, 7] *= 2.0 ** 70
    scales = scales.to(torch.bfloat16)
    w = ops.Weight4(w.packed, scales, K)
    p = w.packed.view(N, -1, 4)
    e = torch.cat([p & 15, p >> 4], dim=2).view(N, G, GROUP).int()
    e = torch.where(e > 7, e - 16, e)
    wv = (e.double() * scales.double().t()[:, :, None]).view(N, -1)
    x, xv = rows8(64, T, K)
    x.scales[:, T // 2] = 0
    xv[T // 2] = 0
    x.scales *= torch.exp2(torch.randint(-15, 1, tuple(x.scales.shape), generator=gen(65), device="cuda").float())
    xv = (x.rows.view(T, G, GROUP).double() * x.scales.double().t()[:, :, None]).view(T, -1)
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.linear(x, w, out_dtype=dtype)
        check_product(y, xv, wv, dtype)
        assert (y[:, 5] == 0).all() and (y[T // 2] == 0).all()
    # what is no number stays with its feature, and with its token
    scales[2, 9] = float("nan")
    x.scales[4, 1] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.linear(x, ops.Weight4(w.packed, scales, K), out_dtype=dtype)
        assert torch.isnan(y[:, 9]).all() and torch.isnan(y[1]).all()
        y[:, 9] = 0
        y[1] = 0
        assert torch.isfinite(y).all()


def test_refusals():
    from pyre_b200.kernels import ops
    w, _ = weight(51, 32, 256)
    x, _ = rows8(53, 3, 256)
    bad = rows8(53, 3, 384)[0]
    with pytest.raises(ValueError, match="inner sizes differ"):
        ops.linear(bad, w)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.linear(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="contiguous"):
        ops.linear(ops.Rows8(x.rows[::2], x.scales[:, ::2].contiguous(), 256), w)
    with pytest.raises(ValueError, match="contiguous"):
        ops.linear(ops.Rows8(x.rows, x.scales.t().contiguous().t(), 256), w)
    with pytest.raises(ValueError, match="contiguous CUDA tensors"):
        ops.Weight4(w.packed[::2], w.scales[:, ::2], 256)
    with pytest.raises(ValueError, match="16-byte"):
        ops.Weight4(torch.zeros(128 * 4 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 128), w.scales[:, :4].contiguous(), 256)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.quantize_rows8(torch.zeros((4, 64), device="cuda").t())
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.quantize_weight4(torch.zeros((4, 64), dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError, match="norm weight"):
        ops.add_rmsnorm_rows8(torch.zeros((2, 64), device="cuda"), None, torch.ones(63, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="delta shape"):
        ops.add_rmsnorm_rows8(torch.zeros((2, 64), device="cuda"), torch.zeros((1, 64), device="cuda", dtype=torch.bfloat16), torch.ones(64, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="delta must be"):
        ops.add_rmsnorm_rows8(torch.zeros((2, 64), device="cuda"), torch.zeros((2, 64), device="cuda"), torch.ones(64, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="even number"):
        ops.gate_rows8(torch.zeros((2, 63), device="cuda"))
    with pytest.raises(ops.UnsupportedSize, match="gate activation"):
        ops.gate_rows8(torch.zeros((2, 64), device="cuda"), kind="tanh")
