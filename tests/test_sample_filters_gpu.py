"""Sampling from the likeliest tokens against a plain evaluation in 64 bits, over every form of row."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _shr(z, by):
    return (z >> by) & ((1 << (64 - by)) - 1)


def _mix(z):
    def signed(v):
        return v - (1 << 64) if v >= 1 << 63 else v
    z = z + signed(0x9E3779B97F4A7C15)
    z = (z ^ _shr(z, 30)) * signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shr(z, 27)) * signed(0x94D049BB133111EB)
    return z ^ _shr(z, 31)


def noise(seeds, index, V):
    """g(seed, index, entry) in 64 bits: [R, V]."""
    h = _mix(seeds[:, None] ^ _mix((index.long()[:, None] << 32) | torch.arange(V, device=seeds.device)))
    return -torch.log(-torch.log((_shr(h, 41).double() + 0.5) / 8388608.0))


def kept(logits, T, k, p, m):
    """Which tokens of each row may be chosen (T > 0), and how far, relative to the mass, the nearest border of p or m is."""
    R, V = logits.shape
    l = torch.where(torch.isnan(logits), float("-inf"), logits).double()
    ordered, at = torch.sort(l, dim=1, descending=True, stable=True)
    d = torch.where(ordered == ordered[:, :1], 0.0, ordered - ordered[:, :1]) / T[:, None].double()
    w = torch.exp(d)
    place = torch.arange(V, device=l.device)
    first = (k[:, None] <= 0) | (place < k[:, None])
    mass = (w * first).cumsum(1)
    whole = mass[:, -1:]
    before = mass - w * first
    p64, m64 = p[:, None].double(), m[:, None].double().clamp(max=1)
    keep = first & ((p64 >= 1) | (before < p64 * whole)) & (w >= m64)
    keep[:, 0] = True
    return torch.zeros_like(keep).scatter_(1, at, keep), w, before, whole


def check(ids, logits, T, seeds, index, k, p, m):
    """The chosen token is the best of the kept ones.  Ties and borders: scores are off by 32-bit roundings (of the distance, below 2^-24 of it,
    and of the noise, below 2^-21 up to 16), so a token within 2^-18 (1 + |score|) of the best one is right too; a border may lie 2^-20 of the mass
    to either side (masses are rounded to 2^-31, their exponentials to 2^-22), so a token kept by either is right."""
    R, V = logits.shape
    l = torch.where(torch.isnan(logits), float("-inf"), logits).double()
    best = l.amax(dim=1, keepdim=True)
    g = noise(seeds, index, V)
    greedy = ~(T > 0)
    safe_T = torch.where(greedy, 1.0, T)
    score = torch.where(l == best, 0.0, l - best) / safe_T[:, None].double() + g
    near = 2.0 ** -20
    strict, _, _, _ = kept(logits, safe_T, k, torch.where(p < 1, p * (1 - near), p), m * (1 + near))
    loose, _, _, _ = kept(logits, safe_T, k, torch.where(p < 1, p * (1 + near), p), m * (1 - near))
    for r in range(R):
        i = int(ids[r])
        assert 0 <= i < V
        if not torch.isfinite(best[r]) and best[r] < 0:
            assert i == 0
            continue
        if greedy[r]:
            assert i == int((l[r] == best[r]).nonzero()[0])
            continue
        assert bool(loose[r, i]), f"row {r}: token {i} may not be chosen"
        top = float(score[r][strict[r]].max())
        assert float(score[r, i]) >= top - 2.0 ** -18 * (1 + abs(top)), f"row {r}: token {i} has {float(score[r, i])}, the best {top}"


def call(logits, T, seeds, index, k, p, m):
    from pyre_b200.kernels import ops
    return ops.sample(logits, T, seeds, index, top_k=k, top_p=p, min_p=m)


def rules(seed, R):
    """Every combination of filters in turn."""
    g = gen(seed)
    kind = torch.arange(R, device="cuda") % 9
    T = torch.where(kind == 0, 0.0, 0.3 + 1.5 * torch.rand(R, generator=g, device="cuda"))
    k = torch.where((kind == 2) | (kind == 5) | (kind == 6) | (kind == 8), torch.randint(1, 60, (R,), generator=g, device="cuda"), 0).to(torch.int32)
    p = torch.where((kind == 3) | (kind == 5) | (kind == 7) | (kind == 8), 0.05 + 0.94 * torch.rand(R, generator=g, device="cuda"), 1.0)
    m = torch.where((kind == 4) | (kind == 6) | (kind == 7) | (kind == 8), 0.2 * torch.rand(R, generator=g, device="cuda"), 0.0)
    seeds = torch.randint(0, 1 << 62, (R,), generator=g, device="cuda")
    index = torch.randint(0, 1000, (R,), generator=g, device="cuda", dtype=torch.int32)
    return T, seeds, index, k, p, m


@pytest.mark.parametrize("R,V", [(1, 1), (9, 2), (18, 7), (9, 130), (18, 512), (27, 1001), (9, 2049), (18, 4097), (90, 5000), (9, 16384), (10, 32769), (9, 152064), (200, 3001),
                                 (9, 300001), (2, 700003)])
@pytest.mark.parametrize("form", ["normal", "coarse", "flat", "equal"])
def test_rows(R, V, form):
    g = gen(R * 1000 + V)
    logits = torch.randn((R, V), generator=g, device="cuda") * 3
    if form == "coarse":
        logits = (logits * 4).round() / 4
    elif form == "flat":
        logits = logits * 1e-3 - 5
    elif form == "equal":
        logits = torch.full_like(logits, 2.5)
    rule = rules(R + V, R)
    check(call(logits, *rule), logits, *rule)


@pytest.mark.parametrize("V", [50, 3000, 40000])
def test_masked_entries_infinities_and_what_is_no_number(V):
    R = 36
    logits = torch.randn((R, V), generator=gen(V), device="cuda") * 3
    logits[:, ::2] = float("-inf")
    logits[3] = float("-inf")                      # nothing left
    logits[4] = torch.finfo(torch.float32).min     # masked by the type's lowest value, all of it
    logits[5, 1:] = torch.finfo(torch.float32).min
    logits[6, V // 2:] = float("nan")
    logits[7] = float("nan")
    logits[8, 1::3] = float("inf")                 # several that are certain
    logits[17, 0], logits[17, 1] = -0.0, 0.0       # equal: the lower index is first
    logits[17, 2:] = -50
    rule = rules(V, R)
    rule[0][17], rule[3][17] = 1.0, 1
    ids = call(logits, *rule)
    check(ids, logits, *rule)
    assert int(ids[17]) == 0


def test_values_at_the_ends_of_the_arguments():
    """p of 0 or less and m of 1 or more leave the best token; k beyond the vocabulary and p of 1 leave all; temperatures of any size."""
    V = 700
    logits = torch.randn((12, V), generator=gen(3), device="cuda")
    T = torch.tensor([1.0, 1, 1, 1, 1, 1, 1e-30, 1e-44, 1e30, float("inf"), 1, 1], device="cuda")
    k = torch.tensor([0, 0, 0, 0, 5000, V, 7, 7, 7, 7, 1, -3], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.0, -1, 1, 1, 1, 1, 0.5, 0.5, 0.5, 0.5, 1, 2.0], device="cuda")
    m = torch.tensor([0.0, 0, 1, 7, 0, 0, 0, 0, 0, 0, 0, -1.0], device="cuda")
    seeds = torch.arange(12, device="cuda")
    index = torch.arange(12, device="cuda", dtype=torch.int32)
    ids = call(logits, T, seeds, index, k, p, m)
    best = logits.argmax(dim=1).int()
    for r in (0, 1, 2, 3, 6, 7, 10):
        assert int(ids[r]) == int(best[r]), r
    check(ids[:6], logits[:6], T[:6], seeds[:6], index[:6], k[:6], p[:6], m[:6])
    check(ids[11:], logits[11:], T[11:], seeds[11:], index[11:], k[11:], p[11:], m[11:])
    for r in (8, 9):       # all of the first seven are as likely; half of their mass is the first four
        assert int(ids[r]) in logits[r].topk(4).indices.tolist()


def test_a_row_without_filters_gets_its_token_with_and_without_the_arguments():
    from pyre_b200.kernels import ops
    for V in (600, 9000, 40000):
        R = 20
        logits = torch.randn((R, V), generator=gen(V), device="cuda") * 2
        T = torch.where(torch.arange(R, device="cuda") % 3 == 0, 0.0, 0.9)
        seeds, index = torch.arange(R, device="cuda") * 77, torch.arange(R, device="cuda", dtype=torch.int32)
        off = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.ones(R, device="cuda"), torch.zeros(R, device="cuda")
        assert torch.equal(ops.sample(logits, T, seeds, index), call(logits, T, seeds, index, *off))


def test_a_rows_token_does_not_depend_on_the_batch():
    """One row alone takes a cluster of CTAs, many rows take one or a few each; rows off 16-byte boundaries, of a wider table."""
    V, R = 20011, 400
    table = torch.randn((R, V + 2), generator=gen(1), device="cuda") * 2
    rule = rules(5, R)
    ids = call(table[:, 1:V + 1], *rule)
    check(ids[:60], table[:60, 1:V + 1], *(t[:60] for t in rule))
    for r in (0, 1, 2, 3, 4, 5, 6, 7, 8, 399):
        one = tuple(t[r:r + 1].contiguous() for t in rule)
        assert int(call(table[r:r + 1, 1:V + 1], *one)) == int(ids[r])
    few = tuple(t[10:50].contiguous() for t in rule)
    assert torch.equal(call(table[10:50, 1:V + 1], *few), ids[10:50])


@pytest.mark.parametrize("form", ["normal", "coarse", "flat", "equal", "peaked"])
def test_any_number_of_ctas_per_row_gives_the_same(form, monkeypatch):
    """Borders are found in whole numbers: 1 to 16 CTAs per row agree to the bit, on rows whose borders lie near the best token or far, or among ties."""
    from pyre_b200.kernels import ops
    R, V = 45, 60001
    logits = torch.randn((R, V), generator=gen(77), device="cuda") * {"normal": 2, "coarse": 2, "flat": 0.01, "equal": 0, "peaked": 0.5}[form]
    if form == "coarse":
        logits = (logits * 2).round() / 2
    if form == "peaked":
        logits[:, 100:140] += 9
    rule = rules(123, R)
    want = None
    for cluster in (0, 1, 2, 4, 8, 16):
        monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", cluster)
        ids = call(logits, *rule)
        if want is None:
            check(ids, logits, *rule)
            want = ids
        assert torch.equal(ids, want), cluster


@pytest.mark.parametrize("form", ["normal", "flat", "equal", "ends"])
def test_long_rows_on_few_ctas(form, monkeypatch):
    """More blocks of 128 entries than a CTA, or a row's first CTA, keeps the largest entries of."""
    from pyre_b200.kernels import ops
    R, V = 9, 700003
    logits = torch.randn((R, V), generator=gen(78), device="cuda") * {"normal": 2, "flat": 0.01, "equal": 0, "ends": 0.5}[form]
    if form == "ends":
        logits[:, -30:] += 9
        logits[:, :5] += 9
    rule = rules(124, R)
    want = None
    for cluster in (1, 2, 4, 0):
        monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", cluster)
        ids = call(logits, *rule)
        if want is None:
            check(ids, logits, *rule)
            want = ids
        assert torch.equal(ids, want), cluster


@pytest.mark.parametrize("V", [11000, 150001])
def test_entries_that_stay_lie_in_one_end_of_a_row(V, monkeypatch):
    """The share of a row's first entries that stay says nothing about the others."""
    from pyre_b200.kernels import ops
    R = 18
    logits = torch.randn((R, V), generator=gen(79), device="cuda") * 0.01
    logits[::2, :V * 2 // 3] -= 40
    logits[1::2, V // 3:] -= 40
    logits[::2, 100] = 0.5
    rule = rules(125, R)
    for cluster in (1, 2, 0):
        monkeypatch.setattr(ops, "_SAMPLE_CLUSTER", cluster)
        check(call(logits, *rule), logits, *rule)


def test_draws_follow_the_distribution():
    """Many draws of one row: frequencies against the renormalised probabilities of the kept tokens.  4,096 draws; a count's deviation is at most
    sqrt(n / 4) = 32, so five of them bound each of the few counts with a chance of error below 1e-5."""
    V, R = 300, 4096
    row = torch.full((V,), -4.0, device="cuda")
    row[[7, 100, 250, 20]] = torch.tensor([2.0, 1.5, 1.0, 0.2], device="cuda")
    logits = row.expand(R, V).contiguous()
    T, one = torch.full((R,), 0.8, device="cuda"), torch.ones(R, device="cuda")
    seeds = torch.full((R,), 42, device="cuda")
    index = torch.arange(R, device="cuda", dtype=torch.int32)
    ids = call(logits, T, seeds, index, torch.full((R,), 3, dtype=torch.int32, device="cuda"), one, one * 0)
    w = torch.exp(torch.tensor([2.0, 1.5, 1.0], dtype=torch.float64) / 0.8)
    for token, share in zip((7, 100, 250), (w / w.sum()).tolist()):
        assert abs(int((ids == token).sum()) - share * R) <= 5 * 32
    assert set(ids.tolist()) == {7, 100, 250}


def test_only_some_of_the_arguments_a_replay_and_another_stream():
    from pyre_b200.kernels import ops
    R, V = 12, 30000
    logits = torch.randn((R, V), generator=gen(9), device="cuda") * 2
    T, seeds, index, k, p, m = rules(9, R)
    zero, one = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.ones(R, device="cuda")
    for kw, full in (({"top_k": k}, (k, one, one * 0)), ({"top_p": p}, (zero, p, one * 0)), ({"min_p": m}, (zero, one, m))):
        ids = ops.sample(logits, T, seeds, index, **kw)
        check(ids, logits, T, seeds, index, *full)
    want = call(logits, T, seeds, index, k, p, m)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = call(logits, T, seeds, index, k, p, m)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(logits, T, seeds, index, k, p, m)
    index += 5
    graph.replay()
    check(out, logits, T, seeds, index, k, p, m)
    assert call(logits[:0], T[:0], seeds[:0], index[:0], k[:0], p[:0], m[:0]).shape == (0,)


def test_rows_far_apart_and_two_streams_at_once():
    """Rows whose offsets pass 32 bits; two streams with rows of their own."""
    V, step, R = 40000, 1100000000, 3
    near = torch.randn((R, V), generator=gen(31), device="cuda") * 2
    far = torch.empty(2 * step + V, device="cuda").as_strided((R, V), (step, 1))
    far.copy_(near)
    rule = tuple(t[5:8].contiguous() for t in rules(33, 9))
    assert torch.equal(call(far, *rule), call(near, *rule))
    del far
    many, each = torch.randn((150, V), generator=gen(35), device="cuda") * 2, rules(37, 150)
    cases = ((near, *rule), (many, *each))
    want = [call(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(ids, want[i]) for ids in got[i])


def test_refusals():
    from pyre_b200.kernels import ops
    logits = torch.zeros((3, 50), device="cuda")
    T, seeds, index, k, p, m = rules(1, 3)
    with pytest.raises(ValueError, match="go with a temperature"):
        ops.sample(logits, top_k=k)
    with pytest.raises(ValueError, match="top_k must be"):
        ops.sample(logits, T, seeds, index, top_k=k.long())
    with pytest.raises(ValueError, match="top_p must be"):
        ops.sample(logits, T, seeds, index, top_p=p.double())
    with pytest.raises(ValueError, match="min_p needs one entry per row"):
        ops.sample(logits, T, seeds, index, min_p=m[:2])
    with pytest.raises(ValueError, match="need an entry"):
        ops.sample(logits[:, :0], T, seeds, index, min_p=m)
    with pytest.raises(ValueError, match="needs seeds"):
        ops.sample(logits, T, top_p=p)
