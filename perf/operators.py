"""The operators of a decoded token with 4-bit weights, each as a user of the engine's kernels calls it: the norm that adds the
residual and leaves rows in 8 bits with scales, the product of such rows with a 4-bit weight, and the choice of a token among the
likeliest ones.

``norm``    x += delta (float32, in place); y = x / sqrt(mean(x^2) + eps) * w; every 128 neighbouring y share a scale max|y| / 127 and are
            held as whole multiples of it.  Returned: the stream, the values that the rows stand for (bfloat16), the scales [groups, rows].
``linear``  rows in 8 bits (scales per 128 elements) times a weight in 4 bits (scales per 128 elements of a feature), in bfloat16 or,
            where the residual stream or the sampler takes the result, in float32.  The weight's bytes: in a word of eight elements byte i holds
            element i in its lower half and element i + 4 in its upper one, two's complement.
``sample``  a token per row of logits: temperature, then the first k, of those the shortest run of the likeliest whose mass is p of theirs, of
            those the ones with at least min_p of the likeliest one's probability; noise from the given (seed, index) and the entry alone.

Sizes are those of the engine's 7B, 14B and 32B shapes and of odd ones between its tiny test models and those.
"""

from __future__ import annotations

import torch

own = False
DEVICE = "cuda:0"
GROUP = 128


def _groups(width: int) -> int:
    return -(-width // GROUP)


def listed() -> list:
    return [
        # one request decodes: a row of the 7B shape
        {"name": "norm_1x3584", "op": "norm", "rows": 1, "width": 3584, "eps": 1e-6},
        # a batch of requests decodes: the 14B shape
        {"name": "norm_48x5120", "op": "norm", "rows": 48, "width": 5120, "eps": 1e-5},
        # a ragged portion, rows that end inside a group and off every vector's boundary
        {"name": "norm_333x1001", "op": "norm", "rows": 333, "width": 1001, "eps": 1e-6},
        # a prompt of the 7B shape
        {"name": "norm_2048x3584", "op": "norm", "rows": 2048, "width": 3584, "eps": 1e-6},
        # one request: the stacked q/k/v projections of the 7B shape
        {"name": "linear_1_3584_4608", "op": "linear", "rows": 1, "inner": 3584, "features": 4608, "out": "bf16"},
        # eight requests: the 7B shape's down projection, which goes on to the residual stream
        {"name": "linear_8_18944_3584", "op": "linear", "rows": 8, "inner": 18944, "features": 3584, "out": "f32"},
        # 24 requests: gates and ups of the 14B shape
        {"name": "linear_24_5120_27648", "op": "linear", "rows": 24, "inner": 5120, "features": 27648, "out": "bf16"},
        # an odd portion of a prompt, features and inner size off every tile
        {"name": "linear_333_1001_4999", "op": "linear", "rows": 333, "inner": 1001, "features": 4999, "out": "f32"},
        # a prompt: gates and ups of the 7B shape
        {"name": "linear_2048_3584_37888", "op": "linear", "rows": 2048, "inner": 3584, "features": 37888, "out": "bf16"},
        # one request draws from the likeliest tokens
        {"name": "sample_1x32768", "op": "sample", "rows": 1, "vocab": 32768, "filter": "top_p", "coarse": False},
        # a batch in which every request has its own rule, greedy and unfiltered ones among them; logits on a coarse grid, so with ties
        {"name": "sample_16x152064", "op": "sample", "rows": 16, "vocab": 152064, "filter": "mixed", "coarse": True},
        # the largest batch, first k and then p
        {"name": "sample_256x152064", "op": "sample", "rows": 256, "vocab": 152064, "filter": "top_k_top_p", "coarse": False},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number whose logarithm is spread evenly."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng) -> dict:
    op = rng.choice(["norm", "linear", "linear", "sample"])
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 2048), "width": _spread(rng, 64, 5120) if rng.random() < 0.5 else 32 * _spread(rng, 2, 160),
                "eps": rng.choice([1e-6, 1e-5])}
    if op == "linear":
        rows = _spread(rng, 1, 2048)
        inner = _spread(rng, 64, 18944) if rng.random() < 0.5 else 128 * _spread(rng, 1, 148)
        most = min(37888, 2048 * 3584 * 37888 // (rows * inner))
        features = _spread(rng, 64, most) if rng.random() < 0.5 else 64 * _spread(rng, 1, most // 64)
        return {"op": op, "rows": rows, "inner": inner, "features": features, "out": rng.choice(["bf16", "f32"])}
    return {"op": op, "rows": _spread(rng, 1, 256), "vocab": _spread(rng, 300, 152064), "coarse": rng.random() < 0.5,
            "filter": rng.choice(["top_k", "top_p", "min_p", "top_k_top_p", "all", "mixed"])}


def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _integers(g, low: int, high: int, *shape, dtype=torch.int64) -> torch.Tensor:
    return torch.randint(low, high, shape, generator=g, device=DEVICE, dtype=dtype)


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "norm":
        T, H = case["rows"], case["width"]
        # a residual stream: some columns are far larger than the others
        gain = 1.0 + 30.0 * (torch.rand(H, generator=g, device=DEVICE) < 0.005).float()
        s["x"] = _normal(g, T, H) * 2.0 * gain
        s["delta"] = (_normal(g, T, H) * 0.5).to(torch.bfloat16)
        s["weight"] = 1.0 + 0.1 * _normal(g, H)
    elif case["op"] == "linear":
        T, K, N = case["rows"], case["inner"], case["features"]
        G = _groups(K)
        live = (torch.arange(G * GROUP, device=DEVICE) < K)
        s["rows8"] = (_normal(g, T, G * GROUP) * 36.0).round_().clamp_(-127, 127).mul_(live).to(torch.int8)
        s["row_scales"] = torch.rand((G, T), generator=g, device=DEVICE) * 0.03 + 0.01
        w = (_normal(g, N, G * GROUP) * 2.6).round_().clamp_(-8, 7).mul_(live).to(torch.int8).view(N, -1, 2, 4)
        s["packed"] = ((w[:, :, 0] & 15) | (w[:, :, 1] << 4)).view(torch.uint8).reshape(N, -1).contiguous()
        s["weight_scales"] = (torch.rand((G, N), generator=g, device=DEVICE) * 0.01 + 0.005).to(torch.bfloat16)
    else:
        R, V = case["rows"], case["vocab"]
        logits = _normal(g, R, V) * 2.0
        # what the context makes likely
        peaks = _integers(g, 0, V, R, 40)
        logits.scatter_add_(1, peaks, 6.0 + 2.0 * _normal(g, R, 40))
        s["logits"] = (logits * 16.0).round_() / 16.0 if case["coarse"] else logits
        f = case["filter"]
        # 0 greedy, 1 no filter, 2 first k, 3 mass, 4 share of the best, 5 all three
        kind = torch.arange(R, device=DEVICE) % 6 if f == "mixed" else \
            torch.full((R,), {"top_k": 2, "top_p": 3, "min_p": 4, "top_k_top_p": 6, "all": 5}[f], device=DEVICE)
        with_k, with_p, with_m = (kind == 2) | (kind >= 5), (kind == 3) | (kind >= 5), (kind == 4) | (kind == 5)
        s["temperature"] = torch.where(kind == 0, 0.0, 0.5 + torch.rand(R, generator=g, device=DEVICE))
        s["top_k"] = torch.where(with_k, _integers(g, 1, 200, R), 0).to(torch.int32)
        s["top_p"] = torch.where(with_p, 0.5 + 0.49 * torch.rand(R, generator=g, device=DEVICE), 1.0)
        s["min_p"] = torch.where(with_m, 0.01 + 0.1 * torch.rand(R, generator=g, device=DEVICE), 0.0)
        s["seeds"] = _integers(g, 0, 1 << 62, R)
        s["token_index"] = _integers(g, 0, 4096, R, dtype=torch.int32)
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_norm(s: dict):
    T, H = s["x"].shape
    s["x"] += s["delta"].float()
    x = s["x"]
    y = x * (1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + s["eps"])) * s["weight"]
    y = torch.nn.functional.pad(y, (0, _groups(H) * GROUP - H)).view(T, -1, GROUP)
    scale = y.abs().amax(dim=2) / 127.0
    q = torch.round(y / torch.where(scale > 0, scale, 1.0)[:, :, None])
    values = (q * scale[:, :, None]).view(T, -1)[:, :H]
    return [x, values.to(torch.bfloat16), scale.t().contiguous()]


def _plain_linear(s: dict):
    T, N, G = s["rows8"].shape[0], s["packed"].shape[0], s["row_scales"].shape[0]
    x = s["rows8"].view(T, G, GROUP).float() * s["row_scales"].t()[:, :, None]
    words = s["packed"].view(N, -1, 1, 4)
    w = torch.cat([words & 15, words >> 4], dim=2).view(N, G, GROUP)
    w = ((w ^ 8).float() - 8.0) * s["weight_scales"].float().t()[:, :, None]
    y = x.view(T, -1) @ w.view(N, -1).t()
    return y.to(torch.bfloat16) if s["out"] == "bf16" else y


def _shifted(z: torch.Tensor, by: int) -> torch.Tensor:
    """Whole numbers of 64 bits shifted to the right, zeros coming in."""
    return (z >> by) & ((1 << (64 - by)) - 1)


def _mixed(z: torch.Tensor) -> torch.Tensor:
    def signed(v):
        return v - (1 << 64) if v >= 1 << 63 else v
    z = z + signed(0x9E3779B97F4A7C15)
    z = (z ^ _shifted(z, 30)) * signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shifted(z, 27)) * signed(0x94D049BB133111EB)
    return z ^ _shifted(z, 31)


def _plain_sample(s: dict):
    logits, T = s["logits"], s["temperature"][:, None]
    R, V = logits.shape
    entry = torch.arange(V, device=logits.device)
    inverse = 1.0 / torch.where(T > 0, T, 1.0)
    noise = _mixed(s["seeds"][:, None] ^ _mixed((s["token_index"].long()[:, None] << 32) | entry))
    noise = -torch.log(-torch.log((_shifted(noise, 41).float() + 0.5) * (1.0 / 8388608.0)))
    ordered, at = torch.sort(logits, dim=1, descending=True, stable=True)
    best = ordered[:, :1]
    mass = torch.exp((ordered - best) * inverse)
    first_k = (s["top_k"][:, None] <= 0) | (entry < s["top_k"][:, None])
    # sums next to a border in 64 bits
    before = (mass.double() * first_k).cumsum(dim=1)
    whole = before[:, -1:]
    before = before - mass.double() * first_k
    p = s["top_p"].double()[:, None]
    kept = first_k & ((p >= 1.0) | (before < p * whole)) & (mass >= s["min_p"][:, None])
    kept[:, 0] = True
    kept = torch.zeros_like(kept).scatter_(1, at, kept)
    filtered = ((s["top_k"] > 0) | (s["top_p"] < 1.0) | (s["min_p"] > 0))[:, None]
    scores = torch.where(filtered, (logits - best) * inverse, logits * inverse) + noise
    scores = torch.where(T > 0, torch.where(kept, scores, float("-inf")), logits)
    return scores.argmax(dim=1).to(torch.int32)


def _own(s: dict):
    from pyre_b200.kernels import ops
    if s["op"] == "norm":
        rows = ops.add_rmsnorm_rows8(s["x"], s["delta"], s["weight"], s["eps"])
        return [s["x"], ops.materialize(rows), rows.scales]
    if s["op"] == "linear":
        x = ops.Rows8(s["rows8"], s["row_scales"], s["inner"])
        w = ops.Weight4(s["packed"], s["weight_scales"], s["inner"])
        return ops.linear(x, w, out_dtype=torch.bfloat16 if s["out"] == "bf16" else torch.float32)
    return ops.sample(s["logits"], s["temperature"], s["seeds"], s["token_index"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def run(state: dict):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "linear": _plain_linear, "sample": _plain_sample}[state["op"]](state)


def work(case: dict) -> dict:
    if case["op"] == "norm":
        n, G = case["rows"] * case["width"], _groups(case["width"])
        # the stream read and written, the branch read, the values written
        return {"bytes": 12 * n + 4 * case["rows"] * G + 4 * case["width"], "flops": 8 * n}
    if case["op"] == "linear":
        T, K, N, G = case["rows"], case["inner"], case["features"], _groups(case["inner"])
        return {"bytes": N * K / 2 + 2 * N * G + T * K + 4 * T * G + (2 if case["out"] == "bf16" else 4) * T * N, "flops": 2 * T * N * K}
    return {"bytes": 4 * case["rows"] * case["vocab"] + 32 * case["rows"], "flops": 4 * case["rows"] * case["vocab"]}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double() + s["delta"].double()
        rms = torch.linalg.vector_norm(x, dim=1).square() / x.shape[1] + case["eps"]
        y = x * s["weight"].double() / rms.sqrt().unsqueeze(1)
        values, scales = torch.empty_like(y), []
        for start in range(0, case["width"], GROUP):
            part = y[:, start:start + GROUP]
            step = torch.linalg.vector_norm(part, ord=float("inf"), dim=1) / 127.0
            values[:, start:start + GROUP] = torch.round(part / step.unsqueeze(1)) * step.unsqueeze(1)
            scales.append(step)
        return [x, values, torch.stack(scales)]
    if case["op"] == "linear":
        nibbles = torch.stack([s["packed"] % 16, s["packed"] // 16]).to(torch.int8)
        nibbles = torch.where(nibbles >= 8, nibbles - 16, nibbles)
        y = torch.zeros((case["rows"], case["features"]), dtype=torch.float64, device=DEVICE)
        for group in range(s["row_scales"].shape[0]):
            rows = s["rows8"][:, group * GROUP:(group + 1) * GROUP].double()
            half = nibbles[:, :, group * GROUP // 2:(group + 1) * GROUP // 2].double()
            # bytes 4j .. 4j + 3 hold elements 8j .. 8j + 3 below and 8j + 4 .. 8j + 7 above
            lower = (torch.arange(GROUP // 2, device=DEVICE) // 4) * 8 + torch.arange(GROUP // 2, device=DEVICE) % 4
            part = rows[:, lower] @ half[0].t() + rows[:, lower + 4] @ half[1].t()
            y += part * s["row_scales"][group].double().unsqueeze(1) * s["weight_scales"][group].double()
        return y
    return None      # whole numbers
