"""The operators of token models that the framework offers, as measurable cases.

Three operators, each in both directions:

  embedding   rows of a table looked up by token and scaled, with or without dropout on the result; its gradient, summed
              over the positions of each token.  Positions outside the table (padding, -1) give zeros and take no part.
  dropout     from a counter-based generator (Philox4x32-10), whose mask is computed again in the backward pass
  group norm  channels last, with an activation; its gradient for the input, the weights and the biases

`run` computes them with elementary torch operations, or, where `own` is true, through vtl_b200.capi.Device.
"""
import math

import torch

own = False
_device = None


def _dev():
    """The one Device (and its context) of the process, as a program keeps it."""
    global _device
    if _device is None:
        from vtl_b200 import capi
        _device = capi.Device(0)
    return _device


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the next token of eight users: eight rows out of a table of 0.8 GB, nothing but latency
        {"name": "embedding_fwd_8", "kind": "embedding_fwd", "n": 8, "d": 4096, "v": 50000, "scale": 64.0, "p": 0.0, "pad": 0.0},
        # sizes that nothing divides, a padded batch, dropout while training
        {"name": "embedding_fwd_odd", "kind": "embedding_fwd", "n": 999, "d": 2047, "v": 3001, "scale": 1.0, "p": 0.1, "pad": 0.25},
        # the benchmark's inference batch: 16384 tokens of width 4096
        {"name": "embedding_fwd_16384", "kind": "embedding_fwd", "n": 16384, "d": 4096, "v": 50000, "scale": 64.0, "p": 0.0, "pad": 0.0},
        # a small classifier of texts: 256 tokens a step, 5000 words
        {"name": "embedding_bwd_256", "kind": "embedding_bwd", "n": 256, "d": 600, "v": 5000, "scale": 1.0, "p": 0.0, "pad": 0.0},
        # sizes that nothing divides, padding, the mask of the forward pass applied again
        {"name": "embedding_bwd_odd", "kind": "embedding_bwd", "n": 8191, "d": 1023, "v": 3001, "scale": 1.0, "p": 0.1, "pad": 0.25},
        # a training step on 16384 tokens: a gradient of 0.8 GB, most of whose rows are zero
        {"name": "embedding_bwd_16384", "kind": "embedding_bwd", "n": 16384, "d": 4096, "v": 50000, "scale": 64.0, "p": 0.0, "pad": 0.0},
        # behind the hidden layer of a small classifier: a batch of 64, 256 features
        {"name": "dropout_fwd_64x256", "kind": "dropout_fwd", "n": 64 * 256, "p": 0.5},
        # the gradient of 16384 tokens of width 4096
        {"name": "dropout_bwd_16384x4096", "kind": "dropout_bwd", "n": 16384 * 4096, "p": 0.1},
        # a small feature map of two images: 8 x 8 positions, 128 channels
        {"name": "groupnorm_fwd_8x8", "kind": "groupnorm_fwd", "b": 2, "s": 64, "c": 128, "groups": 32, "act": "silu"},
        # large feature maps: 64 x 64 positions, 512 channels, 32 images
        {"name": "groupnorm_fwd_64x64", "kind": "groupnorm_fwd", "b": 32, "s": 4096, "c": 512, "groups": 32, "act": "silu"},
        # sizes that nothing divides: 17 x 19 positions, groups of 11 channels
        {"name": "groupnorm_bwd_odd", "kind": "groupnorm_bwd", "b": 3, "s": 323, "c": 330, "groups": 30, "act": "relu"},
        # a training step on 64 maps of 32 x 32 positions
        {"name": "groupnorm_bwd_32x32", "kind": "groupnorm_bwd", "b": 64, "s": 1024, "c": 512, "groups": 32, "act": "silu"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["embedding_fwd", "embedding_bwd", "dropout_fwd", "dropout_bwd", "groupnorm_fwd", "groupnorm_bwd"])
    if kind.startswith("embedding"):
        return {"kind": kind, "n": _log(rng, 1, 16384), "d": _log(rng, 8, 4096), "v": _log(rng, 50, 50000),
                "scale": rng.choice([1.0, 8.0, 0.37]), "p": rng.choice([0.0, 0.1, 0.25]), "pad": rng.choice([0.0, 0.25])}
    if kind.startswith("dropout"):
        return {"kind": kind, "n": _log(rng, 100, 16384 * 4096), "p": rng.choice([0.1, 0.2, 0.5])}
    while True:
        groups, width = rng.choice([1, 2, 4, 8, 16, 32]), _log(rng, 1, 64)
        b, s = _log(rng, 1, 64), _log(rng, 1, 4096)
        if 512 <= b * s * groups * width <= 32 * 4096 * 512 // 2:
            return {"kind": kind, "b": b, "s": s, "c": groups * width, "groups": groups, "act": rng.choice(["none", "relu", "silu"])}


# ---------------------------------------------------------------- inputs
EPS = 1e-5
ACTS = {"none": 0, "relu": 1, "silu": 2}


def _token_weights(v):
    """How often the tokens of a vocabulary are met: the r-th most frequent one with a weight of 1 / (r + 2.7)."""
    return 1.0 / (torch.arange(v, dtype=torch.float64) + 2.7)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    state = {"case": case, "seed": seed * 7919 + 11, "step": seed % 1000}
    kind = case["kind"]
    if kind.startswith("embedding"):
        n, d, v = case["n"], case["d"], case["v"]
        upto = torch.cumsum(_token_weights(v), 0)
        ids = torch.searchsorted((upto / upto[-1]).cuda(), torch.rand(n, device="cuda", dtype=torch.float64, generator=g), right=True)
        ids = ids.clamp(max=v - 1).to(torch.int32)
        ids[torch.rand(n, device="cuda", generator=g) < case["pad"]] = -1
        state["ids"] = ids
        if kind == "embedding_fwd":
            state |= {"table": normal(v, d), "y": torch.empty(n, d, device="cuda")}
        else:
            state |= {"g": normal(n, d), "dtable": torch.empty(v, d, device="cuda")}
    elif kind.startswith("dropout"):
        state |= {"x": normal(case["n"]), "y": torch.empty(case["n"], device="cuda")}
    else:
        b, s, c, groups = (case[k] for k in ("b", "s", "c", "groups"))
        x = normal(b, s, c) * 2 + 0.5
        state |= {"x": x, "gamma": 1 + 0.2 * normal(c), "beta": 0.2 * normal(c), "y": torch.empty_like(x),
                  "mean": torch.empty(b, groups, device="cuda"), "rstd": torch.empty(b, groups, device="cuda")}
        if kind == "groupnorm_bwd":  # what the forward pass has left behind
            xg = x.view(b, s, groups, c // groups).double()
            state["mean"].copy_(xg.mean((1, 3)))
            state["rstd"].copy_((xg.var((1, 3), correction=0) + EPS).rsqrt())
            state |= {"g": normal(b, s, c), "dgamma": torch.empty(c, device="cuda"), "dbeta": torch.empty(c, device="cuda")}
    return state


# ---------------------------------------------------------------- the plain forms
def _philox(n, seed, step):
    """The first n 32-bit numbers of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) with the key `seed`: number i is
    word i % 4 of the block whose counter is i // 4 in its lower and `step` in its upper 64 bits."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device="cuda")
    c0, c1, c2, c3 = block & low, block >> 32, torch.full_like(block, step & low), torch.full_like(block, step >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _drop(x, p, seed, step):
    """Each element is kept, with a probability of 1 - p, and divided by that, or zero."""
    kept = _philox(x.numel(), seed, step).view(x.shape) >= int(p * 2**32)
    return torch.where(kept, x * (1.0 / (1.0 - p)), 0.0)


def _act(z, act):
    return z if act == "none" else torch.where(z < 0, 0.0, z) if act == "relu" else z / (1 + torch.exp(-z))


def _act_slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z >= 0).float()
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain(state, case):
    kind, seed, step = case["kind"], state["seed"], state["step"]
    if kind == "embedding_fwd":
        ids = state["ids"].long()
        inside = (ids >= 0) & (ids < case["v"])
        y = torch.where(inside[:, None], state["table"][torch.where(inside, ids, 0)] * case["scale"], 0.0)
        return _drop(y, case["p"], seed, step) if case["p"] else y
    if kind == "embedding_bwd":
        ids, g = state["ids"].long(), state["g"]
        inside = (ids >= 0) & (ids < case["v"])
        g = _drop(g, case["p"], seed, step) if case["p"] else g
        out = torch.zeros(case["v"], case["d"], device="cuda")
        return out.index_add_(0, ids[inside], g[inside]) * case["scale"]
    if kind.startswith("dropout"):
        return _drop(state["x"], case["p"], seed, step)
    b, s, c, groups = (case[k] for k in ("b", "s", "c", "groups"))
    grouped = (b, s, groups, c // groups)
    x, gamma, beta = state["x"].view(grouped), state["gamma"].view(grouped[2:]), state["beta"].view(grouped[2:])
    if kind == "groupnorm_fwd":
        mean = x.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
        y = _act((x - mean) * rstd * gamma + beta, case["act"])
        return {"y": y.view(b, s, c), "mean": mean.view(b, groups), "rstd": rstd.view(b, groups)}
    mean, rstd = state["mean"].view(b, 1, groups, 1), state["rstd"].view(b, 1, groups, 1)
    h = (x - mean) * rstd
    if case["act"] == "relu":  # which side of zero: in 64 bits
        z = (x.double() - mean.double()) * rstd.double() * gamma.double() + beta.double()
    else:
        z = h * gamma + beta
    dz = state["g"].view(grouped) * _act_slope(z, case["act"])
    dh = dz * gamma
    dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - h * (dh * h).mean((1, 3), keepdim=True))
    return {"dx": dx.view(b, s, c), "dgamma": (dz * h).sum((0, 1)).view(c), "dbeta": dz.sum((0, 1)).view(c)}


# ---------------------------------------------------------------- the framework's calls
def _own(state, case):
    dev, kind = _dev(), case["kind"]
    at = lambda name: state[name].data_ptr()  # noqa: E731
    if kind == "embedding_fwd":
        dev.embedding_fwd_f32(at("table"), case["v"], case["d"], at("ids"), case["n"], at("y"), scale=case["scale"], p=case["p"],
                              seed=state["seed"], step=state["step"], check=False)
        return state["y"]
    if kind == "embedding_bwd":
        dev.embedding_bwd_f32(at("g"), at("ids"), case["n"], case["v"], case["d"], at("dtable"), scale=case["scale"], p=case["p"],
                              seed=state["seed"], step=state["step"])
        return state["dtable"]
    if kind.startswith("dropout"):
        call = dev.dropout_fwd_f32 if kind == "dropout_fwd" else dev.dropout_bwd_f32
        call(at("x"), at("y"), case["n"], case["p"], state["seed"], state["step"])
        return state["y"]
    sizes = tuple(case[k] for k in ("b", "s", "c", "groups"))
    if kind == "groupnorm_fwd":
        dev.groupnorm_fwd_f32(at("x"), *sizes, at("gamma"), at("beta"), EPS, ACTS[case["act"]], at("y"), at("mean"), at("rstd"))
        return {k: state[k] for k in ("y", "mean", "rstd")}
    dev.groupnorm_bwd_f32(at("g"), at("x"), *sizes, at("gamma"), at("beta"), at("mean"), at("rstd"), ACTS[case["act"]], dx=at("y"),
                          dgamma=at("dgamma"), dbeta=at("dbeta"))
    return {"dx": state["y"], "dgamma": state["dgamma"], "dbeta": state["dbeta"]}


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return _plain(state, case)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind.startswith("embedding"):
        n, d, v = case["n"], case["d"], case["v"]
        inside = n * (1 - case["pad"])
        if kind == "embedding_fwd":  # each row of the table that is met, once (their expected number)
            w = _token_weights(v)
            met = float((1 - (1 - w / w.sum()) ** inside).sum())
            return {"bytes": 4 * (met * d + n + n * d), "flops": n * d}
        return {"bytes": 4 * (inside * d + n + v * d), "flops": inside * d}
    if kind.startswith("dropout"):
        return {"bytes": 8 * case["n"], "flops": case["n"]}
    size, c, stats = case["b"] * case["s"] * case["c"], case["c"], 2 * case["b"] * case["groups"]
    if kind == "groupnorm_fwd":
        return {"bytes": 4 * (2 * size + 2 * c + stats), "flops": 8 * size}
    return {"bytes": 4 * (3 * size + 4 * c + stats), "flops": 16 * size}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]

    def keep_factor(n):
        """1 / (1 - p) where an element is kept, 0 where it is dropped: Philox on words cut into halves of 16 bits."""
        def times(x, m):  # the upper and the lower word of x * m
            x0, x1, m0, m1 = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
            mid = x1 * m0 + ((x0 * m0) >> 16)
            mid2 = x0 * m1 + (mid & 0xFFFF)
            return x1 * m1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((x0 * m0) & 0xFFFF)

        count = -(-n // 4)
        words = torch.zeros(4, count, dtype=torch.int64, device="cuda")
        words[0] = torch.arange(count, device="cuda").remainder(2**32)
        words[1] = torch.arange(count, device="cuda").div(2**32, rounding_mode="floor")
        words[2], words[3] = state["step"] % 2**32, state["step"] // 2**32
        for r in range(10):
            key = [(state["seed"] % 2**32 + r * 0x9E3779B9) % 2**32, (state["seed"] // 2**32 + r * 0xBB67AE85) % 2**32]
            (up0, low0), (up2, low2) = times(words[0], 0xD2511F53), times(words[2], 0xCD9E8D57)
            words = torch.stack([up2 ^ words[1] ^ key[0], low2, up0 ^ words[3] ^ key[1], low0])
        dropped = words.t().reshape(-1)[:n] < math.floor(case["p"] * 2**32)
        return (~dropped).double() / (1 - case["p"])

    if kind == "embedding_fwd":
        table = torch.cat([state["table"], torch.zeros(1, case["d"], device="cuda")])  # a last row of zeros for the positions outside
        ids = state["ids"].long()
        y = table[torch.where(ids < 0, case["v"], ids)].double().mul_(case["scale"])
        return y * keep_factor(y.numel()).view(y.shape) if case["p"] else y
    if kind == "embedding_bwd":
        g = state["g"].double()
        if case["p"]:
            g *= keep_factor(g.numel()).view(g.shape)
        ids, order = torch.sort(state["ids"].long(), stable=True)  # the sums of a token's positions, as differences of running sums
        upto = torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device="cuda"), torch.cumsum(g[order], 0)])
        tokens = torch.arange(case["v"], device="cuda")
        first, past = torch.searchsorted(ids, tokens), torch.searchsorted(ids, tokens, right=True)
        out = torch.zeros(case["v"], case["d"], dtype=torch.float64, device="cuda")
        met = torch.nonzero(past > first).view(-1)
        out[met] = (upto[past[met]] - upto[first[met]]) * case["scale"]
        return out
    if kind.startswith("dropout"):
        return state["x"].double() * keep_factor(case["n"])
    b, s, c, groups = (case[k] for k in ("b", "s", "c", "groups"))
    width = c // groups
    rows = lambda t: t.double().view(b, s, groups, width).permute(0, 2, 1, 3).reshape(b * groups, s * width)  # noqa: E731
    back = lambda t: t.view(b, groups, s, width).permute(0, 2, 1, 3).reshape(b, s, c)  # noqa: E731
    per = lambda t: t.double().view(1, groups, 1, width).expand(b, groups, s, width).reshape(b * groups, s * width)  # noqa: E731
    x = rows(state["x"])
    if kind == "groupnorm_fwd":
        mean = x.sum(1) / (s * width)
        rstd = (x.square().sum(1) / (s * width) - mean.square() + EPS) ** -0.5
    else:
        mean, rstd = state["mean"].double().view(-1), state["rstd"].double().view(-1)
    h = (x - mean[:, None]) * rstd[:, None]
    z = h * per(state["gamma"]) + per(state["beta"])
    if kind == "groupnorm_fwd":
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
        return {"y": back(y), "mean": mean.view(b, groups), "rstd": rstd.view(b, groups)}
    sig = torch.sigmoid(z)
    dz = rows(state["g"]) * {"none": lambda: 1.0, "relu": lambda: (z >= 0).double(), "silu": lambda: sig + z * sig * (1 - sig)}[case["act"]]()
    dh = dz * per(state["gamma"])
    n = s * width
    dx = (rstd / n)[:, None] * (n * dh - dh.sum(1, keepdim=True) - h * (dh * h).sum(1, keepdim=True))
    fold = lambda t: back(t).view(b * s, c).sum(0)  # noqa: E731
    return {"dx": back(dx), "dgamma": fold(dz * h), "dbeta": fold(dz)}
