"""Cases, plain forms and exact values of the layer operators: layer normalisation, dropout from a counter-based
generator, and both in one pass, forward and with their gradients.

Rows are network inputs (one per country and world instance, or per replayed transition), columns the units of a
layer.  Widths and row counts come from the worlds and learners of this package -- 6 countries, replay batches of
128 x 4, 4,096 batched worlds of 6 or 200 countries, hidden widths of 128 and 256, feature rows over a sparse world of
20,000 patches -- and from ordinary layer widths beside them."""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
_TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_MASK = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _case(name, op, train, dtype, rows, cols, p=0.0):
    return {"name": name, "op": op, "train": train, "dtype": dtype, "rows": rows, "cols": cols, "p": p}


def listed():
    return [
        # the six countries of the toy world asking for an action: one call per world step, all latency
        _case("norm_six_countries", "norm", False, "f64", 6, 128),
        # one learn call of one agent: 128 transitions times 4 accumulation steps, in the learners' own type
        _case("norm_train_replay", "norm", True, "f64", 512, 128),
        # greedy evaluation of 4,096 worlds of six countries
        _case("norm_rollout", "norm", False, "f32", 24576, 128),
        # a training step over the same rollout with the widest hidden layer of the learners, mixed precision
        _case("norm_train_rollout", "norm", True, "bf16", 24576, 256),
        # an odd width, whose rows start at every alignment
        _case("norm_train_odd", "norm", True, "f16", 3001, 1023),
        # a wide layer at a large batch
        _case("norm_train_wide", "norm", True, "bf16", 16384, 4096),
        # rows that span all patches of a sparse world (one feature per patch)
        _case("norm_patches", "norm", False, "f32", 1021, 20000),
        # dropout in one learn call of one agent
        _case("dropout_replay", "dropout", False, "f64", 512, 128, 0.1),
        # dropout at an odd width, half of the units
        _case("dropout_train_odd", "dropout", True, "f32", 20011, 1001, 0.5),
        # dropout and its gradient over 4,096 worlds of 200 countries
        _case("dropout_train_large", "dropout", True, "bf16", 819200, 128, 0.1),
        # a regularised hidden layer: dropout, then the norm, in one learn call of six agents, 256 transitions each
        _case("both_train_replay", "both", True, "f32", 1536, 128, 0.1),
        # the same over 4,096 worlds of 200 countries
        _case("both_train_large", "both", True, "bf16", 819200, 128, 0.1),
    ]


def draw(rng):
    """One more case: any operator, direction and type; widths from 16 to 24,000 units, sizes up to the largest listed."""
    op = rng.choice(["norm", "norm", "dropout", "both", "both"])
    dtype = rng.choice(["f64", "f32", "bf16", "f16"])
    cols = int(round(math.exp(rng.uniform(math.log(16), math.log(24000)))))
    most = 400_000_000 // _TYPES[dtype].itemsize // 2 // cols
    rows = max(1, min(819200, int(round(math.exp(rng.uniform(0.0, math.log(most)))))))
    p = 0.0 if op == "norm" else rng.choice([0.05, 0.1, 0.2, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    return {"op": op, "train": rng.random() < 0.6, "dtype": dtype, "rows": rows, "cols": cols, "p": p}


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, cols = _TYPES[case["dtype"]], case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    # pre-activations: every unit with a scale and an offset of its own
    x = (normal(rows, cols).mul_(0.5 + torch.rand(cols, generator=gen, device="cuda")).add_(0.5 * normal(cols))).to(dtype)
    state = {"case": case, "x": x, "p": case["p"], "seed": seed * 7919 + 12345, "offset": seed % 5,
             "weight": (1.0 + 0.2 * normal(cols)).to(dtype), "bias": (0.2 * normal(cols)).to(dtype)}
    if case["train"]:
        state["dy"] = (0.1 * normal(rows, cols)).to(dtype)
        for name in ("x", "weight", "bias"):
            state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from epidemicsimulator_amd import layers
    case, x, weight, bias = state["case"], state["x"], state["weight"], state["bias"]
    if case["op"] == "dropout":
        y = layers.dropout(x, state["p"], state["seed"], state["offset"])
        leaves = (x,)
    else:
        y = layers.layer_norm(x, weight, bias, EPS, dropout=state["p"], seed=state["seed"], offset=state["offset"])
        leaves = (x, weight, bias)
    if not case["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, leaves, state["dy"])


def _kept(state, rows, cols):
    """The units that are kept, and the factor that makes up for the others: Philox4x32-10 (Salmon et al., 2011) with
    key = seed and counter = (column / 8, row, offset) gives 8 draws of 16 bits; a draw below p, in units of 2^-16,
    drops its unit."""
    groups = (cols + 7) // 8
    row = torch.arange(rows, device="cuda", dtype=torch.int64).view(rows, 1)
    col = torch.arange(groups, device="cuda", dtype=torch.int64).view(1, groups)
    c0, c1 = col.expand(rows, groups), row.expand(rows, groups)
    c2, c3 = torch.full_like(c0, state["offset"] & _MASK), torch.full_like(c0, state["offset"] >> 32 & _MASK)
    k0, k1 = state["seed"] & _MASK, state["seed"] >> 32 & _MASK
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57   # the low 64 bits: the sign bit is shifted and masked away
        c0, c1, c2, c3 = (b >> 32 & _MASK) ^ c1 ^ k0, b & _MASK, (a >> 32 & _MASK) ^ c3 ^ k1, a & _MASK
        k0, k1 = (k0 + 0x9E3779B9) & _MASK, (k1 + 0xBB67AE85) & _MASK
    draws = torch.stack([half for word in (c0, c1, c2, c3) for half in (word & 0xFFFF, word >> 16)], dim=-1)
    kept = draws.view(rows, groups * 8)[:, :cols] >= round(state["p"] * 65536)
    return kept, 65536.0 / (65536 - round(state["p"] * 65536))


@torch.no_grad()
def _plain(state):
    case = state["case"]
    dtype = _TYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    rows, cols = case["rows"], case["cols"]
    h = state["x"].to(wide)
    dy = state["dy"].to(wide) if case["train"] else None
    if case["op"] != "norm":
        kept, scale = _kept(state, rows, cols)
        h = torch.where(kept, h * scale, 0.0)
    if case["op"] == "dropout":
        y = h.to(dtype)
        return (y, torch.where(kept, dy * scale, 0.0).to(dtype)) if case["train"] else y
    weight, bias = state["weight"].to(wide), state["bias"].to(wide)
    centred = h - h.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    xhat = centred * rstd
    y = (xhat * weight + bias).to(dtype)
    if not case["train"]:
        return y
    g = dy * weight
    dh = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    dx = dh if case["op"] == "norm" else torch.where(kept, dh * scale, 0.0)
    return y, dx.to(dtype), (dy * xhat).sum(dim=0).to(dtype), dy.sum(dim=0).to(dtype)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    size = _TYPES[case["dtype"]].itemsize
    n, cols = case["rows"] * case["cols"], case["cols"]
    norm = case["op"] != "dropout"
    planes = 4 if case["train"] else 2                                    # x, y and with training dy, dx
    vectors = 0 if not norm else 4 if case["train"] else 2                # weight, bias and their gradients
    flops = (7 if norm else 0) + (1 if case["op"] != "norm" else 0)
    if case["train"]:
        flops += (14 if norm else 0) + (1 if case["op"] != "norm" else 0)
    return {"bytes": (planes * n + vectors * cols) * size, "flops": flops * n}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_kept(p, seed, offset, rows, cols):
    """The kept units by the generator's definition, on the host, a band of rows at a time."""
    u = np.uint64
    width, low, threshold = -(-cols // 8), u(_MASK), round(p * 65536)
    kept = np.empty((rows, width, 8), dtype=bool)
    for first in range(0, rows, max(1, 400_000 // width)):
        count = min(max(1, 400_000 // width), rows - first)
        ctr = [np.zeros((count, width), u) for _ in range(4)]
        ctr[0] += np.arange(width, dtype=u)[None, :]
        ctr[1] += np.arange(first, first + count, dtype=u)[:, None]
        ctr[2] += u(offset % 2**32)
        ctr[3] += u(offset // 2**32 % 2**32)
        for r in range(10):
            left, right = ctr[0] * u(3528531795), ctr[2] * u(3449720151)
            ctr = [(right >> u(32)) ^ ctr[1] ^ u((seed + 2654435769 * r) % 2**32), right & low,
                   (left >> u(32)) ^ ctr[3] ^ u((seed // 2**32 + 3144134277 * r) % 2**32), left & low]
        for k in range(8):
            kept[first:first + count, :, k] = (ctr[k // 2] // u(65536 if k % 2 else 1)) % u(65536) >= u(threshold)
    return kept.reshape(rows, width * 8)[:, :cols]


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    n = float(case["cols"])
    x = state["x"].double()
    factor = None
    if case["op"] != "norm":
        kept = _exact_kept(case["p"], state["seed"], state["offset"], case["rows"], case["cols"])
        factor = torch.from_numpy(np.ascontiguousarray(kept)).cuda().double() / (1.0 - round(case["p"] * 65536) / 65536.0)
        x = x * factor
    if case["op"] == "dropout":
        return (x, state["dy"].double() * factor) if case["train"] else x
    weight, bias = state["weight"].double(), state["bias"].double()
    x = x - x.sum(1, keepdim=True) / n
    x = x - x.sum(1, keepdim=True) / n
    deviation = torch.sqrt((x ** 2).sum(1, keepdim=True) / n + EPS)
    unit = x / deviation
    y = torch.addcmul(bias.expand_as(unit), unit, weight)
    if not case["train"]:
        return y
    dy = state["dy"].double()
    dunit = dy * weight
    # d unit / d x = (1 - 1/n - unit unit^T / n) / deviation for every row
    dx = (dunit - dunit.sum(1, keepdim=True) / n - unit * ((dunit * unit).sum(1, keepdim=True) / n)) / deviation
    if factor is not None:
        dx = dx * factor
    return y, dx, (dy * unit).sum(0), dy.sum(0)
