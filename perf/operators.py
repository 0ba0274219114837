"""The channel-last row operators beside the BatchNorm layers, as they are measured: group norm with an activation,
dropout from a counter-based generator, products in 8-bit floats with a scale for each block of 128.

`run` computes a case in its plain form, or with `own` through the package's entry points.  Training cases return the
outputs and every gradient.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases ----------------------------------------------------------------------------------------------------------------

def _norm(name, clouds, rows, channels, groups, dtype, act, train, residual=False, p=0.0, ragged=False):
    return {"name": name, "op": "norm", "clouds": clouds, "rows": rows, "channels": channels, "groups": groups,
            "dtype": dtype, "act": act, "train": train, "residual": residual, "p": p, "ragged": ragged}


def _drop(name, rows, channels, dtype, p, train, residual=False):
    return {"name": name, "op": "dropout", "rows": rows, "channels": channels, "dtype": dtype, "p": p, "train": train,
            "residual": residual}


def _prod(name, rows, k, n, dtype, train, bias=False):
    return {"name": name, "op": "fp8", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train, "bias": bias}


def listed():
    return [
        # one cloud's deepest level (256 centres x 256 channels) at inference: latency
        _norm("norm_one_cloud", 1, 256, 256, 8, "f32", "relu", False),
        # the seed features of four clouds behind a residual branch, a training step in 16 bits
        _norm("norm_seeds_train", 4, 1024, 256, 32, "bf16", "gelu", True, residual=True),
        # clouds of different sizes packed row after row, odd sizes, dropped out in the same pass
        _norm("norm_ragged_train", 7, 50021, 90, 6, "f16", "silu", True, p=0.1, ragged=True),
        # the grouped neighbourhoods of the first set-abstraction level (2048 centres x 64 neighbours, 4 clouds)
        _norm("norm_grouped_train", 4, 131072, 128, 8, "f32", "silu", True),
        # one cloud's seeds in front of a head: latency
        _drop("dropout_seeds", 1024, 256, "f32", 0.1, False),
        # a residual branch of odd width in a training step
        _drop("dropout_residual_train", 65537, 515, "bf16", 0.25, True, residual=True),
        # the largest grouped activation of a training step
        _drop("dropout_grouped_train", 524288, 256, "f32", 0.5, True),
        # a single row through a 1024 x 1024 layer that is kept in 8 bits
        _prod("fp8_one_row", 1, 1024, 1024, "bf16", False),
        # the per-seed head of four clouds: 259 features, 2 + 300 outputs, none a multiple of a tile
        _prod("fp8_head", 4096, 259, 302, "f32", False, bias=True),
        # the pointwise expansion 128 -> 512 of the first level's blocks, a training step
        _prod("fp8_pointwise_train", 8192, 128, 512, "f32", True, bias=True),
        # grouped neighbourhoods: many rows, few channels
        _prod("fp8_grouped_train", 524288, 128, 256, "bf16", True),
        # a wide layer over many rows: the matrix cores
        _prod("fp8_wide_train", 16384, 4096, 4096, "bf16", True),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is uniform."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "fp8", "fp8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if op == "norm":
        groups = rng.choice([1, 2, 4, 6, 8, 16, 32])
        channels = groups * rng.randint(max(1, 16 // groups), max(1, 1024 // groups))
        ragged = rng.random() < 0.4
        clouds = rng.randint(1, 9)
        room = 60_000_000 // (channels * (1 if ragged else clouds))
        case = _norm("", clouds, _spread(rng, 16, min(room, 131072)), channels, groups, dtype,
                     rng.choice(["silu", "gelu", "none"] + ([] if train else ["relu", "leaky_relu"])), train,
                     residual=rng.random() < 0.4, p=rng.choice([0.0, 0.0, 0.1, 0.5]), ragged=ragged)
    elif op == "dropout":
        channels = rng.randint(16, 1024)
        case = _drop("", _spread(rng, 1, 130_000_000 // channels), channels, dtype, rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]),
                     train, residual=rng.random() < 0.5)
    else:
        k, n = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
        most = min(524288, 60_000_000_000 // (k * n), 150_000_000 // max(k, n))
        case = _prod("", _spread(rng, 1, most), k, n, dtype, train, bias=rng.random() < 0.5)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    state = {"case": case}
    if case["op"] == "norm":
        C = case["channels"]
        shape = (case["rows"], C) if case["ragged"] else (case["clouds"], case["rows"], C)
        # what a 1x1 convolution puts out: every channel with an offset and a width of its own
        state["x"] = (normal(*shape) * (0.5 + torch.rand(C, generator=gen, device=dev)) + normal(C)).to(dtype)
        state["weight"] = 1.0 + 0.2 * normal(C)
        state["bias"] = 0.2 * normal(C)
        state["residual"] = normal(*shape).to(dtype) if case["residual"] else None
        state["offsets"] = None
        if case["ragged"]:
            cuts = torch.randint(0, case["rows"] + 1, (case["clouds"] - 1,), generator=gen, device=dev).sort().values
            ends = torch.tensor([0, case["rows"]], device=dev)
            state["offsets"] = torch.cat([ends[:1], cuts, ends[1:]])
        state["rng"] = torch.tensor([seed * 7919 + 13, 5], device=dev) if case["p"] else None
        like = state["x"]
    elif case["op"] == "dropout":
        state["x"] = normal(case["rows"], case["channels"]).to(dtype)
        state["residual"] = normal(case["rows"], case["channels"]).to(dtype) if case["residual"] else None
        state["rng"] = torch.tensor([seed * 7919 + 13, 5], device=dev)
        like = state["x"]
    else:
        # activations behind a norm and an activation function; weights as they are initialised
        state["x"] = torch.nn.functional.silu(normal(case["rows"], case["k"])).to(dtype)
        weight = normal(case["n"], case["k"]) * (2.0 / case["k"]) ** 0.5
        if case["train"]:
            state["weight"] = weight
        else:                          # a served layer is kept in 8 bits: codes padded to whole blocks, and exponents
            state["codes"], state["scales"] = _quantise_weight(weight)
        state["bias"] = normal(case["n"]) if case["bias"] else None
        like = state["x"].new_empty(case["rows"], case["n"])
    if case["train"]:
        state["dy"] = normal(*like.shape).to(dtype)
        for name in ("x", "residual", "weight", "bias"):
            if state.get(name) is not None:
                state[name].requires_grad_()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _run_norm, "dropout": _run_dropout, "fp8": _run_fp8}[state["case"]["op"]](state)


def _run_own(state):
    from graspbalance_amd import fused_rows
    case = state["case"]
    if case["op"] == "norm":
        y = fused_rows.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], act=case["act"],
                                      residual=state["residual"], offsets=state["offsets"], dropout_p=case["p"],
                                      rng=state["rng"])
    elif case["op"] == "dropout":
        y = fused_rows.dropout(state["x"], case["p"], state["rng"], residual=state["residual"])
    elif case["train"]:
        y = fused_rows.fp8_linear(state["x"], state["weight"], state["bias"])
    else:
        y = fused_rows.fp8_linear(state["x"], fused_rows.Fp8Weight(state["codes"], state["scales"], case["k"]), state["bias"])
    if not case["train"]:
        return {"y": y}
    names = [n for n in ("x", "residual", "weight", "bias") if state.get(n) is not None]
    grads = torch.autograd.grad(y, [state[n] for n in names], state["dy"])
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


# the plain forms

def _mul_hi_lo(a, b):
    """The two 32-bit halves of a * b for a 32-bit number a and 32-bit numbers b held in 64 bits."""
    low, high = a * (b & 0xFFFF), a * (b >> 16)
    middle = high + (low >> 16)
    return middle >> 16, ((middle & 0xFFFF) << 16) | (low & 0xFFFF)


def _halfwords(rng, count):
    """The first `count` 16-bit numbers of the call rng = [seed, call]: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011)."""
    block = torch.arange((count + 7) // 8, device=rng.device)
    c = [block & 0xFFFFFFFF, block >> 32, (rng[1] & 0xFFFFFFFF).expand_as(block), ((rng[1] >> 32) & 0xFFFFFFFF).expand_as(block)]
    k0, k1 = rng[0] & 0xFFFFFFFF, (rng[0] >> 32) & 0xFFFFFFFF
    for _ in range(10):
        hi0, lo0 = _mul_hi_lo(0xD2511F53, c[0])
        hi1, lo1 = _mul_hi_lo(0xCD9E8D57, c[2])
        c = [hi1 ^ c[1] ^ k0, lo1, hi0 ^ c[3] ^ k1, lo0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack(c, 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count]


def _factor(rng, p, shape):
    """keep / (1 - p) of every element, p to the nearest 65536th."""
    q = int(p * 65536 + 0.5)
    keep = (_halfwords(rng, math.prod(shape)) >= q).view(shape)
    return torch.where(keep, 65536.0 / (65536 - q), 0.0)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, 0.01 * z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, 0.01)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _per_cloud(rows, clouds, offsets):
    """rows (R, G) summed over the rows of each cloud, in 64 bits: (clouds, G)."""
    if offsets is None:
        return rows.view(clouds, -1, rows.shape[1]).sum(1, dtype=torch.float64)
    upto = torch.nn.functional.pad(rows.t().contiguous().cumsum(1, dtype=torch.float64), (1, 0))
    return (upto[:, offsets[1:]] - upto[:, offsets[:-1]]).t()


def _run_norm(state):
    case, x = state["case"], state["x"]
    shape, C, G = x.shape, case["channels"], case["groups"]
    x = x.float().view(-1, G, C // G)
    offsets = state["offsets"]
    if offsets is None:
        count = float(case["rows"] * (C // G))
        cloud = torch.arange(case["clouds"], device=x.device).repeat_interleave(case["rows"])
    else:
        count = (offsets[1:] - offsets[:-1]).double().clamp(min=1)[:, None] * (C // G)
        cloud = torch.searchsorted(offsets[1:], torch.arange(x.shape[0], device=x.device), right=True)

    def average(values):
        """values (rows, G, C / G) averaged over each cloud and group, for every row."""
        sums = _per_cloud(values.sum(2), case["clouds"], offsets)
        return (sums / count).float()[cloud][:, :, None]

    mean = average(x)
    rstd = torch.rsqrt(average((x - mean) ** 2) + 1e-5)
    xh = (x - mean) * rstd
    weight, bias = state["weight"].view(G, -1), state["bias"].view(G, -1)
    z = xh * weight + bias
    if state["residual"] is not None:
        z = z + state["residual"].float().view_as(z)
    factor = _factor(state["rng"], case["p"], z.shape) if case["p"] else 1.0
    y = (_act(z, case["act"]) * factor).to(state["x"].dtype).view(shape)
    if not case["train"]:
        return {"y": y}
    g = state["dy"].float().view_as(z) * factor * _act_grad(z, case["act"])
    h = g * weight
    out = {"y": y, "dx": ((h - average(h) - xh * average(h * xh)) * rstd).to(state["x"].dtype).view(shape)}
    if state["residual"] is not None:
        out["dresidual"] = g.to(state["residual"].dtype).view(shape)
    out["dweight"] = (g * xh).sum(0, dtype=torch.float64).float().view(C)
    out["dbias"] = g.sum(0, dtype=torch.float64).float().view(C)
    return out


def _run_dropout(state):
    case, x = state["case"], state["x"]
    factor = _factor(state["rng"], case["p"], x.shape)
    y = x.float() * factor
    if state["residual"] is not None:
        y = y + state["residual"].float()
    y = y.to(x.dtype)
    if not case["train"]:
        return {"y": y}
    out = {"y": y, "dx": (state["dy"].float() * factor).to(x.dtype)}
    if state["residual"] is not None:
        out["dresidual"] = state["dy"].clone()
    return out


def _exponent(largest):
    """The least e with largest <= 448 * 2^e, at least -126; 0 for blocks of zeros."""
    mantissa, e = torch.frexp(largest)
    e = torch.where(mantissa <= 0.875, e - 9, e - 8).clamp(min=-126)
    return torch.where(largest == 0, 0, e)


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _padded(x, rows=1):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 128, 0, -x.shape[0] % rows))


def _quantise_weight(weight):
    """Codes (N, K up to whole blocks) and biased exponents, one for each block of 128 x 128."""
    blocks = _padded(weight.float(), 128).unflatten(1, (-1, 128)).unflatten(0, (-1, 128))
    e = _exponent(blocks.abs().amax((1, 3)))
    codes = (blocks * _power(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.flatten(2, 3).flatten(0, 1)[:weight.shape[0]].contiguous(), (e + 127).to(torch.uint8)


def _weight_values(codes, scales, n, k):
    scale = _power(scales.int() - 127).repeat_interleave(128, 0).repeat_interleave(128, 1)
    return (codes.float() * scale[:n, :codes.shape[1]])[:, :k]


def _in_8_bits(x):
    """The values that x has in 8 bits with a power of two for each 128 along its rows."""
    blocks = _padded(x.float()).unflatten(1, (-1, 128))
    e = _exponent(blocks.abs().amax(2, keepdim=True))
    return ((blocks * _power(-e)).to(torch.float8_e4m3fn).float() * _power(e)).flatten(1)[:, :x.shape[1]]


def _run_fp8(state):
    case, x = state["case"], state["x"]
    codes, scales = _quantise_weight(state["weight"]) if case["train"] else (state["codes"], state["scales"])
    w = _weight_values(codes, scales, case["n"], case["k"])
    xq = _in_8_bits(x)
    y = xq @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"]
    y = y.to(x.dtype)
    if not case["train"]:
        return {"y": y}
    dyq = _in_8_bits(state["dy"])
    out = {"y": y, "dx": (dyq @ w).to(x.dtype), "dweight": dyq.t() @ xq}
    if state["bias"] is not None:
        out["dbias"] = state["dy"].sum(0, dtype=torch.float64).float()
    return out


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        return {"norm": _exact_norm, "dropout": _exact_dropout, "fp8": _exact_fp8}[case["op"]](case, state)


def _exact_factor(rng, p, shape):
    q = round(p * 65536)
    seed, call = (int(v) for v in rng)
    count = math.prod(shape)
    i = torch.arange(-(-count // 8), dtype=torch.int64, device=rng.device)
    full = 2 ** 32 - 1
    w = [i & full, i >> 32 & full, torch.full_like(i, call & full), torch.full_like(i, call >> 32 & full)]
    key = [seed & full, seed >> 32 & full]
    for r in range(10):
        a = w[0] * 0xD2511F53      # 64-bit products wrap, so all of their bits are there
        b = w[2] * 0xCD9E8D57
        w = [(b >> 32 & full) ^ w[1] ^ (key[0] + r * 0x9E3779B9 & full), b & full,
             (a >> 32 & full) ^ w[3] ^ (key[1] + r * 0xBB67AE85 & full), a & full]
    numbers = torch.empty(i.numel(), 8, dtype=torch.int64, device=rng.device)
    for j in range(4):
        numbers[:, 2 * j] = w[j] & 65535
        numbers[:, 2 * j + 1] = w[j] >> 16
    return (numbers.flatten()[:count].reshape(shape) >= q).double() / (1 - q / 65536)


def _exact_norm(case, state):
    x = state["x"].double().reshape(-1, case["channels"])
    n, C, G = x.shape[0], case["channels"], case["groups"]
    cuts = state["offsets"].tolist() if case["ragged"] else [i * case["rows"] for i in range(case["clouds"] + 1)]
    w, b = state["weight"].double(), state["bias"].double()
    res = state["residual"].double().reshape(n, C) if case["residual"] else None
    factor = _exact_factor(state["rng"], case["p"], (n, C)) if case["p"] else None
    dy = state["dy"].double().reshape(n, C) if case["train"] else None
    y, dx, dres = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for lo, hi in zip(cuts[:-1], cuts[1:]):
        if lo == hi:
            continue
        part = x[lo:hi].reshape(hi - lo, G, C // G)
        var, mean = torch.var_mean(part, (0, 2), correction=0, keepdim=True)
        normed = ((part - mean) / torch.sqrt(var + 1e-5)).reshape(hi - lo, C)
        z = normed * w + b
        if res is not None:
            z = z + res[lo:hi]
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        sig = 1 / (1 + torch.exp(-z))
        value = {"none": z, "relu": torch.relu(z), "leaky_relu": torch.maximum(z, 0.01 * z), "silu": z * sig, "gelu": z * phi}
        y[lo:hi] = value[case["act"]]
        if dy is not None:
            slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "leaky_relu": 0.01 + 0.99 * (z > 0).double(),
                     "silu": sig + z * sig * (1 - sig), "gelu": phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}
            g = dy[lo:hi] * slope[case["act"]]
            if factor is not None:
                g = g * factor[lo:hi]
            dres[lo:hi] = g
            dw += (g * normed).sum(0)
            db += g.sum(0)
            h, v = (g * w).reshape(part.shape), normed.reshape(part.shape)
            dx[lo:hi] = ((h - h.mean((0, 2), keepdim=True) - v * (h * v).mean((0, 2), keepdim=True))
                         / torch.sqrt(var + 1e-5)).reshape(hi - lo, C)
    if factor is not None:
        y = y * factor
    shape = state["x"].shape
    if not case["train"]:
        return {"y": y.reshape(shape)}
    out = {"y": y.reshape(shape), "dx": dx.reshape(shape)}
    if case["residual"]:
        out["dresidual"] = dres.reshape(shape)
    out["dweight"], out["dbias"] = dw, db
    return out


def _exact_dropout(case, state):
    factor = _exact_factor(state["rng"], case["p"], state["x"].shape)
    y = state["x"].double() * factor
    if case["residual"]:
        y = y + state["residual"].double()
    out = {"y": y}
    if case["train"]:
        out["dx"] = state["dy"].double() * factor
        if case["residual"]:
            out["dresidual"] = state["dy"].double()
    return out


def _exact_8_bits(x, block_rows):
    """x in 64 bits rounded to e4m3 under a power of two for each block of block_rows x 128."""
    rows, cols = x.shape
    out = torch.zeros(-(-rows // block_rows) * block_rows, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    out[:rows, :cols] = x
    b = out.reshape(-1, block_rows, out.shape[1] // 128, 128)
    top = b.abs().amax(dim=(1, 3), keepdim=True)
    e = torch.ceil(torch.log2(top / 448))
    e = torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, e)       # the logarithm may be off by one at a border
    e = torch.where(torch.exp2(e) * 448 < top, e + 1, e).clamp(min=-126)
    scale = torch.where(top > 0, torch.exp2(e), 1.0)
    b = b / scale
    # e4m3: four significant bits, the last place never below 2^-9
    place = torch.exp2(torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(b / place) * place * scale).reshape(out.shape)[:rows, :cols]


def _exact_fp8(case, state):
    x = _exact_8_bits(state["x"].double(), 1)
    if case["train"]:
        w = _exact_8_bits(state["weight"].double(), 128)
    else:
        w = state["codes"].to(torch.float64)[:, :case["k"]]
        rows = torch.arange(case["n"], device=w.device) // 128
        cols = torch.arange(case["k"], device=w.device) // 128
        w = w * torch.exp2(state["scales"].double() - 127)[rows][:, cols]
    y = x @ w.T
    if case["bias"]:
        y += state["bias"].double()
    if not case["train"]:
        return {"y": y}
    dy = _exact_8_bits(state["dy"].double(), 1)
    out = {"y": y, "dx": dy @ w, "dweight": dy.T @ x}
    if case["bias"]:
        out["dbias"] = state["dy"].double().sum(0)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["channels"] * (1 if case["ragged"] else case["clouds"])
        tensors = 2 + case["residual"] + case["train"] * (2 + case["residual"])
        flops = n * ((60 if case["train"] else 20) + (30 if case["p"] else 0))
        return {"bytes": n * size * tensors + 4 * case["channels"] * (2 + 2 * case["train"]), "flops": flops}
    if case["op"] == "dropout":
        n = case["rows"] * case["channels"]
        tensors = 2 + case["residual"] + case["train"] * (2 + case["residual"])
        return {"bytes": n * size * tensors, "flops": n * 20 * (1 + case["train"])}
    p, k, n = case["rows"], case["k"], case["n"]
    if not case["train"]:
        return {"bytes": p * (k + n) * size + k * n + 4 * n * case["bias"], "flops": 2 * p * k * n}
    return {"bytes": 2 * p * (k + n) * size + 2 * 4 * k * n + 8 * n * case["bias"], "flops": 6 * p * k * n}
