"""Work of the low-bit operators as a user's program calls it: the microscaled 4-bit codec, the product of 4-bit
operands, training steps of linear layers whose input is kept in 8 bits, and the device-resident 8-bit cache.

``run`` computes either the plain form (elementary torch operations in fp32) or, with ``own`` set, calls
``tensorcache_b200``.  ``exact`` restates the operators in 64 bits.
"""
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the activations of one token, stored in 4 bits and read back: latency
        {"name": "codec_token", "op": "codec", "rows": 1, "cols": 4096, "dtype": "bf16"},
        # fp32 weights of an odd shape: ragged scale tiles on both sides
        {"name": "codec_ragged", "op": "codec", "rows": 1333, "cols": 4128, "dtype": "f32"},
        # a batch of cached features, 128 samples of [446, 768]
        {"name": "codec_features", "op": "codec", "rows": 57088, "cols": 768, "dtype": "bf16"},
        # one token against a 4-bit weight: the weight's bytes are the work
        {"name": "product_token", "op": "product", "m": 1, "n": 14336, "k": 4096, "dtype": "bf16", "bias": False},
        # one sample through a small head with an odd number of outputs
        {"name": "product_ragged", "op": "product", "m": 446, "n": 1001, "k": 768, "dtype": "f16", "bias": True},
        # a long prompt (the shape of the framework's 8-bit product): matrix rate
        {"name": "product_prompt", "op": "product", "m": 8192, "n": 14336, "k": 4096, "dtype": "bf16", "bias": False},
        # training step of a small layer on one sample: latency of several products
        {"name": "linear_sample", "op": "linear", "source": "x", "m": 446, "n": 768, "k": 768, "group": 16, "bias": True},
        # training step of a 1000-class head on a cached batch of 128 x 446 features: few output tiles, a long sum
        {"name": "linear_probe", "op": "linear", "source": "amo", "m": 57088, "n": 1000, "k": 768, "group": 32, "bias": True},
        # training step of a wide layer whose input is kept in 8 bits: matrix rate
        {"name": "linear_block", "op": "linear", "source": "x", "m": 16384, "n": 4096, "k": 4096, "group": 32, "bias": False},
        # one new feature row into a cache that is then read whole: latency
        {"name": "cache_token", "op": "cache", "rows": 446, "width": 768, "new": 1, "skip": 0, "group": 32, "dtype": "bf16"},
        # odd sizes, rows left out (negative index), fp32 features
        {"name": "cache_ragged", "op": "cache", "rows": 2003, "width": 1560, "new": 1001, "skip": 7, "group": 24, "dtype": "f32"},
        # a batch of 128 x 446 feature rows written in random order, the whole cache read in another
        {"name": "cache_batch", "op": "cache", "rows": 65536, "width": 768, "new": 57088, "skip": 0, "group": 32, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["codec", "product", "linear", "cache"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "codec":
        cols = 32 * _log(rng, 1, 448)
        return {"op": op, "rows": _log(rng, 1, min(57088, 43000000 // cols)), "cols": cols, "dtype": dtype}
    if op == "product":
        k, n = 32 * _log(rng, 2, 128), _log(rng, 1, 14336)
        return {"op": op, "m": _log(rng, 1, 8192), "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
    if op == "linear":
        group = rng.choice([16, 32, 64, 128])
        return {"op": op, "source": rng.choice(["x", "x", "sym", "amo"]), "m": _log(rng, 1, 16384), "n": _log(rng, 1, 4096),
                "k": group * _log(rng, 1, 4096 // group), "group": group, "bias": rng.random() < 0.5}
    group = rng.choice([8, 16, 24, 32, 48, 64, 128])
    width = group * _log(rng, 1, 4096 // group)
    rows = _log(rng, 1, min(65536, 50000000 // width))
    new = _log(rng, 1, rows)
    return {"op": op, "rows": rows, "width": width, "new": new, "skip": rng.randrange(0, new // 8 + 1), "group": group, "dtype": dtype}


def work(case):
    op = case["op"]
    if op == "codec":   # x read once, codes and scales written and read, the values written
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["dtype"]] + 2 * (0.5 + 1 / 32) + 2), "flops": 4 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * SIZE[case["dtype"]] + n * k * (0.5 + 1 / 32) + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "linear":  # y, (dX,) dW: inputs and weight in, y and the gradients out
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        x = case["source"] == "x"
        kept = m * k * (1 + (3 if case["source"] == "amo" else 2) / g)
        moved = (2 * m * k + kept + 2 * m * k if x else kept) + 2 * n * k + 4 * m * n + 2 * n * k + (4 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": (6 if x else 4) * m * n * k}
    t, w, g = case["new"] - case["skip"], case["width"], case["group"]
    return {"bytes": t * w * (SIZE[case["dtype"]] + 1 + 2 / g) + case["rows"] * w * (1 + 2 / g + 2), "flops": 4 * t * w + case["rows"] * w}


# ------------------------------------------------------------------------------------------------ inputs

def _features(g, rows, cols, dtype):
    """Normal values with a spread over the channels, some far out, and some rows of zeros (padding tokens)."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    x = torch.where(torch.rand(rows, cols, generator=g, device=DEV) < 0.001, 20 * x, x)
    x[torch.rand(rows, generator=g, device=DEV) < 0.01] = 0
    return x.to(TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "codec":
        s["x"] = _features(g, case["rows"], case["cols"], case["dtype"])
    elif op == "product":
        s["x"] = _features(g, case["m"], case["k"], case["dtype"])
        s["codes"], s["scales"] = _mx_pack(*_mx_quantize(0.02 * torch.randn(case["n"], case["k"], generator=g, device=DEV)))
        s["b"] = torch.randn(case["n"], generator=g, device=DEV).to(torch.bfloat16) if case["bias"] else None
    elif op == "linear":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        x = _features(g, m, k, "bf16")
        if case["source"] == "x":
            s["x"] = x.requires_grad_(True)
        elif case["source"] == "sym":
            q, scales = _int8_quantize(x, group)
            s["q"], s["scales"], s["zp"] = q.to(torch.int8), scales.reshape(-1), None
        else:
            v = x.float().view(m, k // group, group)
            lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
            scale = ((hi - lo) / 255).clamp(min=1e-8).to(torch.bfloat16)
            zp = torch.round(-lo / scale.float()).clamp(0, 255)
            s["q"] = (torch.round(v / scale.float()) + zp).clamp(0, 255).to(torch.uint8).view(m, k)
            s["scales"], s["zp"] = scale.reshape(-1), zp.to(torch.uint8).reshape(-1)
        s["w"] = (k ** -0.5 * torch.randn(n, k, generator=g, device=DEV)).to(torch.bfloat16).requires_grad_(True)
        s["b"] = torch.randn(n, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True) if case["bias"] else None
        s["dy"] = torch.randn(m, n, generator=g, device=DEV).to(torch.bfloat16)
    else:
        rows, width, new, group = case["rows"], case["width"], case["new"], case["group"]
        s["codes"] = torch.randint(-127, 128, (rows, width), generator=g, device=DEV, dtype=torch.int8)
        s["scales"] = (0.02 * torch.rand(rows, width // group, generator=g, device=DEV)).to(torch.bfloat16)
        s["x"] = _features(g, new, width, case["dtype"])
        s["into"] = torch.randperm(rows, generator=g, device=DEV)[:new]
        s["into"][torch.randperm(new, generator=g, device=DEV)[:case["skip"]]] = -1
        s["order"] = torch.randperm(rows, generator=g, device=DEV)
        if own:
            import tensorcache_b200 as tc
            s["cache"] = tc.DeviceFeatureCache(rows, width, group_size=group, device=DEV)
            s["cache"].codes.copy_(s["codes"])
            s["cache"].scales.copy_(s["scales"])
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _mx_quantize(x):
    """fp32 [r, k] -> values of E2M1 [r, k] and scale bytes (biased exponents) [r, k / 32]."""
    v = x.view(x.shape[0], -1, 32)
    v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    byte = ((v.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=0)
    a = torch.ldexp(v, (127 - byte).unsqueeze(-1))
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))   # the spacing of E2M1 around m
    return torch.copysign((torch.round(m / step) * step).clamp(max=6), a).view(x.shape), byte


def _mx_pack(values, byte):
    """E2M1 values and scale bytes -> two codes a byte (low half first), scales in tiles of 128 rows x 4 blocks."""
    r, k = values.shape
    m = values.abs()
    code = torch.where(m < 2, 2 * m, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(values).to(torch.uint8)
    tiles = torch.zeros(-(-r // 128) * 128, -(-k // 128) * 4, dtype=torch.uint8, device=values.device)
    tiles[:r, :k // 32] = byte.to(torch.uint8)
    tiles = tiles.view(-1, 4, 32, tiles.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return code[:, 0::2] + 16 * code[:, 1::2], tiles.reshape(-1)


def _mx_unpack(codes, scales, k):
    r = codes.shape[0]
    code = torch.stack((codes & 15, codes >> 4), -1).view(r, k)
    m = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)[code.int()]
    rows = scales.view(-(-r // 128), -(-k // 128), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-r // 128) * 128, -1)[:r, :k // 32]
    return torch.ldexp(m.view(r, k // 32, 32), rows.int().unsqueeze(-1) - 127).view(r, k)


def _int8_quantize(x, group):
    """[r, k] -> signed codes (as fp32) and bf16 scales [r, k / group]."""
    v = x.float().view(x.shape[0], -1, group)
    v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    scale = (v.abs().amax(-1).clamp(min=1e-8) / 127).to(torch.bfloat16)
    return torch.round(v / scale.float().unsqueeze(-1)).clamp(-128, 127).view(x.shape), scale


def _int8_values(q, scales, group, zp=None):
    v = q.float().view(q.shape[0], -1, group)
    if zp is not None:
        v = v - zp.float().view(q.shape[0], -1, 1)
    return (v * scales.float().view(q.shape[0], -1, 1)).view(q.shape)


def _plain(s):
    op = s["op"]
    if op == "codec":
        codes, scales = _mx_pack(*_mx_quantize(s["x"].float()))
        return _mx_unpack(codes, scales, s["cols"]).to(torch.bfloat16)
    if op == "product":
        xq, byte = _mx_quantize(s["x"].float())
        x = torch.ldexp(xq.view(s["m"], -1, 32), byte.unsqueeze(-1) - 127).view(xq.shape)
        y = x @ _mx_unpack(s["codes"], s["scales"], s["k"]).t()
        return (y if s["b"] is None else y + s["b"].float()).to(torch.bfloat16)
    if op == "linear":
        w, dy = s["w"].detach().float(), s["dy"].float()
        if s["source"] == "x":
            x = s["x"].detach().float()
            kept = _int8_values(*_int8_quantize(x, s["group"]), s["group"])
        else:
            x = kept = _int8_values(s["q"], s["scales"], s["group"], s["zp"])
        y = x @ w.t()
        out = {"y": y if s["b"] is None else y + s["b"].detach().float(), "dw": dy.t() @ kept}
        if s["b"] is not None:
            out["db"] = dy.sum(0)
        if s["source"] == "x":
            out["dx"] = dy @ w
        return {name: t.to(torch.bfloat16) for name, t in out.items()}
    q, scale = _int8_quantize(s["x"], s["group"])
    live = s["into"] >= 0
    s["codes"][s["into"][live]] = q[live].to(torch.int8)
    s["scales"][s["into"][live]] = scale[live]
    return _int8_values(s["codes"][s["order"]], s["scales"][s["order"]], s["group"]).to(torch.bfloat16)


def _framework(s):
    import tensorcache_b200 as tc

    op = s["op"]
    if op == "codec":
        codes, scales, shape = tc.quantize_mxfp4(s["x"])
        return tc.dequantize_mxfp4(codes, scales, shape)
    if op == "product":
        return tc.mxfp4_matmul(s["x"], s["codes"], s["scales"], bias=s["b"])
    if op == "linear":
        if s["source"] == "x":
            y = tc.int8_checkpoint_linear(s["x"], s["w"], s["b"], group_size=s["group"])
            leaves = {"dw": s["w"], "db": s["b"], "dx": s["x"]}
        else:
            y = tc.fused_dequant_linear(s["q"], s["scales"], s["w"], s["b"], zero_points=s["zp"], group_size=s["group"])
            leaves = {"dw": s["w"], "db": s["b"]}
        leaves = {name: t for name, t in leaves.items() if t is not None}
        return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["dy"])))}
    s["cache"].write(s["into"], s["x"])
    return s["cache"].read(s["order"])


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ 64 bits

def _pow2(e):
    """2^e for whole numbers, exactly (from the bits of a double)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_mx(x):
    """The values that the 4-bit form of x [r, k] stands for, by nearest neighbour on the E2M1 grid."""
    v = x.double().view(x.shape[0], -1, 32)
    v = torch.where(v.isfinite(), v, 0.0)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=v.device)
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))      # max = m * 2^e with m in [0.5, 1)
    unit = _pow2((e - 3).clamp(min=-127))
    a = v.abs() / unit
    low = (torch.searchsorted(grid, a.contiguous(), right=True) - 1).clamp(0, 7)
    high = (low + 1).clamp(max=7)
    below, above = a - grid[low], grid[high] - a
    up = (above < below) | ((above == below) & (low % 2 == 1))
    return (torch.sign(v) * torch.where(up, grid[high], grid[low]) * unit).view(x.shape)


def _exact_int8(x, group):
    """(signed codes, scales) of x in 64 bits; the scale is defined as the bf16 rounding of the fp32 quotient."""
    v = x.detach().double().view(x.shape[0], -1, group)
    v = torch.where(v.isfinite(), v, 0.0)
    scale = (v.abs().amax(-1, keepdim=True).clamp(min=float(torch.tensor(1e-8))) / 127).float().to(torch.bfloat16).double()
    return torch.round((v / scale).float().double()).clamp(-128, 127), scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "codec":
        return _exact_mx(s["x"])
    if op == "product":
        c = s["codes"].long()
        c = torch.stack((c % 16, c // 16), 2).flatten(1)
        r, k = c.shape
        grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        w = torch.tensor(grid + [-v for v in grid], dtype=torch.float64, device=c.device)[c]
        row, blk = torch.arange(r, device=c.device)[:, None], torch.arange(k // 32, device=c.device)[None, :]
        at = (row // 128 * -(-k // 128) + blk // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + blk % 4
        w = w.view(r, -1, 32) * _pow2(s["scales"].long()[at] - 127).unsqueeze(-1)
        y = _exact_mx(s["x"]) @ w.view(r, k).t()
        return y if s["b"] is None else y + s["b"].double()
    if op == "linear":
        w, dy, m = s["w"].detach().double(), s["dy"].double(), case["m"]
        if case["source"] == "x":
            q, scale = _exact_int8(s["x"], case["group"])
            kept, x = (q * scale).view(m, -1), s["x"].detach().double()
        else:
            q = s["q"].double().view(m, -1, case["group"])
            q = q if s["zp"] is None else q - s["zp"].double().view(m, -1, 1)
            kept = x = (q * s["scales"].double().view(m, -1, 1)).view(m, -1)
        out = {"y": x @ w.t(), "dw": dy.t() @ kept}
        if s["b"] is not None:
            out["y"] = out["y"] + s["b"].detach().double()
            out["db"] = dy.sum(0)
        if case["source"] == "x":
            out["dx"] = dy @ w
        return out
    rows = s["codes"].double().view(case["rows"], -1, case["group"]) * s["scales"].double().unsqueeze(-1)
    q, scale = _exact_int8(s["x"], case["group"])
    live = s["into"] >= 0
    rows[s["into"][live]] = (q * scale)[live]
    return rows[s["order"]].view(case["rows"], case["width"])
