"""What is measured of the training operators: group normalisation with an activation (channels last, forward and backward,
with or without dropout of its result) and dropout from a counter-based generator (forward with a block's residual, backward).

`run` computes an operator in its plain form, elementary torch operations in float32 on whatever device the state is on, or,
where `own` is true, through fisr_amd/norm.py.  `exact` is the operator's definition in 64 bits, written apart from both.
"""
import functools

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
LOW = 0xFFFFFFFF


# ---- the cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # Channels and maps are those of this repository's U-Net: 64 / 128 / 256 / 512 channels, training patches of 96 x 96 pixels
        # in a batch of 8 samples x 4 windows = 32 images, inference tiles of 544 x 992 pixels.
        # the bottleneck of the coarsest level of a training step: a map of 3 x 3 pixels, the call's latency is what counts
        dict(name="norm 3x3 f32", op="norm", type="f32", n=32, h=3, w=3, c=512, groups=32, act="relu", p=0.0),
        # the first encoder level of a training step, full resolution
        dict(name="norm train f32", op="norm", type="f32", n=32, h=96, w=96, c=64, groups=8, act="silu", p=0.0),
        # the second encoder level in bfloat16, normalised, activated and dropped in one go before the block's second conv
        dict(name="norm drop train bf16", op="norm", type="bf16", n=32, h=48, w=48, c=128, groups=32, act="silu", p=0.1),
        # serving: one tile of a 4K frame, statistics over half a million pixels and few groups
        dict(name="norm tile f16", op="norm", type="f16", n=1, h=544, w=992, c=64, groups=8, act="gelu", p=0.0),
        # serving: the twelve tiles of a stack of three windows in one call (the largest)
        dict(name="norm 12 tiles f16", op="norm", type="f16", n=12, h=544, w=992, c=64, groups=16, act="relu", p=0.0),
        # ragged: an odd map, channels that fill no whole vector of loads, groups of nine channels
        dict(name="norm ragged f32", op="norm", type="f32", n=5, h=67, w=45, c=36, groups=4, act="gelu", p=0.25),
        # backward of the coarse maps of a training step
        dict(name="norm grad 6x6 f32", op="norm_grad", type="f32", n=32, h=6, w=6, c=256, groups=32, act="silu", p=0.0),
        # backward at full resolution
        dict(name="norm grad train f32", op="norm_grad", type="f32", n=32, h=96, w=96, c=64, groups=8, act="silu", p=0.0),
        # backward of the fused block in bfloat16
        dict(name="norm grad drop bf16", op="norm_grad", type="bf16", n=32, h=48, w=48, c=128, groups=32, act="gelu", p=0.1),
        # the end of a residual block on the bottleneck's map
        dict(name="dropout 3x3 f32", op="dropout", type="f32", n=32, h=3, w=3, c=512, p=0.1, residual=True),
        # the end of a residual block at full resolution in bfloat16
        dict(name="dropout train bf16", op="dropout", type="bf16", n=32, h=96, w=96, c=64, p=0.2, residual=True),
        # its gradient in float32 on a map of odd size and 29 channels (the network's input)
        dict(name="dropout grad odd f32", op="dropout", type="f32", n=13, h=271, w=495, c=29, p=0.5, residual=False),
    ]


def draw(rng):
    """One more case of the listed ones' ranges: maps of one pixel to a tile's, 1 to 32 images, 1 to 1024 channels, every type."""
    op = rng.choice(("norm", "norm", "norm_grad", "norm_grad", "dropout"))
    most = 60e6 if op == "norm" else 30e6                     # elements
    while True:
        side = 2.0 ** rng.uniform(0.0, 9.5)
        h = max(1, round(side * 2.0 ** rng.uniform(-0.5, 0.5)))
        w = max(1, round(side * 2.0 ** rng.uniform(-0.5, 0.5)))
        n = max(1, round(2.0 ** rng.uniform(0.0, 5.0)))
        groups = rng.choice((1, 2, 4, 8, 16, 32))
        c = groups * rng.choice((1, 2, 3, 4, 6, 8, 9, 12, 16, 24, 32))
        # (the gradient of a group of a few values is rounding and little else: no two ways to compute it agree there)
        if 2000 <= n * h * w * c <= most and (op == "dropout" or h * w * (c // groups) >= 32):
            break
    case = dict(op=op, type=rng.choice(("f32", "f16", "bf16")), n=n, h=h, w=w, c=c, p=rng.choice((0.0, 0.0, 0.1, 0.25)))
    if op == "dropout":
        case.update(p=rng.choice((0.05, 0.1, 0.3, 0.5)), residual=rng.random() < 0.5)
    else:
        # (the step of relu's gradient at zero leaves no value that two roundings agree on: the backward cases have smooth ones)
        case.update(groups=groups, act=rng.choice(("none", "relu", "silu", "gelu") if op == "norm" else ("none", "silu", "gelu")))
    return case


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    t = TYPES[case["type"]]
    n, h, w, c = (case[k] for k in "nhwc")

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = dict(case)
    s["p"] = float(case["p"])
    # the generator's key and the number of the call: numbers that a program draws per step
    s["rng_seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) & (2 ** 64 - 1)
    s["rng_offset"] = seed % 1000003
    if case["op"] == "dropout":
        s["x"] = normal(n, h, w, c).to(t)
        s["residual_in"] = normal(n, h, w, c).to(t) if case["residual"] else None
    else:
        # what a conv leaves: every channel has its own mean and spread
        x = normal(n, h, w, c)
        x.mul_(0.5 + torch.rand(c, generator=gen, device=dev)).add_(0.5 + normal(c))
        s["x"] = x.to(t)
        del x
        s["gamma"] = 1.0 + 0.2 * normal(c)
        s["beta"] = 0.2 * normal(c)
    if case["op"] == "norm_grad":
        s["dy"] = normal(n, h, w, c).to(t)
        v = s["x"].double().view(n, h * w, case["groups"], -1)       # the statistics that the forward pass kept
        var, mean = torch.var_mean(v, dim=(1, 3), correction=0)
        s["stats"] = torch.stack((mean, torch.rsqrt(var + EPS))).float()
    return s


def run(s):
    if own:
        return run_own(s)
    if s["op"] == "norm":
        return plain_norm(s)
    if s["op"] == "norm_grad":
        return plain_norm_grad(s)
    y = plain_drop(s["x"].float(), s)
    return (y if s["residual_in"] is None else y + s["residual_in"].float()).to(s["x"].dtype)


@functools.lru_cache(None)
def framework():
    from fisr_amd import norm
    return norm


def run_own(s):
    norm = framework()
    drop = norm.Dropout(s["p"], s["rng_seed"], s["rng_offset"]) if s["p"] else None
    if s["op"] == "norm":
        y, stats = norm.group_norm(s["x"], s["groups"], s["gamma"], s["beta"], eps=EPS, act=s["act"], dropout=drop)
        return {"y": y, "mean": stats[0], "rstd": stats[1]}
    if s["op"] == "norm_grad":
        dx, dgamma, dbeta = norm.group_norm_backward(s["dy"], s["x"], s["stats"], s["groups"], s["gamma"], s["beta"],
                                                     act=s["act"], dropout=drop)
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if s["residual_in"] is None:
        return norm.dropout_backward(s["x"], drop)
    return norm.dropout(s["x"], drop, residual=s["residual_in"])


# ---- the plain form: float32 ---------------------------------------------------------------------------------------------
def mul32(a, m):
    """High and low word of a * m, a: 32-bit words in int64, by 16-bit parts of m (no product passes 2^63)."""
    lo, hi = a * (m & 0xFFFF), a * (m >> 16)
    return (hi + (lo >> 16)) >> 16, (lo + ((hi & 0xFFFF) << 16)) & LOW


def philox_round(state, _):
    """One round of Philox4x32 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, Parallel random numbers: as easy as 1, 2, 3, 2011)."""
    c0, c1, c2, c3, k0, k1 = state
    h0, l0 = mul32(c0, 0xD2511F53)
    h1, l1 = mul32(c2, 0xCD9E8D57)
    return h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0, (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW


def plain_drop(v, s):
    """Element i of the dense tensor is dropped where the 16-bit number i % 8 of Philox block i // 8 is below 65536 p (7 rounds)."""
    t = round(s["p"] * 65536)
    if t == 0:
        return v
    count = v.numel()
    block = torch.arange((count + 7) // 8, device=v.device)
    zero = torch.zeros_like(block)
    start = (block & LOW, block >> 32, zero + (s["rng_offset"] & LOW), zero + (s["rng_offset"] >> 32), s["rng_seed"] & LOW, s["rng_seed"] >> 32)
    words = torch.stack(functools.reduce(philox_round, range(7), start)[:4], 1)
    numbers = torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:count].view(v.shape)
    return torch.where(numbers >= t, v * (65536.0 / (65536 - t)), torch.zeros_like(v))


def plain_act(z, act):
    """act(z) and its derivative's factors are elementary: where, exp, erf."""
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return z


def plain_act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return sg * (1 + z * (1 - sg))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    return torch.ones_like(z)


def spread(v, s):
    """[n, groups] -> what multiplies [n, pixels, groups, channels of a group]."""
    return v.view(s["n"], 1, s["groups"], 1)


def per_group(v, s):
    return v.view(s["n"], s["h"] * s["w"], s["groups"], s["c"] // s["groups"])


def plain_norm(s):
    x = per_group(s["x"].float(), s)
    mean = x.mean(dim=(1, 3))
    d = x - spread(mean, s)
    rstd = 1 / torch.sqrt((d * d).mean(dim=(1, 3)) + EPS)
    z = (d * spread(rstd, s)).view(s["x"].shape) * s["gamma"] + s["beta"]
    return {"y": plain_drop(plain_act(z, s["act"]), s).to(s["x"].dtype), "mean": mean, "rstd": rstd}


def plain_norm_grad(s):
    mean, rstd = s["stats"]
    xh = ((per_group(s["x"].float(), s) - spread(mean, s)) * spread(rstd, s)).view(s["x"].shape)
    z = xh * s["gamma"] + s["beta"]
    dz = plain_drop(s["dy"].float(), s) * plain_act_grad(z, s["act"])
    a, b = dz.sum(dim=(1, 2)), (dz * xh).sum(dim=(1, 2))            # [n, c]
    m = s["h"] * s["w"] * (s["c"] // s["groups"])
    s1 = (a * s["gamma"]).view(s["n"], s["groups"], -1).sum(2) / m
    s2 = (b * s["gamma"]).view(s["n"], s["groups"], -1).sum(2) / m
    dx = spread(rstd, s) * (per_group(dz * s["gamma"], s) - spread(s1, s) - per_group(xh, s) * spread(s2, s))
    return {"dx": dx.reshape(s["x"].shape).to(s["x"].dtype), "dgamma": b.sum(0), "dbeta": a.sum(0)}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    e = case["n"] * case["h"] * case["w"] * case["c"]
    size, drawn = BYTES[case["type"]], 12 if case["p"] else 0        # Philox: 7 rounds of 14 operations for 8 elements
    if case["op"] == "dropout":
        return {"bytes": e * size * (3 if case["residual"] else 2), "flops": e * (2 + drawn)}
    kept = 8 * case["n"] * case["groups"] + 8 * case["c"]            # statistics, gamma and beta
    if case["op"] == "norm":
        return {"bytes": 2 * e * size + kept, "flops": e * (9 + drawn)}
    return {"bytes": 3 * e * size + kept + 8 * case["c"], "flops": e * (20 + drawn)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def kept64(count, s, device):
    """0 where an element is dropped, its factor elsewhere: the generator on 64-bit products that wrap (their bits are the unsigned ones)."""
    t = int(round(65536 * s["p"]))
    i = torch.arange(count, device=device, dtype=torch.int64)
    blk, lane = i // 8, i % 8
    del i
    x = [blk & LOW, (blk >> 32) & LOW, torch.full_like(blk, s["rng_offset"] % 2 ** 32), torch.full_like(blk, s["rng_offset"] // 2 ** 32)]
    key = [s["rng_seed"] % 2 ** 32, s["rng_seed"] // 2 ** 32]
    for r in range(7):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((p1 >> 32) & LOW) ^ x[1] ^ ((key[0] + r * 0x9E3779B9) % 2 ** 32), p1 & LOW,
             ((p0 >> 32) & LOW) ^ x[3] ^ ((key[1] + r * 0xBB67AE85) % 2 ** 32), p0 & LOW]
    word = torch.where(lane < 4, torch.where(lane < 2, x[0], x[1]), torch.where(lane < 6, x[2], x[3]))
    number = (word >> (16 * (lane % 2))) % 65536
    return (number >= t).double() * (65536 / (65536 - t))


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def forward64(x, gamma, beta, s):
    """Rows of one group each: [n * groups, pixels * channels of a group]."""
    n, p, g, d = s["n"], s["h"] * s["w"], s["groups"], s["c"] // s["groups"]
    rows = x.reshape(n, p, g, d).transpose(1, 2).reshape(n * g, p * d)
    mean = rows.sum(1) / (p * d)
    rows = rows - mean[:, None]
    rstd = ((rows ** 2).sum(1) / (p * d) + EPS) ** -0.5
    rows = rows * rstd[:, None]
    y = act64(rows.view(n, g, p, d).transpose(1, 2).reshape(n, p, g * d) * gamma + beta, s["act"])
    if s["p"]:
        y = y * kept64(y.numel(), s, y.device).view(y.shape)
    return y.view(n, s["h"], s["w"], s["c"]), mean.view(n, g), rstd.view(n, g)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "dropout":
        y = x * kept64(x.numel(), s, x.device).view(x.shape)
        return y + s["residual_in"].double() if case["residual"] else y
    gamma, beta = s["gamma"].double(), s["beta"].double()
    if case["op"] == "norm":
        y, mean, rstd = forward64(x, gamma, beta, s)
        return {"y": y, "mean": mean, "rstd": rstd}
    for leaf in (x, gamma, beta):
        leaf.requires_grad_(True)
    with torch.enable_grad():
        y, _, _ = forward64(x, gamma, beta, s)
        dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
