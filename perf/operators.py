"""Performance cases of the norm, activation and dropout passes of a residual block on ragged batches.

A case is one call through the public entry points, for training with the gradients of everything it takes:

``norm``     ``fused_group_norm_act``: group norm per sample of the batch (one group: layer norm; as many groups as channels:
             instance norm), a residual, an activation, and with ``p`` > 0 dropout by element, in one operator
``dropout``  ``fused_dropout``: dropout of elements, of whole channels of a sample or of whole samples (drop path), with the
             residual and the ReLU of a block's tail

The random words come from a seed and an offset that are part of the input: word ``u % 8`` (16 bits, low halves first) of
Philox4x32-10 with the counter (u / 8, offset) and the seed as key decides for element, channel or sample ``u``; it is kept
where the word is at least ``round(65536 p)``, and then scaled by 65536 / (65536 - round(65536 p)).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
MOST_ELEMENTS = 1_100_003 * 64     # of a drawn case, in 16 bits; half of it in 32


def listed():
    return [
        # serving: the deepest stage of one small scene; a call that is bound by latency
        dict(name="norm_infer_deep", kind="norm", points=942, samples=1, empty=False, c=256, groups=32, act="silu", residual=False,
             p=0.0, dtype="bf16", train=False),
        # serving: a block's tail on a whole room
        dict(name="norm_infer_200k_c96", kind="norm", points=200000, samples=1, empty=False, c=96, groups=8, act="relu", residual=True,
             p=0.0, dtype="bf16", train=False),
        # full-precision training of a first experiment; five groups of ten channels, rows that are no multiple of 16 bytes
        dict(name="norm_train_fp32_20k_c50", kind="norm", points=20000, samples=2, empty=True, c=50, groups=5, act="silu",
             residual=False, p=0.0, dtype="fp32", train=True),
        # a middle stage in training: one group, the layer norm, with a residual
        dict(name="norm_train_80k_c128", kind="norm", points=80001, samples=4, empty=False, c=128, groups=1, act="gelu", residual=True,
             p=0.0, dtype="fp16", train=True),
        # object classification: hundreds of small clouds, instance norm
        dict(name="norm_train_objects_c64", kind="norm", points=400000, samples=400, empty=True, c=64, groups=64, act="silu",
             residual=False, p=0.0, dtype="bf16", train=True),
        # the training batch behind the first stage: eight rooms, a block's tail
        dict(name="norm_train_1m_c64", kind="norm", points=1100003, samples=8, empty=False, c=64, groups=8, act="relu", residual=True,
             p=0.0, dtype="bf16", train=True),
        # the same batch between a block's convolutions: activation and dropout in the norm's pass
        dict(name="norm_drop_train_1m_c64", kind="norm", points=1100003, samples=8, empty=False, c=64, groups=8, act="silu",
             residual=False, p=0.1, dtype="bf16", train=True),
        # a deep stage with strong dropout, small enough that launches count
        dict(name="norm_drop_train_5k_c256", kind="norm", points=5000, samples=8, empty=False, c=256, groups=32, act="gelu",
             residual=False, p=0.5, dtype="fp16", train=True),
        # dropout in front of the classifier of the network, training
        dict(name="dropout_train_1m_c96", kind="dropout", points=730000, samples=8, empty=False, c=96, unit="element", residual=False,
             relu=False, p=0.5, dtype="bf16", train=True),
        # a small full-precision layer
        dict(name="dropout_train_fp32_5k_c48", kind="dropout", points=5000, samples=1, empty=False, c=48, unit="element",
             residual=False, relu=False, p=0.2, dtype="fp32", train=True),
        # drop path over a block's branch: residual and ReLU of the tail
        dict(name="drop_path_train_500k_c64", kind="dropout", points=500000, samples=16, empty=False, c=64, unit="sample",
             residual=True, relu=True, p=0.3, dtype="bf16", train=True),
        # feature dropout on rows that are no multiple of 16 bytes
        dict(name="channel_drop_train_80k_c20", kind="dropout", points=80001, samples=3, empty=True, c=20, unit="channel",
             residual=False, relu=False, p=0.25, dtype="fp16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choices(["bf16", "fp16", "fp32"], [5, 2, 3])[0]
    c = rng.choice([6, 20, 32, 33, 48, 50, 64, 96, 100, 128, 192, 256, 384, 512])
    points = _log(rng, 200, min(1_100_000, MOST_ELEMENTS // (c * (2 if dtype == "fp32" else 1))))
    samples = rng.choice([1, 1, 2, 4, 8, max(1, points // 1000)])
    case = dict(points=points, samples=samples, empty=rng.random() < 0.3, c=c, dtype=dtype, train=rng.random() < 0.7)
    p = rng.choice([0.05, 0.1, 0.3, 0.5, 0.9])
    if rng.random() < 0.35:
        residual = rng.random() < 0.5
        # (a sum of 32 bits next to the border of the ReLU is settled by its last bit: 16 bits there)
        return dict(kind="dropout", unit=rng.choice(["element", "element", "channel", "sample"]), residual=residual,
                    relu=residual and dtype != "fp32" and rng.random() < 0.5, p=p, **case)
    groups = rng.choice([g for g in (1, 2, 3, 4, 5, 8, 10, 16, 25, 32, c) if c % g == 0])
    act = rng.choice(["silu", "gelu", "identity"] + (["relu", "relu"] if dtype != "fp32" else []))
    return dict(kind="norm", groups=groups, act=act, residual=rng.random() < 0.4, p=p if rng.random() < 0.4 else 0.0, **case)


# ------------------------------------------------------------------ inputs ----
def _lengths(case):
    """Ragged sizes, between 0.6 and 1.4 times the mean; with ``empty`` one cloud in the middle has no points."""
    n, s = case["points"], case["samples"]
    w = [0.6 + 0.8 * ((b * 0.618) % 1.0) for b in range(s)]
    sizes = [int(n * v / sum(w)) for v in w]
    sizes[0] += n - sum(sizes)
    if case["empty"]:
        sizes.insert(s // 2, 0)
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, c, dtype = case["points"], case["c"], DTYPES[case["dtype"]]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    state = dict(case=case, lengths=torch.tensor(_lengths(case), device="cuda"))
    # channels of a convolution: each with a mean and a spread of its own
    x = rand(n, c).mul_(0.5 + torch.rand(c, generator=gen, device="cuda")).add_(0.5 * rand(c))
    state["x"] = x.to(dtype)
    if case["residual"]:
        state["residual"] = rand(n, c).to(dtype)
    if case["kind"] == "norm":
        state["weight"], state["bias"] = 1 + 0.2 * rand(c), 0.2 * rand(c)
    if case["train"]:
        state["grad"] = rand(n, c).to(dtype)
        for name in ("x", "residual", "weight", "bias"):
            if name in state:
                state[name].requires_grad_()
    state["rng"] = (0x9E3779B97F4A7C15 ^ (seed * 0x10001), 4 * seed + 4)
    return state


# ------------------------------------------------------------- plain forms ----
def _words(units, rng, device):
    """16-bit random words of ``units`` units: Philox4x32-10 in 64-bit integers (products wrap; their halves come out right)."""
    low = 0xFFFFFFFF
    seed, offset = rng
    at = torch.arange((units + 7) // 8, device=device)
    a, b = at & low, at >> 32
    c, d = torch.full_like(at, offset & low), torch.full_like(at, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ d ^ k1, p & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([a, b, c, d], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:units]


def _factor(units, p, rng, device):
    """What dropout multiplies each unit by."""
    t = int(math.floor(65536 * p + 0.5))
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    return torch.where(_words(units, rng, device) >= t, scale, 0.0).float()


def _sample_of(lengths, n):
    return torch.repeat_interleave(torch.arange(lengths.numel(), device=lengths.device), lengths, output_size=n)


def _per_sample(v, sample, samples):
    """Sums of rows by sample, in 64 bits: long sums."""
    return torch.zeros(samples, *v.shape[1:], dtype=torch.float64, device=v.device).index_add_(0, sample, v.double())


def _act(z, kind):
    """The activation and its derivative."""
    if kind == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_norm(s):
    case, x, w, b, lengths = s["case"], s["x"].detach(), s["weight"].detach(), s["bias"].detach(), s["lengths"]
    (n, c), g, dtype, S = x.shape, case["groups"], x.dtype, lengths.numel()
    sample = _sample_of(lengths, n)
    rows = x.float().view(n, g, c // g)
    count = (lengths * (c // g)).clamp_min(1)[:, None].double()
    mean = _per_sample(rows.sum(2, dtype=torch.float64), sample, S) / count
    # the sign of what the ReLU takes is that of 64 bits
    xc = rows.double() - mean[sample][:, :, None] if case["act"] == "relu" else rows - mean.float()[sample][:, :, None]
    rstd = torch.rsqrt(_per_sample(xc.square().sum(2, dtype=torch.float64), sample, S) / count + EPS).to(xc.dtype)[sample][:, :, None]
    xh = xc * rstd
    z = xh.view(n, c) * w + b
    if case["residual"]:
        z = z + s["residual"].detach()
    y, slope = _act(z, case["act"])
    keep = _factor(n * c, case["p"], s["rng"], x.device).view(n, c) if case["p"] else None
    if keep is not None:
        y = y * keep
    out = {"y": y.to(dtype)}
    if case["train"]:
        gz = s["grad"].float() * slope
        if keep is not None:
            gz = gz * keep
        xh_rows = xh.reshape(n, c)
        out["db"], out["dw"] = gz.sum(0, dtype=torch.float64).float(), (gz * xh_rows).sum(0, dtype=torch.float64).float()
        gh = (gz * w).view(n, g, c // g)
        m1 = (_per_sample(gh.sum(2, dtype=torch.float64), sample, S) / count).float()[sample][:, :, None]
        m2 = (_per_sample((gh * xh).sum(2, dtype=torch.float64), sample, S) / count).float()[sample][:, :, None]
        out["dx"] = (rstd * (gh - m1 - xh * m2)).view(n, c).to(dtype)
        if case["residual"]:
            out["dresidual"] = gz.to(dtype)
    return out


def _plain_dropout(s):
    case, x, lengths = s["case"], s["x"].detach(), s["lengths"]
    n, c = x.shape
    if case["unit"] == "element":
        keep = _factor(n * c, case["p"], s["rng"], x.device).view(n, c)
    elif case["unit"] == "channel":
        keep = _factor(lengths.numel() * c, case["p"], s["rng"], x.device).view(-1, c)[_sample_of(lengths, n)]
    else:
        keep = _factor(lengths.numel(), case["p"], s["rng"], x.device)[_sample_of(lengths, n)][:, None]
    y = x.float() * keep
    if case["residual"]:
        y = y + s["residual"].detach().float()
    out = {"y": (y.clamp_min(0) if case["relu"] else y).to(x.dtype)}
    if case["train"]:
        g = s["grad"].float()
        if case["relu"]:
            g = g * (y > 0)
        out["dx"] = (g * keep).to(x.dtype)
        if case["residual"]:
            out["dresidual"] = g.to(x.dtype)
    return out


def run(state):
    case = state["case"]
    if not own:
        return _plain_norm(state) if case["kind"] == "norm" else _plain_dropout(state)
    from pointelligence_b200.layers.dropout import fused_dropout
    from pointelligence_b200.layers.norm import fused_group_norm_act

    x, residual = state["x"], state.get("residual")
    with torch.set_grad_enabled(case["train"]):
        if case["kind"] == "norm":
            y = fused_group_norm_act(x, state["lengths"], case["groups"], state["weight"], state["bias"], EPS, residual=residual,
                                     activation=case["act"], dropout=case["p"], rng=state["rng"] if case["p"] else None)
        else:
            y = fused_dropout(x, case["p"], rng=state["rng"], unit=case["unit"], lengths=state["lengths"], residual=residual,
                              relu=case["relu"])
    out = {"y": y.detach()}
    if case["train"]:
        names = {"dx": "x", "dresidual": "residual", "dw": "weight", "db": "bias"}
        names = {k: v for k, v in names.items() if v in state}
        out.update(zip(names, torch.autograd.grad(y, [state[v] for v in names.values()], state["grad"])))
    return out


def work(case):
    elements = case["points"] * case["c"]
    tensors = 2.0 + case["residual"]                    # x, residual, y
    if case["train"]:
        tensors += 2 + case["residual"]                 # the gradients: of y; of x, of the residual
    norm = case["kind"] == "norm"
    if not norm and case["unit"] == "sample":
        # rows of a dropped sample need not be read: x, or the gradient where no residual takes it
        tensors -= case["p"] * (1 + (case["train"] and not case["residual"]))
    flops = (8 + (16 if case["train"] else 0)) if norm else (2 + (2 if case["train"] else 0))
    if case["p"] and (norm or case["unit"] == "element"):
        flops += 8                                      # a generator call of 60 operations for eight elements
    return {"bytes": tensors * elements * BYTES[case["dtype"]] + (16.0 * case["c"] if norm else 0.0), "flops": float(flops * elements)}


# ---------------------------------------------------- the definition in 64 bits ----
def _kept(units, p, rng):
    """True where a unit is kept, on the host, in unsigned integers."""
    at = np.arange(-(-units // 8), dtype=np.uint64)
    mask = np.uint64(0xFFFFFFFF)
    ctr = [at & mask, at >> np.uint64(32), np.full_like(at, rng[1] % 2 ** 32), np.full_like(at, rng[1] // 2 ** 32 % 2 ** 32)]
    key = [rng[0] % 2 ** 32, rng[0] // 2 ** 32 % 2 ** 32]
    for r in range(10):
        left, right = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        ctr = [(right >> np.uint64(32)) ^ ctr[1] ^ k[0], right & mask, (left >> np.uint64(32)) ^ ctr[3] ^ k[1], left & mask]
    words = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)[:units]
    return words >= round(65536 * p)


def exact(case, seed):
    s = prepare(case, seed)
    lengths, n, c, dev = _lengths(case), case["points"], case["c"], s["x"].device
    leaf = {k: s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "residual", "weight", "bias") if k in s}
    scale = 65536 / (65536 - round(65536 * case["p"]))
    keep = lambda units: torch.from_numpy(_kept(units, case["p"], s["rng"])).to(dev).double() * scale
    parts = torch.split(leaf["x"], lengths)
    if case["kind"] == "norm":
        normed = []
        for part in parts:
            v = part.reshape(len(part), case["groups"], c // case["groups"])
            if len(part):
                var, mean = torch.var_mean(v, dim=(0, 2), correction=0, keepdim=True)
                v = (v - mean) / torch.sqrt(var + EPS)
            normed.append(v.reshape(len(part), c))
        z = torch.cat(normed) * leaf["weight"] + leaf["bias"]
        if case["residual"]:
            z = z + leaf["residual"]
        y = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "identity": lambda v: v}[case["act"]](z)
        if case["p"]:
            y = y * keep(n * c).view(n, c)
    else:
        if case["unit"] == "element":
            y = leaf["x"] * keep(n * c).view(n, c)
        else:
            factors = keep(len(lengths) * (c if case["unit"] == "channel" else 1)).view(len(lengths), -1)
            y = torch.cat([part * f for part, f in zip(parts, factors)])
        if case["residual"]:
            y = y + leaf["residual"]
        if case["relu"]:
            y = torch.relu(y)
    out = {"y": y.detach()}
    if case["train"]:
        names = {"dx": "x", "dresidual": "residual", "dw": "weight", "db": "bias"}
        names = {k: v for k, v in names.items() if v in leaf}
        out.update(zip(names, torch.autograd.grad(y, [leaf[v] for v in names.values()], s["grad"].double())))
    return out
