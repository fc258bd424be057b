"""``fused_group_norm_act`` against its definition in float64."""
import numpy as np
import pytest
import torch

from oracle import norm_act as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RNG = (0x123456789ABCDEF0, 12)


def _make(lengths, C, dtype, seed, shift=0.5, rows_behind=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    N = sum(lengths) + rows_behind
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)
    x = (rand(N, C) * (0.5 + torch.rand(C, device=DEV, generator=g)) + shift * rand(C)).to(dtype)
    return dict(x=x, weight=1 + 0.3 * rand(C), bias=0.3 * rand(C), residual=rand(N, C).to(dtype), grad=rand(N, C).to(dtype))


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _run(t, lengths, groups, act, p=0.0, rng=RNG, affine=True, residual=True, eps=1e-5):
    from pointelligence_b200.layers.norm import fused_group_norm_act

    leaves = {k: t[k].detach().requires_grad_() for k in ("x",) + (("weight", "bias") if affine else ()) + (("residual",) if residual else ())}
    y = fused_group_norm_act(leaves["x"], torch.tensor(lengths, device=DEV), groups, leaves.get("weight"), leaves.get("bias"), eps,
                             residual=leaves.get("residual"), activation=act, dropout=p, rng=rng if p else None)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["grad"])))
    return y.detach(), grads


def _check(t, lengths, groups, act, p=0.0, affine=True, residual=True, got=None):
    """Bounds, element by element.  u = 2^-24 is a rounding of fp32, U one of the type.  z takes the roundings of x - mu (and of mu), of
    the product and the sums, and the relative error of rstd, which is half that of a sum of squares: a chunk's is folded from
    chains of at most 64 terms and trees, so 2^7 u covers it with the rest: dz = 2^-17 (|xh w| + |b| + |res| + |mu| rstd |w|).  Slopes of
    the activations are at most 1.13 and bend by at most 0.8, their values by exp within 4 u: y moves by 2 dz scale, gz by
    (dz + 2^-17) |g| scale, and the means over a group by the largest of those."""
    y, grads = got or _run(t, lengths, groups, act, p, affine=affine, residual=residual)
    lens = list(lengths)
    lens[-1] += t["x"].shape[0] - sum(lens)     # rows behind the last sample are its own
    want = oracle.group_norm_act(_f64(t["x"]), lens, groups, _f64(t["weight"]) if affine else None, _f64(t["bias"]) if affine else None, 1e-5,
                                 _f64(t["residual"]) if residual else None, act, p, RNG, _f64(t["grad"]))
    U, e, scale = oracle.EPS_OF[str(y.dtype).split(".")[1]], 2.0 ** -17, 1 / (1 - p) if p < 1 else 1.0
    w, b = (np.abs(_f64(t["weight"])), np.abs(_f64(t["bias"]))) if affine else (1.0, 0.0)
    x, g = np.abs(_f64(t["x"])), np.abs(_f64(t["grad"]))
    dz = e * (1 + np.abs(want["xh"]) * w + b + (np.abs(_f64(t["residual"])) if residual else 0) + 2 * x * want["rstd"] * w)
    settled = np.abs(want["z"]) > dz if act == "relu" else np.ones_like(dz, bool)
    tiny = 2.0 ** -24 if y.dtype == torch.float16 else 0.0      # below the normal numbers of fp16 steps are absolute

    def close(name, a, ref, bound):
        off = np.abs(_f64(a) - ref) - (U * np.abs(ref) * (1 + e) + bound + tiny)
        worst = np.unravel_index(np.argmax(np.where(settled, off, -1) if off.shape == settled.shape else off), off.shape) if off.size else None
        assert worst is None or off[worst] <= 0 or not (settled[worst] if off.shape == settled.shape else True), (name, worst, _f64(a)[worst], ref[worst])

    close("y", y, want["y"], 2 * dz * scale)
    dgz = (dz + e) * g * scale
    xh = np.abs(want["xh"]) + 1
    close("dx", grads["x"], want["dx"], want["rstd"] * (w * dgz + 2 * xh * (w * dgz).max(initial=0) * xh.max(initial=0) + e * (np.abs(want["gh"]) + np.abs(want["m1"]) + np.abs(want["m2"]) * xh)))
    if residual:
        close("dresidual", grads["residual"], want["dresidual"], dgz)
    if affine:   # (summed in 32 bits, returned in them)
        # a sign that the ReLU's argument does not settle moves a sum by its term
        loose = np.where(settled, 0, g * scale)
        for name, ref, bound in (("bias", want["db"], dgz + e * np.abs(want["dresidual"]) + loose),
                                 ("weight", want["dw"], (dgz + e * np.abs(want["dresidual"]) + loose) * xh)):
            off = np.abs(_f64(grads[name]) - ref) - bound.sum(0) - 1e-30
            assert off.max(initial=-1) <= 0, (name, off.max())
    return y, grads


SHAPES = [([1], 8, 1), ([1], 8, 8), ([2], 6, 3), ([3, 0, 5], 24, 4), ([0, 700, 0, 0, 33, 1], 64, 8), ([3000, 1, 5000, 300, 0, 17], 48, 16),
          ([5000, 1, 8000], 20, 20), ([1234, 4321], 50, 5), ([777], 33, 11), ([300, 500], 2048, 32), ([17, 4], 2056, 8), ([2] * 700, 32, 4),
          ([129, 0, 64], 96, 1), ([9000], 3, 1)]


@pytest.mark.parametrize("lengths,C,groups", SHAPES, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,p", [("silu", 0.0), ("relu", 0.3)])
def test_against_the_definition(lengths, C, groups, dtype, act, p):
    _check(_make(lengths, C, dtype, sum(lengths) + C), lengths, groups, act, p)


@pytest.mark.parametrize("act", ["identity", "relu", "silu", "gelu"])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
def test_every_tail(act, affine, residual, p):
    lengths = [400, 0, 1, 700]
    _check(_make(lengths, 40, torch.bfloat16, 7), lengths, 5, act, p, affine, residual)


@pytest.mark.parametrize("C", [1, 2, 4, 5, 12, 100, 257, 300, 1000, 4100])
def test_widths(C):
    lengths = [50, 31]
    _check(_make(lengths, C, torch.float32, C), lengths, C if C % 2 else C // 2, "gelu", 0.2)


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses_and_strides(offset, dtype):
    """Rows that do not begin at 16 bytes, in every tensor; and a column slice, which is copied."""
    lengths = [300, 45]
    t = _make(lengths, 32, dtype, offset)
    moved = {}
    for k, v in t.items():
        if v.dim() == 2:
            flat = torch.zeros(v.numel() + offset, dtype=dtype, device=DEV)
            flat[offset:] = v.reshape(-1)
            moved[k] = flat[offset:].view(v.shape)
        else:
            moved[k] = v
    _check(moved, lengths, 4, "silu", 0.25)
    wide = {k: torch.cat([v, v], 1)[:, 16:48] if v.dim() == 2 else v for k, v in t.items()}
    assert not wide["x"].is_contiguous()
    _check(wide, lengths, 4, "relu")


def test_rows_behind_the_last_sample_are_its_own():
    lengths = [100, 60]
    _check(_make(lengths, 16, torch.float32, 3, rows_behind=40), lengths, 4, "silu")


@pytest.mark.parametrize("lengths", [[90, 1000, 5], [-7, 130], [0, 0, 0], [2 ** 62, 2 ** 62, 3]])
def test_lengths_that_are_not_the_rows(lengths):
    """They are taken within the rows there are."""
    t = _make([130], 16, torch.float32, 3)
    real, left = [], 130
    for v in lengths:
        real.append(min(max(v, 0), left))
        left -= real[-1]
    real[-1] += left
    _check(t, real, 2, "silu", got=_run(t, lengths, 2, "silu"))


def test_far_from_zero_and_constant():
    """A mean that is 2000 times the spread; rows that are all alike; a first row that is far from the others."""
    lengths = [2000, 500, 900]
    t = _make(lengths, 32, torch.float32, 1)
    t["x"] = t["x"] + 2000
    t["x"][2000:2500] = 7.0
    t["x"][2500] = 1e4
    _check(t, lengths, 4, "silu")


def test_not_a_number_stays_in_its_group():
    lengths = [200, 300, 10]
    t = _make(lengths, 32, torch.float32, 1)
    t["x"][250, 9] = float("inf")
    t["x"][505, 3] = float("nan")
    y, grads = _run(t, lengths, 4, "relu")
    bad = torch.zeros(510, 32, dtype=torch.bool, device=DEV)
    bad[200:500, 8:16] = True
    bad[500:, :8] = True
    assert torch.equal(y.isnan(), bad)
    assert torch.equal(grads["x"].isnan(), bad)
    clean = {k: v.clone() for k, v in t.items()}
    clean["x"][250, 9] = 0.0
    clean["x"][505, 3] = 0.0
    z, dz = _run(clean, lengths, 4, "relu")
    assert torch.equal(y[~bad], z[~bad]) and torch.equal(grads["x"][~bad], dz["x"][~bad])


def test_dropped_elements_are_zero_whatever_they_were():
    t = _make([64], 16, torch.float32, 1)
    t["residual"][:] = float("nan")
    t["grad"][:] = float("inf")
    y, grads = _run(t, [64], 4, "identity", 1.0)
    assert not y.any() and not any(g.any() for g in grads.values())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_every_time(dtype):
    lengths = [20000, 3, 40000, 0, 999]
    t = _make(lengths, 64, dtype, 5)
    first = _run(t, lengths, 8, "silu", 0.1)
    for _ in range(3):
        y, grads = _run(t, lengths, 8, "silu", 0.1)
        assert torch.equal(y, first[0]) and all(torch.equal(grads[k], first[1][k]) for k in grads)


def test_mask_is_that_of_the_dropout_alone():
    from pointelligence_b200.layers.dropout import fused_dropout

    lengths = [500, 77]
    for C, dtype in ((64, torch.bfloat16), (33, torch.float32), (20, torch.float16)):
        t = _make(lengths, C, dtype, C)
        y, _ = _run(t, lengths, C, "identity", 0.4)
        kept = fused_dropout(torch.ones(577, C, device=DEV), 0.4, rng=RNG) != 0
        assert not y[~kept].any() and y[kept].ne(0).float().mean() > 0.99


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_against_differences(act):
    """Central differences in float64 of the definition, along a direction: the formula's own gradient first, then the kernel's."""
    lengths, C, groups = [40, 9], 12, 3
    t = _make(lengths, C, torch.float32, 11)
    _, grads = _run(t, lengths, groups, act, 0.3)
    g = np.random.default_rng(0)
    names = ["x", "weight", "bias", "residual"]
    arrays = {k: _f64(t[k]) for k in names}
    value = lambda a: (oracle.group_norm_act(a["x"], lengths, groups, a["weight"], a["bias"], 1e-5, a["residual"], act, 0.3, RNG, _f64(t["grad"]))["y"] * _f64(t["grad"])).sum()
    for k in names:
        d = g.standard_normal(arrays[k].shape)
        h = 1e-5
        up, down = ({**arrays, k: arrays[k] + s * h * d} for s in (1, -1))
        want = (value(up) - value(down)) / (2 * h)
        got = (_f64(grads[k]) * d).sum()
        # differences: h^2 of the third derivative and 1e-16 / h of rounding; the kernel: 2^-17 of terms of size one
        assert abs(got - want) <= 2e-5 * (np.abs(_f64(grads[k]) * d).sum() + 1), k


def test_without_points_and_statistics_of_empty_samples():
    for lengths in ([0], [0, 0, 0]):
        t = _make(lengths, 16, torch.float32, 0)
        y, grads = _run(t, lengths, 4, "silu")
        assert y.shape == (0, 16) and not grads["weight"].any() and not grads["bias"].any()


def test_only_what_is_asked_for():
    """Gradients of some of the inputs; parameters of 16 bits; int32 lengths; no gradient at all."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    lengths = [100, 50]
    t = _make(lengths, 32, torch.bfloat16, 2)
    full, grads = _run(t, lengths, 4, "silu")
    lens = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    for names in (["x"], ["weight"], ["bias"], ["residual"], ["bias", "residual"]):
        leaves = {k: t[k].detach().requires_grad_(k in names) for k in ("x", "weight", "bias", "residual")}
        y = fused_group_norm_act(leaves["x"], lens, 4, leaves["weight"], leaves["bias"], residual=leaves["residual"])
        assert torch.equal(y, full)
        for k, g in zip(names, torch.autograd.grad(y, [leaves[k] for k in names], t["grad"])):
            assert torch.equal(g, grads[k]), k
    with torch.no_grad():
        half = fused_group_norm_act(t["x"], lens, 4, t["weight"].bfloat16(), t["bias"].bfloat16(), residual=t["residual"].float())
        same = fused_group_norm_act(t["x"], lens, 4, t["weight"].bfloat16().float(), t["bias"].bfloat16().float(), residual=t["residual"])
        assert not half.requires_grad and torch.equal(half, same)
    w = t["weight"].bfloat16().requires_grad_()
    g, = torch.autograd.grad(fused_group_norm_act(t["x"], lens, 4, w, t["bias"]), w, t["grad"])
    assert g.dtype == torch.bfloat16


def test_another_stream_and_a_captured_step():
    """Forward and backward on a side stream, and captured: each replay draws a new mask, which its backward pass takes too."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    lengths = torch.tensor([3000, 900], device=DEV)
    t = _make([3000, 900], 64, torch.bfloat16, 9)
    leaves = [t[k].detach().requires_grad_() for k in ("x", "weight", "bias")]
    step = lambda: (lambda y: (y.detach(),) + torch.autograd.grad(y, leaves, t["grad"]))(
        fused_group_norm_act(leaves[0], lengths, 8, leaves[1], leaves[2], activation="identity", dropout=0.5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append([v.clone() for v in out])
        kept = seen[-1][0] != 0
        assert 0.48 < kept.float().mean() < 0.52
        # the bias's gradient is the sum of what was kept: the backward pass took the same mask
        want = (t["grad"].double() * kept * 2).sum(0)
        assert float((seen[-1][3].double() - want).norm() / want.norm()) < 1e-4
    assert not torch.equal(seen[0][0] != 0, seen[1][0] != 0) and not torch.equal(seen[1][0] != 0, seen[2][0] != 0)


def test_seeds_follow_the_generator():
    from pointelligence_b200.layers.norm import fused_group_norm_act

    t = _make([500], 32, torch.bfloat16, 9)
    call = lambda rng=None: fused_group_norm_act(t["x"], torch.tensor([500], device=DEV), 8, dropout=0.5, rng=rng)
    torch.manual_seed(5)
    a, b = call(), call()
    torch.manual_seed(5)
    assert torch.equal(a, call()) and torch.equal(b, call()) and not torch.equal(a, b)
    pair = torch.tensor([-3, 8], device=DEV)
    assert torch.equal(call(pair), call((-3, 8))) and torch.equal(call((-3, 8)), call((2 ** 64 - 3, 8)))


def test_seed_that_is_written_before_the_backward_pass_is_noticed():
    from pointelligence_b200.layers.norm import fused_group_norm_act

    t = _make([50], 32, torch.bfloat16, 9)
    x, pair = t["x"].requires_grad_(), torch.tensor([1, 8], device=DEV)
    y = fused_group_norm_act(x, torch.tensor([50], device=DEV), 8, dropout=0.5, rng=pair)
    pair += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last sample of a long batch is what it is alone (no dropout: that goes by the place in the batch)."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    C, tail = 64, 3001
    N = 2 ** 32 // C + tail
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(N, C, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=g)
    w, b = torch.randn(C, device=DEV, generator=g), torch.randn(C, device=DEV, generator=g)
    lengths = torch.tensor([N - tail - 5, 5, tail], device=DEV)
    go = torch.zeros_like(x)
    go[-tail:].normal_(generator=g)
    x.requires_grad_()
    y = fused_group_norm_act(x, lengths, 8, w, b)
    dx, = torch.autograd.grad(y, x, go)
    alone = x.detach()[-tail:].clone().requires_grad_()
    y1 = fused_group_norm_act(alone, torch.tensor([tail], device=DEV), 8, w, b)
    dx1, = torch.autograd.grad(y1, alone, go[-tail:])
    # pieces are cut at other rows: statistics differ by roundings of 32 bits, results by one of 16
    assert float((y.detach()[-tail:].double() - y1.detach().double()).norm() / y1.detach().double().norm()) < 2.0 ** -9
    assert float((dx[-tail:].double() - dx1.double()).norm() / dx1.double().norm()) < 2.0 ** -9
    assert not dx[:-tail].any()
