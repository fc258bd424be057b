"""What the activation of ``fused_group_norm_act`` is given, and its signs, where means are far from zero beside the deviation."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step


def _definition(x, lengths, G, w, b, res, eps=1e-5):
    """mean, rstd (rows, C), xh and the argument, in float64."""
    parts = []
    for rows in torch.split(x.double(), lengths):
        v = rows.view(len(rows), G, -1)
        m = v.mean((0, 2), keepdim=True)
        r = torch.rsqrt((v - m).square().mean((0, 2), keepdim=True) + eps)
        parts.append([t.expand_as(v).reshape(len(rows), -1) for t in (m, r, (v - m) * r)])
    mean, rstd, xh = (torch.cat(t) for t in zip(*parts))
    return mean, rstd, xh, xh * w.double() + b.double() + (0 if res is None else res.double())


@pytest.mark.parametrize("far", [1.0, 50.0, 2000.0])
@pytest.mark.parametrize("C,G", [(64, 8), (50, 50), (1032, 4)])
@pytest.mark.parametrize("residual", [False, True])
def test_far_from_zero(far, C, G, residual):
    """Rows of 32 bits.  xc = x - mu and a = rstd w are each a rounding, their product with b another, the residual one more: 2^-24 of
    2 |xh w| + |b| + |t| + |z| with t = xh w + b, whatever the mean; b has the mean's rest in it, 2^-24 of |mean rstd w|.  dx has the
    roundings of its three terms and of the sums, which are means of n terms in 32 bits: 2^-24 of 16 of each."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    lengths = [4000, 1, 900]
    g = torch.Generator(device=DEV).manual_seed(C)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    N = sum(lengths)
    x = (rand(N, C) + far).requires_grad_()
    w, b = (1 + 0.2 * rand(C)).requires_grad_(), (0.2 * rand(C)).requires_grad_()
    res = rand(N, C) if residual else None
    go = rand(N, C)
    y = fused_group_norm_act(x, torch.tensor(lengths, device=DEV), G, w, b, residual=res, activation="identity")
    dx, dw = torch.autograd.grad(y, (x, w), go)
    mean, rstd, xh, z = _definition(x.detach(), lengths, G, w.detach(), b.detach(), res)
    wd, bd, e = w.detach().double(), b.detach().double(), 2.0 ** -24
    t = xh * wd + bd
    rest = e * (mean * rstd * wd).abs()
    bound = e * (2 * (xh * wd).abs() + bd.abs() + rest + t.abs() + 2 * z.abs()) * (1 + 2 ** -20)
    assert bool(((y.detach().double() - z).abs() <= bound).all())
    gh = go.double() * wd
    want = []
    for rows in zip(torch.split(gh, lengths), torch.split(xh, lengths), torch.split(rstd, lengths)):
        h, v, r = (q.view(len(q), G, -1) for q in rows)
        m1, m2 = h.mean((0, 2), keepdim=True), (h * v).mean((0, 2), keepdim=True)
        s1, s2 = h.abs().mean((0, 2), keepdim=True), (h * v).abs().mean((0, 2), keepdim=True)
        want.append([(r * (h - m1 - v * m2)).reshape(len(h), -1), (r * (h.abs() + s1 + v.abs() * s2)).reshape(len(h), -1)])
    want, size = (torch.cat(q) for q in zip(*want))
    assert bool(((dx.double() - want).abs() <= 16 * e * size).all())
    dw_want, dw_size = (go.double() * xh).sum(0), (go.double() * xh).abs().sum(0)
    assert bool(((dw.double() - dw_want).abs() <= 16 * e * dw_size).all())


def _at_the_border(lengths, C, G, dtype, residual, seed):
    """Values of a few steps of the type, as layers of 16 bits have them, and a bias that puts one of them, a few rows in a hundred,
    on the border of the ReLU, so near that 32 bits do not tell on which side: z is what the bias's rounding leaves."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    N = sum(lengths)
    values = torch.tensor([0.0, 1.0, -2.0, 0.5, 3.0, -0.75, 100.0], device=DEV)
    x = values[torch.randint(0, 7, (N, C), generator=g, device=DEV)].to(dtype)
    res = values[torch.randint(0, 3, (N, C), generator=g, device=DEV)].to(dtype) if residual else None
    w = 1 + 0.2 * torch.randn(C, generator=g, device=DEV)
    zero = torch.zeros(C, device=DEV)
    _, _, xh, _ = _definition(x, lengths, G, w, zero, None)
    at = torch.arange(C, device=DEV) % 7       # the value that is on the border, in the batch's first sample
    first = x[:lengths[0]].float()
    row = (first == values[at].to(dtype).float()).int().argmax(0)
    b = -(xh[row, torch.arange(C, device=DEV)] * w.double())
    if residual:
        b = b - values[1].double()             # with a residual of one
    return x, res, w, b.float()


@pytest.mark.parametrize("C,G,lengths", [(64, 8, [3001, 700]), (64, 64, [20000]), (50, 5, [3001, 3, 700]), (33, 1, [2500, 1]), (1032, 4, [900, 80]), (256, 256, [5000, 9])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("residual,p", [(False, 0.0), (True, 0.0), (True, 0.3), (False, 0.3)])
def test_signs_at_the_border(C, G, lengths, dtype, residual, p):
    """Every element of the gradients of x and of the residual, and of the sums, is on the side that float64 gives it; y is the ReLU of an
    argument that is off by some 2^-22 of its terms."""
    _check_signs(C, G, lengths, dtype, residual, p, (5, 8) if p else None)


@pytest.mark.parametrize("C,G", [(8, 2), (24, 3), (100, 4), (130, 13), (512, 8), (688, 1), (1000, 5), (1024, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_signs_at_the_border_of_other_widths(C, G, dtype):
    """With a seed on the device; no wait of a kernel runs out."""
    from pointelligence_b200 import _cabi

    _check_signs(C, G, [1700, 2, 640], dtype, True, 0.3, torch.tensor([5, 8], device=DEV))
    _check_signs(C, G, [1700, 2, 640], dtype, False, 0.0, None)
    assert _cabi.device_status() == 0


def _check_signs(C, G, lengths, dtype, residual, p, rng):
    import numpy as np

    from oracle import norm_act as oracle
    from pointelligence_b200.layers.norm import fused_group_norm_act

    x, res, w, b = _at_the_border(lengths, C, G, dtype, residual, C)
    N = sum(lengths)
    go = (1 + torch.rand(N, C, device=DEV)).to(dtype)      # (no gradient is zero)
    leaves = [t.requires_grad_() for t in (x, w, b)] + ([res.requires_grad_()] if residual else [])
    y = fused_group_norm_act(x, torch.tensor(lengths, device=DEV), G, w, b, residual=res, activation="relu", dropout=p, rng=rng)
    grads = torch.autograd.grad(y, leaves, go)
    _, rstd, xh, z = _definition(x.detach(), lengths, G, w.detach(), b.detach(), None if res is None else res.detach())
    near = z.abs() < 2.0 ** -22
    assert 0.002 < float(near.double().mean())
    # (a constant row or group has z = 0 but for the order of float64's sums)
    told = z.abs() > 2.0 ** -45
    keep = torch.from_numpy(oracle.keep_factor(np.arange(N * C), p, (5, 8))).view(N, C).to(DEV) if p else torch.ones(N, C, dtype=torch.double, device=DEV)
    open_ = (z > 0) & (keep > 0)
    y_want, terms = z.clamp_min(0) * keep, (xh * w.detach().double()).abs() + b.detach().double().abs() + (0 if res is None else res.detach().double().abs())
    assert bool(((y.detach().double() - y_want).abs() <= U[dtype] * y_want + 2.0 ** -22 * terms * keep + 2.0 ** -24 * (dtype == torch.float16)).all())
    if residual:
        assert torch.equal((grads[3] != 0)[told], open_[told])
    gz = go.double() * keep * open_
    unsure = (go.double() * keep * ~told).sum(0)
    size = gz.sum(0)
    # sums of 32 bits in short chains: 16 roundings of 2^-24 of their terms, as many for each part of xh
    assert bool(((grads[2].double() - size).abs() <= 2.0 ** -20 * size + unsure).all())
    assert bool(((grads[1].double() - (gz * xh).sum(0)).abs() <= 2.0 ** -20 * (gz * xh.abs()).sum(0) + unsure * xh.abs().max()).all())
    by_group = lambda t: torch.cat([q.view(len(q), G, -1).mean((0, 2), keepdim=True).expand(len(q), G, C // G).reshape(len(q), C) for q in torch.split(t, lengths)])
    gh = gz * w.detach().double()
    dx = rstd * (gh - by_group(gh) - xh * by_group(gh * xh))
    loose = rstd * (by_group(go.double() * keep * ~told * w.detach().double().abs()) * (1 + xh.abs() * xh.abs().max()))
    bound = U[dtype] * dx.abs() + 2.0 ** -19 * rstd * (gh.abs() + by_group(gh.abs()) + xh.abs() * by_group((gh * xh).abs())) + loose + 2.0 ** -24
    assert bool(((grads[0].double() - dx).abs() <= bound)[told].all())


def _values(kind, z):
    """act(z) and its slope, in float64 on the host, from functions that are right in the tails."""
    import numpy as np
    from scipy import special

    if kind == "silu":
        s = special.expit(z)
        return z * s, s * (1 + z * special.expit(-z)), s * (1 + np.abs(z) * special.expit(-z))
    density = np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    cdf = special.ndtr(z)
    return z * cdf, cdf + z * density, cdf + np.abs(z) * density


def _activated(kind, z, dtype):
    """y and the residual's gradient for arguments z: the offsets of channels whose weight is zero."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    C = len(z)
    x = torch.randn(4, C, device=DEV).to(dtype)
    res = torch.zeros(4, C, device=DEV, dtype=dtype, requires_grad=True)
    y = fused_group_norm_act(x, torch.tensor([4], device=DEV), 8, torch.zeros(C, device=DEV), torch.tensor(z, device=DEV, dtype=torch.float32), residual=res, activation=kind)
    g, = torch.autograd.grad(y, res, torch.ones_like(y))
    return [t.detach().double().cpu().numpy() for t in (y, g)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("C", [1024, 2048])
def test_gelu_in_its_tails(dtype, C):
    """Relative to the value: 2^-20 of the approximation with the reciprocal and the exponential; the exponent z^2 / 2 is three roundings, 2^-23 z^2
    of the result.  Below -12 results leave fp32's normal numbers."""
    import numpy as np

    z = np.linspace(-12, 12, C).astype(np.float32).astype(float)
    y, g = _activated("gelu", z, dtype)
    want, slope, terms = _values("gelu", z)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    e = 2.0 ** -20 + 2.0 ** -23 * z * z
    assert (np.abs(y - want) <= (U[dtype] + e) * np.abs(want) + tiny).all()
    assert (np.abs(g - slope) <= U[dtype] * np.abs(slope) + e * terms + tiny).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("C", [1024, 2048])
def test_silu_in_its_tails(dtype, C):
    """Relative to the value: 2^-20 of the reciprocal and the exponential with its products; the exponent is two roundings, 2^-23 |z|
    of the result.  Below -86 results leave fp32's normal numbers."""
    import numpy as np

    z = np.linspace(-86, 86, C).astype(np.float32).astype(float)
    y, g = _activated("silu", z, dtype)
    want, slope, terms = _values("silu", z)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    e = 2.0 ** -20 + 2.0 ** -23 * np.abs(z)
    assert (np.abs(y - want) <= (U[dtype] + e) * np.abs(want) + tiny).all()
    assert (np.abs(g - slope) <= U[dtype] * np.abs(slope) + e * terms + tiny).all()
    y, g = _activated("silu", np.array([-1e3, -100.0, -0.0, 0.0, 100.0, 1e3, 3e4, -3e4] * 2), dtype)
    assert (y == np.array([0, 0, 0, 0, 100, 1000, float(torch.tensor(3e4).to(dtype)), 0] * 2)).all()
    assert (g == np.array([0, 0, 0.5, 0.5, 1, 1, 1, 0] * 2)).all()


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("C", [24, 25, 1032])
def test_not_a_number_stays_in_its_channel(kind, C):
    """Instance norm: what is no number in one channel leaves its neighbours as they are, in both directions."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    x = torch.randn(500, C, device=DEV).bfloat16()
    res, go = torch.randn_like(x), torch.randn_like(x)

    def run(x, res):
        x, res = x.clone().requires_grad_(), res.clone().requires_grad_()
        y = fused_group_norm_act(x, torch.tensor([500], device=DEV), C, residual=res, activation=kind)
        return (y.detach(),) + torch.autograd.grad(y, (x, res), go)

    clean = run(x, res)
    for value in (float("nan"), float("inf"), -float("inf")):
        bad_x, bad_res = x.clone(), res.clone()
        bad_x[7, 3::8] = value
        bad_res[9, 6::8] = value
        apart = torch.ones(C, dtype=torch.bool, device=DEV)
        apart[3::8] = apart[6::8] = False
        for a, b in zip(run(bad_x, bad_res), clean):
            assert torch.equal(a[:, apart], b[:, apart])


def test_signs_on_two_streams_and_in_a_replayed_graph():
    """The same bits as alone, with many elements at the border."""
    from pointelligence_b200 import _cabi
    from pointelligence_b200.layers.norm import fused_group_norm_act

    cases = []
    for C, G, lengths in ((64, 8, [20000, 9000]), (50, 5, [15000, 3, 12000])):
        x, res, w, b = _at_the_border(lengths, C, G, torch.bfloat16, True, C)
        leaves = [t.requires_grad_() for t in (x, w, b, res)]
        go, lens = torch.randn_like(x), torch.tensor(lengths, device=DEV)
        cases.append(lambda leaves=leaves, go=go, lens=lens, G=G: torch.autograd.grad(
            fused_group_norm_act(leaves[0], lens, G, leaves[1], leaves[2], residual=leaves[3], activation="relu", dropout=0.1, rng=(1, 4)), leaves, go))
    alone = [step() for step in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for stream, step in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for q, r in zip(alone, got) for a, b in zip(q, r))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [step() for step in cases]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for q, r in zip(alone, out) for a, b in zip(q, r))
    assert _cabi.device_status() == 0
