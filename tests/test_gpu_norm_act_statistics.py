"""The statistics that ``pcx_ragged_group_norm_act`` leaves for the backward pass, against two passes in float64."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# samples begin at every part of a chunk of rows, and some of them are many chunks long
RAGGED = [5003, 1, 20011, 37, 0, 700, 1201, 9, 33333, 2, 0, 517]
WIDTHS = [(64, 8), (64, 1), (32, 32), (50, 5), (96, 8), (20, 20), (8, 1), (1032, 4), (6, 3)]


def _rows(lengths, C, dtype, kind, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + C)
    N = sum(lengths)
    x = torch.randn(N, C, generator=g, device=DEV) * (0.5 + torch.rand(C, generator=g, device=DEV)) + 0.5 * torch.randn(C, generator=g, device=DEV)
    at = 0
    for n in lengths:
        rows = x[at:at + n]
        at += n
        if n and kind == "drift":
            rows += torch.linspace(0, 10, n, device=DEV)[:, None]
        elif n and kind == "first row far off":
            rows[0] += 300
        elif n and kind == "first rows far off":
            rows[:n // 20 + 1] -= 30
        elif kind == "nearly constant":
            rows[:] = torch.where(torch.rand(n, 1, generator=g, device=DEV) < 0.003, 1004.0, 1000.0)
        elif kind == "large":
            rows *= 2.0 ** 70
    return x.to(dtype)


def _statistics(x, lengths, G, eps):
    from pointelligence_b200 import _cabi

    h, P = _cabi.lib(), _cabi.ptr
    (N, C), S, code = x.shape, len(lengths), _cabi._DTYPES[x.dtype]
    rows = torch.tensor(lengths, device=DEV)
    y = torch.empty_like(x)
    mean, rstd = (torch.empty(S, G, dtype=torch.double, device=DEV) for _ in range(2))
    ws = torch.empty(h.pcx_ragged_group_norm_act_workspace_bytes(N, S, C, G, code), dtype=torch.uint8, device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _cabi.check(h.pcx_ragged_group_norm_act(P(x), P(rows), None, None, None, P(y), P(mean), P(rstd), N, S, C, G, eps, 0, 0.0, 0, 0, None, code, P(ws), ws.numel(), stream))
    return mean, rstd


@pytest.mark.parametrize("C,G", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "drift", "first row far off", "first rows far off", "nearly constant", "large"])
def test_statistics(C, G, dtype, kind):
    """Sums are in 64 bits: a rounding is 2^-53.  What is squared is less than (n - 1) times the sum of squares M2 about the mean away
    from it, n rows a piece, some 2^12 at most, so that what cancels costs a factor of that, and chains of sums some 2^8 roundings more:
    2^-33 of M2; the inverse root halves it.  The mean is compared with the deviation (and eps)."""
    if kind == "large" and dtype == torch.float16:
        pytest.skip("no such values")
    eps = 1e-5
    x = _rows(RAGGED, C, dtype, kind)
    mean, rstd = _statistics(x, RAGGED, G, eps)
    for s, rows in enumerate(torch.split(x.double(), RAGGED)):
        if len(rows) == 0:
            assert not mean[s].any() and bool((rstd[s] == 1 / math.sqrt(eps)).all())
            continue
        v = rows.view(len(rows), G, C // G)
        m = v.mean((0, 2))
        r = torch.rsqrt((v - m[:, None]).square().mean((0, 2)) + eps)
        assert float(((mean[s] - m) * r).abs().max()) <= 2.0 ** -32, s
        assert float((rstd[s] / r - 1).abs().max()) <= 2.0 ** -32, s


@pytest.mark.parametrize("x", [float("inf"), -float("inf"), float("nan")])
def test_what_is_no_number_is_in_both(x):
    """No statistics of a group with an infinity are numbers, whichever row it is in."""
    for at in (0, 3, 5000):
        rows = torch.randn(6000, 16, device=DEV)
        rows[at, 3] = x
        mean, rstd = _statistics(rows, [6000], 4, 1e-5)
        assert not torch.isfinite(mean[0, 0]) and rstd[0, 0].isnan()
        assert bool(torch.isfinite(mean[0, 1:]).all()) and bool(torch.isfinite(rstd[0, 1:]).all())


def _ragged(points, samples):
    """Between 0.6 and 1.4 times the mean."""
    w = [0.6 + 0.8 * ((b * 0.618) % 1.0) for b in range(samples)]
    sizes = [int(points * v / sum(w)) for v in w]
    sizes[0] += points - sum(sizes)
    return sizes


@pytest.mark.parametrize("points,samples,C,G,dtype,seeds", [(1100003, 8, 64, 8, torch.bfloat16, 8), (678000, 678, 32, 32, torch.float16, 4),
                                                            (550001, 3, 50, 1, torch.float32, 3)])
def test_no_sign_of_a_relu_is_on_the_other_side(points, samples, C, G, dtype, seeds):
    """The gradients of weight and bias are sums over all rows: an element whose argument has the wrong sign moves them by a whole
    gradient, 1e-5 to 1e-4 of their norm.  Sums of 32 bits in short chains round by some 2^-23 of their terms, and those add up as roots:
    2^-20 of the norm."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    lengths = _ragged(points, samples)
    sample = torch.repeat_interleave(torch.arange(samples, device=DEV), torch.tensor(lengths, device=DEV))
    for seed in range(seeds):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
        x = (rand(points, C) * (0.5 + torch.rand(C, generator=g, device=DEV)) + 0.5 * rand(C)).to(dtype)
        res, go = rand(points, C).to(dtype), rand(points, C).to(dtype)
        w, b = (1 + 0.2 * rand(C)).requires_grad_(), (0.2 * rand(C)).requires_grad_()
        y = fused_group_norm_act(x, torch.tensor(lengths, device=DEV), G, w, b, residual=res, activation="relu")
        dw, db = torch.autograd.grad(y, (w, b), go)
        v = x.double().view(points, G, -1)
        count = torch.tensor(lengths, device=DEV).double()[:, None] * (C // G)
        per_sample = lambda t: torch.zeros(samples, G, dtype=torch.double, device=DEV).index_add_(0, sample, t)
        v = v - (per_sample(v.sum(2)) / count)[sample][:, :, None]
        v = (v * torch.rsqrt(per_sample(v.square().sum(2)) / count + 1e-5)[sample][:, :, None]).view(points, C)
        gz = go.double() * (v * w.detach().double() + b.detach().double() + res.double() > 0)
        for got, want in ((db, gz.sum(0)), (dw, (gz * v).sum(0))):
            assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -20, seed


def test_sums_of_pieces_are_of_64_bits():
    """A large gradient in the first row and its opposite in the last: what lies between is summed beside them.  Sums of a piece are exact
    here (multiples of 1/4 below 2^22, or one value and zeros), so that the bias's gradient is within its one rounding."""
    from pointelligence_b200.layers.norm import fused_group_norm_act

    N, C, edge = 3500003, 24, 200000
    x = torch.randn(N, C, device=DEV).bfloat16()
    go = torch.full_like(x, 0.25)
    go[:edge] = 0
    go[-edge:] = 0
    go[0], go[-1] = 2.0 ** 30, -2.0 ** 30
    w, b = torch.ones(C, device=DEV, requires_grad=True), torch.zeros(C, device=DEV, requires_grad=True)
    y = fused_group_norm_act(x, torch.tensor([N], device=DEV), 4, w, b, activation="identity")
    db, = torch.autograd.grad(y, b, go)
    want = go.double().sum(0)
    assert bool(((db.double() - want).abs() <= 2.0 ** -24 * want).all())
