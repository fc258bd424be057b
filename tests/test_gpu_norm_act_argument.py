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
