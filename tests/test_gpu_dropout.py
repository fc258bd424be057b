"""``fused_dropout`` against its definition: the mask bit for bit, the values to a rounding."""
import numpy as np
import pytest
import torch

from oracle import norm_act as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RNG = (2 ** 64 - 12345, 2 ** 33 + 8)


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check(lengths, C, dtype, unit, p, residual, relu, move=0):
    from pointelligence_b200.layers.dropout import fused_dropout

    g = torch.Generator(device=DEV).manual_seed(sum(lengths) + C)
    N = sum(lengths)

    def make():
        flat = torch.randn(N * C + move, device=DEV, generator=g).to(dtype)
        return flat[move:].view(N, C).requires_grad_()

    x, res, go = make(), make(), make()
    lens = torch.tensor(lengths, device=DEV)
    y = fused_dropout(x, p, rng=RNG, unit=unit, lengths=lens if unit != "element" else None, residual=res if residual else None, relu=relu)
    leaves = [x] + ([res] if residual else [])
    grads = torch.autograd.grad(y, leaves, go.detach())
    want = oracle.dropout(_f64(x), p, RNG, unit, lengths, _f64(res) if residual else None, relu, _f64(go))
    # a product and a sum in fp32, then one rounding; next to the border of the ReLU its sign may be that of either
    U = oracle.EPS_OF[str(dtype).split(".")[1]]
    size = (np.abs(_f64(x)) / (1 - p if p < 1 else 1) + (np.abs(_f64(res)) if residual else 0)) * 2.0 ** -23
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    assert (np.abs(_f64(y) - want[0]) <= U * np.abs(want[0]) + size + tiny).all()
    settled = np.abs(want[0]) > size if relu else np.ones((N, C), bool)
    # (where the rounded result is zero, the ReLU's gradient is)
    settled &= ~((_f64(y) == 0) & (want[0] > 0))
    for a, ref in zip(grads, want[1:]):
        assert (np.abs(_f64(a) - ref) <= U * np.abs(ref) + 2.0 ** -23 * np.abs(ref) + tiny)[settled].all()
    if not relu and not residual and p:
        kept = oracle.dropout(np.ones((N, C)), p, RNG, unit, lengths, None, False, np.ones((N, C)))[0] > 0
        assert np.array_equal(_f64(y) != 0, kept & (_f64(x) != 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("unit", ["element", "channel", "sample"])
@pytest.mark.parametrize("lengths,C", [([1], 1), ([3, 0, 6], 7), ([1000, 1, 0, 300], 64), ([513], 20), ([40] * 70, 33), ([11, 22], 2500)], ids=lambda v: str(v)[:20])
def test_against_the_definition(dtype, unit, lengths, C):
    _check(lengths, C, dtype, unit, 0.3, False, False)
    _check(lengths, C, dtype, unit, 0.3, True, True)


@pytest.mark.parametrize("unit", ["element", "channel", "sample"])
@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
@pytest.mark.parametrize("residual,relu", [(False, False), (True, False), (False, True)])
def test_probabilities(unit, p, residual, relu):
    _check([500, 0, 1500] + [20] * 30, 24, torch.bfloat16, unit, p, residual, relu)


@pytest.mark.parametrize("unit", ["element", "channel", "sample"])
@pytest.mark.parametrize("move", [1, 2, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses(unit, move, dtype):
    _check([100, 31], 48, dtype, unit, 0.4, True, True, move)


def test_dropped_is_zero_and_dropped_samples_are_not_read():
    from pointelligence_b200.layers.dropout import fused_dropout

    for unit in ("element", "channel", "sample"):
        x = torch.full((300, 16), float("nan"), device=DEV)
        lens = torch.tensor([100, 200], device=DEV)
        assert not fused_dropout(x, 1.0, rng=RNG, unit=unit, lengths=lens).any()
        kept = fused_dropout(torch.ones_like(x), 0.5, rng=RNG, unit=unit, lengths=lens) != 0
        assert torch.equal(fused_dropout(x, 0.5, rng=RNG, unit=unit, lengths=lens).isnan(), kept)


def test_relu_hands_nan_on():
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.tensor([[float("nan"), -1.0, 2.0, -float("inf")]], device=DEV)
    assert torch.equal(fused_dropout(x, 0.0, relu=True).nan_to_num(9.0), torch.tensor([[9.0, 0.0, 2.0, 0.0]], device=DEV))


def test_any_shape_by_element_and_higher_gradients():
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.randn(3, 5, 7, device=DEV).requires_grad_()
    y = fused_dropout(x, 0.5, rng=RNG)
    keep = torch.from_numpy(oracle.keep_factor(np.arange(105), 0.5, RNG)).float().view(3, 5, 7).to(DEV)
    assert torch.equal(y, x * keep)
    for relu in (False, True):
        y = fused_dropout(x * x, 0.5, rng=RNG, relu=relu)
        gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        ggx, = torch.autograd.grad(gx.sum(), x)
        # (x^2 keep)^2: 4 x^3 keep^2 and 12 x^2 keep^2, in a dozen roundings of 32 bits
        assert torch.allclose(gx, 4 * x ** 3 * keep ** 2, rtol=2.0 ** -20, atol=0) and torch.allclose(ggx, 12 * x ** 2 * keep ** 2, rtol=2.0 ** -20, atol=0)
    z = fused_dropout(x.permute(2, 0, 1), 0.5, rng=RNG)     # read in its own order
    assert torch.equal(z.reshape(-1), x.permute(2, 0, 1).reshape(-1) * keep.reshape(-1))


def test_no_points():
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.zeros(0, 16, device=DEV).requires_grad_()
    for unit in ("element", "channel", "sample"):
        y = fused_dropout(x, 0.5, unit=unit, lengths=torch.tensor([0, 0], device=DEV), residual=torch.zeros_like(x), relu=True)
        assert y.shape == (0, 16) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 16)


def test_generator_streams_and_capture():
    """A module under a captured step: every replay has its own mask, and the backward pass the same."""
    from pointelligence_b200.layers import RaggedDropout

    torch.manual_seed(3)
    x, lens = torch.ones(4000, 32, device=DEV).requires_grad_(), torch.tensor([1000] * 4, device=DEV)
    layer, path = RaggedDropout(0.25), RaggedDropout(0.5, "sample")
    a = layer(x).detach()
    torch.manual_seed(3)
    assert torch.equal(a, layer(x)) and not torch.equal(a, layer(x))
    assert layer.eval()(x) is x
    layer.train()

    def step():
        y = path(layer(x), lens, residual=x)
        return y.detach(), torch.autograd.grad(y.sum(), x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    masks = []
    for _ in range(8):
        graph.replay()
        assert torch.equal(out[0], out[1])      # of ones, the result is the gradient
        masks.append(out[0].clone())
    assert all(not torch.equal(m, masks[0]) for m in masks[1:])


def test_share_and_independence_of_offsets():
    """2^24 elements: the share that is kept is that of the probability in use within five deviations, and masks of two offsets or
    two seeds agree as often as independent ones."""
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.ones(2 ** 24, device=DEV)
    p = 0.3
    q = 1 - round(65536 * p) / 65536
    masks = [fused_dropout(x, p, rng=r) != 0 for r in ((7, 0), (7, 4), (8, 0))]
    sigma = (q * (1 - q) / x.numel()) ** 0.5
    for m in masks:
        assert abs(float(m.double().mean()) - q) < 5 * sigma
    agree = q * q + (1 - q) ** 2
    for m in masks[1:]:
        assert abs(float((m == masks[0]).double().mean()) - agree) < 5 * (agree * (1 - agree) / x.numel()) ** 0.5


def test_offsets_past_32_bits():
    from pointelligence_b200.layers.dropout import fused_dropout

    n = 2 ** 32 + 4096 + 5
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = fused_dropout(x, 0.5, rng=RNG)
    for lo in (0, 2 ** 31 - 8, 2 ** 32 - 8, n - 4000):
        want = oracle.keep_factor(np.arange(lo, min(n, lo + 4000)), 0.5, RNG)
        assert np.array_equal(_f64(y[lo:lo + 4000]), want)
