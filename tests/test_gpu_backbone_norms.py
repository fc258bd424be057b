"""Group norm with activation and dropout, and drop path, as a network uses them together."""
import numpy as np
import pytest
import torch

from oracle import norm_act as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_a_block_of_them_against_float64(act):
    """norm, activation, dropout -> product -> norm -> drop path, residual, ReLU: the result and every gradient.

    Each stage is right to 2^-17 of its terms (roundings of 2^-24 through sums of squares, exponentials and slopes); there are six
    of them forward and as many backward, norms pass errors on by factors of at most two: 2^-17 12 2 < 2^-12."""
    from pointelligence_b200.layers.dropout import fused_dropout
    from pointelligence_b200.layers.norm import fused_group_norm_act

    lengths, C, p, q = [900, 0, 333, 50, 2000, 700, 1], 48, 0.25, 0.4
    first, path = (11, 4), (12, 8)
    n = sum(lengths)
    g = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    leaves = [rand(n, C), 1 + 0.2 * rand(C), 0.2 * rand(C), rand(C, C) / C ** 0.5, 1 + 0.2 * rand(C), 0.2 * rand(C)]
    leaves = [t.requires_grad_() for t in leaves]
    go, lens = rand(n, C), torch.tensor(lengths, device=DEV)

    def own(x, w1, b1, m, w2, b2):
        h = fused_group_norm_act(x, lens, 6, w1, b1, activation=act, dropout=p, rng=first) @ m
        h = fused_group_norm_act(h, lens, 1, w2, b2, activation="identity")
        return fused_dropout(h, q, rng=path, unit="sample", lengths=lens, residual=x, relu=True)

    def plain(x, w1, b1, m, w2, b2):
        def norm(v, groups, w, b):
            parts = []
            for s in torch.split(v, lengths):
                s = s.view(len(s), groups, C // groups)
                if len(s):
                    s = (s - s.mean((0, 2), keepdim=True)) / torch.sqrt(s.var((0, 2), correction=0, keepdim=True) + 1e-5)
                parts.append(s.reshape(len(s), C))
            return torch.cat(parts) * w + b

        keep = torch.from_numpy(oracle.keep_factor(np.arange(n * C), p, first)).view(n, C).to(DEV)
        kept = torch.from_numpy(oracle.keep_factor(np.repeat(np.arange(len(lengths)), lengths), q, path))[:, None].to(DEV)
        h = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](norm(x, 6, w1, b1)) * keep @ m
        return torch.relu(norm(h, 1, w2, b2) * kept + x)

    y = own(*leaves)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    ref = plain(*exact)
    # an element whose sign the ReLU's argument does not settle in 32 bits is left out of the comparison of gradients
    settled = ((y > 0) == (ref > 0)).double()
    assert settled.mean() > 0.9999
    got, want = torch.autograd.grad(y, leaves, go * settled.float()), torch.autograd.grad(ref, exact, go.double() * settled)
    for a, b in zip((y,) + got, (ref,) + want):
        assert float((a.double() - b).norm()) <= 2.0 ** -12 * float(b.norm())


@pytest.mark.parametrize("options", [dict(norm_groups=8, activation="silu", dropout=0.1, drop_path=0.2), dict(dropout=0.3), dict(drop_path=0.5),
                                     dict(norm_groups=4), dict(activation="gelu", drop_path=0.1)], ids=str)
def test_network_with_them_trains(options):
    from pointelligence_b200 import _cabi
    from pointelligence_b200.backbone import ResUNet
    from pointelligence_b200.synthetic import indoor_scene, ragged_batch

    pts, inds, sizes = (torch.from_numpy(a).to(DEV) for a in ragged_batch([indoor_scene(4000, 1), indoor_scene(3000, 2)]))
    feat = torch.randn(len(pts), 3, device=DEV)
    torch.manual_seed(0)
    net = ResUNet(in_channels=3, num_classes=20, **options).to(DEV)
    _cabi.profile_enable(True)
    logits = net(feat, pts, inds, sizes, 0.02)
    names = {name for name, _ in _cabi.profile_records()}
    _cabi.profile_enable(False)
    plain_norms = set(options) <= {"drop_path"}
    assert ("group_norm_act(fwd)" in names) != plain_norms and ("dropout(fwd)" in names) == ("drop_path" in options)
    assert logits.shape == (len(pts), 20)
    logits.float().square().mean().backward()
    for name, w in net.named_parameters():
        assert w.grad is not None and torch.isfinite(w.grad).all(), name
    net.eval()
    with torch.no_grad():
        a, b = (net(feat, pts, inds, sizes, 0.02).float() for _ in range(2))
    # nothing is dropped any more: two passes differ by the order of the convolutions' sums, which bf16 layers round
    assert float((a - b).norm()) <= 0.05 * float(a.norm())


def test_drop_path_of_all_branches_leaves_the_identity():
    from pointelligence_b200.backbone import BasicBlock

    block = BasicBlock(32, 32, drop_path=1.0).to(DEV)
    x, lens = torch.randn(100, 32, device=DEV).bfloat16(), torch.tensor([40, 60], device=DEV)
    identity = torch.randn_like(x)
    assert torch.equal(block._tail(x, identity, lens), identity.relu())
    block.eval()
    assert not torch.equal(block._tail(x, identity, lens), identity.relu())
