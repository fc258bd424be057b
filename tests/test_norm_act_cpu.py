"""Host side of the group norm with activation and of dropout: refusals before any kernel, and the generator's known answers."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import norm_act as oracle
from pointelligence_b200 import _cabi
from pointelligence_b200.layers import RaggedDropout
from pointelligence_b200.layers.dropout import draw_rng, fused_dropout
from pointelligence_b200.layers.norm import fused_group_norm_act

LENGTHS = torch.tensor([4])


@pytest.mark.parametrize("counter,key,words", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0], [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])])
def test_known_answers_of_the_generator(counter, key, words):
    """(The vectors that the generator's authors publish with it.)"""
    assert oracle.philox4x32_10(np.array(counter), key).tolist() == words


def test_unknown_names():
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="activation"):
        fused_group_norm_act(x, LENGTHS, 2, activation="tanh")
    with pytest.raises(ValueError, match="unit"):
        fused_dropout(x, 0.5, unit="row")
    with pytest.raises(ValueError, match="unit"):
        RaggedDropout(0.5, "row")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            RaggedDropout(p)


def test_no_cpu_tensors():
    x = torch.randn(4, 8)
    for call in (lambda: fused_group_norm_act(x, LENGTHS, 2), lambda: fused_group_norm_act(x, LENGTHS, 2, dropout=0.5),
                 lambda: fused_dropout(x, 0.5), lambda: fused_dropout(x, 0.5, rng=(1, 2)), lambda: draw_rng(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_bad_arguments():
    x = torch.randn(4, 8)
    for rng, error in (("ab", TypeError), ((1, 2, 3), TypeError), (5, TypeError), ((1.5, 2), TypeError), (torch.zeros(2), ValueError),
                       (torch.zeros(3, dtype=torch.int64), ValueError)):
        with pytest.raises(error):
            fused_dropout(x, 0.5, rng=rng)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            fused_dropout(x, p, rng=(1, 2))
        with pytest.raises(ValueError):
            fused_group_norm_act(x, LENGTHS, 2, dropout=p, rng=(1, 2))
    for shape in ((8,), (4, 2, 4)):
        with pytest.raises(ValueError, match="rows"):
            fused_group_norm_act(torch.randn(shape), LENGTHS, 2)


def test_transforms_are_refused():
    x = torch.randn(4, 8)
    for call in (lambda v: fused_group_norm_act(v, LENGTHS, 2), lambda v: fused_dropout(v, 0.5, rng=(1, 2))):
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.vmap(call)(x[None])
        with torch.no_grad(), pytest.raises(RuntimeError, match="functorch"):
            torch.func.jvp(call, (x,), (x,))



def test_c_entry_refuses_before_it_launches():
    """Sizes, null pointers, alignment and capacities are looked at before anything is enqueued (there is no device here)."""
    at = ctypes.c_void_p(4096)
    L = _cabi.lib()
    ws = L.pcx_ragged_group_norm_act_workspace_bytes(10, 2, 8, 4, 0)
    assert ws > 0

    def forward(x=at, lengths=at, w=at, b=at, N=10, S=2, C=8, G=4, act=2, p=0.0, dtype=0, work=at, size=ws):
        return L.pcx_ragged_group_norm_act(x, lengths, w, b, None, at, at, at, N, S, C, G, 1e-5, act, p, 0, 0, None, dtype, work, size, None)

    bad = [dict(N=-1), dict(S=0), dict(C=0), dict(G=3), dict(G=0), dict(C=1 << 17, G=1), dict(act=4), dict(act=-1), dict(dtype=3), dict(p=1.5),
           dict(p=-0.5), dict(x=None), dict(lengths=None), dict(w=None), dict(b=None), dict(work=None), dict(work=ctypes.c_void_p(4100)),
           dict(N=2 ** 61)]
    for change in bad:
        with pytest.raises(ValueError):
            _cabi.check(forward(**change))
    with pytest.raises(RuntimeError, match="workspace"):
        _cabi.check(forward(size=ws - 1))
    for sizes in ((-1, 2, 8, 4, 0), (10, 0, 8, 4, 0), (10, 2, 8, 3, 0), (10, 2, 8, 4, 7)):
        assert L.pcx_ragged_group_norm_act_workspace_bytes(*sizes) == 0

    def backward(g=at, x=at, gw=at, gb=at, G=4, size=ws):
        return L.pcx_ragged_group_norm_act_backward(g, x, None, at, at, at, at, at, at, gw, gb, None, 10, 2, 8, G, 2, 0.0, 0, 0, None, 0, at, size, None)

    for change in (dict(g=None), dict(x=None), dict(gw=None), dict(gb=None), dict(G=5)):
        with pytest.raises(ValueError):
            _cabi.check(backward(**change))
    with pytest.raises(RuntimeError, match="workspace"):
        _cabi.check(backward(size=0))

    need = L.pcx_dropout_workspace_bytes(2, 1)
    assert need > 0 and L.pcx_dropout_workspace_bytes(2, 0) == 0

    def drop(x=at, lengths=at, N=10, S=2, C=8, unit=1, p=0.5, dtype=0, work=at, size=need):
        return L.pcx_dropout(x, lengths, None, at, N, S, C, unit, 0, p, 0, 0, None, dtype, work, size, None)

    for change in (dict(x=None), dict(lengths=None), dict(N=-1), dict(S=0), dict(C=0), dict(unit=3), dict(p=2.0), dict(dtype=5), dict(work=None),
                   dict(work=ctypes.c_void_p(4100)), dict(N=2 ** 61)):
        with pytest.raises(ValueError):
            _cabi.check(drop(**change))
    with pytest.raises(RuntimeError, match="workspace"):
        _cabi.check(drop(size=need - 1))
    with pytest.raises(ValueError):
        _cabi.check(L.pcx_dropout_backward(at, None, None, at, None, 10, 0, 8, 0, 1, 0.5, 0, 0, None, 0, None, 0, None))   # the ReLU's result
    with pytest.raises(ValueError):
        _cabi.check(L.pcx_rng_state(None, at, 0, at, None))


def test_module_without_training_is_the_tail_alone():
    x, res = torch.randn(4, 8), torch.randn(4, 8)
    layer = RaggedDropout(0.5, "sample").eval()
    assert layer(x) is x and torch.equal(layer(x, residual=res, relu=True), (x + res).relu())
    assert RaggedDropout(0.0)(x) is x
    assert "p=0.5" in repr(layer)


def test_network_arguments():
    from pointelligence_b200.backbone import ResUNet

    plain, grouped = ResUNet(), ResUNet(norm_groups=8, activation="silu", dropout=0.1, drop_path=0.2)
    assert {k: v.shape for k, v in plain.state_dict().items()} == {k: v.shape for k, v in grouped.state_dict().items()}
    for bad in (dict(activation="tanh"), dict(dropout=1.5), dict(drop_path=-0.1), dict(norm_groups=7)):
        with pytest.raises(ValueError):
            ResUNet(**bad)


def test_rows_too_long():
    x = torch.zeros(1, dtype=torch.float16).expand(4, 2 ** 32 + 8)
    with pytest.raises(ValueError, match="channels"):
        fused_group_norm_act(x, LENGTHS, 2)


def test_the_layer_keeps_its_type_without_training():
    layer = RaggedDropout(0.5).eval()
    y = layer(torch.ones(2, 3, dtype=torch.bfloat16), residual=torch.full((2, 3), 0.25), relu=True)
    assert y.dtype == torch.bfloat16 and bool((y == 1.25).all())
