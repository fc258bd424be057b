"""``fused_dropout`` by channel and by sample where rows are no multiple of 16 bytes, and samples end inside of those."""
import pytest
import torch

from test_gpu_dropout import DEV, RNG, _check

pytestmark = pytest.mark.gpu
RAGGED = [1, 1, 2, 3, 0, 5, 7, 1, 11, 2003, 0, 1, 4, 9]


@pytest.mark.parametrize("C", [1, 2, 3, 5, 6, 7, 12, 20, 33, 50, 100, 257, 3001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("unit", ["channel", "sample"])
def test_rows_side_by_side(C, dtype, unit):
    _check(RAGGED, C, dtype, unit, 0.5, False, False)
    _check(RAGGED, C, dtype, unit, 0.5, True, True)


@pytest.mark.parametrize("N", range(1, 18))
def test_ends_of_a_tensor(N):
    for C in (1, 5, 6):
        for unit in ("channel", "sample"):
            _check([N], C, torch.bfloat16, unit, 0.5, True, False)


@pytest.mark.parametrize("unit", ["channel", "sample"])
@pytest.mark.parametrize("C", [33, 50])
def test_neighbours_and_rows_not_read(unit, C):
    """What is dropped is zero whatever it was, and what is beside it in 16 bytes stays what it is."""
    from pointelligence_b200.layers.dropout import fused_dropout

    lengths = torch.tensor([1] * 200 + [3, 5, 7] * 20, device=DEV)
    x = torch.randn(int(lengths.sum()), C, device=DEV).bfloat16()
    y = fused_dropout(x, 0.5, rng=RNG, unit=unit, lengths=lengths)
    dropped = fused_dropout(torch.ones_like(x), 0.5, rng=RNG, unit=unit, lengths=lengths) == 0
    assert 0.3 < dropped.float().mean() < 0.7
    bad = torch.where(dropped, torch.full_like(x, float("nan")), x)
    assert torch.equal(fused_dropout(bad, 0.5, rng=RNG, unit=unit, lengths=lengths), y)


def test_rows_too_long():
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.zeros(1, dtype=torch.float16, device=DEV).expand(4, 2 ** 32 + 8)
    for unit in ("channel", "sample"):
        with pytest.raises(ValueError, match="channels"):
            fused_dropout(x, 0.5, unit=unit, lengths=torch.tensor([4], device=DEV))
