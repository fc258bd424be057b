"""Limits of the group norm with activation, looked at before anything is enqueued (there is no device here)."""
import ctypes

import pytest

from pointelligence_b200 import _cabi


def test_samples_times_channels():
    at, L = ctypes.c_void_p(4096), _cabi.lib()
    assert L.pcx_ragged_group_norm_act_workspace_bytes(10, 2 ** 20, 2047, 1, 0) > 0
    for samples, channels in ((2 ** 20, 2048), (2 ** 31, 1), (2 ** 60, 64)):
        assert L.pcx_ragged_group_norm_act_workspace_bytes(10, samples, channels, 1, 0) == 0
        with pytest.raises(ValueError, match="2\\^31"):
            _cabi.check(L.pcx_ragged_group_norm_act(at, at, None, None, None, at, at, at, 10, samples, channels, 1, 1e-5, 2, 0.0, 0, 0, None, 0, at, 0, None))
        with pytest.raises(ValueError, match="2\\^31"):
            _cabi.check(L.pcx_ragged_group_norm_act_backward(at, at, None, at, None, None, at, at, at, None, None, None, 10, samples, channels, 1, 2, 0.0, 0, 0, None, 0,
                                                             at, 0, None))
