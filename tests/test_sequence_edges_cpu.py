"""Sequence operators without a device: calls at the edges of what is allowed, which launch nothing or are refused on the host."""
import ctypes as C

import pytest

import freesound_classification_amd as pkg
from freesound_classification_amd import _lib


def _conv(**kw):
    return _lib.CausalConvArgs(**dict(dict(batch=2, length=200, channels=8, taps=4, weight=64), **kw))


def _scan(**kw):
    return _lib.ScanArgs(**dict(dict(batch=2, length=200, channels=8, states=16, groups=1, a_log=64), **kw))


@pytest.mark.parametrize("empty", [dict(batch=0), dict(channels=0), dict(batch=0, channels=0), dict(length=0)])
@pytest.mark.parametrize("length", [1, 64, 5000])
def test_sizes_of_empty_calls(length, empty):
    """The queries a caller makes in front of a launch: lengths at which time would be cut into segments, were there anything to cut."""
    lib = pkg.load_library()
    kw = dict(dict(length=length), **empty)
    assert lib.fsc_selective_scan_checkpoint_bytes(C.byref(_scan(**kw))) == 0
    assert lib.fsc_selective_scan_workspace_bytes(C.byref(_scan(**kw)), 0) == 0
    # (one share of the parameters' sums a sequence: 64 channels of 16 states, skip and bias)
    assert lib.fsc_selective_scan_workspace_bytes(C.byref(_scan(**kw)), 1) == (4 * 2 * 64 * 18 if empty == dict(length=0) else 0)
    # (one share of the filters' and biases' sums)
    assert lib.fsc_causal_conv_bwd_workspace_bytes(C.byref(_conv(**kw))) == (0 if "channels" in empty else 4 * 5 * 8)
    assert lib.fsc_causal_conv_fwd(C.byref(_conv(**kw)), None) == 0
    assert lib.fsc_selective_scan_fwd(C.byref(_scan(**kw)), None) == 0
