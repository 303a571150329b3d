"""Device memory that entry points clear: with a kernel, whose status is its own and which replays of a recorded graph run like any other."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd import _lib  # noqa: E402
from freesound_classification_amd._lib import call, stream_ptr  # noqa: E402

DEV = "cuda:0"


def test_an_older_error_is_not_taken_for_a_failed_clearing():
    """An error that somebody else's call left behind (a device number that does not exist) is not this call's."""
    lib = _lib.load()
    lib.hipGetLastError.restype = lib.hipSetDevice.restype = C.c_int
    lib.hipSetDevice.argtypes = [C.c_int]
    nbytes = lib.fsc_bn_workspace_bytes(24)
    workspace = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    try:
        assert lib.hipSetDevice(10 ** 6) != 0
        assert lib.fsc_bn_workspace_reset(workspace.data_ptr(), 24, stream_ptr()) == 0, lib.fsc_last_error_string()
    finally:
        lib.hipGetLastError()
    torch.cuda.synchronize()
    at = lib.fsc_bn_workspace_ticket_offset(24)
    assert not workspace[at:at + 24 * 4].any() and bool((workspace[:at] == 0xFF).all())


def test_cleared_sums_in_a_replayed_graph():
    """The gradients of a LayerNorm's parameters are cleared and then added to: every replay gives the eager sums (of whole numbers: exact in
    any order), with eager work in between."""
    rows, c = 300, 200
    gen = torch.Generator(device=DEV).manual_seed(3)
    x, ones = torch.randn(rows, c, generator=gen, device=DEV), torch.ones(c, device=DEV)
    mean, rstd = torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    sets = [torch.randint(-4, 5, (rows, c), generator=gen, device=DEV).float() for _ in range(3)]

    def backward(dy, dx, dgamma, dbeta):
        call("fsc_layernorm_bwd", dy.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ones.data_ptr(), dx.data_ptr(), dgamma.data_ptr(),
             dbeta.data_ptr(), rows, c, stream_ptr())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        static = sets[0].clone()
        dx, dgamma, dbeta = torch.empty_like(x), torch.full((c,), 7.0, device=DEV), torch.full((c,), 7.0, device=DEV)
        backward(static, dx, dgamma, dbeta)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            backward(static, dx, dgamma, dbeta)
        for turn in (1, 2, 0, 1):
            static.copy_(sets[turn])
            graph.replay()
            more = torch.empty_like(dbeta)
            backward(sets[turn], torch.empty_like(x), torch.empty_like(dgamma), more)
            torch.cuda.synchronize()
            assert torch.equal(dbeta, sets[turn].sum(0)) and torch.equal(more, dbeta)
