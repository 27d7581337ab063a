"""The kernel switch of the group norm (ops.gn_config) belongs to the thread that sets it."""
import threading

import pytest

from complex_yolov4_pytorch_amd import ops
from complex_yolov4_pytorch_amd.ops import CY_F16

SHAPE = (16, 152, 152, 128, 32, CY_F16)      # one launch by default; its workspace is not that of three launches


@pytest.fixture(autouse=True)
def default_after():
    yield
    ops.gn_config()


def _in_another_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


def test_a_setting_does_not_reach_another_threads_calls():
    default = ops.gn_workspace_bytes(*SHAPE)
    other = []
    for kw in (dict(mode=0), dict(width=16, chunks=8), dict(chunks=8)):
        ops.gn_config(**kw)
        assert _in_another_thread(lambda: ops.gn_workspace_bytes(*SHAPE)) == default
        other.append(ops.gn_workspace_bytes(*SHAPE))
    ops.gn_config()
    assert any(n != default for n in other)
    _in_another_thread(lambda: ops.gn_config(width=16, chunks=8))
    assert ops.gn_workspace_bytes(*SHAPE) == default


@pytest.mark.parametrize('kw', [dict(mode=0), dict(width=8, chunks=16), dict(chunks=8), dict(polls=0)])
@pytest.mark.parametrize('shape', [SHAPE, (1, 19, 19, 1024, 32, CY_F16), (2, 9, 7, 24, 8, CY_F16), (1, 160, 150, 64, 32, CY_F16)])
def test_a_workspace_serves_the_default_kernels_too(shape, kw):
    """A model's backward pass runs in a thread of autograd's."""
    default = ops.gn_workspace_bytes(*shape)
    ops.gn_config(**kw)
    assert ops.gn_workspace_bytes(*shape) >= default
