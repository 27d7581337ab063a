"""Group norm + activation where the result is known to the last bits.  e = 2^-24 is half a step of float32; storage adds half a step of its
type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
from complex_yolov4_pytorch_amd.ops import CY_BF16, CY_F16, CY_F32  # noqa: E402
from tests.test_gpu_layers import DEV, E, EPS, Strided, _close, _gen, _workspace, kernels  # noqa: E402, F401

TYPES = pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
SHAPES = pytest.mark.parametrize('shape', [(2, 40, 41, 64, 8), (1, 50, 50, 30, 5), (2, 13, 17, 64, 16), (1, 19, 19, 96, 3)],
                                 ids=['rows16', 'ragged', 'narrow', 'wide'])
R = 1 / (EPS ** 0.5)


LEVELS = [1000.0, -8.125, 60000.0, 0.1, -333.25, 12345.0, 0.0, 3e-5, 1.0]


def _one_value_groups(N, HW, C, G, t):
    """-> values [N, G], x [N, HW, C]"""
    levels = torch.tensor(LEVELS).to(t)
    which = torch.randint(0, len(levels), (N, G), generator=_gen(1))
    which[0, 0], which[0, 1] = 0, 2
    v = levels[which]
    return v, v[:, None, :, None].expand(N, HW, G, C // G).reshape(N, HW, C)


@SHAPES
@TYPES
def test_statistics_of_groups_of_one_value(shape, dt, kernels):  # noqa: F811
    """Deviations from one of the values are all 0: the mean is that value, the variance 0."""
    N, H, W, C, G = shape
    v, x = _one_value_groups(N, H * W, C, G, ops.torch_dtype(dt))
    xs, ys, stats = Strided(N, H, W, C, dt, fill=x), Strided(N, H, W, C, dt), torch.empty(N, G, 2, device=DEV)
    ops.gn_act_fwd(xs.view, ys.view, None, torch.ones(C, device=DEV), torch.zeros(C, device=DEV), G, EPS, 0, stats, _workspace(N, H, W, C, G, dt))
    assert torch.equal(stats[..., 0].cpu(), v.float())
    _close(stats[..., 1].cpu(), torch.full((N, G), R, dtype=torch.float64), torch.full((N, G), 4 * E * R, dtype=torch.float64), 'r')
