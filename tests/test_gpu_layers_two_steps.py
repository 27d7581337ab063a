"""Images of many blocks, and such whose blocks meet in two steps, in both directions, with blocks that wait and blocks that never do (the last one out
then combines both steps by itself): against the 64-bit formulas, and the same bits either way."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
from complex_yolov4_pytorch_amd.ops import CY_BF16, CY_F16, CY_F32, View  # noqa: E402
from tests.test_gpu_layers import COUNTERS, DEV, EPS, NAMES, _problem, _workspace, test_many_images_blocks_and_columns as _against_the_formulas  # noqa: E402
from tests.test_layers_plans import TWO_STEPS  # noqa: E402

CASES = pytest.mark.parametrize('shape,dt', [(s, dt) for s, dt, _ in TWO_STEPS], ids=['%dx%dx%dx%d_g%d_%s' % (*s, NAMES[dt]) for s, dt, _ in TWO_STEPS])


@CASES
@pytest.mark.parametrize('config', [{}, dict(polls=0)], ids=['policy', 'nowait'])
def test_against_the_formulas(shape, dt, config):
    _against_the_formulas((*shape, 0, 0), dt, config)


@pytest.mark.parametrize('shape,dt', [((1, 530, 520, 32, 8), CY_F16),      # one launch with all chunks forward, three launches backward
                                      ((1, 500, 500, 32, 8), CY_BF16),     # one launch with all chunks both ways
                                      ((1, 400, 420, 64, 16), CY_F16)],    # half a line to a block backward
                         ids=['530x520x32', '500x500x32', '400x420x64'])
def test_large_images_of_a_batch_of_one(shape, dt):
    _against_the_formulas((*shape, 0, 0), dt, {})


@CASES
def test_the_same_bits_whoever_finishes(shape, dt):
    N, H, W, C, G = shape
    x, dy, res, gamma, beta = (t.to(DEV) for t in _problem((*shape, 0, 0), dt, 17))
    view = lambda t: View(t, 0, N, H, W, C, C, dt)      # noqa: E731
    rng = ops.dropout_state(3, DEV)
    runs = []
    for config in ({}, dict(polls=0), dict(polls=3), {}):
        y, dx, rg = torch.empty_like(x), torch.empty_like(x), torch.zeros_like(x)
        stats, gg = torch.empty(N, G, 2, device=DEV), torch.empty(2, C, device=DEV)
        ops.gn_config(**config)
        try:
            ws = _workspace(N, H, W, C, G, dt)
            for _ in range(2):      # (the second call finds the workspace as the first left it)
                rg.zero_()
                ops.gn_act_fwd(view(x), view(y), view(res), gamma, beta, G, EPS, 2, stats, ws, 0.2, rng, 1)
                ops.gn_act_bwd(view(x), view(dy), view(dx), view(rg), True, gamma, beta, stats, G, 2, gg[0], gg[1], 1.0, False, ws, 0.2, rng, 1)
            torch.cuda.synchronize()
            assert int(ws[:COUNTERS].max()) == 0
        finally:
            ops.gn_config()
        runs.append((y, stats, dx, rg, gg))
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)
