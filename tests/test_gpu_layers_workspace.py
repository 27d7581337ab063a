"""A group norm workspace that is not as the caller should have left it: results are not defined, but nothing outside the workspace and
the outputs is written, and the same workspace zeroed again serves as before."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
from complex_yolov4_pytorch_amd.ops import CY_F16, View  # noqa: E402
from tests.test_gpu_layers import COUNTERS, DEV, EPS, _gen  # noqa: E402

LINES = 512 * 17                          # counters in cache lines of 32 words, 17 to a cluster: the list's length is the first line's word 1


@pytest.mark.parametrize('length', [1, 40, 1 << 20, (1 << 32) - 2])
@pytest.mark.parametrize('entries', [0, 7, 0xFFFFFFFF])
def test_the_list_of_blocks_stays_in_bounds(length, entries):
    N, H, W, C, G = 2, 100, 90, 32, 8
    need, guard = ops.gn_workspace_bytes(N, H, W, C, G, CY_F16), 1 << 20
    buf = torch.zeros(need + 2 * guard, dtype=torch.uint8, device=DEV)
    buf[:guard], buf[guard + need:] = 0xA5, 0xA5
    ws = buf[guard:guard + need]
    mk = lambda s: torch.randn(N * H * W * C, generator=_gen(s)).half().to(DEV)      # noqa: E731
    x, dy, gamma, beta = mk(1), mk(2), torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    outs = [torch.full((N * H * W * C + 8192,), 9.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    stats, gg = torch.empty(N, G, 2, device=DEV), torch.empty(2, C, device=DEV)
    view = lambda t, off=0: View(t, off, N, H, W, C, C, CY_F16)      # noqa: E731

    def nothing():
        pass

    def poison():
        ws[:LINES * 128].view(torch.int32).view(512, 17, 32)[:, 0, 1] = length - (1 << 32) if length >> 31 else length
        ws[COUNTERS:].view(torch.int32).fill_(entries - (1 << 32) if entries >> 31 else entries)

    def run(before=nothing):
        before()
        ops.gn_act_fwd(view(x), view(outs[0], 4096), None, gamma, beta, G, EPS, 2, stats, ws)
        before()
        ops.gn_act_bwd(view(x), view(dy), view(outs[1], 4096), None, False, gamma, beta, stats, G, 2, gg[0], gg[1], 1.0, False, ws)
        torch.cuda.synchronize()
        return [o.clone() for o in outs] + [stats.clone(), gg.clone()]
    want = run()
    assert int(ws[:COUNTERS].max()) == 0
    for polls in (0, -1):
        ops.gn_config(polls=polls)
        try:
            run(poison)
        finally:
            ops.gn_config()
        assert bool((buf[:guard] == 0xA5).all()) and bool((buf[guard + need:] == 0xA5).all())
        for o in outs:
            assert bool((o[:4096] == 9).all()) and bool((o[-4096:] == 9).all())
        ws.zero_()
        assert all(torch.equal(a, b) for a, b in zip(want, run()))
