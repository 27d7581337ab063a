"""Group norm + activation and dropout on the device against the 64-bit oracle (oracle/layers_ref.py).

Tolerances count roundings.  Storage: half a step of the type relative to the value (2^-11, 2^-8, 2^-24; half a step of the subnormal
spacing below the normal range).  Arithmetic: float32 throughout, e = 2^-24 per operation: a normalised value takes the rounding of
the statistics, a subtraction, two products, a sum and the activation (an exponential and a reciprocal at 1 - 2 e each): below 16 e
of the largest magnitude that enters -- |mean| r gamma, |xh gamma|, |beta|, the value itself.  A sum of n terms t is off by at most
(depth of the additions) e sum |t|; depth <= 64 at these sizes (a thread's pixels + the tree; the folds are double)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
from complex_yolov4_pytorch_amd.ops import CY_BF16, CY_F16, CY_F32, View  # noqa: E402
from oracle import layers_ref as ref  # noqa: E402

DEV = 'cuda'
E = 2.0 ** -24
EPS = 1e-5
HALF_STEP = {CY_F16: 2.0 ** -11, CY_BF16: 2.0 ** -8, CY_F32: 2.0 ** -24}
SUBNORMAL = {CY_F16: 2.0 ** -25, CY_BF16: 2.0 ** -134, CY_F32: 2.0 ** -150}
NAMES = {CY_F16: 'f16', CY_BF16: 'bf16', CY_F32: 'f32'}
SEED, STEP, LAYER = 0x9E3779B97F4A7C15, 5, 9


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Strided:
    """A view with its own row stride and offset inside a buffer whose other elements must keep their values."""

    def __init__(self, N, H, W, C, dt, pad=0, off=0, fill=None, seed=0):
        ld = C + pad
        t = ops.torch_dtype(dt)
        host = torch.randn(off + N * H * W * ld + 16, generator=_gen(seed)).to(t)
        self.view = View(host.to(DEV), off, N, H, W, C, ld, dt)
        self.idx = (off + torch.arange(N * H * W)[:, None] * ld + torch.arange(C)[None]).reshape(-1)
        if fill is not None:
            self.view.buf[self.idx.to(DEV)] = fill.reshape(-1).to(t).to(DEV)
        self.before = self.view.buf.cpu()
        self.shape = (N, H * W, C)

    def get(self):
        return self.view.buf.cpu()[self.idx].view(self.shape)

    def check_outside(self):
        now, mask = self.view.buf.cpu(), torch.ones(self.view.buf.numel(), dtype=torch.bool)
        mask[self.idx] = False
        bits = torch.int32 if now.dtype == torch.float32 else torch.int16
        assert torch.equal(now.view(bits)[mask], self.before.view(bits)[mask]), 'wrote outside the view'


def _workspace(N, H, W, C, G, dt):
    ws = ops.gn_workspace(N, H, W, C, G, dt)
    assert int(ws[:COUNTERS].max()) == 0
    ws[COUNTERS:].fill_(0xFF)      # (behind the counters the contents are arbitrary: NaN in every type)
    return ws


COUNTERS = 512 * 17 * 128 + 384 * 1024 * 8

# the three-launch kernels; one launch by the library's own rule, with few and many blocks to an image, and with blocks that never wait
# for the others (the last of an image's blocks then finishes all of them)
KERNELS = {'general': dict(mode=0), 'policy': {}, 'chunks8': dict(chunks=8), 'chunks16': dict(chunks=16), 'nowait': dict(polls=0, chunks=8)}


@pytest.fixture(params=list(KERNELS))
def kernels(request):
    kw = dict(KERNELS[request.param])
    ops.gn_config(**kw)
    yield request.param
    ops.gn_config()


def _stored(exact, dt):
    return HALF_STEP[dt] * exact.abs() + SUBNORMAL[dt]


def _close(got, exact, tol, what):
    got = got.double()
    bad = ~((got - exact).abs() <= tol)
    assert not bool(bad.any()), '%s: %d of %d off, worst %.3g over its tolerance %.3g' % (
        what, int(bad.sum()), bad.numel(), float((got - exact).abs()[bad].max()), float((tol + 0 * exact)[bad].min()))


# N, H, W, C, G, pad of the rows, offset of the first element
SHAPES = [
    (1, 19, 19, 1024, 32, 0, 0),       # the deepest stage
    (2, 13, 17, 64, 16, 0, 0),         # groups narrower than a 16-byte access
    (3, 8, 9, 96, 8, 32, 8),           # a slice of a concatenation
    (2, 7, 5, 144, 9, 0, 0),           # 18 accesses of 16 bytes per pixel: 256 threads are not a multiple of them
    (2, 9, 7, 24, 8, 0, 0),            # groups of 3
    (1, 33, 31, 30, 6, 7, 0),          # rows of 37 elements
    (2, 5, 5, 20, 4, 0, 1),            # first element off every 16-byte boundary
    (3, 1, 1, 512, 32, 0, 0),          # one pixel
    (2, 1, 1, 8, 8, 0, 0),             # groups of one value: the output is act(beta)
    (1, 1, 2, 6, 1, 0, 0),
    (1, 57, 1, 16, 1, 0, 0),           # one group
    (2, 6, 6, 2056, 8, 0, 0),          # more columns than a block has threads (16-bit: 257)
    (1, 3, 3, 1030, 2, 0, 0),          # the same, one element at a time
    (40, 2, 3, 32, 32, 0, 0),          # a group per channel
    (2, 50, 45, 64, 4, 0, 0),          # several blocks to an image in every kernel
    (1, 160, 150, 64, 32, 0, 0),       # many blocks and many groups: they meet in two steps
    (2, 100, 90, 32, 8, 0, 0),         # several pixel ranges per image
    (1, 1, 1, 1, 1, 0, 0),
]
IDS = ['%dx%dx%dx%d_g%d_p%d_o%d' % s for s in SHAPES]


def _problem(shape, dt, seed, shift=0.0):
    N, H, W, C, G, pad, off = shape
    g = _gen(seed)
    t = ops.torch_dtype(dt)
    x = (torch.randn(N, H * W, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + 0.5 * torch.randn(C, generator=g) + shift).to(t)
    dy = torch.randn(N, H * W, C, generator=g).to(t)
    res = torch.randn(N, H * W, C, generator=g).to(t)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    return x, dy, res, gamma, beta


def _stats_tol(x, G):
    """mean: rounding of the result + depth e of the mean magnitude; r: relative error of the variance / 2 + rounding."""
    N, HW, C = x.shape
    v = x.double().reshape(N, HW, G, -1)
    return 64 * E * v.abs().mean((1, 3)), 64 * E


@pytest.mark.parametrize('drop', [0.0, 0.2], ids=['', 'drop'])
@pytest.mark.parametrize('act', [0, 1, 2], ids=['linear', 'leaky', 'mish'])
@pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('shape', SHAPES, ids=IDS)
def test_group_norm_act(shape, dt, act, drop, kernels):
    N, H, W, C, G, pad, off = shape
    x, dy, res, gamma, beta = _problem(shape, dt, 100 + C)
    use_res = act != 1
    q = ops.dropout_q(drop)
    fac = ref.drop_factor((N, H * W, C), q, SEED, STEP, LAYER) if q else torch.ones((), dtype=torch.float64)
    rng = ops.dropout_state(SEED, DEV, STEP)
    xs, ys = Strided(N, H, W, C, dt, pad, off, x), Strided(N, H, W, C, dt, pad, off, seed=1)
    rs = Strided(N, H, W, C, dt, pad, off, res, seed=2)
    ga, be = gamma.to(DEV), beta.to(DEV)
    stats = torch.full((N, G, 2), float('nan'), device=DEV)
    ws = _workspace(N, H, W, C, G, dt)
    ops.gn_act_fwd(xs.view, ys.view, rs.view if use_res else None, ga, be, G, EPS, act, stats, ws, drop, rng, LAYER)
    want, n = ref.gn_act(x, gamma, beta, G, EPS, act, fac, res if use_res else None)
    mt, rt = _stats_tol(x, G)
    st = stats.cpu().double()
    _close(st[..., 0], n['mean'], mt + E * n['mean'].abs(), 'mean')
    # (variance near zero beside eps: the centred sum is exact to 64 e of the second moment about a value of the data)
    m2 = (x.double().reshape(N, H * W, G, -1) - n['mean'][:, None, :, None]).pow(2).mean((1, 3))
    _close(st[..., 1], n['rstd'], n['rstd'] * (rt * m2 / (m2 + EPS) + 4 * E + 0.5 * n['rstd'] ** 2 * (mt + E * n['mean'].abs()) ** 2), 'r')
    per_c = lambda t: t.repeat_interleave(C // G, -1)[:, None, :]      # noqa: E731
    big = per_c(n['rstd']) * (per_c(n['mean'].abs() + mt / (16 * E)) + x.double().abs()) * gamma.double().abs() + beta.double().abs() + n['z'].abs()
    tol = _stored(want, dt) + (16 * E * big) * 1.1 * fac.max() + (8 * E * (want.abs() + (res.double().abs() if use_res else 0)))
    _close(ys.get(), want, tol, 'y')
    ys.check_outside()
    # the eval form: no statistics kept, the same values; and in place
    y2 = Strided(N, H, W, C, dt, pad, off, seed=1)
    ops.gn_act_fwd(xs.view, y2.view, rs.view if use_res else None, ga, be, G, EPS, act, None, ws, drop, rng, LAYER)
    assert torch.equal(y2.get(), ys.get())
    x2 = Strided(N, H, W, C, dt, pad, off, x)
    ops.gn_act_fwd(x2.view, x2.view, rs.view if use_res else None, ga, be, G, EPS, act, stats, ws, drop, rng, LAYER)
    assert torch.equal(x2.get(), ys.get())
    x2.check_outside()

    # ---- gradient, from the statistics the forward pass left
    dys, dxs = Strided(N, H, W, C, dt, pad, off, dy), Strided(N, H, W, C, dt, pad, off, seed=3)
    old_rg = torch.randn(N, H * W, C, generator=_gen(7)).to(ops.torch_dtype(dt))
    rg = Strided(N, H, W, C, dt, pad, off, old_rg)
    g0 = torch.randn(2, C, generator=_gen(8))
    gg = g0.to(DEV)
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, rg.view, True, ga, be, stats, G, act, gg[0], gg[1], 0.5, True, ws, drop, rng, LAYER)
    o = ref.gn_act_grad(x, dy, gamma, beta, G, EPS, act, fac)
    # a leaky value within the error of zero may take either slope
    zerr = 16 * E * big
    kink = (o['z'].abs() <= zerr) if act == 1 else torch.zeros_like(o['z'], dtype=torch.bool)
    slack = torch.where(kink, 0.9 * (dy.double() * fac).abs(), torch.zeros(())) + 3 * zerr * (dy.double() * fac).abs() * (act == 2)
    hs = o['h'].abs() + slack * gamma.double().abs()
    grp = lambda t: t.reshape(N, H * W, G, -1)      # noqa: E731
    mean_abs = grp(hs * (1 + o['xh'].abs())).mean((1, 3))
    mean_slack = grp(slack * gamma.double().abs() * (1 + o['xh'].abs())).mean((1, 3))
    xe = per_c(n['rstd']) * 16 * E * (per_c(n['mean'].abs() + mt / (16 * E)) + x.double().abs()) + 64 * E * o['xh'].abs()      # error of xh
    mean_xe = grp(hs * xe).mean((1, 3))
    S2 = per_c(o['s2'].abs())
    tol = per_c(n['rstd']) * (slack * gamma.double().abs() + per_c(mean_slack + mean_xe) * (1 + o['xh'].abs()) + S2 * xe
                              + 80 * E * (hs + per_c(mean_abs) * (1 + o['xh'].abs()))) + 80 * E * o['dx'].abs() + _stored(o['dx'], dt)
    _close(dxs.get(), o['dx'], tol, 'dx')
    dxs.check_outside()
    _close(rg.get(), old_rg.double() + dy.double(), _stored(old_rg.double() + dy.double(), dt) + 2 * E * (old_rg.double().abs() + dy.double().abs()), 'res')
    got = gg.cpu().double()
    for k, name, terms, err in ((0, 'ggamma', o['dz'] * o['xh'], slack * o['xh'].abs() + (o['dz'].abs() + slack) * xe), (1, 'gbeta', o['dz'], slack)):
        want_g = g0[k].double() + 0.5 * terms.sum((0, 1))
        t = 0.5 * (err.sum((0, 1)) + 80 * E * terms.abs().sum((0, 1))) + 4 * E * (want_g.abs() + g0[k].double().abs())
        _close(got[k], want_g, t, name)
    # dx over dy, shortcut gradient stored, parameter gradients stored
    dy2, rg2, gg2 = Strided(N, H, W, C, dt, pad, off, dy), Strided(N, H, W, C, dt, pad, off, seed=4), torch.full((2, C), float('nan'), device=DEV)
    ops.gn_act_bwd(xs.view, dy2.view, dy2.view, rg2.view, False, ga, be, stats, G, act, gg2[0], gg2[1], 1.0, False, ws, drop, rng, LAYER)
    assert torch.equal(dy2.get(), dxs.get()) and torch.equal(rg2.get(), dy)
    dy2.check_outside()
    rg2.check_outside()
    gg3 = torch.full((2, C), float('nan'), device=DEV)
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, ga, be, stats, G, act, None, gg3[1], 1.0, False, ws, drop, rng, LAYER)
    assert torch.equal(gg3[1], gg2[1]) and bool(gg3[0].isnan().all())
    assert int(ws[:COUNTERS].max()) == 0      # (as it was: the next call finds its counters)
    _close(gg2.cpu().double() * 0.5 + g0.double(), got, 4 * E * (got.abs() + g0.double().abs()), 'stored gradients')


@pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('shape', [(2, 40, 41, 64, 8, 0, 0), (1, 50, 50, 30, 5, 0, 0)], ids=['rows16', 'ragged'])
def test_statistics_beside_a_large_mean(shape, dt, kernels):
    """Deviations of a step or two of the type beside the mean: sums of squares of the values would lose them all."""
    N, H, W, C, G, pad, off = shape
    g = _gen(5)
    step = {CY_F16: 2.0 ** -10, CY_BF16: 2.0 ** -7, CY_F32: 2.0 ** -23}[dt] * 1024
    x = (1024 + step * torch.randint(0, 8, (N, H * W, C), generator=g).double()).to(ops.torch_dtype(dt))
    x[:, 0] = 0 if dt == CY_F32 else x[:, 0]      # the first pixel far away from the rest
    xs, ys = Strided(N, H, W, C, dt, fill=x), Strided(N, H, W, C, dt)
    stats = torch.empty(N, G, 2, device=DEV)
    ops.gn_act_fwd(xs.view, ys.view, None, torch.ones(C, device=DEV), torch.zeros(C, device=DEV), G, EPS, 0, stats, _workspace(N, H, W, C, G, dt))
    n = ref.group_norm(x, torch.ones(C), torch.zeros(C), G, EPS)
    st = stats.cpu().double()
    _close(st[..., 0], n['mean'], 2 * E * n['mean'].abs(), 'mean')
    # a thread's centred sum: at most (values it holds <= 512) e of the column's own; means merged to e |mean| each
    merged = (4 * E * n['mean']) ** 2 * n['rstd'] ** 2
    _close(st[..., 1], n['rstd'], n['rstd'] * (512 * E + merged), 'r')


@pytest.mark.parametrize('config', [{}, dict(mode=0), dict(width=256)], ids=['policy', 'general', 'wide'])
@pytest.mark.parametrize('shape,dt', [
    ((300, 11, 100, 4, 1, 0, 0), CY_F32),       # 600 blocks' sums per channel: parameter gradients in two slices
    ((16, 512, 512, 4, 2, 0, 0), CY_F32),       # 2048: in eight
    ((70, 9, 9, 24, 8, 0, 0), CY_BF16),         # more images than lanes that add them
    ((16, 76, 76, 255, 17, 0, 0), CY_F16),      # element by element, more blocks than fit at a time
    ((2, 7, 9, 2048, 2048, 0, 0), CY_F16),      # the widest block: 2048 groups of one channel
    ((9, 19, 19, 512, 32, 0, 0), CY_BF16),      # blocks alone with their columns, more of them than compute units
], ids=lambda v: '%dx%dx%dx%d_g%d' % v[:5] if isinstance(v, tuple) else NAMES[v])
def test_many_images_blocks_and_columns(shape, dt, config):
    """Against the 64-bit formulas on the device.  A sum's depth here: at most 64 values of a thread and 256 rows of a block (the rest is
    in double), so 320 e of the sum of magnitudes; a column of the general kernels adds up to 512 pixels per thread and eight levels."""
    N, H, W, C, G, pad, off = shape
    x, dy, _, gamma, beta = (t.to(DEV) for t in _problem(shape, dt, 31))
    xs, dys = View(x, 0, N, H, W, C, C, dt), View(dy, 0, N, H, W, C, C, dt)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    stats, gg = torch.empty(N, G, 2, device=DEV), torch.empty(2, C, device=DEV)
    ops.gn_config(**config)
    try:
        ws = _workspace(N, H, W, C, G, dt)
        ops.gn_act_fwd(xs, View(y, 0, N, H, W, C, C, dt), None, gamma, beta, G, EPS, 2, stats, ws)
        ops.gn_act_bwd(xs, dys, View(dx, 0, N, H, W, C, C, dt), None, False, gamma, beta, stats, G, 2, gg[0], gg[1], 1.0, False, ws)
        torch.cuda.synchronize()
        assert int(ws[:COUNTERS].max()) == 0
    finally:
        ops.gn_config()
    one = torch.ones((), dtype=torch.float64, device=DEV)
    want, n = ref.gn_act(x, gamma, beta, G, EPS, 2, one)
    per_c = lambda t: t.repeat_interleave(C // G, -1)[:, None, :]      # noqa: E731
    xe = 64 * E * (per_c(n['rstd'] * (1 + n['mean'].abs())) * (1 + x.double().abs()))      # error of xh
    _close(y, want, _stored(want, dt) + 1.1 * (xe * gamma.double().abs() + 16 * E * (beta.double().abs() + n['z'].abs())) + 8 * E * want.abs(), 'y')
    o = ref.gn_act_grad(x, dy, gamma, beta, G, EPS, 2, one)
    ze = xe * gamma.double().abs() + 16 * E * (beta.double().abs() + n['z'].abs())
    dze = 3 * ze * dy.double().abs() + 16 * E * o['dz'].abs()
    depth = (520 if config.get('mode') == 0 else 320) * E
    for k, name, t, err in ((0, 'ggamma', o['dz'] * o['xh'], dze * o['xh'].abs() + (o['dz'].abs() + dze) * xe), (1, 'gbeta', o['dz'], dze)):
        _close(gg[k], t.sum((0, 1)), err.sum((0, 1)) + depth * t.abs().sum((0, 1)), name)
    grp = lambda t: t.reshape(N, H * W, G, -1).mean((1, 3))      # noqa: E731
    he, h = dze * gamma.double().abs(), o['h'].abs()
    sums = per_c(grp(he) + depth * grp(h)) + o['xh'].abs() * per_c(grp(he * o['xh'].abs() + (h + he) * xe) + depth * grp(h * o['xh'].abs()))
    tol = per_c(n['rstd']) * (he + sums + xe * per_c(o['s2'].abs()) + 16 * E * (h + per_c(grp(h)))) + 80 * E * o['dx'].abs()
    _close(dx, o['dx'], tol + _stored(o['dx'], dt), 'dx')


def test_non_finite_values_stay_in_their_group():
    N, H, W, C, G = 2, 6, 6, 32, 4
    x, dy, _, gamma, beta = _problem((N, H, W, C, G, 0, 0), CY_F16, 3)
    x[0, 5, 3], x[1, 7, 30] = float('nan'), float('inf')
    xs, ys, dys, dxs = (Strided(N, H, W, C, CY_F16, fill=f) for f in (x, x, dy, dy))
    stats, ws, gg = torch.empty(N, G, 2, device=DEV), _workspace(N, H, W, C, G, CY_F16), torch.empty(2, C, device=DEV)
    ops.gn_act_fwd(xs.view, ys.view, None, gamma.to(DEV), beta.to(DEV), G, EPS, 2, stats, ws)
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, gamma.to(DEV), beta.to(DEV), stats, G, 2, gg[0], gg[1], 1.0, False, ws)
    for t in (ys.get(), dxs.get()):
        bad = ~t.isfinite().view(N, H * W, G, C // G)
        assert bool(bad[0, :, 0].all()) and bool(bad[1, :, 3].all()) and not bool(bad[0, :, 1:].any()) and not bool(bad[1, :, :3].any())
    assert not bool(gg[:, 8:24].isnan().any()) and bool(gg[:, :8].isnan().all()) and bool(gg[:, 24:].isnan().all())


@pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
def test_mish_far_out(dt):
    """Values whose exponential over- or underflows: mish(z) is z above and -0 below, the derivative 1 and 0.  A hardware exponential below
    2^-126 is 0 (it has no subnormals): mish, z e^z there, is then off by at most |z| 2^-126, which no z below -87.3 makes more than
    120 x 2^-126 of (e^z halves with every 0.7)."""
    z = torch.tensor([0.0, -1e-6, 20.5, -20.5, 88.0, -88.0, 104.0, -104.0, 3e4, -3e4] + ([1e20, -1e20, 3e38, -3e38] if dt != CY_F16 else [6e4, -6e4]))
    C = z.numel()
    x = torch.tensor([[1.0], [-1.0]]).repeat(1, C)[None].to(ops.torch_dtype(dt))      # xh = +-1 / sqrt(1 + eps) in every channel
    dy = torch.ones(1, 2, C).to(ops.torch_dtype(dt))
    xs, ys, dys, dxs = (Strided(1, 2, 1, C, dt, fill=f) for f in (x, x, dy, dy))
    stats, ws, gg = torch.empty(1, C, 2, device=DEV), _workspace(1, 2, 1, C, C, dt), torch.empty(2, C, device=DEV)
    ga, be = torch.zeros(C, device=DEV), z.to(DEV)                                     # gamma = 0: z is beta
    ops.gn_act_fwd(xs.view, ys.view, None, ga, be, C, EPS, 2, stats, ws)
    zd = z.double()
    want = ref.act(zd, 2)[None, None].expand(1, 2, C)
    _close(ys.get(), want, _stored(want, dt) + 16 * E * want.abs() + 120 * 2.0 ** -126, 'y')
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, ga, be, stats, C, 2, gg[0], gg[1], 1.0, False, ws)
    slope = ref.act_grad(zd.clamp(-700, 700), 2)
    _close(gg[1].cpu(), 2 * slope, 16 * E * (slope.abs() + zd.abs().clamp(max=100) * (zd < 0)) + 16 * E, 'sum of the derivative')


def test_everything_dropped():
    N, H, W, C, G = 2, 5, 7, 32, 8
    x, dy, res, gamma, beta = _problem((N, H, W, C, G, 0, 0), CY_BF16, 4)
    rng = ops.dropout_state(1, DEV)
    xs, ys, rs, dys, dxs = (Strided(N, H, W, C, CY_BF16, fill=f) for f in (x, x, res, dy, dy))
    stats, ws, gg = torch.empty(N, G, 2, device=DEV), _workspace(N, H, W, C, G, CY_BF16), torch.full((2, C), float('nan'), device=DEV)
    ops.gn_act_fwd(xs.view, ys.view, rs.view, gamma.to(DEV), beta.to(DEV), G, EPS, 2, stats, ws, 1.0, rng)
    assert torch.equal(ys.get(), res)
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, gamma.to(DEV), beta.to(DEV), stats, G, 2, gg[0], gg[1], 1.0, False, ws, 1.0, rng)
    assert float(dxs.get().abs().max()) == 0 and float(gg.abs().max()) == 0
    ops.dropout_fwd(xs.view, ys.view, 1.0, rng)
    assert float(ys.get().abs().max()) == 0


def test_no_images_and_no_pixels():
    ws = torch.empty(16, dtype=torch.uint8, device=DEV)
    ga, be = torch.ones(8, device=DEV), torch.zeros(8, device=DEV)
    for N, H, W in ((0, 4, 4), (2, 0, 4)):
        v = View(torch.empty(0, dtype=torch.float16, device=DEV), 0, N, H, W, 8, 8, CY_F16)
        assert ops.gn_workspace(N, H, W, 8, 2, CY_F16).numel() >= 8
        st = torch.empty(N, 2, 2, device=DEV)
        gg = torch.full((2, 8), 3.0, device=DEV)
        ops.gn_act_fwd(v, v, None, ga, be, 2, EPS, 2, st, ws)
        ops.gn_act_bwd(v, v, v, None, False, ga, be, st, 2, 2, gg[0], gg[1], 1.0, True, ws)
        assert float((gg - 3).abs().max()) == 0
        ops.gn_act_bwd(v, v, v, None, False, ga, be, st, 2, 2, gg[0], gg[1], 1.0, False, ws)
        assert float(gg.abs().max()) == 0
        ops.dropout_fwd(v, v, 0.5, ops.dropout_state(0, DEV))


def test_offsets_beyond_32_bits():
    """Rows 2^18 elements apart: the last pixels lie 4.3 GB into the buffer (2^31 elements and more)."""
    H, W, C, G, ld = 96, 96, 16, 2, 1 << 18
    buf = torch.zeros(H * W * ld, dtype=torch.float16, device=DEV)
    x = torch.randn(1, H * W, C, generator=_gen(6)).half()
    torch.as_strided(buf, (H * W, C), (ld, 1)).copy_(x[0].to(DEV))
    v, y = View(buf, 0, 1, H, W, C, ld, CY_F16), View(buf, 64, 1, H, W, C, ld, CY_F16)
    ga, be = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    stats, ws, gg = torch.empty(1, G, 2, device=DEV), _workspace(1, H, W, C, G, CY_F16), torch.empty(2, C, device=DEV)
    ops.gn_act_fwd(v, y, None, ga, be, G, EPS, 2, stats, ws)
    want, n = ref.gn_act(x, torch.ones(C), torch.zeros(C), G, EPS, 2)
    got = torch.as_strided(buf, (H * W, C), (ld, 1), 64).cpu()
    _close(got[None], want, _stored(want, CY_F16) + 32 * E * (1 + n['z'].abs()), 'y')
    dx = View(buf, 128, 1, H, W, C, ld, CY_F16)
    ops.gn_act_bwd(v, y, dx, None, False, ga, be, stats, G, 2, gg[0], gg[1], 1.0, False, ws)
    o = ref.gn_act_grad(x, got[None], torch.ones(C), torch.zeros(C), G, EPS, 2)
    _close(torch.as_strided(buf, (H * W, C), (ld, 1), 128).cpu()[None], o['dx'], _stored(o['dx'], CY_F16) + 2.0 ** -16 * n['rstd'].max() * (1 + o['xh'].abs()), 'dx')
    ops.dropout_fwd(v, dx, 0.5, ops.dropout_state(SEED, DEV, STEP), LAYER)
    fac = ref.drop_factor((1, H * W, C), 32768, SEED, STEP, LAYER)
    assert torch.equal(torch.as_strided(buf, (H * W, C), (ld, 1), 128).cpu()[None].double(), x.double() * fac)


# ---- dropout -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize('p', [0.0, 0.1, 0.5, 0.9])
@pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('shape', [(1, 19, 19, 512, 0, 0), (2, 7, 9, 24, 8, 8), (3, 5, 5, 30, 7, 0), (1, 1, 1, 1, 0, 0), (2, 3, 3, 20, 0, 1),
                                   (1, 1, 1, 8, 0, 0), (1, 300, 300, 40, 24, 0)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_dropout(shape, dt, p):
    N, H, W, C, pad, off = shape
    x = torch.randn(N, H * W, C, generator=_gen(C)).to(ops.torch_dtype(dt))
    x[0, 0, 0] = 0.0
    q = ops.dropout_q(p)
    rng = ops.dropout_state(SEED, DEV, (1 << 32) + STEP)      # (the step counts modulo 2^32)
    fac = ref.drop_factor((N, H * W, C), q, SEED, STEP, LAYER)
    xs, ys = Strided(N, H, W, C, dt, pad, off, x), Strided(N, H, W, C, dt, pad, off, seed=1)
    ops.dropout_fwd(xs.view, ys.view, p, rng, LAYER)
    want = x.double() * fac
    _close(ys.get(), want, _stored(want, dt) + 2 * E * want.abs(), 'y')      # (the factor and the product, in float32)
    assert torch.equal(ys.get() == 0, want == 0)
    ys.check_outside()
    old = torch.randn(N, H * W, C, generator=_gen(1)).to(ops.torch_dtype(dt))
    for acc in (False, True):
        g = Strided(N, H, W, C, dt, pad, off, old)
        ops.dropout_bwd(xs.view, g.view, acc, p, rng, LAYER)
        wg = want + (old.double() if acc else 0)
        _close(g.get(), wg, _stored(wg, dt) + 3 * E * (want.abs() + old.double().abs()), 'gradient')
        g.check_outside()
    ops.dropout_fwd(xs.view, xs.view, p, rng, LAYER)
    assert torch.equal(xs.get(), ys.get())


def test_dropped_nan_is_gone_and_kept_nan_stays():
    N, H, W, C = 1, 16, 16, 64
    x = torch.full((N, H * W, C), float('nan')).half()
    xs, ys = Strided(N, H, W, C, CY_F16, fill=x), Strided(N, H, W, C, CY_F16)
    ops.dropout_fwd(xs.view, ys.view, 0.5, ops.dropout_state(SEED, DEV, STEP), LAYER)
    keep = ref.keep_mask(H * W * C, 32768, SEED, STEP, LAYER).view(N, H * W, C)
    assert torch.equal(ys.get().isnan(), keep) and float(ys.get()[~keep].abs().max()) == 0


def test_mask_is_the_same_in_every_type_and_kernel():
    """The mask belongs to the dense element index: not to the storage type, the row stride or the kernel that ran."""
    N, H, W, C = 2, 11, 13, 40
    one = torch.ones(N, H * W, C)
    rng = ops.dropout_state(77, DEV, 3)
    masks = []
    for dt in (CY_F16, CY_BF16, CY_F32):
        for pad, off in ((0, 0), (8, 0), (3, 1)):
            a, b = Strided(N, H, W, C, dt, pad, off, one), Strided(N, H, W, C, dt, pad, off)
            ops.dropout_fwd(a.view, b.view, 0.3, rng, 2)
            masks.append(b.get() != 0)
            # fused behind a group norm: gamma = 0, beta = 1 gives ones to drop from
            st, ws = torch.empty(N, 8, 2, device=DEV), _workspace(N, H, W, C, 8, dt)
            ops.gn_act_fwd(a.view, b.view, None, torch.zeros(C, device=DEV), torch.ones(C, device=DEV), 8, EPS, 0, st, ws, 0.3, rng, 2)
            masks.append(b.get() != 0)
    assert all(torch.equal(m, masks[0]) for m in masks) and 0.2 < float((~masks[0]).double().mean()) < 0.4


# ---- streams, recording, graphs ----------------------------------------------------------------------------

def _run_block(b):
    """A block as a training step runs it: norm + activation + dropout + shortcut, its gradient, a dropout behind it and its gradient."""
    ops.gn_act_fwd(b['x'], b['y'], b['res'], b['ga'], b['be'], 8, EPS, 2, b['stats'], b['ws'], 0.2, b['rng'], 1)
    ops.dropout_fwd(b['y'], b['d'], 0.4, b['rng'], 2)
    ops.dropout_bwd(b['dy'], b['g'], False, 0.4, b['rng'], 2)
    ops.gn_act_bwd(b['x'], b['g'], b['dx'], b['rg'], True, b['ga'], b['be'], b['stats'], 8, 2, b['gg'][0], b['gg'][1], 1.0, False, b['ws'], 0.2, b['rng'], 1)


def _block(seed=0, dt=CY_F16):
    N, H, W, C = 4, 38, 38, 64
    mk = lambda s: View((torch.randn(N * H * W * C, generator=_gen(s))).to(ops.torch_dtype(dt)).to(DEV), 0, N, H, W, C, C, dt)      # noqa: E731
    b = dict(x=mk(seed), res=mk(seed + 1), dy=mk(seed + 2), y=mk(9), d=mk(9), g=mk(9), dx=mk(9), rg=mk(9))
    b.update(ga=1 + 0.1 * torch.randn(C, generator=_gen(3)).to(DEV), be=torch.randn(C, generator=_gen(4)).to(DEV), stats=torch.empty(N, 8, 2, device=DEV),
             ws=ops.gn_workspace(N, H, W, C, 8, dt), gg=torch.empty(2, C, device=DEV), rng=ops.dropout_state(42, DEV))
    return b


OUT = ('y', 'd', 'g', 'dx', 'rg')


def _results(b):
    return [b[k].buf.clone() for k in OUT] + [b['stats'].clone(), b['gg'].clone()]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _reset(b):
    b['rg'].buf.zero_()


def test_repeats_are_bit_identical_and_streams_are_honoured():
    b = _block()
    _reset(b)
    _run_block(b)
    first = _results(b)
    for _ in range(3):
        _reset(b)
        _run_block(b)
        assert _same(first, _results(b))
    # another stream, its input produced there behind a long kernel
    s = torch.cuda.Stream()
    a = torch.randn(4096, 4096, device=DEV)
    keep = b['x'].buf.clone()
    b['x'].buf.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(8):
            a = (a @ a).clamp_(-1, 1)
        b['x'].buf.copy_(keep)
        _reset(b)
        _run_block(b)
        out = _results(b)
    s.synchronize()
    assert _same(first, out)


def test_two_streams_at_once():
    blocks = [_block(seed=10 * i) for i in range(2)]
    want = []
    for b in blocks:
        _reset(b)
        _run_block(b)
        want.append(_results(b))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    for _ in range(20):
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                _reset(b)
                _run_block(b)
    torch.cuda.synchronize()
    assert all(_same(w, _results(b)) for w, b in zip(want, blocks))


def test_recorded_launch_list():
    b = _block()
    _reset(b)
    ops.start_recording()
    _run_block(b)
    prog = ops.stop_recording()
    first = _results(b)
    b['rng'][1] += 1
    _reset(b)
    prog.run()
    second = _results(b)
    assert not _same(first, second)      # (the step is read on the device)
    b['rng'][1] -= 1
    _reset(b)
    prog.run()
    assert _same(first, _results(b))


def test_captured_graph_replays():
    b = _block()
    want = []
    for _ in range(4):
        b['rng'][1] += 1
        _reset(b)
        _run_block(b)
        want.append(_results(b))
    b['rng'][1] -= 4
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b['rng'][1:].add_(1)
        b['rg'].buf.zero_()
        _run_block(b)
    for w in want:
        for k in OUT:
            if k != 'rg':
                b[k].buf.fill_(float('nan'))
        graph.replay()
        torch.cuda.synchronize()
        assert _same(w, _results(b))
        eager = _block(seed=50)      # other work between the replays, on buffers of its own
        _run_block(eager)


def test_two_graphs_with_a_workspace_each_and_one_shared_in_turn():
    blocks = [_block(seed=20 + i) for i in range(2)]
    blocks[1]['ws'] = blocks[0]['ws']      # one after the other on one stream: shared
    want = []
    for b in blocks:
        _reset(b)
        _run_block(b)
        want.append(_results(b))
    torch.cuda.synchronize()
    graphs = []
    for b in blocks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b['rg'].buf.zero_()
            _run_block(b)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(_same(w, _results(b)) for w, b in zip(want, blocks))
