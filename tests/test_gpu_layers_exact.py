"""Group norm + activation where the result is known to the last bits: groups of one value, values a few steps of the type apart beside a
large mean, and the derivative of mish far below zero.  e = 2^-24 is half a step of float32; storage adds half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
from complex_yolov4_pytorch_amd.ops import CY_BF16, CY_F16, CY_F32  # noqa: E402
from oracle import layers_ref as ref  # noqa: E402
from tests.test_gpu_layers import DEV, E, EPS, Strided, _close, _gen, _stored, _workspace, kernels  # noqa: E402, F401

TYPES = pytest.mark.parametrize('dt', [CY_F16, CY_BF16, CY_F32], ids=['f16', 'bf16', 'f32'])
ACTS = pytest.mark.parametrize('act', [0, 1, 2], ids=['linear', 'leaky', 'mish'])
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


@SHAPES
@ACTS
@TYPES
def test_groups_of_one_value(shape, dt, act, kernels):  # noqa: F811
    """A dead group: x - mean is 0, so z is beta and what is left is the activation (an exponential and a reciprocal at 1 - 2 e each, five
    operations: 16 e) and storage, however large the value beside the deviation of sqrt(eps)."""
    N, H, W, C, G = shape
    t = ops.torch_dtype(dt)
    _, x = _one_value_groups(N, H * W, C, G, t)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=_gen(2)), 0.3 * torch.randn(C, generator=_gen(3))
    dy = torch.randn(N, H * W, C, generator=_gen(4)).to(t)
    xs, ys, dys, dxs = Strided(N, H, W, C, dt, fill=x), Strided(N, H, W, C, dt), Strided(N, H, W, C, dt, fill=dy), Strided(N, H, W, C, dt)
    stats, ws, gg = torch.empty(N, G, 2, device=DEV), _workspace(N, H, W, C, G, dt), torch.empty(2, C, device=DEV)
    ga, be = gamma.to(DEV), beta.to(DEV)
    ops.gn_act_fwd(xs.view, ys.view, None, ga, be, G, EPS, act, stats, ws)
    want = ref.act(beta.double(), act).expand(N, H * W, C)
    _close(ys.get(), want, _stored(want, dt) + 16 * E * beta.double().abs(), 'y')
    # gradient: xh is 0.  A block's sum takes at most 64 additions in a row (this file's sizes), the rest is in double
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, ga, be, stats, G, act, gg[0], gg[1], 1.0, False, ws)
    assert float(gg[0].abs().max()) == 0
    slope = ref.act_grad(beta.double(), act)
    dz = dy.double() * slope
    dze = 16 * E * dy.double().abs() * (slope.abs() + beta.double().abs() * (act == 2))
    _close(gg[1].cpu(), dz.sum((0, 1)), (dze + 64 * E * dz.abs()).sum((0, 1)), 'gbeta')
    grp = lambda a: a.reshape(N, H * W, G, -1)      # noqa: E731
    h, he = grp(dz * gamma.double()), grp(dze * gamma.double().abs())
    dx = R * (h - h.mean((1, 3), keepdim=True))
    tol = R * (he + he.mean((1, 3), keepdim=True) + 80 * E * (h.abs() + h.abs().mean((1, 3), keepdim=True)))
    _close(dxs.get(), dx.reshape(N, H * W, C), tol.reshape(N, H * W, C) + _stored(dx.reshape(N, H * W, C), dt), 'dx')


@SHAPES
@ACTS
@TYPES
def test_outputs_beside_a_large_mean(shape, dt, act, kernels):  # noqa: F811
    """Values up to seven steps of the type apart at 1024.  The mean is a float32 number: e |mean| of its own rounding and as much again from
    the means of blocks; x - mean takes e of the distance, the rest is as everywhere (16 e of the terms)."""
    N, H, W, C, G = shape
    step = {CY_F16: 2.0 ** -10, CY_BF16: 2.0 ** -7, CY_F32: 2.0 ** -23}[dt] * 1024
    x = (1024 + step * torch.randint(0, 8, (N, H * W, C), generator=_gen(5)).double()).to(ops.torch_dtype(dt))
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=_gen(2)), 0.3 * torch.randn(C, generator=_gen(3))
    xs, ys = Strided(N, H, W, C, dt, fill=x), Strided(N, H, W, C, dt)
    ops.gn_act_fwd(xs.view, ys.view, None, gamma.to(DEV), beta.to(DEV), G, EPS, act, None, _workspace(N, H, W, C, G, dt))
    want, n = ref.gn_act(x, gamma, beta, G, EPS, act)
    per_c = lambda t: t.repeat_interleave(C // G, -1)[:, None, :]      # noqa: E731
    xe = 2 * E * per_c(n['mean'].abs() * n['rstd']) + (64 + 512) * E * n['xh'].abs()      # (r: 512 e, as the statistics' own test has it)
    ze = xe * gamma.double().abs() + 16 * E * ((n['xh'] * gamma.double()).abs() + beta.double().abs())
    _close(ys.get(), want, _stored(want, dt) + 1.1 * ze + 16 * E * want.abs(), 'y')


@TYPES
def test_mish_derivative_below_zero(dt, kernels):  # noqa: F811
    """gamma = 0 makes z = beta.  mish' = tanh s + z (1 - tanh^2 s) sigmoid(z), s = log(1 + e^z): far below zero both terms are e^z times a
    small power of z and of one sign, so nothing may cancel.  e^z: the exponent z log2(e) is rounded twice (2 |z| e of e^z), an
    exponential and a reciprocal at 2 e, eight operations: (2 |z| + 16) e of the two terms' sum.  The hardware's exponential is 0
    below 2^-126."""
    z = torch.cat([torch.linspace(-20, 3, 93), torch.linspace(-110, -20.5, 35)])
    C, HW = z.numel(), 6
    sign = torch.tensor([1.0, -1.0] * 3)
    x = sign[None, :, None].repeat(1, 1, C).to(ops.torch_dtype(dt))                         # xh = +-1 / sqrt(1 + eps) in every channel
    dy = torch.tensor([1.0, -0.5] * 3)[None, :, None].repeat(1, 1, C).to(ops.torch_dtype(dt))
    xs, dys, dxs = Strided(1, HW, 1, C, dt, fill=x), Strided(1, HW, 1, C, dt, fill=dy), Strided(1, HW, 1, C, dt)
    stats, ws, gg = torch.empty(1, C, 2, device=DEV), _workspace(1, HW, 1, C, C, dt), torch.empty(2, C, device=DEV)
    ga, be = torch.zeros(C, device=DEV), z.to(DEV)
    ops.gn_act_fwd(xs.view, dxs.view, None, ga, be, C, EPS, 2, stats, ws)
    ops.gn_act_bwd(xs.view, dys.view, dxs.view, None, False, ga, be, stats, C, 2, gg[0], gg[1], 1.0, False, ws)
    zd = z.double()
    n = zd.exp()
    w = n * (n + 2)
    t = w / (w + 2)
    second = zd * (4 * (w + 1) / (w + 2) ** 2) * torch.sigmoid(zd)      # (1 - tanh^2 = 4 (w + 1) / (w + 2)^2)
    slope = t + second
    xh = 1 / (1 + EPS) ** 0.5
    tol = (2 * zd.abs() + 16) * E * (t + second.abs()) + 120 * 2.0 ** -126
    _close(gg[1].cpu(), 1.5 * slope, 3 * 1.5 * tol + 8 * E * slope.abs(), 'gbeta')
    _close(gg[0].cpu(), 4.5 * slope * xh, 4.5 * (tol + 8 * E * slope.abs()), 'ggamma')
