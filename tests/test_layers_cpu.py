"""Per-image layers without a GPU: the oracle's generator against published vectors and its gradients against differences, the
refusals of the operator layer and of the C ABI (all of them before any launch)."""
import ctypes

import numpy as np
import pytest
import torch

from complex_yolov4_pytorch_amd import _lib, ops
from complex_yolov4_pytorch_amd.ops import CY_BF16, CY_F16, CY_F32, View
from oracle import layers_ref as ref


@pytest.mark.parametrize('ctr,key,want', [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_generator_gives_the_published_vectors(ctr, key, want):
    got = ref.philox4x32(np.array([ctr], dtype=np.uint32), key)[0]
    assert tuple(int(v) for v in got) == want


def test_mask_share_and_independence():
    n = 1 << 16
    a = ref.keep_mask(n, 6554, 1234567890123456789, 3, 1)
    # 65536 draws of probability 0.1: standard deviation of the share 0.0012
    assert abs(float((~a).double().mean()) - 0.1) < 5 * 0.0012
    for other in (ref.keep_mask(n, 6554, 1234567890123456789, 4, 1), ref.keep_mask(n, 6554, 1234567890123456789, 3, 2),
                  ref.keep_mask(n, 6554, 1234567890123456788, 3, 1)):
        both = float((~a & ~other).double().mean())
        assert abs(both - 0.01) < 5 * 0.0004      # sqrt(0.01 * 0.99 / 65536)
    assert torch.equal(ref.keep_mask(64, 6554, 5, 6, 7, first=128), ref.keep_mask(192, 6554, 5, 6, 7)[128:])


@pytest.mark.parametrize('kind', [0, 1, 2])
def test_oracle_gradient_against_differences(kind):
    g = torch.Generator().manual_seed(3 + kind)
    x = torch.randn(2, 5, 6, generator=g, dtype=torch.float64)
    gamma, beta = 1 + 0.3 * torch.randn(6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 5, 6, generator=g, dtype=torch.float64)
    fac = ref.drop_factor((2, 5, 6), 20000, 11, 2, 4)
    loss = lambda x_, ga, be: float((ref.gn_act(x_, ga, be, 3, 1e-5, kind, fac)[0] * dy).sum())      # noqa: E731
    out = ref.gn_act_grad(x, dy, gamma, beta, 3, 1e-5, kind, fac)
    h = 1e-6

    def central(make):      # error of a central difference: third derivative * h^2 / 6 + 2^-52 * |loss| / h, both below 1e-8
        return (make(h) - make(-h)) / (2 * h)
    for i in [(0, 0, 0), (0, 3, 5), (1, 2, 2), (1, 4, 3)]:
        e = torch.zeros_like(x)
        e[i] = 1
        assert abs(central(lambda d: loss(x + d * e, gamma, beta)) - float(out['dx'][i])) < 1e-6
    for c in range(6):
        e = torch.zeros(6, dtype=torch.float64)
        e[c] = 1
        assert abs(central(lambda d: loss(x, gamma + d * e, beta)) - float(out['ggamma'][c])) < 1e-6
        assert abs(central(lambda d: loss(x, gamma, beta + d * e)) - float(out['gbeta'][c])) < 1e-6


# ---- C ABI: rejected before any launch -------------------------------------------------------------------

P = ctypes.c_void_p(4096)      # never dereferenced: every call below is refused


def _fwd(x=P, ldx=16, y=P, ldy=16, res=None, ldres=0, N=1, HW=4, C=16, G=4, gamma=P, beta=P, eps=1e-5, act=2, dt=0, stats=P, q=0, rng=None,
         id=0, ws=P, nb=1 << 20):
    return _lib.lib().raw('cy_gn_act_fwd')(x, ldx, y, ldy, res, ldres, N, HW, C, G, gamma, beta, eps, act, dt, stats, q, rng, id, ws, nb, None)


def _bwd(x=P, ldx=16, dy=P, lddy=16, dx=P, lddx=16, rg=None, ldrg=0, acc=0, N=1, HW=4, C=16, G=4, gamma=P, beta=P, stats=P, act=2, dt=0,
         gg=P, gb=P, gs=1.0, accumulate=0, q=0, rng=None, id=0, ws=P, nb=1 << 20):
    return _lib.lib().raw('cy_gn_act_bwd')(x, ldx, dy, lddy, dx, lddx, rg, ldrg, acc, N, HW, C, G, gamma, beta, stats, act, dt, gg, gb, gs,
                                           accumulate, q, rng, id, ws, nb, None)


BAD_SIZES = [dict(N=-1), dict(HW=-1), dict(C=0), dict(G=0), dict(G=3), dict(G=32), dict(ldx=15), dict(act=3), dict(act=-1), dict(dt=3),
             dict(q=-1, rng=P), dict(q=65537, rng=P), dict(q=5), dict(gamma=None), dict(beta=None), dict(ws=None), dict(nb=8),
             dict(x=None), dict(x=ctypes.c_void_p(4097)), dict(ws=ctypes.c_void_p(4100))]


@pytest.mark.parametrize('bad', BAD_SIZES + [dict(ldy=15), dict(y=None), dict(res=P, ldres=15), dict(eps=-1.0), dict(eps=float('nan')),
                                             dict(stats=ctypes.c_void_p(4100)), dict(y=ctypes.c_void_p(4097)),
                                             dict(N=1 << 30, HW=1, G=16, nb=1 << 62)])
def test_forward_refusals(bad):
    assert _fwd(**bad) == -1


@pytest.mark.parametrize('bad', BAD_SIZES + [dict(lddy=15), dict(lddx=15), dict(rg=P, ldrg=15), dict(dy=None), dict(dx=None), dict(stats=None),
                                             dict(dy=ctypes.c_void_p(4097)), dict(dx=ctypes.c_void_p(4099))])
def test_backward_refusals(bad):
    assert _bwd(**bad) == -1


@pytest.mark.parametrize('bad', [dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(M=-1), dict(C=0), dict(q=-1), dict(q=65537),
                                 dict(rng=None), dict(dt=3), dict(x=ctypes.c_void_p(4097)), dict(y=ctypes.c_void_p(4097))])
def test_dropout_refusals(bad):
    a = dict(x=P, ldx=8, y=P, ldy=8, M=4, C=8, q=100, rng=P, id=0, acc=0, dt=0)
    a.update(bad)
    assert _lib.lib().raw('cy_dropout')(a['x'], a['ldx'], a['y'], a['ldy'], a['M'], a['C'], a['q'], a['rng'], a['id'], a['acc'], a['dt'], None) == -1


def test_nothing_to_do_is_no_error():
    assert _fwd(N=0, x=None, y=None, ws=None) == 0 and _fwd(HW=0, x=None, y=None, ws=None) == 0
    assert _bwd(N=0, x=None, dy=None, dx=None, accumulate=1) == 0
    assert _lib.lib().raw('cy_dropout')(None, 8, None, 8, 0, 8, 5, P, 0, 0, 0, None) == 0


def test_workspace_sizes():
    raw = _lib.lib().raw('cy_gn_workspace')
    for bad in ((-1, 4, 8, 2, 0), (1, -1, 8, 2, 0), (1, 4, 8, 3, 0), (1, 4, 0, 1, 0), (1, 4, 8, 0, 0), (1, 4, 8, 2, 5)):
        assert raw(*bad) == -1
    for dt in (CY_F16, CY_BF16, CY_F32):
        for N, HW, C, G in ((1, 1, 1, 1), (1, 361, 1024, 32), (16, 608 * 608, 32, 8), (3, 3225, 30, 6), (32, 4, 1024, 1), (65536, 1, 8, 8)):
            n = raw(N, HW, C, G, dt)
            assert 0 < n < 8 * N * C * (HW + 2) + 8 * N * G + (64 << 20)


# ---- operator layer: refused on the host -----------------------------------------------------------------

@pytest.fixture
def on_cpu(monkeypatch):
    """The operator layer's checks with host tensors standing in for device tensors; a call that reaches the library fails the test."""
    monkeypatch.setattr(ops, '_require_gpu', lambda: None)
    monkeypatch.setattr(ops, 'check_device_tensor', lambda t, who: None)
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: -1)      # what a host tensor's get_device() says

    class NoCalls:
        def call(self, name, *a):
            raise AssertionError('%s was called' % name)

        def raw(self, name):
            return _lib.lib().raw(name)
    monkeypatch.setattr(ops, 'lib', lambda: NoCalls())


def _v(N=2, H=3, W=3, C=8, ld=None, dt=CY_F16, off=0, n=None):
    ld = ld or C
    t = ops.torch_dtype(dt)
    return View(torch.zeros(n if n is not None else off + N * H * W * ld, dtype=t), off, N, H, W, C, ld, dt)


def _gn(**kw):
    a = dict(x=_v(), y=_v(), res=None, gamma=torch.ones(8), beta=torch.zeros(8), groups=2, eps=1e-5, act=2, stats=torch.zeros(2, 2, 2),
             ws=torch.zeros(1 << 16, dtype=torch.uint8), drop=0.0, rng=None, drop_id=0)
    a.update(kw)
    ops.gn_act_fwd(**a)


def _gnb(**kw):
    a = dict(x=_v(), dy=_v(), dx=_v(), res_grad=None, res_accum=False, gamma=torch.ones(8), beta=torch.zeros(8), stats=torch.zeros(2, 2, 2),
             groups=2, act=2, ggamma=torch.zeros(8), gbeta=torch.zeros(8), gscale=1.0, accumulate=True, ws=torch.zeros(1 << 16, dtype=torch.uint8),
             drop=0.0, rng=None, drop_id=0)
    a.update(kw)
    ops.gn_act_bwd(**a)


STATE = torch.zeros(2, dtype=torch.int64)
COMMON = [dict(groups=3), dict(groups=0), dict(act=3), dict(act='mish'), dict(gamma=torch.ones(7)), dict(gamma=torch.ones(8).half()),
          dict(beta=None), dict(beta=torch.zeros(16)[::2]), dict(stats=torch.zeros(2, 2)), dict(x=_v(H=4)), dict(x=_v(dt=CY_BF16)),
          dict(x=_v(n=100)), dict(x=_v(off=-8)), dict(x=_v(ld=7, n=1000)), dict(ws=None), dict(drop=0.5), dict(drop=1.5, rng=STATE),
          dict(drop=-0.1, rng=STATE), dict(drop=float('nan'), rng=STATE), dict(drop=0.5, rng=torch.zeros(2)), dict(drop=0.5, rng=torch.zeros(3, dtype=torch.int64))]


@pytest.mark.parametrize('kw', COMMON + [dict(res=_v(C=16)), dict(y=_v(N=1)), dict(eps=-1.0), dict(eps=float('nan'))])
def test_operator_layer_refuses_forward(on_cpu, kw):
    with pytest.raises(ops.CyoloError):
        _gn(**kw)


@pytest.mark.parametrize('kw', COMMON + [dict(stats=None), dict(dy=_v(W=4)), dict(dx=_v(dt=CY_F32)), dict(res_grad=_v(C=16)), dict(ggamma=torch.zeros(4)),
                                         dict(gbeta=torch.zeros(8).double())])
def test_operator_layer_refuses_backward(on_cpu, kw):
    with pytest.raises(ops.CyoloError):
        _gnb(**kw)


@pytest.mark.parametrize('kw', [dict(rng=None), dict(p=1.01), dict(p=-0.01), dict(rng=torch.zeros(2)), dict(y=_v(C=16)), dict(y=_v(dt=CY_F32))])
def test_operator_layer_refuses_dropout(on_cpu, kw):
    for fn in (lambda x, y, p, rng: ops.dropout_fwd(x, y, p, rng), lambda x, y, p, rng: ops.dropout_bwd(x, y, True, p, rng)):
        a = dict(x=_v(), y=_v(), p=0.3, rng=STATE)
        a.update(kw)
        with pytest.raises(ops.CyoloError):
            fn(**a)


def test_another_device_than_the_current_one_is_refused(on_cpu, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 1)
    for call in (_gn, _gnb, lambda: ops.dropout_fwd(_v(), _v(), 0.5, STATE)):
        with pytest.raises(ops.CyoloError, match='current device'):
            call()


def test_probability_is_resolved_to_65536ths():
    assert [ops.dropout_q(p) for p in (0, 0.1, 0.25, 0.5, 1.0, 2.0 ** -17, 2.0 ** -18)] == [0, 6554, 16384, 32768, 65536, 1, 0]


def test_state_takes_any_64_bit_seed():
    for seed in (0, 1, (1 << 63) - 1, 1 << 63, (1 << 64) - 1):
        assert int(ops.dropout_state(seed, 'cpu', step=5)[0]) % (1 << 64) == seed
    assert ops.dropout_state(3, 'cpu', step=5).tolist() == [3, 5]


@pytest.mark.skipif(torch.cuda.is_available(), reason='checks the no-device behaviour')
def test_no_cpu_fallback():
    with pytest.raises(ops.CyoloError):
        _gn()
    with pytest.raises(ops.CyoloError):
        ops.dropout_fwd(_v(), _v(), 0.5, STATE)
