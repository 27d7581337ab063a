"""Cfgs with group_normalize / [dropout] blocks in every position the plan treats differently, and the CPU restatement of the layer
operators for tests/opsim.py's kind of run (test infrastructure only)."""
import os
import tempfile

import torch

import complex_yolov4_pytorch_amd.ops as real
from oracle import layers_ref
from tests import opsim
from tests.util import _yolo


def _conv(f, k, s=1, act='mish', bn=0, gn=0):
    return ('[convolutional]\n' + ('batch_normalize=1\n' if bn else '') + ('group_normalize=%d\n' % gn if gn else '') +
            'filters=%d\nsize=%d\nstride=%d\npad=1\nactivation=%s\n' % (f, k, s, act))


def _drop(p):
    return '[dropout]\nprobability=%s\n' % p


# module index in the comment; grids are S/4 (head 1) and S/2 (head 2).  {p}: drop probability
BLOCKS = [
    '[net]\nwidth=64\nheight=64\nchannels=3\n',
    _conv(32, 3, 1, gn=8),                             # 0   first layer, group norm
    _conv(32, 3, 2, bn=1),                             # 1   S/2, batch norm between group norms
    _conv(64, 3, 2, gn=32),                            # 2   S/4, two channels to a group
    _conv(32, 1, gn=4),                                # 3
    _conv(64, 3, gn=16),                               # 4
    '[shortcut]\nfrom=-3\nactivation=linear\n',        # 5   4 + 2 (folded into 4's pass)
    _conv(64, 1, gn=1),                                # 6   one group
    '{drop}',                                          # 7   folded into 6
    _conv(64, 3, gn=64),                               # 8   a group per channel
    '{drop}',                                          # 9   folded into 8 ...
    '[shortcut]\nfrom=-3\nactivation=linear\n',        # 10  ... and 8 + 7 with it
    _conv(32, 1, bn=1),                                # 11
    '{drop}',                                          # 12  behind a batch norm: a pass of its own
    '[route]\nlayers=-1,-3\n',                         # 13  cat(12, 10)
    '{drop}',                                          # 14  behind a concatenation
    _conv(64, 1, gn=8),                                # 15
    '[maxpool]\nstride=1\nsize=5\n',                   # 16
    '{drop}',                                          # 17
    '[route]\nlayers=-1,-3\n',                         # 18  cat(17, 15)
    _conv(64, 1, gn=8, act='leaky'),                   # 19
    _conv(30, 1, act='linear'),                        # 20
    _yolo('3,4,5'),                                    # 21
    '[route]\nlayers=-3\n',                            # 22  -> 19
    _conv(32, 1, gn=2, act='linear'),                  # 23  no activation
    '[upsample]\nstride=2\n',                          # 24  S/2
    '[route]\nlayers=-1,1\n',                          # 25  cat(24, 1)
    _conv(64, 3, gn=8),                                # 26
    '{drop}',                                          # 27
    _conv(30, 1, act='linear'),                        # 28
    _yolo('0,1,2'),                                    # 29
]


def cfg_path(p=0.25, tag=''):
    path = os.path.join(tempfile.gettempdir(), 'cyolo_layers_%d_%s%s.cfg' % (os.getpid(), p, tag))
    with open(path, 'w') as f:
        f.write('\n'.join(_drop(p) if b == '{drop}' else b for b in BLOCKS))
    return path


def write_cfg(blocks, tag):
    path = os.path.join(tempfile.gettempdir(), 'cyolo_layers_%d_%s.cfg' % (os.getpid(), tag))
    with open(path, 'w') as f:
        f.write('\n'.join(blocks))
    return path


# ---- operator layer on the CPU -------------------------------------------------------------------------

def _rows(v):
    return opsim._t(v).reshape(v.N, v.H * v.W, v.C)


def _put(v, t, accumulate=False):
    dst = opsim._t(v)
    t = t.reshape(v.N, v.H, v.W, v.C)
    dst.copy_((dst.double() + t if accumulate else t).to(dst.dtype))


def _factor(v, p, rng, layer):
    q = real.dropout_q(p)
    if not q:
        return 1.0
    return layers_ref.drop_factor((v.N, v.H * v.W, v.C), q, int(rng[0]) % (1 << 64), int(rng[1]), layer)


def gn_act_fwd(x, y, res, gamma, beta, groups, eps, act, stats, ws, drop=0.0, rng=None, drop_id=0):
    out, n = layers_ref.gn_act(_rows(x), gamma, beta, groups, eps, act, _factor(x, drop, rng, drop_id), None if res is None else _rows(res))
    if stats is not None:
        stats.copy_(torch.stack((n['mean'], n['rstd']), -1).float())
    _put(y, out)


def gn_act_bwd(x, dy, dx, res_grad, res_accum, gamma, beta, stats, groups, act, ggamma, gbeta, gscale, accumulate, ws, drop=0.0, rng=None,
               drop_id=0):
    g = _rows(dy).clone()
    o = layers_ref.gn_act_grad(_rows(x), g, gamma, beta, groups, 1e-5, act, _factor(x, drop, rng, drop_id))
    assert torch.allclose(stats[..., 0].double(), o['mean'], atol=1e-5), 'statistics of another forward pass'
    if res_grad is not None:
        _put(res_grad, g.double(), accumulate=bool(res_accum))
    _put(dx, o['dx'])
    for t, v in ((ggamma, o['ggamma']), (gbeta, o['gbeta'])):
        if t is not None:
            t.copy_((t.double() if accumulate else 0) + gscale * v)


def dropout_fwd(x, y, p, rng, drop_id=0):
    _put(y, _rows(x).double() * _factor(x, p, rng, drop_id))


def dropout_bwd(dy, dx, accumulate, p, rng, drop_id=0):
    _put(dx, _rows(dy).double() * _factor(dy, p, rng, drop_id), accumulate=bool(accumulate))


def install(monkeypatch):
    opsim.install(monkeypatch)
    for n in ('gn_act_fwd', 'gn_act_bwd', 'dropout_fwd', 'dropout_bwd'):
        monkeypatch.setattr(real, n, globals()[n])
