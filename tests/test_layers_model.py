"""group_normalize and [dropout] through the cfg, the plan and the engine, on a CPU restatement of the operator layer: lowering, buffer
wiring, gradient fan-in, state dict, .weights files, the generator's position.  float32 on both sides."""
import numpy as np
import pytest
import torch

import complex_yolov4_pytorch_amd.synthetic as syn
from complex_yolov4_pytorch_amd.models.darknet2pytorch import Darknet
from complex_yolov4_pytorch_amd.models.darknet_utils import parse_cfg
from complex_yolov4_pytorch_amd.models.graph import Plan
from oracle import darknet_ref
from tests import layer_nets
from tests.util import grad_rel_errors


def _model(path, **kw):
    m = Darknet(path, use_giou_loss=True, dtype='f32', **kw)
    sd = m.state_dict()
    sd.update({k: syn.fill_tensor(k, tuple(v.shape)) for k, v in sd.items() if v.dtype.is_floating_point})
    m.load_state_dict(sd)
    return m


def test_plan_of_the_layer_cfg():
    plan = Plan(parse_cfg(layer_nets.cfg_path()), 64, 64, 4)
    by = {r['idx']: r for r in plan.fwd if r['op'] == 'conv'}
    assert plan.has_dropout and plan.dropped_by == {7: 6, 9: 8, 27: 26}
    assert plan.fused_into == {4: 5, 8: 10}
    assert [r['idx'] for r in plan.fwd if r['op'] == 'dropout'] == [12, 14, 17]
    assert [(by[i]['drop'], by[i]['drop_id']) for i in (6, 8, 26, 15)] == [(0.25, 7), (0.25, 9), (0.25, 27), (0.0, 0)]
    assert by[8]['res'] is by[6]['out'] and plan.out[10] is by[8]['out'] and plan.out[9] is None
    # batch norm's sums may still ride on a group-normalised neighbour's input gradient, never the other way round
    for b in plan.bwd:
        for L in b.get('dx_sums', {}).values():
            assert L['bn']
        if b['op'] == 'conv_bwd' and b['fwd']['gn']:
            assert b['sums_from'] is None
    assert not Plan(parse_cfg(layer_nets.cfg_path(0.0)), 64, 64, 4).has_dropout


@pytest.mark.parametrize('bad', [
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(32, 3, bn=1, gn=4)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(32, 3, gn=5)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(32, 3, gn=-1)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._drop(0.5)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(32, 3, gn=4), layer_nets._drop(1.0)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(32, 3, gn=4), layer_nets._drop(-0.1)],
    ['[net]\nwidth=64\nheight=64\nchannels=3\n', layer_nets._conv(30, 1, act='linear'), layer_nets._drop(0.5)],
], ids=['both norms', 'groups', 'negative', 'first', 'p1', 'negative p', 'head'])
def test_cfg_refusals(bad):
    with pytest.raises(ValueError):
        Plan(parse_cfg(layer_nets.write_cfg(bad, 'bad')), 64, 64, 4)


@pytest.mark.parametrize('p', [0.0, 0.25])
@pytest.mark.parametrize('dgrad_sums', [0, 2])
def test_training_step_against_the_oracle(monkeypatch, p, dgrad_sums):
    layer_nets.install(monkeypatch)
    monkeypatch.setenv('CY_DGRAD_BN_SUMS', str(dgrad_sums))
    path = layer_nets.cfg_path(p)
    model = _model(path)
    model.train()
    model.seed_dropout(1234, step=6)
    x, tg = syn.bev_images(2, 64, seed=5, sparsity=0.5), syn.targets(2, 3, 64, seed=5, collide=True)
    net = darknet_ref.DarknetRef(parse_cfg(path))
    ps, bs = net.param_shapes()
    params = {k: v.requires_grad_(True) for k, v in syn.fill_state_dict(ps).items()}
    bufs = syn.fill_state_dict(bs)
    for step in (7, 8):      # (the step counts training forwards: other masks every time; gradients accumulate)
        loss, out = model(x, tg)
        loss.backward()
        o_ref, l_ref, _ = net.forward(params, x, tg, True, True, bufs, drop=(1234, step))
        l_ref.sum().backward()
        np.testing.assert_allclose(float(loss.detach()), float(l_ref.detach()), rtol=1e-4)
        np.testing.assert_allclose(out.numpy(), o_ref.detach().numpy(), rtol=2e-3, atol=2e-3)
    errs = grad_rel_errors([(n, q.grad) for n, q in model.named_parameters()], {k: v.grad for k, v in params.items()})
    assert max(errs.values()) < 5e-3, sorted(errs.items(), key=lambda kv: -kv[1])[:5]
    if p:
        assert model.dropout_position() == (1234, 8)
    # evaluation: no dropout, no statistics of the batch
    model.eval()
    with torch.no_grad():
        got = model(x).clone()      # (on the CPU the result is the engine's own buffer)
        want = net.forward(params, x, None, True, False, bufs)[0]
    np.testing.assert_allclose(got.numpy(), want.detach().numpy(), rtol=2e-3, atol=2e-3)
    one = torch.cat([model(x[i:i + 1]).clone() for i in range(2)])
    np.testing.assert_allclose(one.numpy(), got.numpy(), rtol=1e-4, atol=1e-4)


def test_training_mode_without_targets(monkeypatch):
    layer_nets.install(monkeypatch)
    path = layer_nets.cfg_path()
    model = _model(path)
    model.train()
    model.seed_dropout(5)
    net = darknet_ref.DarknetRef(parse_cfg(path))
    ps, bs = net.param_shapes()
    x = syn.bev_images(1, 64, seed=2, sparsity=0.5)
    with torch.no_grad():
        want = net.forward(syn.fill_state_dict(ps), x, None, True, True, syn.fill_state_dict(bs), drop=(5, 1))[0]
        np.testing.assert_allclose(model(x).numpy(), want.numpy(), rtol=2e-3, atol=2e-3)


def test_state_dict_and_weights_file(monkeypatch, tmp_path):
    path = layer_nets.cfg_path()
    model = _model(path)
    net = darknet_ref.DarknetRef(parse_cfg(path))
    ps, bs = net.param_shapes()
    sd = model.state_dict()
    assert set(ps) | set(bs) <= set(sd) and 'models.0.gn1.weight' in sd and 'models.0.conv1.bias' not in sd
    f = tmp_path / 'w.weights'
    model.save_weights(str(f))
    other = Darknet(path, use_giou_loss=True, dtype='f32')
    n = other.load_weights(str(f))
    assert n == sum(v.numel() for k, v in sd.items() if v.dtype.is_floating_point)
    for k, v in other.state_dict().items():
        if v.dtype.is_floating_point:
            assert torch.equal(v, sd[k]), k


def test_dropout_position_and_default_seed(monkeypatch):
    model = _model(layer_nets.cfg_path())
    assert model.dropout_position() == (None, 0)
    torch.manual_seed(77)
    st = model._dropout_state(torch.device('cpu'))
    assert st.tolist() == [77, 0]
    st[1] += 3
    assert model.dropout_position() == (77, 3)
    again = _model(layer_nets.cfg_path())
    again.seed_dropout(*model.dropout_position())
    assert again._dropout_state(torch.device('cpu')).tolist() == [77, 3]
    monkeypatch.setattr(torch.distributed, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.distributed, 'get_rank', lambda: 3)
    third = _model(layer_nets.cfg_path())
    assert int(third._dropout_state(torch.device('cpu'))[0]) % (1 << 64) == (77 + 3 * 0x9E3779B97F4A7C15) % (1 << 64)


def test_optimizer_groups_take_the_new_parameters(monkeypatch):
    from complex_yolov4_pytorch_amd.utils.train_utils import create_optimizer

    class C:
        optimizer_type, lr, momentum, weight_decay, fused_optimizer = 'adam', 1e-3, 0.9, 5e-4, False
    model = _model(layer_nets.cfg_path())
    groups = create_optimizer(C, model).param_groups
    name = {id(q): n for n, q in model.named_parameters()}
    kinds = [sorted({name[id(q)].split('.')[2].rstrip('0123456789') + '.' + name[id(q)].split('.')[3] for q in g['params']}) for g in groups]
    assert kinds == [['bn.weight', 'gn.weight'], ['conv.weight'], ['bn.bias', 'conv.bias', 'gn.bias']]
    assert [g['weight_decay'] for g in groups] == [0, 5e-4, 0]
