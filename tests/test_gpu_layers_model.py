"""group_normalize and [dropout] through Darknet on the device: a net with both in every position against the oracle (float32), the
recorded launch lists and captured steps against eager ones (bit for bit), the generator's state across engines."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
import complex_yolov4_pytorch_amd.synthetic as syn  # noqa: E402
from complex_yolov4_pytorch_amd.models.darknet2pytorch import Darknet  # noqa: E402
from complex_yolov4_pytorch_amd.models.darknet_utils import parse_cfg  # noqa: E402
from oracle import darknet_ref  # noqa: E402
from tests import layer_nets  # noqa: E402
from tests.util import grad_rel_errors  # noqa: E402

DEV = 'cuda'


def _model(path, dtype='f32', **kw):
    m = Darknet(path, use_giou_loss=True, dtype=dtype, **kw)
    sd = m.state_dict()
    sd.update({k: syn.fill_tensor(k, tuple(v.shape)) for k, v in sd.items() if v.dtype.is_floating_point})
    m.load_state_dict(sd)
    return m.to(DEV)


@pytest.mark.parametrize('p', [0.0, 0.25])
@pytest.mark.parametrize('deterministic', [False, True])
def test_training_and_evaluation_against_the_oracle(p, deterministic):
    path = layer_nets.cfg_path(p)
    model = _model(path, deterministic=deterministic)
    model.train()
    model.seed_dropout(1234, step=6)
    x, tg = syn.bev_images(2, 64, seed=5, sparsity=0.5), syn.targets(2, 3, 64, seed=5, collide=True)
    net = darknet_ref.DarknetRef(parse_cfg(path))
    ps, bs = net.param_shapes()
    params = {k: v.requires_grad_(True) for k, v in syn.fill_state_dict(ps).items()}
    bufs = syn.fill_state_dict(bs)
    for step in range(7, 11):      # (the third and fourth passes are replayed from recorded lists)
        loss, out = model(x.to(DEV), tg.to(DEV))
        loss.backward()
        o_ref, l_ref, _ = net.forward(params, x, tg, True, True, bufs, drop=(1234, step))
        l_ref.sum().backward()
        np.testing.assert_allclose(float(loss.detach()), float(l_ref.detach()), rtol=1e-4)
        np.testing.assert_allclose(out.cpu().numpy(), o_ref.detach().numpy(), rtol=2e-3, atol=2e-3)
    errs = grad_rel_errors([(n, q.grad.cpu()) for n, q in model.named_parameters()], {k: v.grad for k, v in params.items()})
    assert max(errs.values()) < 5e-3, sorted(errs.items(), key=lambda kv: -kv[1])[:5]
    assert sum(e.replayed for e in model._engines.values()) > 0
    if p:
        assert model.dropout_position() == (1234, 10)
    model.eval()
    with torch.no_grad():
        got = model(x.to(DEV))
        want = net.forward(params, x, None, True, False, bufs)[0]
        one = torch.cat([model(x[i:i + 1].to(DEV)) for i in range(2)])
    np.testing.assert_allclose(got.numpy(), want.detach().numpy(), rtol=2e-3, atol=2e-3)
    np.testing.assert_allclose(one.numpy(), got.numpy(), rtol=1e-3, atol=1e-3)


def _steps(model, batches):
    out = []
    for x, tg in batches:
        for q in model.parameters():
            q.grad = None
        loss, _ = model(x, tg)
        loss.backward()
        out.append((loss.detach().clone(), model.flat_grad.clone()))
    return out


@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
def test_recorded_lists_equal_eager_passes(monkeypatch, dtype):
    path = layer_nets.cfg_path(0.25)
    batches = [(syn.bev_images(2, 96, seed=i, sparsity=0.5).to(DEV), syn.targets(2, 3, 96, seed=i).to(DEV)) for i in range(5)]
    runs = []
    for replay in ('0', '1'):
        monkeypatch.setenv('CY_PLAN_REPLAY', replay)
        model = _model(path, dtype, deterministic=True)
        model.train()
        model.seed_dropout(3)
        runs.append(_steps(model, batches))
        eng = next(iter(model._engines.values()))
        assert (eng.replayed > 0) == (replay == '1')
        assert all(bool(torch.isfinite(g).all()) for _, g in runs[-1])
    for (la, ga), (lb, gb) in zip(*runs):
        assert torch.equal(la, lb) and torch.equal(ga, gb)


def test_masks_differ_from_step_to_step_and_follow_the_seed():
    path = layer_nets.cfg_path(0.25)
    b = [(syn.bev_images(2, 64, seed=1, sparsity=0.5).to(DEV), syn.targets(2, 3, 64, seed=1).to(DEV))] * 2
    model = _model(path, deterministic=True)
    model.train()
    model.seed_dropout(9)
    first = _steps(model, b)
    assert not torch.equal(first[0][0], first[1][0])
    model.seed_dropout(9)
    again = _steps(model, b)
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(first, again))
    model.seed_dropout(10)
    assert not torch.equal(_steps(model, b)[0][0], first[0][0])


def test_a_backward_pass_uses_its_own_forwards_masks():
    """Two geometries in flight: the second forward moves the model's counter, the first one's backward has kept its own."""
    path = layer_nets.cfg_path(0.25)
    a = (syn.bev_images(2, 64, seed=1, sparsity=0.5).to(DEV), syn.targets(2, 3, 64, seed=1).to(DEV))
    c = (syn.bev_images(1, 96, seed=2, sparsity=0.5).to(DEV), syn.targets(1, 3, 96, seed=2).to(DEV))
    model = _model(path, deterministic=True)
    model.train()
    model.seed_dropout(4)
    want = _steps(model, [a])[0]
    model.seed_dropout(4)
    for q in model.parameters():
        q.grad = None
    loss, _ = model(*a)
    model(*c)
    loss.backward()
    assert torch.equal(loss.detach(), want[0]) and torch.equal(model.flat_grad, want[1])


def test_captured_steps_equal_eager_steps():
    from complex_yolov4_pytorch_amd.graphed import GraphedTrainStep
    from complex_yolov4_pytorch_amd.optim import FusedAdam
    path = layer_nets.cfg_path(0.25)
    batches = [(syn.bev_images(2, 96, seed=40 + i, sparsity=0.5).to(DEV), syn.targets(2, 3, 96, seed=40 + i).to(DEV)) for i in range(5)]
    runs = []
    for graphed in (False, True):
        model = _model(path, 'f16', deterministic=True)
        model.train()
        model.seed_dropout(21)
        opt = FusedAdam(model.parameters(), lr=1e-3, capturable=True)

        def eager(x, tg, model=model, opt=opt):
            opt.zero_grad(set_to_none=True)
            loss, _ = model(x, tg)
            loss.backward()
            opt.step()
            return loss
        step = GraphedTrainStep(model, opt, warmup=1) if graphed else eager
        losses = []
        for x, tg in batches:
            losses.append(float(step(x, tg).detach()))
            torch.randn(1000, device=DEV).sum().item()      # (eager work between the replays)
        assert not graphed or step.replays == 4
        assert model.dropout_position() == (21, 5)
        runs.append((losses, copy.deepcopy({k: v.detach().clone() for k, v in model.state_dict().items()})))
    assert runs[0][0] == runs[1][0]
    for k, v in runs[0][1].items():
        assert torch.equal(v, runs[1][1][k]), k


def test_engine_buffers_are_not_left(monkeypatch):
    """Red zones around every engine buffer (the group norm workspace among them): intact, and the guarded run equals the plain one."""
    from complex_yolov4_pytorch_amd.models.engine import Engine
    path = layer_nets.cfg_path(0.25)
    b = [(syn.bev_images(2, 96, seed=i, sparsity=0.5).to(DEV), syn.targets(2, 3, 96, seed=i).to(DEV)) for i in range(3)]
    runs = []
    for guard in (0, 1 << 16):
        monkeypatch.setattr(Engine, 'GUARD_BYTES', guard)
        model = _model(path, 'f16', deterministic=True)
        model.train()
        model.seed_dropout(2)
        runs.append(_steps(model, b))
        if guard:
            assert [v for e in model._engines.values() for v in e.arena.violations()] == []
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(*runs))


def test_one_image_steps_and_another_stream():
    """Batch 1 -- what group norm is for -- on a stream of its own, equal to the same step on the default stream."""
    path = layer_nets.cfg_path(0.25)
    b = [(syn.bev_images(1, 128, seed=7, sparsity=0.5).to(DEV), syn.targets(1, 3, 128, seed=7).to(DEV))] * 3
    runs = []
    for own in (False, True):
        model = _model(path, 'bf16', deterministic=True)
        model.train()
        model.seed_dropout(2)
        s = torch.cuda.Stream() if own else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            runs.append(_steps(model, b))
        torch.cuda.synchronize()
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(*runs))
