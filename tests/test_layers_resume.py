"""The position of the [dropout] masks through checkpoints, models that have not run yet, and ranks."""
import pytest
import torch

import complex_yolov4_pytorch_amd.synthetic as syn
from complex_yolov4_pytorch_amd.models.darknet2pytorch import Darknet
from complex_yolov4_pytorch_amd.utils.train_utils import get_saved_state, save_checkpoint
from tests import layer_nets
from tests.util import mini_cfg_path

CPU = torch.device('cpu')


def _model(path=None):
    return Darknet(path or layer_nets.cfg_path(), use_giou_loss=True, dtype='f32')


def _saved(model, epoch=3):
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    return get_saved_state(model, opt, torch.optim.lr_scheduler.LambdaLR(opt, lambda e: 1.0), epoch, {'lr': 1e-3})


def test_the_position_of_a_new_model_can_be_taken_over():
    a, b = _model(), _model()
    b.seed_dropout(5, step=9)
    b.seed_dropout(*a.dropout_position())
    assert b.dropout_position() == (None, 0)
    torch.manual_seed(31)
    assert b._dropout_state(CPU).tolist() == [31, 0]
    b.seed_dropout(None, step=2)      # (beside a state that exists: the default seed again)
    assert b._dropout_state(CPU).tolist() == [31, 2]


def test_a_resumed_run_continues_the_masks(monkeypatch, tmp_path):
    layer_nets.install(monkeypatch)
    x, tg = syn.bev_images(1, 64, seed=5, sparsity=0.5), syn.targets(1, 3, 64, seed=5)

    def step(m):
        for p in m.parameters():
            p.grad = None
        loss, _ = m(x, tg)
        loss.backward()
        return float(loss.detach())
    first = _model()
    first.train()
    torch.manual_seed(12)
    losses = [step(first) for _ in range(2)]
    msd, usd = _saved(first)
    save_checkpoint(str(tmp_path), 'run', msd, usd, 3)
    losses += [step(first) for _ in range(2)]
    torch.manual_seed(99)
    second = _model()
    second.train()
    second.load_state_dict(torch.load(str(tmp_path / 'Model_run_epoch_3.pth')))
    second.seed_dropout(**torch.load(str(tmp_path / 'Utils_run_epoch_3.pth'), weights_only=True)['dropout'])
    # (no optimizer step: the parameters are the same throughout, the masks alone differ)
    assert [step(second) for _ in range(2)] == losses[2:] and len(set(losses)) == 4


def test_checkpoints_of_models_without_dropout_are_as_before():
    for path in (mini_cfg_path(), layer_nets.cfg_path(0.0)):
        assert set(_saved(_model(path))[1]) == {'epoch', 'configs', 'optimizer', 'lr_scheduler'}


def test_every_rank_of_a_resumed_run_has_its_own_masks(monkeypatch):
    """The checkpoint is rank 0's."""
    rank = [0]
    monkeypatch.setattr(torch.distributed, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.distributed, 'get_rank', lambda: rank[0])
    torch.manual_seed(77)
    before = []
    for r in range(3):
        rank[0] = r
        m = _model()
        before.append(m._dropout_state(CPU).tolist())
        m._dropout_state(CPU)[1] += 4
        if r == 0:
            state = _saved(m)[1]['dropout']
    assert state == {'seed': 77, 'step': 4, 'per_rank': True}
    torch.manual_seed(5)
    for r in range(3):
        rank[0] = r
        m = _model()
        m.seed_dropout(**state)
        assert m._dropout_state(CPU).tolist() == [before[r][0], 4]
    assert len({s for s, _ in before}) == 3
    # a seed that is given is every rank's, unless asked otherwise
    m.seed_dropout(8)
    assert m._dropout_state(CPU).tolist() == [8, 0] and m.dropout_position() == (8, 0)


@pytest.mark.parametrize('seed', [0, -1, 1 << 63, (1 << 64) - 1])
def test_positions_come_back_as_they_were_given(seed):
    m = _model()
    m.seed_dropout(seed, 7)
    assert m.dropout_position() == (seed, 7)
    assert int(m._dropout_state(CPU)[0]) % (1 << 64) == seed % (1 << 64)
