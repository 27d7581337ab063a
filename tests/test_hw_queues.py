"""The number of hardware queues: one rule for every program that imports the package, bench.py among them, with a way to keep one's own."""
import os
import subprocess
import sys

import pytest

import complex_yolov4_pytorch_amd as pkg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CASES = [({}, '8'), ({'GPU_MAX_HW_QUEUES': '4'}, '4'), ({'GPU_MAX_HW_QUEUES': '4', 'WORLD_SIZE': '1'}, '4'),
         ({'GPU_MAX_HW_QUEUES': '4', 'WORLD_SIZE': '8'}, '8'), ({'GPU_MAX_HW_QUEUES': '4', 'CY_DDP_FORCE': '1'}, '8'),
         ({'GPU_MAX_HW_QUEUES': '4', 'CY_DDP_FORCE': '1', 'CY_KEEP_HW_QUEUES': '1'}, '4'), ({'CY_KEEP_HW_QUEUES': '1'}, None),
         ({'GPU_MAX_HW_QUEUES': '6', 'WORLD_SIZE': '8'}, '6'), ({'GPU_MAX_HW_QUEUES': '4', 'WORLD_SIZE': ''}, '4')]


@pytest.mark.parametrize('env,want', CASES)
def test_rule(env, want):
    env = dict(env)
    pkg._hardware_queues(env)
    assert env.get('GPU_MAX_HW_QUEUES') == want


@pytest.mark.parametrize('module', ['bench', 'complex_yolov4_pytorch_amd'])
@pytest.mark.parametrize('case', [4, 5])
def test_programs_follow_it(module, case):
    add, want = CASES[case]
    env = {k: v for k, v in os.environ.items() if k not in ('GPU_MAX_HW_QUEUES', 'WORLD_SIZE', 'CY_DDP_FORCE', 'CY_KEEP_HW_QUEUES')}
    out = subprocess.run([sys.executable, '-c', 'import os, %s; print(os.environ.get("GPU_MAX_HW_QUEUES"))' % module], cwd=ROOT, env={**env, **add},
                         capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.split()[-1] == want, out.stderr
