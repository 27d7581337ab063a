#!/usr/bin/env python3
"""Headline benchmark: BEV images/s of a 608x608 Complex-YOLOv4 TRAIN step.

  python bench.py --gpus N --steps K --warmup W [--config train608|infer32|train1024] [--dtype f16|bf16|f32]
  N > 1: either under the launcher (python -m torch.distributed.run --nnodes=1 --nproc-per-node N --master-addr 127.0.0.1
  --master-port P bench.py --gpus N ...; RANK / LOCAL_RANK / WORLD_SIZE / MASTER_* from the environment) or plainly as
  `python bench.py --gpus N`: without WORLD_SIZE in the environment the script starts its own N ranks (one process per GPU,
  the reference's mp.spawn in src/train.py:46-52) and rank 0 prints the line.

train608 (default): one step = forward + GIoU loss + backward + Adam update of complex_yolov4.cfg on a
fixed synthetic batch of 16 BEV images per GPU; inputs are resident in HBM before the timed region.  Weak scaling: every
rank runs its own 16 images, gradients are averaged over RCCL (parallel.RcclDataParallel).  Rank 0 prints ONE JSON line
with `roofline` (the implicit-GEMM conv kernel family, timed with HIP events on its launch stream) and `cpu_baseline`
(the oracle -- a CPU restatement of the reference -- timed on this host's cores on a bounded sample).
infer32: model.eval()(imgs) + post_processing_v2 (rotated merge-NMS on the device), batch 32.
train1024: the train step at 1024x1024, batch 8.
The default single-GPU run also measures the other configurations briefly -- each in a fresh process of this same script -- and
reports them under `other_configs`, so the one driver line carries configs[1], [3], [4] and configs[2]'s per-GPU work.

Process layout (round 5): the command is a SUPERVISOR without a GPU context; everything that touches the GPU runs in a worker
process (`--worker`, same script).  A GPU memory-access fault kills the process it happens in -- that is how round 4's driver run
ended with nothing on stdout -- so the supervisor retries a dead worker once (single GPU), maps the fault address onto the
worker's named device buffers, and ALWAYS prints one JSON line (`fault_retries`, `faults`; `error` if no attempt measured).
Under a launcher every rank is such a pair; rank 0's supervisor prints the line.  profiles/r05_fault_hunt.txt has the story.
"""
import argparse
import json
import os
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

# Before the HIP runtime comes up: the package sets the number of hardware queues (the step uses two streams and a third for the gradient
# all-reduce; rocprofv3 timeline under CY_DDP_FORCE=1: 686 images/s with four queues for 765).
import complex_yolov4_pytorch_amd  # noqa: E402,F401
# dmabuf IPC is what RCCL needs on this driver; the HSA runtime reads it when it initialises (the first HIP call), so here, not later
os.environ.setdefault('HSA_ENABLE_IPC_MODE_LEGACY', '0')

import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

import complex_yolov4_pytorch_amd.ops as ops  # noqa: E402
import complex_yolov4_pytorch_amd.synthetic as syn  # noqa: E402
from complex_yolov4_pytorch_amd.models.darknet2pytorch import Darknet  # noqa: E402
from complex_yolov4_pytorch_amd.parallel import RcclDataParallel  # noqa: E402
from complex_yolov4_pytorch_amd.utils.train_utils import create_optimizer  # noqa: E402

CFG = os.path.join(ROOT, 'complex-yolov4-pytorch_amd', 'config', 'cfg', 'complex_yolov4.cfg')
MFMA_PEAK_TFLOPS = {'f16': 2500.0, 'bf16': 2500.0, 'f32': 157.3}     # dense peaks, /opt/skills/guides/MI355X_MICROARCH.md
CONFIGS = {'train608': dict(kind='train', batch=16, size=608), 'infer32': dict(kind='infer', batch=32, size=608),
           'train1024': dict(kind='train', batch=8, size=1024),
           # BASELINE configs[2]'s per-GPU work with "mosaic aug on" (reference kitti_dataset.py:123-173): every sample is a
           # 1216 x 1216 canvas of four 608 x 608 BEV maps, built on the device inside the step from a resident pool
           'train1216': dict(kind='train', batch=16, size=1216, mosaic=True)}
HBM_PEAK_GBS = 8000.0
HBM_PEAK_BPS = HBM_PEAK_GBS * 1e9


class _OptCfg:
    optimizer_type, lr, momentum, weight_decay = 'adam', 1e-3, 0.949, 5e-4     # reference train_config.py:82-94


_T0 = time.time()


def stage(msg):
    """Progress marker on stderr (never stdout: that carries the ONE JSON line): where a run was when it died."""
    sys.stderr.write('[bench %7.2fs] %s\n' % (time.time() - _T0, msg))
    sys.stderr.flush()


def emit(line):
    """The ONE JSON line, last on stdout: RCCL writes its version banner through C stdio, which would otherwise be flushed
    after Python's buffer at exit -- flush both first."""
    import ctypes
    sys.stdout.flush()
    try:
        ctypes.CDLL(None).fflush(None)
    except OSError:
        pass
    print(json.dumps(line), flush=True)


def usable_cores(cap=32):
    """Cores this process may really use: affinity mask and cgroup CPU quota, capped (oversubscribed OpenMP teams on
    a 256-thread host made a single oracle step take minutes)."""
    n = len(os.sched_getaffinity(0)) if hasattr(os, 'sched_getaffinity') else (os.cpu_count() or 1)
    try:
        with open('/sys/fs/cgroup/cpu.max') as f:
            quota, period = f.read().split()
            if quota != 'max':
                n = min(n, max(1, int(int(quota) / int(period))))
    except (OSError, ValueError):
        pass
    return max(1, min(n, cap))


def kernel_sources_sha():
    """sha256 over the HIP sources the measured kernels are built from (what a committed PMC figure / tune table is valid for)."""
    from complex_yolov4_pytorch_amd import tune
    return tune.sources_sha()


PMC_FILE = 'profiles/r06_pmc_hbm_traffic.json'
SQ_FILE = 'profiles/r06_sq_counters.json'


def pmc_traffic(kernel, a):
    """HBM bytes PER STEP of the kernel family from the committed rocprofv3 PMC passes (FETCH_SIZE and WRITE_SIZE in
    separate runs of this same command; FETCH doubled per the gfx950 correction of MI355X_MICROARCH.md).  PMC counters
    cannot be read from inside the process, so this is the recorded figure for the default workload -- and only while the
    kernel sources are the ones it was measured on (tools/pmc_traffic.sh stamps their hash and the git head): a stale
    file yields null, never an old number.  The caller divides by ITS launch count, so that `traffic` and the algorithmic
    bytes of the roofline object sit on one basis (round 2 mixed rocprof dispatches with bench brackets)."""
    if (a.batch, a.size, a.dtype, a.config) != (16, 608, 'f16', 'train608'):
        return None
    path = os.path.join(ROOT, PMC_FILE)
    try:
        with open(path) as f:
            doc = json.load(f)
        if doc.get('kernel_sources_sha') != kernel_sources_sha():
            return dict(bytes_per_step=None, stale=True, measured_on=doc.get('kernel_sources_sha'), now=kernel_sources_sha(),
                        source=PMC_FILE)
        d = doc[kernel]
        steps = float(doc.get('steps_counted', 1))
        fetch = d['fetch_bytes_per_launch_corrected'] * d['launches'] / steps
        write = d['write_bytes_per_launch'] * d['launches'] / steps
        whole = sum((v['fetch_bytes_per_launch_corrected'] + v['write_bytes_per_launch']) * v['launches'] / steps
                    for v in doc.values() if isinstance(v, dict) and 'launches' in v)
        return dict(bytes_per_step=round(fetch + write), fetch_per_step=round(fetch), write_per_step=round(write),
                    dispatches_per_step=round(d['launches'] / steps, 1), whole_step_bytes=round(whole), unit='bytes',
                    git_head=doc.get('git_head'), kernel_sources_sha=doc.get('kernel_sources_sha'),
                    source=PMC_FILE + ' (rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE, tools/pmc_traffic.sh)')
    except (OSError, KeyError, ValueError):
        return None


def sq_counters(a):
    """BASELINE's "MFMA utilisation % (rocprof)": the committed SQ-counter passes of this same workload (tools/pmc_sq.sh:
    SQ_VALU_MFMA_BUSY_CYCLES / (32 x SQ_BUSY_CYCLES) per kernel family, LDS array activity, wave-cycle shares) -- like the PMC
    traffic only while the kernel sources are the ones it was measured on; a stale file yields a note, never an old number."""
    if (a.batch, a.size, a.dtype, a.config) != (16, 608, 'f16', 'train608'):
        return None
    try:
        with open(os.path.join(ROOT, SQ_FILE)) as f:
            doc = json.load(f)
        if doc.get('kernel_sources_sha') != kernel_sources_sha():
            return dict(stale=True, measured_on=doc.get('kernel_sources_sha'), now=kernel_sources_sha(), source=SQ_FILE)
        fam = doc['families']
        pick = lambda d: {k: (round(v, 4) if isinstance(v, float) else v) for k, v in d.items() if k in ('mfma_busy', 'lds_array_active', 'launches_per_step')}
        return dict(conv_fwd_dgrad=pick(fam.get('conv fwd/dgrad', {})), wgrad=pick(fam.get('wgrad', {})), whole_step=pick(fam.get('whole step', {})),
                    definition=doc['definitions']['mfma_busy'], kernel_sources_sha=doc.get('kernel_sources_sha'), git_head=doc.get('git_head'),
                    source=SQ_FILE + ' (rocprofv3 --pmc SQ_*, tools/pmc_sq.sh; per kernel in the file)')
    except (OSError, KeyError, ValueError):
        return None


def step_flops(model):
    """Algorithmic FLOPs of one train step of the model's engines: 2 M Cout k^2 Cin per conv with the REAL channel counts, once
    for the forward, the input gradient (not for the first layer) and the weight gradient."""
    total = 0.0
    for e in model._engines.values():
        if e.training:
            for rec in e.plan.convs:
                fl = e._conv_work(rec)[0]
                total += fl * (2.0 if rec['first'] else 3.0)
    return total


def cpu_baseline(batch, size, seconds_budget=20.0):
    """Oracle train step (forward + GIoU loss + backward) on the host cores, bounded sample."""
    from complex_yolov4_pytorch_amd.models.darknet_utils import parse_cfg
    from oracle import darknet_ref
    cores = usable_cores()
    torch.set_num_threads(cores)
    net = darknet_ref.DarknetRef(parse_cfg(CFG))
    ps, bs = net.param_shapes()
    params = {k: v.requires_grad_(True) for k, v in syn.fill_state_dict(ps).items()}
    bufs = syn.fill_state_dict(bs)
    x, tg = syn.bev_images(batch, size, seed=0), syn.targets(batch, 6, size, seed=0)

    def step():
        for p in params.values():
            p.grad = None
        _, loss, _ = net.forward(params, x, tg, True, True, bufs)
        loss.sum().backward()

    t0 = time.time()
    step()                                  # warm-up (also sizes the sample: a slow host gets one timed step)
    warm = time.time() - t0
    t0, n = time.time(), 0
    while n < 1 or (n < 8 and (time.time() - t0) + warm < seconds_budget):
        step()
        n += 1
    dt = (time.time() - t0) / n
    return dict(value=round(batch / dt, 4), unit='images/s', cores=torch.get_num_threads(), kind='port',
                sample='%d timed train steps (fwd+GIoU loss+bwd) of complex_yolov4.cfg, batch %d, %dx%d, fp32, torch-CPU oracle'
                       % (n, batch, size, size))


EVAL_GOLDEN = os.path.join(ROOT, 'tests', 'golden', 'darknet_eval.npz')


def calibrated_eval_model(dev, dtype):
    """complex_yolov4.cfg in eval mode with the seeded weights and the BatchNorm running statistics THE REFERENCE calibrated for
    tests/golden/darknet_eval.npz (tests/golden/make_golden_eval.py: a train-mode forward of the reference with momentum 1), the
    golden's confidence / NMS thresholds and its seeded batch: the network whose eval outputs look like a network's (objectness
    spread around 0.5, ~67 candidate rows and ~67 detections per image) instead of random-init's saturated sigmoids.
    -> (model, images or None, conf_thresh, nms_thresh, reference detection count) -- (None, ...) without the fixture."""
    import numpy as np
    if not os.path.exists(EVAL_GOLDEN):
        return None
    g = np.load(EVAL_GOLDEN, allow_pickle=False)
    torch.manual_seed(0)
    model = Darknet(CFG, use_giou_loss=True, dtype=dtype)
    sd = model.state_dict()
    sd.update({k: syn.fill_tensor(k, tuple(v.shape)) for k, v in sd.items() if v.dtype.is_floating_point})
    off = 0
    for name, n in zip(g['bn_names'], g['bn_sizes']):
        sd[str(name)] = torch.from_numpy(g['bn_values'][off:off + int(n)].copy())
        off += int(n)
    model.load_state_dict(sd)
    return model.to(dev).eval(), float(g['conf_thresh'][0]), float(g['nms_thresh'][0]), int(g['det_count'].sum()), int(g['out_shape'][0])


def measure_inference(dev, batch, size, dtype, steps, warmup, with_contract=True):
    """BASELINE configs[3], the reference's pipeline (evaluate.py:32-45): ``outputs = model(imgs)`` in eval mode, then
    ``post_processing_v2(outputs, conf_thresh, nms_thresh)`` -- the rotated merge-NMS runs on THE MODEL'S OWN OUTPUT of every
    batch.  The network is the seeded one with the reference-calibrated BatchNorm statistics of tests/golden/darknet_eval.npz and
    the golden's thresholds, so the NMS stage sees what a network produces (~67 candidates per image), not saturated random-init
    sigmoids; its detection count is reported beside the reference's own on the same batch.  Without the fixture (or at another
    batch / size than the golden's 32 x 608^2): random-init weights and synthetic predictions, said so in `workload`."""
    from complex_yolov4_pytorch_amd.utils.evaluation_utils import post_processing_v2, post_processing_v2_device
    cal = calibrated_eval_model(dev, dtype) if (size == 608) else None
    if cal is not None:
        model, conf, nms, ref_dets, gb = cal
        x = syn.bev_images(max(batch, gb), size, seed=33)[:batch].to(dev)      # the golden's batch (a prefix of it below batch 32)
        pred = None
    else:
        torch.manual_seed(0)
        model = Darknet(CFG, use_giou_loss=True, dtype=dtype).to(dev).eval()
        conf, nms, ref_dets = 0.5, 0.5, None
        x = syn.bev_images(batch, size, seed=0).to(dev)
        pred = syn.nms_predictions(batch, 3 * ((size // 8) ** 2 + (size // 16) ** 2 + (size // 32) ** 2), 256, seed=4).to(dev)
    model.cpu_outputs = False
    model.static_eval_weights = True           # serving: parameters do not change between batches
    ndet = [0]

    def step():
        with torch.no_grad():
            out = model(x)
            dets, _ = post_processing_v2_device(out if pred is None else pred, conf, nms)
            ndet[0] = sum(0 if d is None else int(d.shape[0]) for d in dets)
        return out

    for _ in range(warmup):
        step()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        step()
    torch.cuda.synchronize()
    dt = (time.perf_counter() - t0) / steps
    # the two stages apart (events on the launch stream): how much of the step is the conv stack, how much the NMS
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    with torch.no_grad():
        ev[0].record(); out = model(x); ev[1].record(); post_processing_v2_device(out if pred is None else pred, conf, nms); ev[2].record()
    torch.cuda.synchronize()
    fwd_ms, nms_ms = ev[0].elapsed_time(ev[1]), ev[1].elapsed_time(ev[2])
    gflop = sum(e._conv_work(rec)[0] for e in model._engines.values() for rec in e.plan.convs) / 1e9
    algo_bytes = sum(e._conv_work(rec)[1] for e in model._engines.values() for rec in e.plan.convs)
    # the reference's own contract (evaluate.py:32-45): model(x) hands its outputs to the HOST (darknet2pytorch.py:228), and
    # post_processing_v2 starts from that host tensor (here: H2D + select + merge-NMS on the device + detections back to the host)
    model.cpu_outputs = True

    def ref_step():
        with torch.no_grad():
            out = model(x)
            post_processing_v2(out if pred is None else pred.cpu(), conf, nms)
        return out

    nref, dt_ref = 0, float('nan')
    if with_contract:       # (profiling runs -- --no-roofline -- leave this leg out: every forward under the tracer is a timed step)
        for _ in range(max(1, warmup // 2)):
            ref_step()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        nref = max(2, steps // 2)
        for _ in range(nref):
            ref_step()
        torch.cuda.synchronize()
        dt_ref = (time.perf_counter() - t0) / nref
    nlaunch = sum(len(e.plan.convs) for e in model._engines.values())
    model.release_engines()
    what = ('post_processing_v2 on the device over the OUTPUT OF model(x) itself (seeded weights + the BatchNorm running statistics the reference '
            'calibrated for tests/golden/darknet_eval.npz, its thresholds %.4f / %.2f)' % (conf, nms)) if pred is None else \
           'post_processing_v2 on the device over SYNTHETIC predictions with 256 candidates/image (random-init weights: no fixture for this shape)'
    return dict(metric='BEV images/s (%dx%d) inference + rotated NMS' % (size, size), value=round(batch / dt, 2), unit='images/s',
                ms_per_step=round(1e3 * dt, 3), steps=steps, dtype=dtype, step_gflop=round(gflop, 1),
                step_tflops=round(gflop / dt / 1e3, 1), step_frac=round(gflop / dt / 1e3 / MFMA_PEAK_TFLOPS[dtype], 4),
                roofline=dict(bound='mfma', achieved=round(gflop / fwd_ms, 1), peak=MFMA_PEAK_TFLOPS[dtype], unit='TFLOP/s',
                              frac=round(gflop / fwd_ms / MFMA_PEAK_TFLOPS[dtype], 4), traffic=None,
                              kernel='the eval forward (conv + BN + activation fused per layer, %d launches): algorithmic FLOPs over its '
                                     'HIP-event time on the launch stream' % nlaunch,
                              forward_ms=round(fwd_ms, 3), nms_ms=round(nms_ms, 3),
                              algorithmic_gbs=round(algo_bytes / fwd_ms / 1e6, 1), hbm_frac=round(algo_bytes / fwd_ms / 1e6 / HBM_PEAK_GBS, 4)),
                detections=ndet[0], reference_detections=ref_dets if batch == 32 else None,
                reference_contract=None if not with_contract else dict(value=round(batch / dt_ref, 2), unit='images/s', ms_per_step=round(1e3 * dt_ref, 3), steps=nref,
                                        workload='model(x) returns its [%d, N, 10] fp32 outputs on the HOST (D2H, reference '
                                                 'darknet2pytorch.py:228), post_processing_v2 takes that HOST tensor (H2D + device select / '
                                                 'merge-NMS + detections to the host)' % batch),
                workload='complex_yolov4.cfg model.eval() forward, batch %d, %dx%d (outputs stay on the device: no 29 MB D2H) + %s, both '
                         'stages in every timed step' % (batch, size, size, what))


def batch_source(dev, batch, size, mosaic, seed=0):
    """() -> (images [B,3,S,S], targets [nT,8]) on the device.  Plain: one resident synthetic batch.  mosaic: a resident pool
    of 4*B maps of (S/2)^2 with 6 targets each; every call assembles B canvases with the device mosaic kernels
    (data_process/transformation.py::make_mosaic, centre drawn per canvas like the reference's load_mosaic)."""
    if not mosaic:
        x, tg = syn.bev_images(batch, size, seed=seed).to(dev), syn.targets(batch, 6, size, seed=seed).to(dev)
        return lambda: (x, tg)
    import random
    from complex_yolov4_pytorch_amd.data_process.transformation import make_mosaic
    half = size // 2
    pool = syn.bev_images(4 * batch, half, seed=seed).to(dev)
    rows = syn.targets(4 * batch, 6, half, seed=seed)
    per_tile = [rows[rows[:, 0] == i].clone() for i in range(4 * batch)]
    rng = random.Random(seed)

    def make():
        random.seed(rng.random())
        canvases, tgs = [], []
        for b in range(batch):
            c, t = make_mosaic([pool[4 * b + k] for k in range(4)], [per_tile[4 * b + k] for k in range(4)], half, random_padding=True)
            t[:, 0] = b
            canvases.append(c)
            tgs.append(t)
        return torch.stack(canvases), torch.cat(tgs, 0)
    return make


def measure_other(config, dtype, steps, warmup):
    """One of the other configurations, measured by this same script in a fresh process (its ONE JSON line, reduced)."""
    import subprocess
    cmd = [sys.executable, os.path.abspath(__file__), '--worker', '--config', config, '--dtype', dtype, '--steps', str(steps),
           '--warmup', str(warmup), '--no-extra', '--no-cpu-baseline'] + ([] if config in ('train1024', 'infer32') else ['--no-roofline'])
    try:
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=900, cwd=ROOT)
        if r.returncode != 0:
            return dict(error='%s: worker exit status %d' % (config, r.returncode), stderr_tail=r.stderr[-400:])
        d = json.loads(r.stdout.strip().splitlines()[-1])
        out = dict(metric=d['metric'], value=d['value'], unit=d['unit'], ms_per_step=d['ms_per_step'], steps=d['steps'], dtype=d['dtype'],
                   workload=d['config']['workload'], loss_final=d['config'].get('loss_final'), process='fresh')
        # roofline of the configuration: its whole-step algorithmic FLOPs over its wall clock against the dense MFMA peak
        out.update({k: d['step'][k] for k in ('step_gflop', 'step_tflops', 'step_frac') if d.get('step') and k in d['step']})
        if d.get('reference_contract'):
            out['reference_contract'] = d['reference_contract']
        # the configuration's own roofline object (inference: the eval forward against the MFMA peak, HIP events; training: the
        # conv family like the headline's), detection counts of the inference pipeline
        for k in ('roofline', 'detections', 'reference_detections'):
            if d.get(k) is not None:
                out[k] = d[k]
        if isinstance(out.get('roofline'), dict):      # (the configuration's conv-family roofline, without the headline's long notes)
            out['roofline'] = {k: v for k, v in out['roofline'].items() if k in (
                'bound', 'achieved', 'peak', 'unit', 'frac', 'traffic', 'launches_per_step', 'avg_launch_us', 'hbm_gbs_algorithmic',
                'algorithmic_bytes_per_step', 'by_bound', 'conv_ms_per_step', 'forward_ms', 'nms_ms', 'algorithmic_gbs', 'hbm_frac', 'kernel')}
        return out
    except Exception as e:      # noqa: BLE001 -- the headline line must still be printed
        return dict(error='%s: %r' % (config, e))


def _free_port():
    import socket
    s = socket.socket()
    s.bind(('127.0.0.1', 0))
    p = s.getsockname()[1]
    s.close()
    return p


def self_launch(n, argv, script=None, need_gpus=True):
    """`python bench.py --gpus N` without a launcher: start N ranks of this script, one per GPU (what the reference's
    mp.spawn does, src/train.py:46-52), through torch.distributed.run on 127.0.0.1; rank 0's JSON line is the children's
    stdout, passed through.  -> exit status.  (`script` / `need_gpus`: tests/test_bench_launch.py starts CPU ranks of
    tests/bench_sim.py through the same function.)"""
    import subprocess
    if need_gpus:
        have = torch.cuda.device_count()
        if have < n:
            sys.stderr.write('bench.py: --gpus %d needs %d GPUs on this node, %d visible (HIP_VISIBLE_DEVICES / ROCR_VISIBLE_DEVICES?)\n'
                             % (n, n, have))
            return 2
    env = dict(os.environ)
    env.setdefault('HSA_ENABLE_IPC_MODE_LEGACY', '0')
    env.setdefault('OMP_NUM_THREADS', str(max(1, usable_cores(256) // n)))
    cmd = [sys.executable, '-m', 'torch.distributed.run', '--nnodes=1', '--nproc-per-node', str(n), '--master-addr', '127.0.0.1',
           '--master-port', str(_free_port()), os.path.abspath(script or __file__)] + list(argv)
    return subprocess.run(cmd, env=env).returncode


def parse_args(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument('--gpus', type=int, default=1)
    ap.add_argument('--steps', type=int, default=30)
    ap.add_argument('--warmup', type=int, default=5)
    ap.add_argument('--config', default='train608', choices=sorted(CONFIGS))
    ap.add_argument('--batch', type=int, default=None, help='images per GPU (default: the configuration\'s)')
    ap.add_argument('--size', type=int, default=None)
    ap.add_argument('--dtype', default='f16', choices=['f16', 'bf16', 'f32'])
    ap.add_argument('--deterministic', action='store_true', help='bit-reproducible reductions (Darknet(..., deterministic=True))')
    ap.add_argument('--no-cpu-baseline', action='store_true')
    ap.add_argument('--no-roofline', action='store_true')
    ap.add_argument('--no-extra', action='store_true', help='skip the brief measurement of the other configurations')
    ap.add_argument('--graph', type=int, default=0, help='1: the step as one captured hipGraph (graphed.GraphedTrainStep); default 0 = '
                    'eager launches: on ROCm 7.2 the replay of the 660-node, two-stream graph takes 33.1 ms against 19.2 ms eager '
                    '(DESIGN.md section 5), so the measured configuration is the eager one')
    ap.add_argument('--worker', action='store_true', help='internal: the measuring process (owns the GPU context); the plain command '
                    'is a supervisor that starts it, retries it once after a GPU fault and assembles the line')
    ap.add_argument('--map-file', default=None, help='internal: where the worker leaves its device buffer map for the supervisor')
    a = ap.parse_args(argv)
    cfg = CONFIGS[a.config]
    a.batch = a.batch or cfg['batch']
    a.size = a.size or cfg['size']
    return a


def main():
    a = parse_args()
    if a.gpus > 1 and 'WORLD_SIZE' not in os.environ:
        sys.exit(self_launch(a.gpus, sys.argv[1:]))
    world = int(os.environ.get('WORLD_SIZE', 1))
    if a.gpus != world and (a.gpus > 1 or world > 1):
        sys.exit('bench.py: --gpus %d but the launcher started WORLD_SIZE=%d ranks (use --nproc-per-node %d)' % (a.gpus, world, a.gpus))
    if a.worker:
        return worker(a)
    sys.exit(supervise(a, sys.argv[1:]))


def worker(a):
    """The measurement itself, in a process of its own: everything that touches the GPU.  Prints the line of ITS part (the
    headline configuration with `roofline`); the supervisor adds `other_configs` and `cpu_baseline`."""
    import faulthandler
    faulthandler.enable(all_threads=False)      # a GPU fault ends in abort(): leave the Python stack of the main thread on stderr
    cfg = CONFIGS[a.config]
    rank = int(os.environ.get('RANK', 0))
    local = int(os.environ.get('LOCAL_RANK', 0))
    world = int(os.environ.get('WORLD_SIZE', 1))
    if a.gpus != world and (a.gpus > 1 or world > 1):
        sys.exit('bench.py: --gpus %d but the launcher started WORLD_SIZE=%d ranks (use --nproc-per-node %d)' % (a.gpus, world, a.gpus))
    if torch.cuda.device_count() <= local:
        sys.exit('bench.py: rank %d needs GPU %d but this node exposes %d device(s)' % (rank, local, torch.cuda.device_count()))
    torch.cuda.set_device(local)
    dev = torch.device('cuda', local)
    force_ddp = os.environ.get('CY_DDP_FORCE') == '1'
    if world > 1 or force_ddp:
        os.environ.setdefault('MASTER_ADDR', '127.0.0.1')
        os.environ.setdefault('MASTER_PORT', '29511')
        os.environ.setdefault('RANK', '0')
        os.environ.setdefault('WORLD_SIZE', '1')
        os.environ.setdefault('HSA_ENABLE_IPC_MODE_LEGACY', '0')      # dmabuf IPC: what RCCL needs on this driver
        dist.init_process_group('nccl', device_id=dev)

    if cfg['kind'] == 'infer':
        # replicas: every rank serves its own batches, no exchange
        r = measure_inference(dev, a.batch, a.size, a.dtype, a.steps, a.warmup, with_contract=not a.no_roofline)
        t = torch.tensor([r['ms_per_step']], device=dev, dtype=torch.float64)
        if world > 1:
            dist.all_reduce(t, op=dist.ReduceOp.MAX)
        if rank == 0:
            ms = float(t)
            line = {'metric': r['metric'], 'value': round(world * a.batch / (ms * 1e-3), 3), 'unit': 'images/s',
                    'n_gpus': world, 'steps': a.steps, 'warmup': a.warmup, 'ms_per_step': round(ms, 3),
                    'higher_is_better': True, 'scaling': 'weak', 'vs_baseline': None, 'dtype': a.dtype,
                    'data': 'synthetic', 'config': {'workload': r['workload'], 'global_batch': world * a.batch,
                                                    'parallelism': 'replicas%d' % world},
                    'roofline': r['roofline'], 'cpu_baseline': None,
                    'step': {k: r[k] for k in ('step_gflop', 'step_tflops', 'step_frac')},
                    'detections': r['detections'], 'reference_detections': r['reference_detections'],
                    'reference_contract': r['reference_contract']}
        if dist.is_initialized():
            dist.destroy_process_group()
        if rank == 0:
            emit(line)
        return

    stage('device up, building the model')
    torch.manual_seed(0)
    model = Darknet(CFG, use_giou_loss=True, dtype=a.dtype, deterministic=a.deterministic).to(dev)
    model.train()
    net = RcclDataParallel(model) if (world > 1 or force_ddp) else model
    opt = create_optimizer(_OptCfg, model)          # FusedAdam (cy_adam_multi) on the device
    source = batch_source(dev, a.batch, a.size, bool(cfg.get('mosaic')), seed=rank)
    use_graph = bool(a.graph) and world == 1 and not force_ddp and hasattr(opt, 'capturable')
    graphed, graph_note = None, 'eager launches'
    if use_graph:
        from complex_yolov4_pytorch_amd.graphed import GraphedTrainStep
        opt.capturable = True
        graphed = GraphedTrainStep(model, opt)

    def eager_step():
        opt.zero_grad(set_to_none=True)
        x, tg = source()
        loss, _ = net(x, tg)
        loss.backward()
        opt.step()
        return loss

    def step():
        if graphed is not None:
            return graphed(*source())       # the whole step = one hipGraphLaunch (captured at the first call of a shape)
        return eager_step()

    if graphed is not None:
        try:
            step()
            graph_note = 'one captured hipGraph per step (graphed.GraphedTrainStep)'
        except Exception as e:      # noqa: BLE001 -- a capture failure must not cost the measurement
            graphed, graph_note = None, 'eager launches (graph capture failed: %r)' % (e,)
            opt.capturable = False

    def sync():
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize()

    for i in range(a.warmup):
        stage('warm-up step %d' % i)
        step()
    if isinstance(net, RcclDataParallel):
        net.exposed_events = []      # (before, after) the compute stream's wait for the all-reduce stream, one pair per step
    # (the supervisor's buffer map is host-side bookkeeping, tens of milliseconds with the allocator's snapshot: written while the
    # queued warm-up steps are still executing, not between the synchronisation and the first timed step -- the GPU would sit
    # idle there and start the timed region from a lowered clock)
    if a.map_file and a.warmup > 0:
        write_buffer_map(a.map_file, model, opt)
    sync()
    if a.map_file and a.warmup == 0:
        write_buffer_map(a.map_file, model, opt)
    stage('timed region: %d steps' % a.steps)
    t0 = time.perf_counter()
    for _ in range(a.steps):
        loss = step()
    sync()
    mine = time.perf_counter() - t0
    stage('timed region done: %.3f ms per step' % (1e3 * mine / a.steps))
    elapsed = torch.tensor([mine], device=dev, dtype=torch.float64)
    per_rank_ms, exposed_ms = None, None
    if isinstance(net, RcclDataParallel):
        # how long the compute stream stood still at the end of backward waiting for the gradient all-reduce (the part of
        # the collective that backward did NOT hide), averaged over the timed steps; max over ranks below
        ex = [e0.elapsed_time(e1) for e0, e1 in (net.exposed_events or [])]
        net.exposed_events = None
        exposed = torch.tensor([sum(ex) / max(1, len(ex))], device=dev, dtype=torch.float64)
    if world > 1:
        every = [torch.zeros_like(elapsed) for _ in range(world)]
        dist.all_gather(every, elapsed)
        per_rank_ms = [round(1e3 * float(t) / a.steps, 3) for t in every]
        dist.all_reduce(elapsed, op=dist.ReduceOp.MAX)
        dist.all_reduce(exposed, op=dist.ReduceOp.MAX)
    if isinstance(net, RcclDataParallel):
        exposed_ms = round(float(exposed), 3)
    elapsed = float(elapsed)
    final_loss = float(loss.detach().reshape(-1)[0])
    if rank == 0:
        # the headline is safe from here on: the supervisor falls back to this line if a later leg of the worker dies
        emit({'partial': True, 'value': round(world * a.batch * a.steps / elapsed, 3), 'ms_per_step': round(1e3 * elapsed / a.steps, 3),
              'loss_final': round(final_loss, 4), 'per_rank_ms_per_step': per_rank_ms, 'allreduce_exposed_ms_per_step': exposed_ms})

    roofline = None
    summ, by_bound = {}, None
    if not a.no_roofline:
        # exclusive kernel durations: the probe steps issue the weight-gradient kernels on the main stream (in the timed
        # region they overlap the dgrad/BN kernels from a side stream, which stretches every kernel's own duration).
        # EVERY rank runs the probe steps (a step contains the gradient all-reduce); only rank 0 brackets its launches.
        stage('roofline probe steps (single stream, bracketed launches)')
        sides = [(e, e.side) for e in model._engines.values()]
        for e, _ in sides:
            e.side = None
        if rank == 0:
            ops.PROFILER = ops.LaunchProfiler()
        for _ in range(2):
            eager_step()        # (the launch brackets are host-side event records: the probe steps run eagerly)
        summ = ops.PROFILER.summary() if rank == 0 else {}
        if rank == 0:
            # the same launches split by which roof bounds them: arithmetic intensity above / below the ridge point.
            # Durations are the RAW event brackets (two event records included, ~5 us): a conservative rate; the figure
            # with the empty-bracket duration taken out is reported beside it (rocprofv3's exclusive durations of the
            # same run, profiles/r02_*, sit between the two).
            ridge = MFMA_PEAK_TFLOPS[a.dtype] * 1e12 / HBM_PEAK_BPS
            acc = {'mfma': [0.0, 0.0, 0.0, 0], 'hbm': [0.0, 0.0, 0.0, 0]}
            # the HBM-bound class again by launch size: a launch that moves < 64 MB lasts 9-25 us, 6-8 us of which are fixed
            # (dispatch, prologue, pipeline fill, tail: DESIGN.md section 5) -- its rate says nothing about the memory system
            size = {'large (>= 64 MB algorithmic)': [0.0, 0.0, 0], 'small': [0.0, 0.0, 0]}
            for kind, fl, nb, ev0, ev1 in ops.PROFILER.records:
                if kind not in ('igemm', 'igemm_sums') or nb <= 0:
                    continue
                k = 'mfma' if fl / nb >= ridge else 'hbm'
                t = max(ev0.elapsed_time(ev1), 1e-6)
                acc[k][0] += fl; acc[k][1] += nb; acc[k][2] += t; acc[k][3] += 1
                if k == 'hbm':
                    sz = size['large (>= 64 MB algorithmic)' if nb >= 64e6 else 'small']
                    sz[0] += nb; sz[1] += t; sz[2] += 1
            by_bound = {}
            for k, (fl, nb, ms, n) in acc.items():
                if n:
                    by_bound[k] = dict(launches_per_step=n // 2, ms_per_step=round(ms / 2, 3),
                                       tflops=round(fl / (ms * 1e-3) / 1e12, 1), gbs_algorithmic=round(nb / (ms * 1e-3) / 1e9, 1),
                                       frac=round((fl / (ms * 1e-3)) / (MFMA_PEAK_TFLOPS[a.dtype] * 1e12), 4) if k == 'mfma'
                                       else round((nb / (ms * 1e-3)) / HBM_PEAK_BPS, 4))
            if 'hbm' in by_bound:
                by_bound['hbm']['by_size'] = {k: dict(launches_per_step=n // 2, ms_per_step=round(ms / 2, 3),
                                                      gbs_algorithmic=round(nb / (ms * 1e-3) / 1e9, 1), avg_launch_us=round(1e3 * ms / n, 1))
                                              for k, (nb, ms, n) in size.items() if n}
        ops.PROFILER = None
        for e, sd in sides:
            e.side = sd
        sync()
    if rank == 0 and not a.no_roofline:
        plain, fused = summ.get('igemm'), summ.get('igemm_sums')
        # the conv family = every forward / dgrad launch as it runs in the step; the dgrad launches that also take the
        # BatchNorm-backward sums of the producer layer in their epilogue (cy_conv_dgrad_bn_sums) are bracketed apart so
        # that the cost of that epilogue is visible (`epilogue_split`)
        ig = {k: plain[k] + (fused[k] if fused else 0) for k in ('flops', 'bytes', 'ms', 'ms_raw', 'launches')} if plain else None
        if ig:
            ach = ig['flops'] / (ig['ms_raw'] * 1e-3) / 1e12
            peak = MFMA_PEAK_TFLOPS[a.dtype]
            tr = pmc_traffic('igemm', a)
            brackets = ig['launches'] // 2                     # launches of the family per step as the engine issues them
            tr_launch = round(tr['bytes_per_step'] / brackets) if tr and tr.get('bytes_per_step') else None
            roofline = dict(bound='mfma', kernel='implicit-GEMM conv kernels (forward + dgrad launches: igemm_fast_kernel / igemm_kernel '
                                                 '4-wave tiles, igemm_pipe_kernel 8-wave tiles, direct3x3 / direct1x1 streaming kernels for the small-Cin and big-grid 1x1 layers, chosen per layer; dgrad launches that also accumulate BatchNorm-backward sums included)',
                            achieved=round(ach, 2), peak=peak, unit='TFLOP/s', frac=round(ach / peak, 4),
                            traffic=tr_launch, traffic_detail=tr,
                            traffic_over_algorithmic=round(tr_launch / (ig['bytes'] / ig['launches']), 3) if tr_launch else None,
                            algorithmic_bytes_per_step=round(ig['bytes'] / 2),
                            launches_per_step=ig['launches'] // 2, avg_launch_us=round(1e3 * ig['ms_raw'] / ig['launches'], 2),
                            hbm_gbs_algorithmic=round(ig['bytes'] / (ig['ms_raw'] * 1e-3) / 1e9, 1),
                            algorithmic_bytes_per_launch=round(ig['bytes'] / ig['launches']),
                            measured='HIP events around every launch of the family on its launch stream (raw brackets, event records '
                                     'included); 2 extra single-stream steps after the timed region',
                            achieved_minus_event_overhead=round(ig['flops'] / (ig['ms'] * 1e-3) / 1e12, 2),
                            avg_launch_us_minus_event_overhead=round(1e3 * ig['ms'] / ig['launches'], 2))
            wg = summ.get('wgrad')
            if wg:
                roofline['wgrad_kernel'] = dict(achieved=round(wg['flops'] / (wg['ms_raw'] * 1e-3) / 1e12, 2), unit='TFLOP/s',
                                                launches_per_step=wg['launches'] // 2,
                                                avg_launch_us=round(1e3 * wg['ms_raw'] / wg['launches'], 2))
            roofline['conv_ms_per_step'] = round((ig['ms_raw'] + (wg['ms_raw'] if wg else 0)) / 2, 3)
            roofline['epilogue_split'] = {
                name: dict(launches_per_step=f['launches'] // 2, avg_launch_us=round(1e3 * f['ms_raw'] / f['launches'], 2),
                           achieved=round(f['flops'] / (f['ms_raw'] * 1e-3) / 1e12, 2), unit='TFLOP/s')
                for name, f in (('conv_only', plain), ('dgrad_with_bn_backward_sums', fused)) if f}
            roofline['by_bound'] = by_bound   # launches above the ridge point against the MFMA peak, the rest against HBM
            sq = sq_counters(a)
            roofline['mfma_busy'] = (sq or {}).get('conv_fwd_dgrad', {}).get('mfma_busy') if sq and not sq.get('stale') else None
            roofline['sq_counters'] = sq      # MFMA pipe busy / LDS activity per family from the committed rocprofv3 SQ passes
            # BASELINE's "MFMA util %": the WHOLE train step's algorithmic FLOPs (forward + input gradient + weight gradient of
            # every conv) over the timed region's wall clock, against the dense MFMA peak
            sf = step_flops(model)
            roofline['step_tflops'] = round(sf / (elapsed / a.steps) / 1e12, 1)
            roofline['step_frac'] = round(sf / (elapsed / a.steps) / (peak * 1e12), 4)
            roofline['step_gflop'] = round(sf / 1e9, 1)
    if world > 1:
        dist.barrier()

    fused_layers = max((len(e._sums_fused) for e in model._engines.values()), default=0)
    replayed = sum(getattr(e, 'replayed', 0) for e in model._engines.values())
    passes = sum(getattr(e, 'passes', 0) for e in model._engines.values())
    for e in model._engines.values():
        e.check_grid_waits()
    sf_all = step_flops(model)         # per-GPU algorithmic FLOPs of one step (weak scaling: the same on every rank)
    if rank == 0:
        imgs = world * a.batch * a.steps
        line = {
            'metric': 'BEV images/s (%dx%d) train step' % (a.size, a.size), 'value': round(imgs / elapsed, 3), 'unit': 'images/s',
            'n_gpus': world, 'steps': a.steps, 'warmup': a.warmup, 'ms_per_step': round(1e3 * elapsed / a.steps, 3),
            'higher_is_better': True, 'scaling': 'weak', 'vs_baseline': None,
            'dtype': a.dtype, 'data': 'synthetic',
            'config': {'workload': 'complex_yolov4.cfg train step (%sfwd + rotated-GIoU loss + bwd + Adam), batch %d per GPU, %dx%dx3 synthetic BEV, %d targets/image'
                                   % ('device mosaic of four maps per sample + ' if cfg.get('mosaic') else '', a.batch, a.size, a.size, 24 if cfg.get('mosaic') else 6),
                       'global_batch': world * a.batch, 'parallelism': 'dp%d' % world, 'loss_final': round(final_loss, 4),
                       'deterministic': bool(a.deterministic),
                       'issue': graph_note if graphed is not None or not replayed else
                       'recorded launch lists replayed from C (cy_run_plan): every kernel still launches eagerly, %d of %d passes replayed' % (replayed, passes),
                       'dgrad_bn_sums_layers': fused_layers,
                       'yolo_outputs': 'stay on the device in training (the reference copies 14.6 MB to the host every step, '
                                       'darknet2pytorch.py:228, and train.py discards them)'},
            'roofline': roofline, 'cpu_baseline': None,
            'step': dict(step_gflop=round(sf_all / 1e9, 1), step_tflops=round(sf_all / (elapsed / a.steps) / 1e12, 1),
                         step_frac=round(sf_all / (elapsed / a.steps) / (MFMA_PEAK_TFLOPS[a.dtype] * 1e12), 4)),
        }
        if per_rank_ms is not None:
            line['per_rank_ms_per_step'] = per_rank_ms
        if exposed_ms is not None:
            line['allreduce_exposed_ms_per_step'] = exposed_ms      # 0 = fully hidden behind backward
    if dist.is_initialized():
        dist.destroy_process_group()
    if rank == 0:
        emit(line)


def write_buffer_map(path, model, opt):
    """Every device buffer of the step by name -> `path` (JSON): the supervisor maps the address of a GPU memory-access fault
    onto it.  Host-side bookkeeping only (data_ptr / sizes / the caching allocator's segment list)."""
    rows = []
    try:
        for key, e in model._engines.items():
            rows += [('engine%r.%s' % (key[:3], n), p_, b) for n, p_, b in e.buffer_map()]
        for n, t in list(model.named_parameters()) + list(model.named_buffers()):
            rows.append(('param ' + n, t.data_ptr(), t.numel() * t.element_size()))
        if model.flat_grad is not None:
            rows.append(('flat_grad', model.flat_grad.data_ptr(), model.flat_grad.numel() * 4))
        for st in getattr(opt, 'state', {}).values():
            for k, v in st.items():
                if isinstance(v, torch.Tensor) and v.is_cuda:
                    rows.append(('optimizer.' + k, v.data_ptr(), v.numel() * v.element_size()))
        segs = [(sg['address'], sg['total_size']) for sg in torch.cuda.memory_snapshot()]
        with open(path, 'w') as f:
            json.dump({'buffers': rows, 'segments': segs}, f)
    except Exception as e:      # noqa: BLE001 -- diagnostics must never cost the measurement
        stage('buffer map not written: %r' % (e,))


def diagnose_fault(stderr_text, map_file):
    """What the worker's stderr and its buffer map say about a GPU fault: the address, the buffer it falls into (or the nearest
    ones), the last stage marker and the main thread's Python stack (faulthandler)."""
    import re
    d = {}
    m = re.search(r'Memory access fault by GPU node-(\d+).*?on address (0x[0-9a-fA-F]+)\. Reason: ([^\n]*)', stderr_text)
    stages = re.findall(r'\[bench +[0-9.]+s\] ([^\n]*)', stderr_text)
    if stages:
        d['last_stage'] = stages[-1]
    fh = stderr_text.find('Current thread')
    if fh < 0:
        fh = stderr_text.find('Fatal Python error')
    if fh >= 0:
        d['python_stack'] = [ln.strip() for ln in stderr_text[fh:].splitlines()[1:9]]
    if not m:
        d['stderr_tail'] = stderr_text[-600:]
        return d
    addr = int(m.group(2), 16)
    d.update(address=m.group(2), reason=m.group(3).strip())
    try:
        with open(map_file) as f:
            doc = json.load(f)
        inside = [(n, p_, b) for n, p_, b in doc['buffers'] if p_ <= addr < p_ + b]
        if inside:
            n, p_, b = min(inside, key=lambda r: r[2])
            d['buffer'] = '%s + %d of %d bytes' % (n, addr - p_, b)
        else:
            below = max([r for r in doc['buffers'] if r[1] + r[2] <= addr], key=lambda r: r[1] + r[2], default=None)
            above = min([r for r in doc['buffers'] if r[1] > addr], key=lambda r: r[1], default=None)
            d['buffer'] = None
            if below:
                d['nearest_below'] = '%s ends %d bytes before the address' % (below[0], addr - below[1] - below[2])
            if above:
                d['nearest_above'] = '%s starts %d bytes after the address' % (above[0], above[1] - addr)
        d['in_allocator_segment'] = any(a0 <= addr < a0 + sz for a0, sz in doc['segments'])
    except (OSError, ValueError, KeyError) as e:
        d['map'] = 'unavailable (%r): the fault came before the end of the warm-up' % (e,)
    return d


def run_worker(argv, map_file, timeout=1500, script=None):
    """One worker process of this script -> (exit status, last complete JSON line or None, last partial line or None, stderr).
    stderr is forwarded line by line (stage markers stay visible while the run is alive) and kept for the diagnosis."""
    import subprocess
    import threading
    cmd = [sys.executable, os.path.abspath(script or __file__), '--worker', '--map-file', map_file] + [x for x in argv if x != '--worker']      # (script: tests)
    def die_with_parent():       # (a supervisor killed by its caller must not leave a worker holding the GPU)
        try:
            import ctypes
            import signal
            ctypes.CDLL(None).prctl(1, signal.SIGKILL)      # PR_SET_PDEATHSIG
        except Exception:      # noqa: BLE001
            pass
    p = subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, cwd=ROOT, preexec_fn=die_with_parent)
    err = []

    def pump():
        for ln in p.stderr:
            err.append(ln)
            sys.stderr.write(ln)
            sys.stderr.flush()
    t = threading.Thread(target=pump, daemon=True)
    t.start()
    # (one reader per pipe: the thread owns stderr, this thread stdout -- communicate() would read stderr too and swallow lines)
    killed = []
    timer = threading.Timer(timeout, lambda: (killed.append(1), p.kill()))
    timer.start()
    out = p.stdout.read()
    p.wait()
    timer.cancel()
    t.join(timeout=5)
    if killed:
        err.append('bench.py supervisor: worker killed after %d s\n' % timeout)
    full = part = None
    for ln in (out or '').splitlines():
        if ln.startswith('{'):
            try:
                d = json.loads(ln)
            except ValueError:
                continue
            if d.get('partial'):
                part = d
            else:
                full = d
    return p.returncode, full, part, ''.join(err)


def supervise(a, argv):
    """What `python bench.py ...` is: a process WITHOUT a GPU context that starts the measuring worker, and -- because a GPU
    memory-access fault kills the process it happens in (round 4's driver run ended that way, BENCH_r04.json, with nothing on
    stdout) -- survives it: the worker is retried once (single GPU), every fault is reported on the line (`fault_retries`,
    `faults` with the address mapped onto the worker's buffers), and rank 0 ALWAYS prints one JSON line, with `error` if no
    attempt produced a measurement.  Under a launcher every rank is such a pair."""
    import tempfile
    rank, world = int(os.environ.get('RANK', 0)), int(os.environ.get('WORLD_SIZE', 1))
    map_file = os.path.join(tempfile.gettempdir(), 'cy_bench_map_%d.json' % os.getpid())
    faults, full, part, tries = [], None, None, 0
    attempts = 2 if world == 1 else 1       # (a retry under a launcher would need every rank to agree on it)
    if rank == 0:
        # under a launcher a rank that dies makes the launcher terminate the others -- rank 0's supervisor included; a single-GPU
        # supervisor can be terminated by its caller's timeout.  Either way it must still leave ONE line saying so
        import signal

        def terminated(signum, frame):
            emit({'metric': 'BEV images/s (%dx%d) train step' % (a.size, a.size), 'value': None, 'unit': 'images/s', 'n_gpus': world,
                  'steps': a.steps, 'warmup': a.warmup, 'ms_per_step': None, 'higher_is_better': True, 'scaling': 'weak', 'vs_baseline': None,
                  'dtype': a.dtype, 'data': 'synthetic', 'config': {'workload': a.config, 'global_batch': world * a.batch},
                  'roofline': None, 'cpu_baseline': None,
                  'error': ('rank 0 was terminated by the launcher (signal %d) before its worker finished: another rank died' if world > 1 else
                            'the supervisor was terminated (signal %d) before its worker finished') % signum})
            os._exit(1)
        signal.signal(signal.SIGTERM, terminated)
    for attempt in range(attempts):
        tries += 1
        rc, f2, p2, err = run_worker(argv, map_file)
        part = p2 or part
        full = f2 if f2 is not None else full      # (a worker that printed its line and died at teardown still measured)
        if rc != 0 or (rank == 0 and f2 is None):
            d = diagnose_fault(err, map_file)
            d.update(attempt=attempt, exit_status=rc)
            faults.append(d)
            stage('worker attempt %d ended with status %s: %s' % (attempt, rc, json.dumps(d)[:600]))
        if full is not None or (rank != 0 and rc == 0):
            break
    try:
        os.remove(map_file)
    except OSError:
        pass
    if rank != 0:
        return 0 if not faults or full is not None else 1
    cfg = CONFIGS[a.config]
    if full is None:
        line = {'metric': 'BEV images/s (%dx%d) %s' % (a.size, a.size, 'train step' if cfg['kind'] == 'train' else 'inference + rotated NMS'),
                'value': part['value'] if part else None, 'unit': 'images/s', 'n_gpus': world, 'steps': a.steps, 'warmup': a.warmup,
                'ms_per_step': part['ms_per_step'] if part else None, 'higher_is_better': True, 'scaling': 'weak', 'vs_baseline': None,
                'dtype': a.dtype, 'data': 'synthetic', 'config': {'workload': a.config, 'global_batch': world * a.batch},
                'roofline': None, 'cpu_baseline': None,
                'error': 'the measuring worker died in every attempt' + ('' if part is None else ' AFTER the timed region: value / ms_per_step are '
                         'the completed timed region of the last attempt, the roofline leg is missing')}
    else:
        line = full
    line['fault_retries'] = tries - 1
    if faults:
        line['faults'] = faults
    if full is None:
        # every attempt died (a wedged GPU after a memory-access fault, say): the line goes out NOW -- the other configurations
        # would only spend their 900 s timeouts on the same GPU while an outer timeout kills the supervisor first
        emit(line)
        return 1
    if world == 1 and a.config == 'train608' and cfg['kind'] == 'train':
        if not a.no_extra:
            # configs[3], configs[4], the bf16 mode and configs[2]'s per-GPU work, briefly -- each in a FRESH PROCESS (one process
            # per configuration: tools/order_probe.py, profiles/r03_order_probe.txt, shows train1216 at 234 images/s as the first
            # 54 GB allocation of a process and 200 after a 17 GB configuration was allocated and freed before it)
            stage('other configurations in fresh processes')
            others = {'infer32': measure_other('infer32', a.dtype, 8, 3),
                      'train1024': measure_other('train1024', a.dtype, 5, 2)}
            if a.dtype == 'f16':
                # the only mode that meets north_star's 1e-4 / 1e-3 parity bars (exact-f32 MFMA at 1/16 of the f16 rate): what it costs
                others['train608_f32'] = measure_other('train608', 'f32', 3, 2)
                others['train608_f32']['note'] = 'the parity mode: the reference-golden tests hold their 1e-4 loss / 1e-3 logit bounds in THIS mode only'
                others['train608_bf16'] = measure_other('train608', 'bf16', 6, 3)
                others['train608_bf16']['note'] = ('EXPERIMENTAL: one-step gradient cosine vs fp32 0.71-0.80 on a conditioned net (f16: 0.96-0.97), '
                                                  'equal to ideal bf16 storage of this function (DESIGN.md section 4); not a drop-in for f16')
            others['train1216_mosaic'] = measure_other('train1216', a.dtype, 4, 3)
            line['other_configs'] = others
        if not a.no_cpu_baseline:
            stage('cpu_baseline (oracle on the host cores)')
            # (torch's autograd engine asks the HIP runtime for its device count the first time backward() runs: hide the GPUs
            # from THIS process -- every GPU process of the run has already been started -- so that the supervisor stays without
            # any GPU state to the end)
            os.environ['HIP_VISIBLE_DEVICES'] = os.environ['ROCR_VISIBLE_DEVICES'] = ''
            try:
                line['cpu_baseline'] = cpu_baseline(2, a.size)
            except Exception as e:      # noqa: BLE001
                line['cpu_baseline'] = dict(error=repr(e))
    emit(line)
    return 0 if full is not None else 1


if __name__ == '__main__':
    main()
