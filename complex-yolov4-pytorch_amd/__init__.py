"""MI355X-native hot path for Complex-YOLOv4.  Host-side mirror of the reference's
model / geometry / post-processing interfaces over the C-ABI library ``libcyolo_hip.so``."""
__version__ = '0.1.0'

import os as _os


def _hardware_queues(env):
    """The engine runs weight gradients on a side HIP stream and the data-parallel wrapper its all-reduce on another.  HIP maps streams
    onto GPU_MAX_HW_QUEUES hardware queues (default 4) and, with RCCL's streams in the process, all three land on one queue and
    serialise: 794 images/s for 878 (complex_yolov4.cfg, batch 16, one rank through RcclDataParallel).  So: 8 where the environment
    says nothing, and where it spells out the default of 4 on a data-parallel path (several ranks, or CY_DDP_FORCE=1).
    CY_KEEP_HW_QUEUES=1 leaves the variable alone.  This only has an effect before the HIP runtime initialises: import this package, or
    set the variable, before the first device call."""
    if env.get('CY_KEEP_HW_QUEUES') == '1':
        return
    ranks = env.get('WORLD_SIZE', '1')
    parallel = env.get('CY_DDP_FORCE') == '1' or (ranks.isdigit() and int(ranks) > 1)
    if 'GPU_MAX_HW_QUEUES' not in env or (env['GPU_MAX_HW_QUEUES'] == '4' and parallel):
        env['GPU_MAX_HW_QUEUES'] = '8'


_hardware_queues(_os.environ)
