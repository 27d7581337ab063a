#!/bin/bash
# One box: pytest -m gpu -x, smoke(), one bench line.  Ends at the first step that fails.
set -e -o pipefail
out=gpurun_out/${1:-v1}; mkdir -p $out
timeout -k 10 1800 python -u -m pytest tests/ -x -q -m gpu > $out/pytest.log 2>&1
timeout -k 10 300 python -u -c "import __graft_entry__ as g; g.smoke()"
timeout -k 10 600 python3 -u bench.py --gpus 1 --steps 20 --warmup 5 > $out/bench.json 2> $out/bench.err
cut -c1-260 $out/bench.json
