"""`python bench.py --gpus N` starts its own ranks: what a rank that fails had to say survives in a file of its own."""
import glob
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="the ranks are to fail for want of a device")
def test_a_failed_ranks_stderr_is_kept(tmp_path):
    env = {k: v for k, v in os.environ.items() if k not in ("WORLD_SIZE", "RANK", "LOCAL_RANK")}
    env.update(LIBRA_DIST_BACKEND="gloo", LIBRA_RANK_LOGS=str(tmp_path))
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--gpus", "2", "--steps", "1", "--warmup", "1", "--no-cpu-baseline"],
                       capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode != 0 and str(tmp_path) in r.stderr and not r.stdout.strip(), (r.stdout[-500:], r.stderr[-2000:])
    logs = {f: open(f).read() for f in glob.glob(os.path.join(str(tmp_path), "**", "stderr.log"), recursive=True)}
    assert len(logs) == 2 and any("Traceback" in text for text in logs.values()), logs
