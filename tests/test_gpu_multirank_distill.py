"""The distill objective over two ranks: each sets its own queries' teacher. A rank without one is an error on every
rank, not a wait; with all of them the ranks grow the trees of one GPU."""

from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
from synth import ranking_binned

from silvic_b200 import B200Backend, SilvicError, TeacherTop, params_from_dict

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_two_ranks_agree_on_the_teacher(device, tmp_path):
    import torch

    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    out = tmp_path / "result.json"
    cmd = ["timeout", "-k", "30", "300", sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2",
           "--master-addr", "127.0.0.1", f"--master-port={29500 + (os.getpid() + 301) % 2000}",
           str(ROOT / "tests" / "multirank_distill_worker.py"), str(out)]
    run = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, NCCL_NVLS_ENABLE="0", PYTHONPATH=str(ROOT)), capture_output=True,
                         text=True, timeout=400)
    assert run.returncode == 0, (run.stdout[-4000:], run.stderr[-4000:])
    got = json.loads(out.read_text())
    assert "another rank has no teacher" in got["errors"][0] and "has no teacher" in got["errors"][1], got
    assert got["trees"] == [3, 3] and not got["differences"], got


def test_one_rank_without_a_teacher_trains_once_it_has_one(device):
    data = ranking_binned(3_000, [31] * 4, seed=8, mean_query=40.0)
    queries = len(data.query_boundaries) - 1
    p = params_from_dict({"objective": "distill", "num_leaves": 7, "num_iterations": 2})
    with B200Backend(device) as b:
        b.load(data, "distill", params=p)
        b.join_ranks(B200Backend.nccl_unique_id(), 1, 0)
        with pytest.raises(SilvicError, match="no teacher"):
            b.train(p, 0.0)
        b.set_teacher(TeacherTop(np.zeros((queries, 1), np.int32), np.zeros((queries, 1), np.float32)))
        assert len(b.train(p, 0.0).trees) == 2
