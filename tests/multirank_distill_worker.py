"""One rank of tests/test_gpu_multirank_distill.py, launched by torchrun (one process per GPU): its shard of a ranking
dataset, cut at query boundaries, under the distill objective.

First the last rank has no teacher, and every rank's training must return a configuration error; then each rank sets its
queries' teacher, the ranks train, and rank 0 trains the whole dataset on its one GPU. Rank 0 writes the ranks' errors and
whether the trees are equal as JSON to the output path.

usage: torchrun ... multirank_distill_worker.py <output.json>
"""

from __future__ import annotations

import datetime
import json
import os
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))
sys.path.insert(0, str(ROOT / "tests"))


def main():
    import numpy as np
    import oracle_lib as orc
    import torch
    import torch.distributed as dist
    from synth import ranking_binned

    from silvic_b200 import B200Backend, SilvicError, TeacherTop, params_from_dict

    rank, world, local = (int(os.environ[k]) for k in ("RANK", "WORLD_SIZE", "LOCAL_RANK"))
    torch.cuda.set_device(local)
    dist.init_process_group("nccl", timeout=datetime.timedelta(seconds=120))
    try:
        data = ranking_binned(60_000, [255] * 6 + [63] * 2, seed=5, mean_query=120.0)
        bounds = data.query_boundaries.astype(np.int64)
        rng = np.random.RandomState(4)
        ids = np.stack([rng.choice(int(n), 20, replace=False) if n >= 20 else np.full(20, -1) for n in np.diff(bounds)])
        teacher = TeacherTop(ids.astype(np.int32), rng.randn(*ids.shape).astype(np.float32))
        queries = len(bounds) - 1
        a, e = queries * rank // world, queries * (rank + 1) // world
        mine = TeacherTop(teacher.ids[a:e], teacher.logits[a:e])
        p = params_from_dict({"objective": "distill", "num_leaves": 63, "num_iterations": 3})
        b = B200Backend(local)
        b.load(data.shard(int(bounds[a]), int(bounds[e])), "distill", params=p)
        uid = [B200Backend.nccl_unique_id() if rank == 0 else None]
        dist.broadcast_object_list(uid, src=0)
        b.join_ranks(uid[0], world, rank)
        if rank != world - 1:
            b.set_teacher(mine)
        error = ""
        try:
            b.train(p, 0.0)
        except SilvicError as err:
            error = str(err)
        errors = [None] * world
        dist.all_gather_object(errors, error)
        b.set_teacher(mine)
        model = b.train(p, 0.0)
        b.close()
        dist.barrier()
        if rank == 0:
            with B200Backend(local) as one:
                one.load(data, "distill", params=p)
                one.set_teacher(teacher)
                single = one.train(p, 0.0)
            differences = [f"tree {k}: {d}" for k, (x, y) in enumerate(zip(model.trees, single.trees))
                           if (d := orc.trees_equal(x, y))]
            Path(sys.argv[1]).write_text(json.dumps({"errors": errors, "trees": [len(model.trees), len(single.trees)],
                                                     "differences": differences}))
        dist.barrier()
    finally:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
