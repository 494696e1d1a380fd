"""The softmax operators over lists where their kernels pass from one way of working to another, and where inputs come
near what f32 holds; against the definitions in 64 bits (lists_reference.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_lists import TYPES, backend, check_distill, check_log_probs, dense, random_teacher, rows_of  # noqa: F401

from silvic_b200 import TeacherTop

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("top", [20, 33, 128])
@pytest.mark.parametrize("width", [100, 257, 512, 513, 1024, 1025])
def test_a_warp_s_lanes_share_the_teacher(backend, width, top, rest, type_):  # noqa: F811
    """Marks and ids set by one lane and read by the others: repeated indices everywhere in the top, 19 lists (not a
    multiple of the lists a CTA takes)."""
    rng = np.random.RandomState(width + top)
    scores = dense(rng, 19, width, type_, 1)
    teacher = random_teacher(rng, [width] * 19, top, type_, rest, 1.3)
    ids = teacher.ids.contiguous()
    k = min(top, width)
    ids[::2, k // 2: k // 2 + 5] = ids[::2, :5]
    ids[3, :k] = ids[3, 0]
    ids[4, k - 1] = ids[4, 0]
    teacher = TeacherTop(ids, teacher.logits.contiguous(), teacher.log_sum, 1.3)
    for _ in range(3):
        check_distill(scores, teacher, backend.distill(scores, teacher, hessian=True), None, None, type_)


@pytest.mark.parametrize("lists,width", [(3, 700), (300, 9001), (5, 40000), (160, 2049)])
def test_equal_scores_are_counted_by_whole_warps(backend, lists, width):  # noqa: F811
    """More equal scores than a CTA gathers: the alternatives come from counts of digits, by warps of which some lanes
    have no entry left."""
    rng = np.random.RandomState(width)
    scores = torch.from_numpy(rng.randint(0, 2, (lists, width)).astype(np.float32)).cuda()
    scores[0] = 1.0
    scores[1, ::3] = -np.inf
    some = min(lists, 6)
    for top in (31, 128):
        got = backend.log_probs(scores, top=top)
        check_log_probs(scores[:some], rows_of(scores[:some]), None, top, 1.0,
                        type(got)(None, got.entropy[:some], got.log_sum[:some], got.top_ids[:some], got.top[:some]))
