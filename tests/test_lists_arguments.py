"""Arguments of the softmax operators over lists that the binding refuses or converts, without a GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from silvic_b200 import TeacherTop, lists


def test_more_lists_than_a_call_takes_are_refused():
    """A count that its 32 bits would cut."""
    assert lists.lists_arg(torch.empty(2 ** 32 - 1, 0), None).num_lists == 2 ** 32 - 1
    for rows in (2 ** 32, 2 ** 32 + 3):
        with pytest.raises(ValueError, match="lists"):
            lists.lists_arg(torch.empty(rows, 0), None)
        with pytest.raises(ValueError, match="lists"):
            lists.lists_arg(torch.empty(4), torch.empty(rows + 1, dtype=torch.int32, device="meta"))


def test_a_training_teacher_s_ids_are_not_cut():
    """Ids that 32 bits would cut to others, and ids that are no whole numbers."""
    logits = np.zeros((1, 2), np.float32)
    ids, _, _ = lists.host_teacher(TeacherTop(np.array([[7, -1]], np.int64), logits))
    assert ids.dtype == np.int32 and ids.tolist() == [[7, -1]]
    assert lists.host_teacher(TeacherTop(np.array([[7, 2 ** 31 - 1]], np.uint64), logits))[0].tolist() == [[7, 2 ** 31 - 1]]
    for bad in ([[2 ** 32, 1]], [[0, -2 ** 31 - 1]], [[2 ** 31, 0]], [[0.5, 1.0]], [[True, False]]):
        with pytest.raises(ValueError, match="ids"):
            lists.host_teacher(TeacherTop(np.array(bad), logits))
    assert lists.host_teacher(TeacherTop(np.zeros((0, 3)), np.zeros((0, 3))))[0].shape == (0, 3)


def test_tensors_without_entries_are_taken_whatever_their_strides():
    for shape in ((0, 4), (4, 0), (0, 0)):
        for strides in ((1, 1), (0, 7), (3, 2)):
            arg = lists.lists_arg(torch.empty_strided(shape, strides), None)
            assert (arg.num_lists, arg.width, arg.stride) == (shape[0], shape[1], shape[1])
    t, _ = lists.teacher_arg(TeacherTop(torch.empty_strided((0, 4), (1, 1), dtype=torch.int32), torch.empty(0, 4)), 0)
    assert (t.top, t.stride) == (4, 4)
