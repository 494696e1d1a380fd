"""The softmax operators over lists without a GPU: the reference's gradients against differences, and the refusals that
the binding makes before a handle is asked."""

from __future__ import annotations

import ctypes as C

import lists_reference as ref
import numpy as np
import pytest
import torch

from silvic_b200 import SilvicError, TeacherTop, _abi, build, lists, params_from_dict


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("t", [1.0, 2.5])
def test_the_gradient_is_the_loss_s_derivative(rest, t):
    r = np.random.RandomState(3)
    z = r.randn(17)
    ids, logits = [4, 9, -1, 0, 9], r.randn(5) * 2
    log_sum = float(np.log(np.exp(logits / t).sum()) + 0.4) if rest else None
    got = ref.distill(z, ids, logits, t, log_sum, 0.7)
    h = 1e-5
    for j in range(len(z)):
        up, down = z.copy(), z.copy()
        up[j] += h
        down[j] -= h
        d = (ref.distill(up, ids, logits, t, log_sum, 0.7)["loss"] - ref.distill(down, ids, logits, t, log_sum, 0.7)["loss"]) / (2 * h)
        assert abs(d - got["grad"][j]) < 1e-8  # h^2 of the third derivative, and 1e-16 / h
    assert abs(got["grad"].sum()) < 1e-12  # a shift of all scores changes nothing


def test_a_student_that_equals_its_teacher_has_loss_and_gradient_0():
    z = np.random.RandomState(1).randn(40) * 3
    order = np.argsort(-z)[:10]
    total = ref.softmax(z, 1.5)[2]
    got = ref.distill(z, order, z[order], 1.5, total)
    assert abs(got["loss"]) < 1e-12 and np.abs(got["grad"]).max() < 1e-12
    full = ref.distill(z, np.arange(40), z, 1.5)
    assert abs(full["loss"]) < 1e-12 and np.abs(full["grad"]).max() < 1e-12


def test_lists_arg_takes_rows_and_runs():
    a = lists.lists_arg(torch.zeros(3, 10, dtype=torch.bfloat16)[:, :7], None)
    assert (a.type, a.num_lists, a.width, a.stride, a.boundaries_dev) == (_abi.BF16, 3, 7, 10, None)
    a = lists.lists_arg(torch.zeros(1, 5), None)
    assert (a.type, a.num_lists, a.width, a.stride) == (_abi.F32, 1, 5, 5)
    bounds = torch.tensor([0, 2, 9], dtype=torch.int32)
    a = lists.lists_arg(torch.zeros(9, dtype=torch.float16), bounds)
    assert (a.type, a.num_lists, a.width, a.boundaries_dev) == (_abi.F16, 2, 9, bounds.data_ptr())


@pytest.mark.parametrize("scores,bounds", [
    (torch.zeros(3, 4, dtype=torch.float64), None),                                # another type
    (torch.zeros(3, 4, dtype=torch.int32), None),
    (torch.zeros(4), None),                                                        # 1-D without boundaries
    (torch.zeros(2, 3, 4), None),
    (torch.zeros(4, 3).t(), None),                                                 # columns are not contiguous
    (torch.zeros(1, 4).expand(3, 4), None),                                        # rows that overlap
    (torch.zeros(3, 4), torch.tensor([0, 4], dtype=torch.int32)),                  # 2-D with boundaries
    (torch.zeros(8)[::2], torch.tensor([0, 4], dtype=torch.int32)),
    (torch.zeros(4), torch.tensor([0, 4])),                                        # int64 boundaries
    (torch.zeros(4), torch.tensor([], dtype=torch.int32)),
    (torch.zeros(4), torch.zeros(2, 2, dtype=torch.int32)),
    (torch.zeros(4), torch.zeros(6, dtype=torch.int32)[::2]),
])
def test_lists_arg_refuses(scores, bounds):
    with pytest.raises(ValueError):
        lists.lists_arg(scores, bounds)


def test_given_and_weights_are_checked():
    assert lists.given_arg(torch.zeros(3, dtype=torch.int32), 3).shape == (3, 1)
    assert lists.given_arg(torch.zeros(5, 3, dtype=torch.int32).t(), 3).is_contiguous()
    for bad in (torch.zeros(3), torch.zeros(2, dtype=torch.int32), torch.zeros(3, 1, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            lists.given_arg(bad, 3)
    for bad in (torch.zeros(3, dtype=torch.float64), torch.zeros(4), torch.zeros(3, 1)):
        with pytest.raises(ValueError):
            lists.per_list_arg(bad, 3, "weight")


def test_teacher_arg_takes_slices_and_refuses():
    ids, logits = torch.zeros(3, 20, dtype=torch.int32), torch.zeros(3, 20, dtype=torch.bfloat16)
    t, keep = lists.teacher_arg(TeacherTop(ids[:, :8], logits[:, :8]), 3)
    assert (t.top, t.stride, t.type, t.log_sum_dev) == (8, 20, _abi.BF16, None) and len(keep) == 2
    t, keep = lists.teacher_arg(TeacherTop(ids[:, :8], logits[:, :8].contiguous(), torch.zeros(3)), 3)
    assert (t.top, t.stride) == (8, 8) and t.log_sum_dev == keep[2].data_ptr()
    for bad in (TeacherTop(ids.long(), logits), TeacherTop(ids, logits.double()), TeacherTop(ids[:2], logits[:2]),
                TeacherTop(ids, logits[:, :4]), TeacherTop(ids[:, :0], logits[:, :0]),
                TeacherTop(torch.zeros(3, 129, dtype=torch.int32), torch.zeros(3, 129)), TeacherTop(ids[0], logits[0]),
                TeacherTop(ids, logits, torch.zeros(4)), TeacherTop(ids, logits, torch.zeros(3, dtype=torch.float64)),
                TeacherTop(ids.t()[:3], logits.t()[:3])):
        with pytest.raises(ValueError):
            lists.teacher_arg(bad, 3)


def test_host_teacher_and_device_are_checked():
    ids, logits, log_sum = lists.host_teacher(TeacherTop([[0, 1]], [[0.5, 1.0]], [2.0]))
    assert ids.dtype == np.int32 and logits.dtype == np.float32 and log_sum.shape == (1,)
    for bad in (TeacherTop([0, 1], [0.5, 1.0]), TeacherTop([[0, 1]], [[0.5]]), TeacherTop([[0]], [[0.5]], [1.0, 2.0])):
        with pytest.raises(ValueError):
            lists.host_teacher(bad)
    with pytest.raises(ValueError, match="cuda:0"):
        lists.check_device(0, [torch.zeros(3)])


def test_the_entry_points_refuse_a_missing_handle():
    lib = _abi.load_library(build.build())
    arg, teacher = _abi.Lists(), _abi.Teacher()
    assert lib.sb2_log_probs(None, C.byref(arg), 1.0, None, 0, 0, None, None, None, None, None, None) == _abi.EDEVICE
    assert lib.sb2_distill(None, C.byref(arg), C.byref(teacher), 1.0, None, None, None, None, 0, None) == _abi.EDEVICE
    assert lib.sb2_set_teacher(None, None, None, None, 0, 1, 1.0) == _abi.EDEVICE


def test_distill_is_an_objective_with_initial_score_0():
    lib = _abi.load_library(build.build())
    p = params_from_dict({"objective": "distill"})
    assert p.objective == _abi.DISTILL
    out = C.c_double(5.0)
    assert lib.sb2_boost_from_average(C.byref(p), (C.c_float * 2)(3.0, 4.0), None, 2, C.byref(out)) == 0
    assert out.value == 0.0
    with pytest.raises(SilvicError):
        params_from_dict({"objective": "distil"})
