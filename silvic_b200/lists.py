"""Softmax operators over lists of candidates: what `B200Backend.log_probs` and `B200Backend.distill` take and return,
and the checks of their arguments.

A list is a row of a matrix (a position's logits over a vocabulary) or, with `boundaries`, a run of a flat tensor (a
query's documents: `query_boundaries` of a `BinnedDataset`). No counterpart in the reference.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import numpy as np

from . import _abi

MAX_TOP = 128  # most alternatives of a list, and most entries of a teacher's top
MAX_LISTS = 2 ** 32 - 1  # of one call


@dataclass
class LogProbs:
    """softmax(scores / temperature) of every list (CUDA tensors, f32; ids int32)."""

    given: Any      # [lists, given]: log probabilities of the given entries; None without any
    entropy: Any    # [lists], in nats
    log_sum: Any    # [lists]: ln sum exp(scores / temperature)
    top_ids: Any    # [lists, top]: the likeliest entries, ties by the lower index, -1 behind the last; None for top 0
    top: Any        # [lists, top]: their log probabilities; None for top 0


@dataclass
class TeacherTop:
    """A teacher's top logits of every list: `ids` int32 [lists, top] (an entry's index in its list, -1: padding) and
    `logits` [lists, top], up to any constant a list. Without `log_sum` the top is the whole teacher (renormalised);
    with it (f32 [lists], ln sum exp(logits / temperature) over the teacher's whole list, as `LogProbs.log_sum`; 0 for
    logits that are log probabilities) the rest of its mass is one more class. `temperature` softens both sides.

    CUDA tensors for `B200Backend.distill`, numpy arrays (f32 logits) for the training objective."""

    ids: Any
    logits: Any
    log_sum: Any = None
    temperature: float = 1.0


@dataclass
class Distilled:
    """The distillation loss of every list, and its derivatives in the scores' shape and type."""

    loss: Any               # f32 [lists]
    gradient: Any = None
    hessian: Any = None


# torch's part of this module, looked up by the first call: the package itself does without torch.
_torch = None
_TYPES: dict = {}


def _use_torch():
    global _torch
    if _torch is None:
        import torch

        _TYPES.update({torch.float32: _abi.F32, torch.bfloat16: _abi.BF16, torch.float16: _abi.F16})
        _torch = torch
    return _torch


def torch_float32():
    return _use_torch().float32


def stream(device: int) -> int:
    """torch's current stream of a device, as a cudaStream_t."""
    return _torch._C._cuda_getCurrentRawStream(device)


def _type_of(tensor, what: str) -> int:
    _use_torch()
    code = _TYPES.get(getattr(tensor, "dtype", None))
    if code is None:
        raise ValueError(f"{what}: a float32, bfloat16 or float16 tensor")
    return code


def _row_stride(tensor, what: str) -> int:
    """Entries from one row of a 2-D tensor to the next; its rows are contiguous and lie apart."""
    rows, cols = tensor.shape
    step, one = tensor.stride()
    if rows == 0 or cols == 0:  # whatever its strides
        return cols
    if cols > 1 and one != 1:
        raise ValueError(f"{what}: rows of contiguous entries")
    if rows <= 1:
        return cols
    if step < cols:
        raise ValueError(f"{what}: rows that do not overlap")
    return step


def lists_arg(scores, boundaries) -> _abi.Lists:
    """The lists of a 2-D tensor's rows, or of a 1-D tensor cut at `boundaries`."""
    code = _type_of(scores, "scores")
    if boundaries is None:
        if scores.dim() != 2:
            raise ValueError("scores: a 2-D tensor, or a 1-D one with boundaries")
        rows, cols = scores.shape
        if rows > MAX_LISTS:
            raise ValueError(f"{rows} lists; {MAX_LISTS} at most in one call")
        return _abi.Lists(scores.data_ptr(), code, rows, cols, _row_stride(scores, "scores"), None)
    torch = _torch
    if scores.dim() != 1 or (scores.shape[0] > 1 and scores.stride(0) != 1):
        raise ValueError("scores: a contiguous 1-D tensor with boundaries")
    if boundaries.dim() != 1 or boundaries.shape[0] < 1 or boundaries.dtype not in (torch.int32, torch.uint32) \
            or not boundaries.is_contiguous():
        raise ValueError("boundaries: a contiguous 1-D int32 or uint32 tensor of one entry more than lists")
    if boundaries.shape[0] - 1 > MAX_LISTS:
        raise ValueError(f"{boundaries.shape[0] - 1} lists; {MAX_LISTS} at most in one call")
    return _abi.Lists(scores.data_ptr(), code, boundaries.shape[0] - 1, scores.shape[0], 0, boundaries.data_ptr())


def output(scores, rows: int, columns: int = 0, ids: bool = False):
    """Memory for an output beside the scores, f32 or int32 [rows, columns], [rows] without columns. One of its own each,
    so that what is done to one output in place, or how long it is kept, is no matter of the others'."""
    return _torch.empty_strided((rows, columns) if columns else (rows,), (columns, 1) if columns else (1,),
                                dtype=_torch.int32 if ids else _torch.float32, device=scores.device)


def like(scores, rows: int, width: int, stride: int):
    """Memory for derivatives of `scores`: rows `stride` entries apart, or (1-D scores) a flat copy of it."""
    if scores.dim() == 1:  # (without lists nothing is launched)
        return scores.new_empty(scores.shape[0]) if rows > 0 else scores.new_zeros(scores.shape[0])
    if stride == width:
        return scores.new_empty((rows, width))
    return scores.new_empty((rows, stride)).as_strided((rows, width), (stride, 1))


def given_arg(given, num_lists: int):
    """The given entries as a contiguous int32 [lists, n] tensor (a 1-D one: an entry a list)."""
    if given.dtype != _use_torch().int32:
        raise ValueError("given: an int32 tensor")
    if given.dim() == 1:
        given = given[:, None]
    if given.dim() != 2 or given.shape[0] != num_lists:
        raise ValueError(f"given of shape {tuple(given.shape)} for {num_lists} lists")
    return given.contiguous()


def per_list_arg(values, num_lists: int, what: str):
    """An f32 value a list, contiguous."""
    if values.dtype != _use_torch().float32 or values.dim() != 1 or values.shape[0] != num_lists:
        raise ValueError(f"{what}: a float32 tensor of {num_lists} values")
    return values.contiguous()


def teacher_arg(teacher: TeacherTop, num_lists: int):
    """(the C struct, the tensors it points to) of a teacher's CUDA tensors."""
    ids, logits = teacher.ids, teacher.logits
    code = _type_of(logits, "the teacher's logits")
    if ids.dtype != _torch.int32 or ids.dim() != 2:
        raise ValueError("the teacher's ids: a 2-D int32 tensor")
    if ids.shape[0] != num_lists or ids.shape != logits.shape:
        raise ValueError(f"a teacher of ids {tuple(ids.shape)} and logits {tuple(logits.shape)} for {num_lists} lists")
    if not 1 <= ids.shape[1] <= MAX_TOP:
        raise ValueError(f"a teacher's top of {ids.shape[1]} entries; 1 to {MAX_TOP} are taken")
    stride = _row_stride(ids, "the teacher's ids")
    if stride != _row_stride(logits, "the teacher's logits"):
        ids, logits = ids.contiguous(), logits.contiguous()
        stride = ids.shape[1]
    log_sum = None if teacher.log_sum is None else per_list_arg(teacher.log_sum, num_lists, "the teacher's log sums")
    keep = [ids, logits] + ([] if log_sum is None else [log_sum])
    return _abi.Teacher(ids.data_ptr(), logits.data_ptr(), code, ids.shape[1], stride,
                        None if log_sum is None else log_sum.data_ptr()), keep


def check_device(device: int, tensors):
    """Every tensor on the handle's device; last among the checks."""
    for t in tensors:
        if t is not None and (not t.is_cuda or t.get_device() != device):
            raise ValueError(f"a tensor on {t.device}, not on the handle's device cuda:{device}")


def host_teacher(teacher: TeacherTop):
    """(ids, logits, log_sum or None) of a training teacher as C-contiguous numpy arrays."""
    ids = np.asarray(teacher.ids)
    if ids.size and (ids.dtype.kind not in "iu" or ids.min() < -2 ** 31 or ids.max() >= 2 ** 31):
        raise ValueError(f"the teacher's ids: whole numbers of 32 bits, not {ids.dtype} from {ids.min()} to {ids.max()}")
    ids = np.ascontiguousarray(ids, dtype=np.int32)
    logits = np.ascontiguousarray(teacher.logits, dtype=np.float32)
    if ids.ndim != 2 or ids.shape != logits.shape:
        raise ValueError(f"a teacher of ids {ids.shape} and logits {logits.shape}")
    log_sum = None
    if teacher.log_sum is not None:
        log_sum = np.ascontiguousarray(teacher.log_sum, dtype=np.float32)
        if log_sum.shape != ids.shape[:1]:
            raise ValueError(f"the teacher's log sums of shape {log_sum.shape} for {ids.shape[0]} lists")
    return ids, logits, log_sum
