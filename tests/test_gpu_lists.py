"""The softmax operators over lists of candidates on the device, against their definitions in 64 bits
(lists_reference.py, which derives the tolerances)."""

from __future__ import annotations

import ctypes as C

import lists_reference as ref
import numpy as np
import pytest
import torch
from synth import ranking_binned

from silvic_b200 import B200Backend, SilvicError, TeacherTop, _abi, init_score, params_from_dict, train

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def backend(device):
    with B200Backend(device) as b:
        yield b


def dense(rng, lists, width, type_, pad=0, offset=0, scale=3.0):
    """[lists, width] scores of a type in rows width + pad apart that start `offset` entries into their memory."""
    flat = torch.zeros(offset + lists * (width + pad), dtype=TYPES[type_], device="cuda")
    view = flat[offset:].view(lists, width + pad)
    view.copy_(torch.from_numpy(rng.randn(lists, width + pad) * scale).to(TYPES[type_]))
    return view[:, :width]


def host(t):
    return None if t is None else t.double().cpu().numpy()


def check_log_probs(scores, rows, given, top, t, got):
    got = {k: host(getattr(got, k)) for k in ("given", "entropy", "log_sum", "top_ids", "top")}
    for i, z in enumerate(rows):
        ref.check_log_probs(z, t, [] if given is None else given[i], top,
                            {k: None if v is None else v[i] for k, v in got.items()})


def rows_of(scores, boundaries=None):
    z = host(scores)
    return list(z) if boundaries is None else [z[a:b] for a, b in zip(boundaries[:-1], boundaries[1:])]


def tolerance(type_):
    """(relative half step, half the smallest step) of a gradient's type."""
    return {"f32": (2.0 ** -24, 0.0), "bf16": (2.0 ** -8, 0.0), "f16": (2.0 ** -11, 2.0 ** -25)}[type_]


def check_distill(scores, teacher, got, weight=None, boundaries=None, type_="f32"):
    rows = rows_of(scores, boundaries)
    ids, logits, log_sum = host(teacher.ids), host(teacher.logits), host(teacher.log_sum)
    loss, w = host(got.loss), host(weight)
    parts = {k: None if v is None else rows_of(v, boundaries) for k, v in (("grad", got.gradient), ("hess", got.hessian))}
    step, least = tolerance(type_)
    for i, z in enumerate(rows):
        ref.check_distill(z, ids[i], logits[i], teacher.temperature, None if log_sum is None else float(log_sum[i]),
                          1.0 if w is None else float(w[i]),
                          {"loss": loss[i], **{k: None if v is None else v[i] for k, v in parts.items()}}, step, least)


def random_teacher(rng, sizes, top, type_="f32", rest=False, t=1.0, pad=0):
    """Distinct ids of each list (-1 behind a short one's last), logits, and a log sum that leaves a rest."""
    ids = np.full((len(sizes), top + pad), -1, np.int32)
    for i, n in enumerate(sizes):
        k = min(top, int(n))
        ids[i, :k] = rng.choice(int(n), k, replace=False) if n > 0 else []
    logits = torch.from_numpy(rng.randn(len(sizes), top + pad) * 2 + 1).to(TYPES[type_]).cuda()
    ids = torch.from_numpy(ids).cuda()
    log_sum = None
    if rest:
        x = torch.where(ids >= 0, logits.double() / t, -np.inf)[:, :top]
        log_sum = torch.logsumexp(x, 1) + 0.3
        log_sum = torch.where(torch.isfinite(log_sum), log_sum, 0.0).float()
    return TeacherTop(ids[:, :top], logits[:, :top], log_sum, t)


# ---- log probabilities ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lists,width,pad,offset,top,given", [
    (1, 1, 0, 0, 1, 1), (3, 2, 0, 0, 5, 2), (5, 31, 0, 1, 3, 1), (4, 33, 3, 0, 33, 2), (2, 128, 0, 0, 128, 1),
    (7, 255, 1, 3, 0, 1), (3, 1000, 0, 0, 20, 8), (200, 1025, 7, 0, 10, 1), (2, 4099, 0, 5, 64, 0), (1, 32769, 0, 0, 128, 3),
    (160, 5000, 0, 0, 7, 1), (2, 70001, 0, 1, 20, 2), (1, 300007, 0, 0, 20, 1), (400, 64, 0, 0, 8, 1)])
@pytest.mark.parametrize("type_", ["f32", "bf16", "f16"])
def test_log_probs_dense(backend, lists, width, pad, offset, top, given, type_):
    rng = np.random.RandomState(lists * 7 + width)
    scores = dense(rng, lists, width, type_, pad, offset)
    ids = rng.randint(-1, width + 1, (lists, given)).astype(np.int32) if given else None
    got = backend.log_probs(scores, given=None if ids is None else torch.from_numpy(ids).cuda(), top=top, temperature=0.8)
    check_log_probs(scores, rows_of(scores), ids, top, 0.8, got)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[0, 1, 0, 3, 0], [5] * 40, [1, 32, 33, 1024, 1025, 0, 7, 2000, 64, 65, 4097, 1],
                                   [20000, 3, 9000, 1, 1]])
def test_log_probs_ragged(backend, sizes, type_):
    rng = np.random.RandomState(len(sizes))
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    scores = torch.from_numpy(np.round(rng.randn(bounds[-1]) * 20) / 8).to(TYPES[type_]).cuda()  # many ties
    ids = np.array([[rng.randint(0, max(n, 1)), n] for n in sizes], np.int32)
    for dtype in (torch.int32, torch.uint32):
        got = backend.log_probs(scores, given=torch.from_numpy(ids).cuda(), top=12, temperature=1.5,
                                boundaries=torch.from_numpy(bounds.astype(np.int32)).to(dtype).cuda())
        check_log_probs(scores, rows_of(scores, bounds), ids, 12, 1.5, got)


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("width", [17, 900, 9001, 66000])
def test_log_probs_masks_ties_and_orders(backend, type_, width):
    """Masked entries (-inf and the type's lowest value), whole rows of them, equal scores, -0 beside 0, scores in
    ascending and descending order, and every large score in one stretch."""
    rng = np.random.RandomState(width)
    z = rng.randn(10, width) * 2
    z[0] = -np.inf
    z[1, 1:] = -np.inf
    z[2, rng.rand(width) < 0.9] = -np.inf
    z[3] = 0.0
    z[3, ::2] = -0.0
    z[4] = torch.finfo(TYPES[type_]).min
    z[5, ::3] = torch.finfo(TYPES[type_]).min
    z[6] = np.sort(z[6])
    z[7] = np.sort(z[7])[::-1]
    z[8, width // 2: width // 2 + 100] += 20
    z[9, ::max(1, width // 64)] += 20
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    ids = np.stack([np.arange(10) % width, np.full(10, width - 1)], 1).astype(np.int32)
    for top in (5, 64, 128):
        got = backend.log_probs(scores, given=torch.from_numpy(ids).cuda(), top=top)
        check_log_probs(scores, rows_of(scores), ids, top, 1.0, got)


def test_log_probs_of_nan_and_inf(backend):
    z = torch.randn(4, 700, device="cuda")
    z[0, 3] = float("nan")
    z[1, 690] = float("inf")
    z[2, 5] = float("-inf")
    got = backend.log_probs(z, given=torch.zeros(4, 1, dtype=torch.int32, device="cuda"), top=3)
    for v in (got.entropy, got.log_sum, got.given[:, 0]):
        assert torch.isnan(v[:2]).all() and torch.isfinite(v[2:]).all()
    assert got.top_ids[1, 0] == 690  # +inf is the likeliest entry
    row = host(z)
    for i in (2, 3):
        assert np.array_equal(host(got.top_ids)[i], np.argsort(-row[i], kind="stable")[:3])


def test_log_probs_of_a_slice_of_positions(backend):
    """The last position's logits of a [batch, positions, vocabulary] tensor: rows far apart."""
    whole = torch.randn(3, 50, 2001, device="cuda").to(torch.bfloat16)
    got = backend.log_probs(whole[:, -1, :], top=4)
    check_log_probs(whole[:, -1, :], rows_of(whole[:, -1, :]), None, 4, 1.0, got)


def test_log_probs_past_32_bit_offsets(backend):
    """Rows behind 2^32 bytes and 2^31 entries of a cache."""
    stride = (1 << 31) + 24
    whole = torch.zeros(stride + 5000, dtype=torch.bfloat16, device="cuda")
    rows = whole.as_strided((2, 5000), (stride, 1))
    rows.copy_(torch.randn(2, 5000, device="cuda"))
    got = backend.log_probs(rows, given=torch.tensor([[1], [4999]], dtype=torch.int32, device="cuda"), top=6)
    check_log_probs(rows, rows_of(rows), np.array([[1], [4999]]), 6, 1.0, got)


# ---- distillation --------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lists,width,pad,offset,top", [
    (1, 1, 0, 0, 1), (3, 2, 0, 0, 5), (5, 31, 0, 1, 3), (4, 33, 3, 0, 33), (2, 128, 0, 0, 128), (7, 255, 1, 3, 16),
    (3, 1000, 0, 0, 20), (200, 1025, 7, 0, 10), (2, 4099, 0, 5, 64), (1, 32769, 0, 0, 128), (160, 5000, 0, 0, 7),
    (2, 70001, 0, 1, 100), (1, 300007, 0, 0, 20), (400, 64, 0, 0, 8)])
@pytest.mark.parametrize("type_", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_dense(backend, lists, width, pad, offset, top, type_, rest):
    rng = np.random.RandomState(lists * 5 + width)
    scores = dense(rng, lists, width, type_, pad, offset)
    teacher = random_teacher(rng, [width] * lists, top, type_, rest, 1.7)
    weight = torch.from_numpy(rng.rand(lists) + 0.5).float().cuda()
    got = backend.distill(scores, teacher, weight=weight, hessian=True)
    assert got.gradient.dtype == got.hessian.dtype == scores.dtype and got.gradient.shape == scores.shape
    check_distill(scores, teacher, got, weight, None, type_)
    alone = backend.distill(scores, teacher, weight=weight, gradient=False)
    assert alone.gradient is None and alone.hessian is None
    check_distill(scores, teacher, alone, weight, None, type_)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("sizes", [[0, 1, 0, 3, 0], [5] * 40, [1, 32, 33, 1024, 1025, 0, 7, 2000, 64, 65, 4097, 1],
                                   [20000, 3, 9000, 1, 1]])
def test_distill_ragged(backend, sizes, rest):
    rng = np.random.RandomState(len(sizes) + rest)
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    scores = torch.from_numpy(np.round(rng.randn(bounds[-1]) * 20) / 8).float().cuda()
    teacher = random_teacher(rng, sizes, 12, "f32", rest)
    got = backend.distill(scores, teacher, boundaries=torch.from_numpy(bounds.astype(np.int32)).cuda(), hessian=True)
    check_distill(scores, teacher, got, None, bounds)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("width", [40, 3001, 140001])
def test_distill_masks_duplicates_and_padding(backend, type_, width):
    rng = np.random.RandomState(width)
    z = rng.randn(9, width) * 2
    top = 6
    ids = np.stack([rng.choice(width, top, replace=False) for _ in range(9)]).astype(np.int32)
    logits = rng.randn(9, top)
    z[0] = -np.inf                                  # an empty list
    z[1, rng.rand(width) < 0.8] = -np.inf           # masked, some of the teacher's entries too
    z[2, ids[2, 0]] = -np.inf                       # the teacher's own entry masked: loss +inf
    ids[3] = -1                                     # no teacher
    ids[4, 2:] = -1
    ids[5, 3:] = [width, -7, 2 ** 31 - 1]           # outside the list: padding
    ids[6] = ids[6, 0]                              # one entry, named six times
    logits[7] = -np.inf                             # a teacher that gives its top nothing
    logits[8, ::2] = -np.inf
    z[8, [j for j in range(width) if j not in ids[8]]] = -np.inf  # no mass outside the top
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    for log_sum in (None, torch.full((9,), 3.0, device="cuda")):
        teacher = TeacherTop(torch.from_numpy(ids).cuda(), torch.from_numpy(logits).float().cuda(), log_sum, 1.25)
        got = backend.distill(scores, teacher, hessian=True)
        check_distill(scores, teacher, got, None, None, type_)


def test_distill_of_nan_and_inf_stays_in_its_list(backend):
    z = torch.randn(4, 700, device="cuda")
    z[0, 3] = float("nan")
    z[1, 690] = float("inf")
    teacher = random_teacher(np.random.RandomState(0), [700] * 4, 5)
    teacher.logits[2, 1] = float("nan")
    got = backend.distill(z, teacher, hessian=True)
    assert torch.isnan(got.loss[:3]).all() and torch.isfinite(got.loss[3])
    assert torch.isnan(got.gradient[:2]).all() and torch.isfinite(got.gradient[3]).all()


def test_a_learned_teacher_has_loss_and_gradient_near_0(backend):
    """The operators together: a teacher's logits -> its top log probabilities and log sum -> a student at the
    teacher's own scores. Nothing is left to learn; a teacher elsewhere is checked against the definition."""
    rng = np.random.RandomState(5)
    teacher_logits = dense(rng, 6, 20011, "bf16")
    t = 2.0
    lp = backend.log_probs(teacher_logits, top=32, temperature=t)
    top = TeacherTop(lp.top_ids, torch.gather(teacher_logits, 1, lp.top_ids.long()), lp.log_sum, t)
    got = backend.distill(teacher_logits.float().contiguous(), top)
    # q and p come from the same scores; each ln is off by ref.slack and 4 U of itself (|x| <= 16 here) at most
    assert host(got.loss).__abs__().max() <= 4 * ref.slack(20011) + 8 * 16 * ref.U
    student = dense(rng, 6, 20011, "f32")
    # Log probabilities in the place of logits, as an API returns them: a log sum of 0 and temperature 1.
    lp = backend.log_probs(teacher_logits, top=20)
    told = TeacherTop(lp.top_ids, lp.top, torch.zeros(6, device="cuda"))
    check_distill(student, told, backend.distill(student, told, hessian=True))
    assert torch.equal(lp.top_ids, backend.log_probs(teacher_logits.contiguous(), top=20).top_ids)


def test_gaps_between_lists_stay_as_they_are(backend):
    """Straight through the C entry: entries between dense rows, and behind the last boundary, are not written."""
    scores = torch.randn(5, 40, device="cuda")
    grad = torch.full((5, 48), 7.0, device="cuda")
    teacher = random_teacher(np.random.RandomState(1), [33] * 5, 4)
    lists = _abi.Lists(scores.data_ptr(), _abi.F32, 5, 33, 40, None)
    t = _abi.Teacher(teacher.ids.data_ptr(), teacher.logits.data_ptr(), _abi.F32, 4, 4, None)
    backend._check(backend._lib.sb2_distill(backend._h, C.byref(lists), C.byref(t), 1.0, None, None, grad.data_ptr(), None,
                                            48, None))
    torch.cuda.synchronize()
    assert (grad[:, 33:] == 7.0).all() and (grad[:, :33] != 7.0).all()
    assert torch.equal(grad[:, :33], backend.distill(scores[:, :33], teacher).gradient)
    bounds = torch.tensor([3, 40, 60], dtype=torch.int32, device="cuda")
    lists = _abi.Lists(scores.data_ptr(), _abi.F32, 2, 200, 0, bounds.data_ptr())
    flat = torch.full((200,), 7.0, device="cuda")
    t = _abi.Teacher(teacher.ids.data_ptr(), teacher.logits.data_ptr(), _abi.F32, 4, 4, None)
    backend._check(backend._lib.sb2_distill(backend._h, C.byref(lists), C.byref(t), 1.0, None, None, flat.data_ptr(), None,
                                            0, None))
    torch.cuda.synchronize()
    assert (flat[:3] == 7.0).all() and (flat[60:] == 7.0).all() and (flat[3:60] != 7.0).all()


def test_boundaries_outside_the_entries_are_cut_off(backend):
    """Boundaries are device memory: whatever they hold, no entry outside the tensor is read or written."""
    scores = torch.randn(100, device="cuda")
    bounds = torch.tensor([0, 60, 40, 90, 1000, 2000], dtype=torch.int32, device="cuda")
    want = [(0, 60), (60, 60), (40, 90), (90, 100), (100, 100)]
    got = backend.log_probs(scores, top=2, boundaries=bounds)
    check_log_probs(scores, [host(scores)[a:b] for a, b in want], None, 2, 1.0, got)
    # gradients of lists that do not share entries
    bounds = torch.tensor([10, 60, 60, 1000, 2000], dtype=torch.int32, device="cuda")
    teacher = random_teacher(np.random.RandomState(2), [50, 0, 40, 0], 4)
    got = backend.distill(scores, teacher, boundaries=bounds)
    ref_grad = host(got.gradient)
    for i, (a, b) in enumerate([(10, 60), (60, 60), (60, 100), (100, 100)]):
        ref.check_distill(host(scores)[a:b], host(teacher.ids)[i], host(teacher.logits)[i], 1.0, None, 1.0,
                          {"loss": host(got.loss)[i], "grad": ref_grad[a:b]}, 2.0 ** -24)


# ---- streams, graphs, repeated calls -------------------------------------------------------------------------------


def test_calls_follow_torch_s_current_stream(backend):
    side = torch.cuda.Stream()
    x = torch.zeros(64, 40001, device="cuda", dtype=torch.bfloat16)
    teacher = random_teacher(np.random.RandomState(4), [40001] * 64, 9, "bf16", True)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        x.copy_(torch.randn(x.shape, device="cuda"))
        lp, d = backend.log_probs(x, top=3), backend.distill(x, teacher)
    side.synchronize()
    again, d2 = backend.log_probs(x, top=3), backend.distill(x, teacher)
    for a, b in [(lp.entropy, again.entropy), (lp.log_sum, again.log_sum), (lp.top, again.top), (d.loss, d2.loss),
                 (d.gradient, d2.gradient)]:
        assert torch.equal(a, b)
    assert torch.equal(lp.top_ids, again.top_ids)


def test_two_streams_at_once_do_not_disturb_one_another(backend):
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [torch.randn(300, 30011, device="cuda"), torch.randn(2, 200003, device="cuda")]
    teachers = [random_teacher(np.random.RandomState(i), [x.shape[1]] * x.shape[0], 30, "f32", True) for i, x in enumerate(xs)]
    torch.cuda.synchronize()
    want = [(backend.log_probs(x, top=9), backend.distill(x, t)) for x, t in zip(xs, teachers)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for s, x, t in zip(streams, xs, teachers):
            with torch.cuda.stream(s):
                got.append((backend.log_probs(x, top=9), backend.distill(x, t)))
    torch.cuda.synchronize()
    for i, (lp, d) in enumerate(got):
        a, b = want[i % 2]
        assert torch.equal(lp.top_ids, a.top_ids) and torch.equal(lp.entropy, a.entropy) and torch.equal(lp.top, a.top)
        assert torch.equal(d.loss, b.loss) and torch.equal(d.gradient, b.gradient)


def test_captured_graphs_replay_on_new_inputs(backend):
    """Two graphs, captured one after the other and replayed in turn, against eager calls on the same inputs."""
    shapes = [(3, 50257), (500, 130)]
    graphs, state = [], []
    for lists, width in shapes:
        x = torch.randn(lists, width, device="cuda")
        teacher = random_teacher(np.random.RandomState(width), [width] * lists, 11, "f32", True)
        backend.distill(x, teacher), backend.log_probs(x, top=5)  # warm
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = backend.log_probs(x, top=5), backend.distill(x, teacher, hessian=True)
        graphs.append(g)
        state.append((x, teacher, out))
    for turn in range(3):
        for g, (x, teacher, (lp, d)) in zip(graphs, state):
            x.copy_(torch.randn_like(x) * (turn + 1))
            g.replay()
            lp2, d2 = backend.log_probs(x, top=5), backend.distill(x, teacher, hessian=True)
            assert torch.equal(lp.top_ids, lp2.top_ids) and torch.equal(lp.top, lp2.top) and torch.equal(lp.entropy, lp2.entropy)
            assert torch.equal(d.loss, d2.loss) and torch.equal(d.gradient, d2.gradient) and torch.equal(d.hessian, d2.hessian)


def test_a_list_s_results_do_not_depend_on_its_neighbours(backend):
    """A query's gradients are the same bits in any shard of the rows."""
    rng = np.random.RandomState(9)
    sizes = rng.poisson(120, 60)
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    scores = torch.from_numpy(rng.randn(bounds[-1])).float().cuda()
    teacher = random_teacher(rng, sizes, 30, "f32", True)
    whole = backend.distill(scores, teacher, boundaries=torch.from_numpy(bounds.astype(np.int32)).cuda(), hessian=True)
    for first in (7, 31):
        part = slice(int(bounds[first]), int(bounds[-1]))
        t = TeacherTop(teacher.ids[first:], teacher.logits[first:], teacher.log_sum[first:])
        b = torch.from_numpy((bounds[first:] - bounds[first]).astype(np.int32)).cuda()
        got = backend.distill(scores[part].clone(), t, boundaries=b, hessian=True)
        assert torch.equal(got.loss, whole.loss[first:]) and torch.equal(got.gradient, whole.gradient[part])
        assert torch.equal(got.hessian, whole.hessian[part])


def test_no_lists_and_no_entries(backend):
    for shape in [(0, 10), (3, 0)]:
        x = torch.zeros(shape, device="cuda")
        got = backend.log_probs(x, given=torch.zeros(shape[0], 1, dtype=torch.int32, device="cuda"), top=2)
        assert got.top_ids.shape == (shape[0], 2) and (got.top_ids == -1).all() and (got.given == -np.inf).all()
        assert (got.entropy == 0).all() and (got.log_sum == -np.inf).all()
        t = TeacherTop(torch.zeros(shape[0], 2, dtype=torch.int32, device="cuda"), torch.zeros(shape[0], 2, device="cuda"))
        d = backend.distill(x, t, hessian=True)
        assert d.gradient.shape == shape and (d.loss == 0).all()


# ---- refusals ------------------------------------------------------------------------------------------------------


def test_the_entry_points_refuse(backend):
    x = torch.randn(4, 100, device="cuda")
    teacher = random_teacher(np.random.RandomState(0), [100] * 4, 5)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        with pytest.raises(SilvicError, match="temperature"):
            backend.log_probs(x, temperature=t)
        with pytest.raises(SilvicError, match="temperature"):
            backend.distill(x, TeacherTop(teacher.ids, teacher.logits, None, t))
    for top in (-1, 129):
        with pytest.raises(ValueError, match="alternatives"):
            backend.log_probs(x, top=top)
    with pytest.raises(ValueError, match="device"):
        backend.log_probs(x.cpu())
    with pytest.raises(ValueError, match="device"):
        backend.distill(x, TeacherTop(teacher.ids.cpu(), teacher.logits))
    with pytest.raises(ValueError, match="device"):
        backend.distill(x, teacher, weight=torch.ones(4))

    def log_probs(lists, top=0, ids=None, out=None):
        backend._check(backend._lib.sb2_log_probs(backend._h, C.byref(lists), 1.0, None, 0, top, None, None, None, ids, out,
                                                  None))

    def distill(lists, t, grad=None, hess=None, stride=0):
        backend._check(backend._lib.sb2_distill(backend._h, C.byref(lists), C.byref(t), 1.0, None, None, grad, hess, stride,
                                                None))

    host_memory = np.zeros(400, np.float32)
    ok = _abi.Lists(x.data_ptr(), _abi.F32, 4, 100, 100, None)
    t = _abi.Teacher(teacher.ids.data_ptr(), teacher.logits.data_ptr(), _abi.F32, 5, 5, None)
    for lists, code in [(_abi.Lists(host_memory.ctypes.data, _abi.F32, 4, 100, 100, None), _abi.EDATA),
                        (_abi.Lists(None, _abi.F32, 4, 100, 100, None), _abi.EDATA),
                        (_abi.Lists(x.data_ptr(), 9, 4, 100, 100, None), _abi.EDATA),
                        (_abi.Lists(x.data_ptr() + 2, _abi.F32, 4, 99, 99, None), _abi.EDATA),
                        (_abi.Lists(x.data_ptr(), _abi.F32, 4, 100, 50, None), _abi.EDATA),
                        (_abi.Lists(x.data_ptr(), _abi.F32, 1, 1 << 31, 0, None), _abi.EUNSUPPORTED),
                        (_abi.Lists(x.data_ptr(), _abi.F32, 4, 100, 1 << 62, None), _abi.EUNSUPPORTED),
                        (_abi.Lists(x.data_ptr(), _abi.F32, 4, 1 << 32, 0, x.data_ptr()), _abi.EUNSUPPORTED),
                        (_abi.Lists(x.data_ptr(), _abi.F32, 4, 100, 0, host_memory.ctypes.data), _abi.EDATA)]:
        for call in (lambda: log_probs(lists), lambda: distill(lists, t)):
            with pytest.raises(SilvicError) as e:
                call()
            assert e.value.code == code
    with pytest.raises(SilvicError, match="alternatives"):
        log_probs(ok, 129, x.data_ptr(), x.data_ptr())
    with pytest.raises(SilvicError, match="null"):
        log_probs(ok, 3)
    with pytest.raises(SilvicError, match="device memory"):
        log_probs(ok, 3, host_memory.ctypes.data, host_memory.ctypes.data)
    grad = torch.empty_like(x)
    for top, stride in [(0, 5), (129, 129), (5, 4)]:
        with pytest.raises(SilvicError):
            distill(ok, _abi.Teacher(teacher.ids.data_ptr(), teacher.logits.data_ptr(), _abi.F32, top, stride, None))
    with pytest.raises(SilvicError, match="overlap"):
        distill(ok, t, x.data_ptr())
    with pytest.raises(SilvicError, match="overlap"):
        distill(ok, t, x.data_ptr() + 4 * 399)
    with pytest.raises(SilvicError, match="overlap"):
        distill(ok, t, grad.data_ptr(), grad.data_ptr())
    with pytest.raises(SilvicError):
        distill(ok, t, grad.data_ptr(), None, 99)
    with pytest.raises(SilvicError, match="device memory"):
        distill(ok, t, host_memory.ctypes.data)
    assert backend.log_probs(x).entropy.shape == (4,)  # the handle goes on


# ---- the training objective ----------------------------------------------------------------------------------------


def ranking_teacher(rng, bounds, top, rest):
    t = random_teacher(rng, np.diff(bounds), top, "f32", rest, 1.5)
    return TeacherTop(t.ids.cpu().numpy(), t.logits.cpu().numpy(), None if t.log_sum is None else t.log_sum.cpu().numpy(), 1.5)


def check_gradients(data, teacher, scores, g, h):
    bounds = data.query_boundaries.astype(np.int64)
    for q in range(len(bounds) - 1):
        a, b = bounds[q], bounds[q + 1]
        w = data.weight[a:b].astype(np.float64) if data.weight is not None else np.ones(b - a)
        ls = None if teacher.log_sum is None else float(teacher.log_sum[q])
        # a row's weight multiplies after the list's derivatives: one more rounding, within `relative`'s constant
        ref.check_distill(scores[a:b].astype(np.float64), teacher.ids[q], teacher.logits[q], 1.5, ls, 1.0,
                          {"grad": g[a:b] / w, "hess": h[a:b] / w}, 2.0 ** -23)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_objective_gradients(device, rest, weighted):
    rng = np.random.RandomState(3)
    data = ranking_binned(3_000, [31] * 4, seed=8, mean_query=40.0)
    bounds = data.query_boundaries.astype(np.int64)
    data.query_boundaries = np.concatenate([[0, 1], bounds[1:]]).astype(np.uint32)  # a single-row query first
    if weighted:
        data.weight = (rng.rand(data.num_rows) + 0.5).astype(np.float32)
    teacher = ranking_teacher(rng, data.query_boundaries.astype(np.int64), 6, rest)
    with B200Backend(device) as b:
        b.load(data, "distill")
        with pytest.raises(SilvicError, match="no teacher"):
            b.compute_gradients()
        b.set_teacher(teacher)
        for value in (0.0, -3.25):
            b.init_scores(0, value)
            most_g, most_h = b.compute_gradients()
            g, h = b.read_gradients()
            check_gradients(data, teacher, np.full(data.num_rows, value, np.float32), g, h)
            assert most_g == np.abs(g).max() and most_h == np.abs(h).max()


@pytest.mark.parametrize("rest", [False, True])
def test_training_takes_the_teacher_s_gradients(device, rest):
    """Each iteration's gradients are those at the scores of the trees before it, and a run of more iterations starts
    with the trees of a shorter one; a long query (5,000 rows) among the others."""
    rng = np.random.RandomState(4)
    data = ranking_binned(30_000, [255] * 6 + [63] * 2, seed=5, mean_query=120.0)
    bounds = data.query_boundaries.astype(np.int64)
    keep = bounds[(bounds == 0) | (bounds >= 5_000)]
    data.query_boundaries = keep.astype(np.uint32)
    teacher = ranking_teacher(rng, keep, 30, rest)
    p = params_from_dict({"objective": "distill", "num_leaves": 31, "num_iterations": 3})
    with B200Backend(device) as b:
        b.load(data, "distill", params=p)
        with pytest.raises(SilvicError, match="no teacher"):
            b.train(p, 0.0)
        b.set_teacher(teacher)
        assert init_score(p, data.label) == 0.0
        models = []
        for n in (3, 4):
            if models:
                scores = b.scores()
            p.num_iterations = n
            models.append(b.train(p, 0.0))
        g, h = b.read_gradients()
        check_gradients(data, teacher, scores, g, h)
        after = b.scores()
    short, long = models
    assert len(short.trees) == 3 and len(long.trees) == 4 and all(t.num_leaves > 1 for t in long.trees)
    for a, c in zip(short.trees, long.trees):
        for name in a.FIELDS:
            assert np.array_equal(getattr(a, name), getattr(c, name)), name
    again = train({"objective": "distill", "num_leaves": 31, "num_iterations": 4}, data, device, teacher)
    for a, c in zip(again.trees, long.trees):
        for name in a.FIELDS:
            assert np.array_equal(getattr(a, name), getattr(c, name)), name
    # the trained ranker's answers: its scores are lists again
    with B200Backend(device) as b:
        lists = torch.from_numpy(after).cuda()
        got = b.log_probs(lists, top=5, boundaries=torch.from_numpy(keep.astype(np.int32)).cuda())
        check_log_probs(lists, rows_of(lists, keep), None, 5, 1.0, got)
    text = long.to_lightgbm_string(data, p)
    assert "\nobjective=lambdarank\n" in text and "[objective: custom]" in text and "[sigmoid" not in text


def test_objective_refuses_bad_queries_and_teachers(device):
    data = ranking_binned(1_000, [31] * 3, seed=2)
    bounds = data.query_boundaries.astype(np.int64)
    rng = np.random.RandomState(0)
    with B200Backend(device) as b:
        with pytest.raises(SilvicError, match="before load"):
            b.set_teacher(ranking_teacher(rng, bounds, 4, False))
        b.load(data, "lambdarank")
        with pytest.raises(SilvicError, match="another objective"):
            b.set_teacher(ranking_teacher(rng, bounds, 4, False))
        bad = ranking_binned(1_000, [31] * 3, seed=2)
        bad.query_boundaries = np.array([0, 10, 900], dtype=np.uint32)
        with pytest.raises(SilvicError, match="query boundaries"):
            b.load(bad, "distill")
        bad.query_boundaries = None
        with pytest.raises(SilvicError, match="query information"):
            b.load(bad, "distill")
        b.load(data, "distill")

        def teacher(**change):
            t = ranking_teacher(np.random.RandomState(1), bounds, 4, True)
            for name, (at, value) in change.items():
                getattr(t, name)[at] = value
            return t

        for change, match in [(dict(ids=((0, 0), 100_000)), "names row"), (dict(ids=((2, 1), -5)), "names row"),
                              (dict(logits=((0, 0), np.nan)), "logit"), (dict(logits=((0, 0), np.inf)), "logit"),
                              (dict(log_sum=(1, np.nan)), "log sum")]:
            with pytest.raises(SilvicError, match=match):
                b.set_teacher(teacher(**change))
            with pytest.raises(SilvicError, match="no teacher"):
                b.compute_gradients()
        t = teacher()
        for bad_t, match in [(TeacherTop(t.ids[:-1], t.logits[:-1]), "queries"),
                             (TeacherTop(t.ids, t.logits, None, 0.0), "temperature"),
                             (TeacherTop(np.full((len(bounds) - 1, 129), -1), np.zeros((len(bounds) - 1, 129))), "129")]:
            with pytest.raises(SilvicError, match=match):
                b.set_teacher(bad_t)
        b.set_teacher(t)
        b.compute_gradients()
        b.load(data, "distill")  # a new dataset asks for its teacher again
        with pytest.raises(SilvicError, match="no teacher"):
            b.compute_gradients()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("lists,width", [(3, 5000), (300, 20011)])
def test_log_probs_of_far_scores(backend, type_, lists, width):
    """Scores so far from 0 that m log2(e) / T rounds by whole units, or passes f32; first entries all masked; a list
    that climbs far above its first entries."""
    rng = np.random.RandomState(width)
    z = rng.randn(lists, width) * 3
    z[0] = -1.0e30
    z[0, ::7] *= 1.0 + 2.0 ** -7
    z[1] += 4.0e6
    z[2, : width - 50] = -np.inf
    if lists > 3:
        z[3] += np.linspace(-300, 300, width)
        z[4, : width - 40] = -np.inf
        z[4, width - 40:] = torch.finfo(TYPES[type_]).min
        z[5, : width - 40] = -1.0e5
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    ids = np.stack([np.arange(lists) % width, np.full(lists, width - 1)], 1).astype(np.int32)
    for t in (1.0, 0.01):
        got = backend.log_probs(scores, given=torch.from_numpy(ids).cuda(), top=9, temperature=t)
        check_log_probs(scores[:12], rows_of(scores[:12]), ids, 9, t,
                        type(got)(*[v[:12] for v in (got.given, got.entropy, got.log_sum, got.top_ids, got.top)]))


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("lists,width", [(3, 5000), (300, 20011)])
def test_distill_of_far_scores(backend, lists, width, type_, rest):
    """The lists of test_log_probs_of_far_scores, the loss alone and with its gradients."""
    rng = np.random.RandomState(width)
    z = rng.randn(lists, width) * 3
    z[0] = -1.0e30
    z[0, ::7] *= 1.0 + 2.0 ** -7
    z[1] += 4.0e6
    z[2, : width - 50] = -np.inf
    if lists > 3:
        z[3] += np.linspace(-300, 300, width)
        z[4, : width - 40] = -np.inf
        z[4, width - 40:] = torch.finfo(TYPES[type_]).min
        z[5, : width - 40] = -1.0e5
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    ids = np.stack([width - 1 - rng.choice(40, 6, replace=False) for _ in range(lists)]).astype(np.int32)
    logits = rng.randn(lists, 6) * 2
    logits = torch.from_numpy(logits).float().cuda()
    log_sum = torch.logsumexp(logits.double(), 1).float() + 0.3 if rest else None
    teacher = TeacherTop(torch.from_numpy(ids).cuda(), logits, log_sum)
    some = TeacherTop(teacher.ids[:12], logits[:12], None if log_sum is None else log_sum[:12])
    for gradient in (False, True):
        got = backend.distill(scores, teacher, gradient=gradient)
        check_distill(scores[:12], some, type(got)(got.loss[:12], got.gradient[:12] if gradient else None), type_=type_)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("width,pad", [(700, 0), (9001, 3), (40000, 0), (150001, 0)])
def test_log_probs_of_equal_scores(backend, type_, width, pad):
    """Lists of a few distinct scores, whole lists of one score among them: ties go to the lower index."""
    rng = np.random.RandomState(width)
    scores = dense(rng, 300, width, type_, pad)
    scores[:] = torch.from_numpy(rng.randint(0, 3, (300, width))).to(scores.dtype).cuda()
    scores[0] = 0.5
    scores[1] = -4.0
    scores[1, width - 1] = 1.0
    scores[2, ::2] = -np.inf
    scores[3] = torch.arange(width, device="cuda").float() / width * 3
    ids = torch.zeros(300, 1, dtype=torch.int32, device="cuda")
    for some in (scores, scores[:5]):  # a CTA a list; clusters
        for top in (1, 40, 128):
            got = backend.log_probs(some, given=ids[: len(some)], top=top)
            check_log_probs(some[:5], rows_of(some[:5]), host(ids)[:5].astype(int), top, 1.0,
                            type(got)(*[v[:5] for v in (got.given, got.entropy, got.log_sum, got.top_ids, got.top)]))


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("top", [32, 33, 100, 128])
@pytest.mark.parametrize("width", [20, 100, 130, 300, 512, 631, 1100])
def test_log_probs_of_many_alternatives(backend, type_, top, width):
    """Short lists with more alternatives than a warp has lanes, masked entries and ties among them."""
    rng = np.random.RandomState(width + top)
    scores = dense(rng, 40, width, type_, 1)
    scores[::3, ::4] = -np.inf
    scores[::5] = torch.round(scores[::5])
    got = backend.log_probs(scores, top=top)
    check_log_probs(scores, rows_of(scores), None, top, 1.0, got)


@pytest.mark.parametrize("sizes", [[200, 3, 400, 40], [700, 5000]])
def test_distill_teachers_that_name_an_entry_twice(backend, sizes):
    """Tops of more than 32 entries with repeated indices, in the warp's lists and longer ones."""
    rng = np.random.RandomState(len(sizes))
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    scores = torch.from_numpy(rng.randn(bounds[-1])).float().cuda()
    for rest in (False, True):
        teacher = random_teacher(rng, sizes, 70, "f32", rest)
        ids = teacher.ids.clone()
        ids[:, 65] = ids[:, 1]
        ids[0, 40] = ids[0, 3]
        ids[:, 69] = ids[:, 1]
        teacher = TeacherTop(ids, teacher.logits, teacher.log_sum)
        got = backend.distill(scores, teacher, boundaries=torch.from_numpy(bounds.astype(np.int32)).cuda(), hessian=True)
        check_distill(scores, teacher, got, None, bounds)


@pytest.mark.parametrize("rest", [False, True])
def test_objective_gradients_do_not_depend_on_the_shard(device, rest):
    """Queries of very different lengths: a rank that holds the short ones, or the long ones, has the same bits."""
    rng = np.random.RandomState(12)
    sizes = np.array([40] * 30 + [130, 300, 500, 512, 513, 700, 2_000, 6_000, 1, 3_000, 90])
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    n = int(bounds[-1])
    teacher = ranking_teacher(rng, bounds, 20, rest)

    def gradients(first, last):
        a, b = int(bounds[first]), int(bounds[last])
        data = ranking_binned(b - a, [31] * 2, seed=8, mean_query=40.0)
        data.query_boundaries = (bounds[first:last + 1] - a).astype(np.uint32)
        part = TeacherTop(teacher.ids[first:last], teacher.logits[first:last],
                          None if teacher.log_sum is None else teacher.log_sum[first:last], teacher.temperature)
        with B200Backend(device) as back:
            back.load(data, "distill")
            back.set_teacher(part)
            back.init_scores(0, 0.0)
            back.compute_gradients()
            return back.read_gradients()

    whole = gradients(0, len(sizes))
    for first, last in ((0, 30), (30, len(sizes)), (34, 38)):
        a, b = int(bounds[first]), int(bounds[last])
        part = gradients(first, last)
        for x, y in zip(whole, part):
            assert np.array_equal(x[a:b].view(np.uint32), y.view(np.uint32))
    assert n == len(whole[0])
