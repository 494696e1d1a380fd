"""The softmax operators over lists where their kernels pass from one way of working to another, and where inputs come
near what f32 holds; against the definitions in 64 bits (lists_reference.py)."""

from __future__ import annotations

import ctypes as C

import lists_reference as ref
import numpy as np
import pytest
import torch
from synth import ranking_binned
from test_gpu_lists import TYPES, backend, check_distill, check_log_probs, dense, random_teacher, rows_of  # noqa: F401

from silvic_b200 import B200Backend, SilvicError, TeacherTop, _abi, params_from_dict

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


# ---- the rest of a confident student -------------------------------------------------------------------------------


def check_rest(z, ids, logits, t, log_sum, w, loss, grad, hess, type_):
    """A list whose mass P outside the top is small, against the definition. p is off by 4 slack(n) and 4 U x of itself
    (x its distance from the maximum over T: four roundings of the exponent), p / P alike about the maximum outside the
    top, the teacher's sums by (k + 32 + 4 arg) U, and r = 1 - sum q by as much of 1. An exponential below 2^-126 of its
    maximum's is 0. Then half a step of the type."""
    with np.errstate(over="ignore"):  # r / P times p, at the top's own
        want = ref.distill(z, ids, logits, t, log_sum, w)
    q, inside, held, _ = ref.teach(len(z), ids, logits, t, log_sum)
    p, lp, _ = ref.softmax(z, t)
    rest_p = p[~inside].sum()
    live = [abs(float(v)) / t for i, v in zip(ids, logits) if 0 <= int(i) < len(z)]
    own = (len(ids) + 32 + 4 * (max(live, default=0.0) + abs(log_sum))) * ref.U
    relative = 4 * ref.slack(len(z)) + own
    assert np.isfinite(loss) and abs(loss - want["loss"]) <= 2 * relative * want["terms"] + 1e-37, (loss, want["loss"])
    step, least = {"f32": (2.0 ** -24, 2.0 ** -150), "bf16": (2.0 ** -8, 2.0 ** -134), "f16": (2.0 ** -11, 2.0 ** -25)}[type_]
    fine = np.isfinite(z)
    x = np.where(fine, -np.where(fine, lp, 0.0), 0.0)
    mass, scale, tiny = held, w / t, 2.0 ** -125 * w / t * (1 + held)
    of_rest, x_rest = np.zeros(len(z)), np.zeros(len(z))
    if rest_p > 0 and held < 1:
        mass = 1.0
        of_rest = np.where(inside, 0.0, p / rest_p)
        x_rest = np.where(fine & ~inside, (z[~inside].max() - np.where(fine, z, 0.0)) / t, 0.0)
    if grad is not None:
        tol = scale * (mass * p * (relative + 4 * ref.U * x) + q * relative + of_rest * (own + relative + 4 * ref.U * x_rest))
        tol = tol + step * 1.001 * np.abs(want["grad"]) + least + tiny
        bad = ~(np.abs(grad - want["grad"]) <= tol)
        assert not bad.any(), (np.nonzero(bad)[0][:5], grad[bad][:5], want["grad"][bad][:5], tol[bad][:5])
    if hess is not None:
        tol = scale / t * p * ((relative + 4 * ref.U * x) * (1 + p) + 4 * ref.U) * max(mass, 1.0)
        tol = tol + step * 1.001 * np.abs(want["hess"]) + least + tiny / t
        bad = ~(np.abs(hess - want["hess"]) <= tol)
        assert not bad.any(), (np.nonzero(bad)[0][:5], hess[bad][:5], want["hess"][bad][:5], tol[bad][:5])


GAPS = [80.0, 86.0, 90.0, 300.0, 700.0, 20.0, 30.0, 60.0]


def confident(rng, n, t, i, top, type_):
    """Scores of n entries and the top's ids: the others lie GAPS nats below the top, some of them masked; of every
    eleventh list all of them, of the next all by the type's lowest value (no mass in 64 bits either)."""
    ids = rng.choice(n, min(top, n), replace=False)
    z = rng.randn(n) * 2 * t
    z[ids] += (GAPS[i % len(GAPS)] + 8.0) * t
    outside = np.setdiff1d(np.arange(n), ids)
    if len(outside) > 1:
        z[outside[1:][rng.rand(len(outside) - 1) < 0.3]] = -np.inf
    if i % 11 == 9:
        z[outside] = -np.inf
    if i % 11 == 10:
        z[outside] = torch.finfo(TYPES[type_]).min
    return z, ids


@pytest.mark.parametrize("weight", [1.0, 65536.0])
@pytest.mark.parametrize("t", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("type_,sizes", [
    ("f32", [300] * 12), ("bf16", [513] * 11), ("f16", [1000] * 12), ("f32", [5000] * 5), ("bf16", [5001] * 300),
    ("bf16", [40001] * 3), ("f32", [20011] * 300), ("f16", [70001] * 160), ("f32", [300007] * 2), ("f32", [500003] * 2),
    ("f32", [5, 300, 700, 5000, 0, 130, 90000, 2000]), ("f32", [7, 40, 3, 600] * 6), ("f16", [900, 3000, 200])])
def test_the_rest_of_a_confident_student(backend, type_, sizes, t, weight):  # noqa: F811
    rng = np.random.RandomState(len(sizes) + sizes[0])
    if type_ == "f16":
        weight = min(weight, 4.0)  # gradients of weight / T
    few = min(len(sizes), 12)
    uneven = len(set(sizes)) > 1
    top = 6
    made = [confident(rng, n, t, i, top, type_) if n else (np.zeros(0), np.zeros(0, int)) for i, n in enumerate(sizes[:few])]
    ids = np.full((len(sizes), top), -1, np.int32)
    for i in range(len(sizes)):
        some = made[i % few][1]
        ids[i, : len(some)] = some
    rows = [torch.from_numpy(made[i % few][0]).to(TYPES[type_]) for i in range(len(sizes))]
    boundaries = None
    if uneven:
        scores = torch.cat(rows).cuda()
        bounds = np.concatenate([[0], np.cumsum(sizes)])
        boundaries = torch.from_numpy(bounds.astype(np.int32)).cuda()
    else:
        scores = torch.stack(rows).cuda()
    logits = torch.from_numpy(rng.randn(len(sizes), top) * 2 * t).float()
    x = torch.where(torch.from_numpy(ids) >= 0, logits.double() / t, -np.inf)
    log_sum = torch.logsumexp(x, 1) + 0.3
    log_sum = torch.where(torch.isfinite(log_sum), log_sum, 0.0).float()
    teacher = TeacherTop(torch.from_numpy(ids).cuda(), logits.cuda(), log_sum.cuda(), t)
    w = torch.full((len(sizes),), weight, device="cuda")
    both = backend.distill(scores, teacher, boundaries=boundaries, weight=w, hessian=True)
    alone = backend.distill(scores, teacher, boundaries=boundaries, weight=w, gradient=False)
    grad_only = backend.distill(scores, teacher, boundaries=boundaries, weight=w)
    for got in (both, alone, grad_only):
        parts = [None if v is None else v.double().cpu().numpy() for v in (got.loss, got.gradient, got.hessian)]
        for i in range(few):
            z = rows[i].double().numpy()
            at = slice(bounds[i], bounds[i + 1]) if uneven else i
            check_rest(z, ids[i], logits[i].numpy(), t, float(log_sum[i]), weight, parts[0][i],
                       None if parts[1] is None else parts[1][at], None if parts[2] is None else parts[2][at], type_)


def test_the_rest_of_a_confident_student_in_training(device):
    """Scores 90 and 0 by a tree, the teacher's top the high rows: the gradients of the low ones, and their maximum."""
    data = ranking_binned(2_000, [31] * 3, seed=4, mean_query=40.0)
    bounds = data.query_boundaries.astype(np.int64)
    rng = np.random.RandomState(1)
    node = _abi.DeviceNode()
    node.split.left_bins[0] = 0x3FF  # of group 0's column 0
    node.left, node.right = ~0, ~1
    with B200Backend(device) as b:
        b.load(data, "distill")
        b.add_tree([node], [0.0, 90.0])
        scores = b.scores()
        assert set(np.unique(scores)) == {0.0, 90.0}
        ids = np.full((len(bounds) - 1, 100), -1, np.int32)
        for i, (a, e) in enumerate(zip(bounds[:-1], bounds[1:])):
            high = np.nonzero(scores[a:e] == 90.0)[0]
            ids[i, : len(high)] = high
        logits = rng.randn(*ids.shape).astype(np.float32)
        total = np.log(np.where(ids >= 0, np.exp(logits.astype(np.float64)), 0.0).sum(1) + 1e-300)
        log_sum = np.where(total > -100, total + 0.4, 0.0).astype(np.float32)
        b.set_teacher(TeacherTop(ids, logits, log_sum))
        most_g, most_h = b.compute_gradients()
        g, h = b.read_gradients()
    assert most_g == np.abs(g).max() and most_h == np.abs(h).max() and np.isfinite([most_g, most_h]).all()
    for i, (a, e) in enumerate(zip(bounds[:-1], bounds[1:])):
        if (ids[i] >= 0).any():
            loss = ref.distill(scores[a:e].astype(np.float64), ids[i], logits[i], 1.0, float(log_sum[i]))["loss"]
            check_rest(scores[a:e].astype(np.float64), ids[i], logits[i], 1.0, float(log_sum[i]), 1.0, loss, g[a:e], h[a:e], "f32")


# ---- the hessian's sign --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("lists,width,uneven", [(400, 600, True), (400, 900, False), (300, 1500, True), (300, 5000, False),
                                                (3, 40001, False)])
def test_the_hessian_is_never_negative(backend, lists, width, uneven, rest):  # noqa: F811
    """One entry with nearly all of the mass, whose p rounds to 1 or past it."""
    rng = np.random.RandomState(width)
    z = rng.randn(lists, width) * 3 + rng.randn(lists, 1) * 40
    ids = rng.randint(0, width, (lists, 3)).astype(np.int32)
    z[np.arange(lists), ids[:, 0]] += 20 + rng.rand(lists) * 60
    scores = torch.from_numpy(z).float().cuda()
    boundaries = None
    if uneven:
        scores = scores.flatten()
        boundaries = torch.arange(0, lists * width + 1, width, dtype=torch.int32, device="cuda")
    log_sum = torch.full((lists,), 3.0, device="cuda") if rest else None
    for t in (1.0, 0.3):
        teacher = TeacherTop(torch.from_numpy(ids).cuda(), torch.from_numpy(rng.randn(lists, 3)).float().cuda(), log_sum, t)
        got = backend.distill(scores, teacher, boundaries=boundaries, hessian=True)
        assert (got.hessian >= 0).all() and (got.hessian > 0).any()


# ---- a teacher without mass on masked entries ----------------------------------------------------------------------


@pytest.mark.parametrize("rest,logit", [(False, -np.inf), (True, -np.inf), (True, -400.0)])
@pytest.mark.parametrize("lists,width", [(3, 40001), (300, 40001), (300, 5000), (4, 700)])
def test_a_teacher_without_mass_on_masked_entries(backend, lists, width, rest, logit):  # noqa: F811
    """The first nine tenths of each list are masked, the whole top among them, and the teacher gives that nothing: the
    loss is the rest's alone (0 without one)."""
    rng = np.random.RandomState(width)
    z = rng.randn(lists, width) * 2
    z[:, : width * 9 // 10] = -np.inf
    scores = torch.from_numpy(z).float().cuda()
    ids = torch.from_numpy(rng.randint(0, width * 9 // 10, (lists, 4)).astype(np.int32)).cuda()
    log_sum = torch.full((lists,), 2.0, device="cuda") if rest else None
    teacher = TeacherTop(ids, torch.full((lists, 4), logit, device="cuda"), log_sum, 0.5)
    for gradient in (False, True):
        got = backend.distill(scores, teacher, gradient=gradient, hessian=gradient)
        assert torch.isfinite(got.loss).all()
        cut = type(got)(got.loss[:4], got.gradient[:4] if gradient else None, got.hessian[:4] if gradient else None)
        check_distill(scores[:4], TeacherTop(ids[:4], teacher.logits[:4], None if log_sum is None else log_sum[:4], 0.5), cut)


# ---- a handle whose second load fails ------------------------------------------------------------------------------


def test_a_failed_load_leaves_no_dataset_behind(device):
    """The second dataset's queries are taken before its features are refused: nothing works on a mixture of the two."""
    data = ranking_binned(3_000, [31] * 3, seed=2, mean_query=10.0)
    queries = len(data.query_boundaries) - 1
    teacher = TeacherTop(np.zeros((queries, 1), np.int32), np.zeros((queries, 1), np.float32))
    p = params_from_dict({"objective": "distill", "num_leaves": 4, "num_iterations": 1})
    for objective in ("lambdarank", "distill"):
        bad = ranking_binned(500, [31] * 3, seed=3, mean_query=40.0)
        bad.features[1].upper_bounds = bad.features[1].upper_bounds[:2]
        with B200Backend(device) as b:
            b.load(data, "distill", params=p)
            b.set_teacher(teacher)
            b.compute_gradients()
            want = b.read_gradients()
            with pytest.raises(SilvicError, match="upper bounds"):
                b.load(bad, objective)
            for call in (lambda: b.set_teacher(teacher), b.compute_gradients, lambda: b.train(p, 0.0), b.scores):
                with pytest.raises(SilvicError, match="before load"):
                    call()
            b.load(data, "distill", params=p)
            b.set_teacher(teacher)
            b.compute_gradients()
            for x, y in zip(want, b.read_gradients()):
                assert np.array_equal(x, y)


def test_the_most_lists_of_a_call(backend):  # noqa: F811
    """2^32 - 1 lists without entries and without outputs: nothing is written, and nothing is refused."""
    lists = _abi.Lists(None, _abi.F32, 2 ** 32 - 1, 0, 0, None)
    backend._check(backend._lib.sb2_log_probs(backend._h, C.byref(lists), 1.0, None, 0, 0, None, None, None, None, None, None))
    torch.cuda.synchronize()


def test_misaligned_pointers_are_refused(backend):  # noqa: F811
    """Every pointer of 4-byte entries, 2 bytes off; the calls are refused before a launch."""
    x = torch.zeros(4096, device="cuda")
    ok, off = x.data_ptr(), x.data_ptr() + 4096 + 2
    lists = _abi.Lists(ok, _abi.F32, 2, 8, 8, None)
    runs = _abi.Lists(ok, _abi.F32, 2, 8, 0, off)
    lib, h = backend._lib, backend._h

    def log_probs(a=lists, **at):
        p = dict(given=ok + 1000, given_out=ok + 2000, entropy=ok + 3000, log_sum=ok + 4000, ids=ok + 5000, out=ok + 6000)
        p.update(at)
        return lib.sb2_log_probs(h, C.byref(a), 1.0, p["given"], 1, 2, p["given_out"], p["entropy"], p["log_sum"], p["ids"], p["out"],
                                 None)

    def distill(a=lists, **at):
        p = dict(ids=ok + 1000, log_sum=ok + 2000, weight=ok + 3000, loss=ok + 4000)
        p.update(at)
        t = _abi.Teacher(p["ids"], ok + 512, _abi.F32, 2, 2, p["log_sum"])
        return lib.sb2_distill(h, C.byref(a), C.byref(t), 1.0, p["weight"], p["loss"], None, None, 0, None)

    for call, names in ((log_probs, ("given", "given_out", "entropy", "log_sum", "ids", "out")),
                        (distill, ("ids", "log_sum", "weight", "loss"))):
        assert call(runs) == _abi.EDATA
        for name in names:
            assert call(**{name: off}) == _abi.EDATA, name
            with pytest.raises(SilvicError, match="aligned"):
                backend._check(call(**{name: off}))
        assert call() == _abi.OK
    torch.cuda.synchronize()


# ---- entries of no list --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("bounds,total", [([3, 40, 60], 200), ([0, 700, 700, 1200], 1201), ([5], 9), ([2000, 9000], 300_000),
                                          ([0, 5000, 9001], 9001), ([7, 7, 7], 11), ([0, 90_000], 90_000),
                                          ([1, 60_000, 130_001], 130_005)])
def test_entries_of_no_list_have_gradient_0(backend, bounds, total, type_):  # noqa: F811
    """The tensors' memory held other values before: what is before the first list and behind the last is 0."""
    rng = np.random.RandomState(total)
    scores = torch.from_numpy(rng.randn(total)).to(TYPES[type_]).cuda()
    sizes = np.diff(bounds)
    teacher = random_teacher(rng, sizes, 4)
    for _ in range(3):
        junk = [torch.full((total,), float("nan"), dtype=TYPES[type_], device="cuda") for _ in range(4)]
        del junk
        got = backend.distill(scores, teacher, boundaries=torch.tensor(bounds, dtype=torch.int32, device="cuda"), hessian=True)
        for v in (got.gradient, got.hessian):
            assert v.shape == (total,)
            assert (v[: bounds[0]] == 0).all() and (v[bounds[-1]:] == 0).all()
        if len(sizes):
            check_distill(scores, teacher, got, None, bounds, type_)


# ---- outputs -------------------------------------------------------------------------------------------------------


def test_outputs_are_tensors_of_their_own(backend):  # noqa: F811
    """What is done to one in place leaves the others, and what autograd saved of them, alone."""
    x = torch.randn(5, 900, device="cuda")
    got = backend.log_probs(x, given=torch.zeros(5, 2, dtype=torch.int32, device="cuda"), top=3)
    parts = [got.given, got.entropy, got.log_sum, got.top_ids, got.top]
    assert len({v.untyped_storage().data_ptr() for v in parts}) == 5
    assert [v.untyped_storage().nbytes() for v in parts] == [40, 20, 20, 60, 60] and all(v.is_contiguous() for v in parts)
    w = torch.ones(5, 2, device="cuda", requires_grad=True)
    loss = (w * got.given).sum()
    got.entropy.mul_(2.0)
    got.top.add_(1.0)
    loss.backward()
    assert torch.equal(w.grad, got.given)
    none = backend.log_probs(x, given=torch.zeros(5, 0, dtype=torch.int32, device="cuda"))
    assert none.given.shape == (5, 0) and none.top is None and none.top_ids is None


# ---- given entries -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("given", [3, 700])
@pytest.mark.parametrize("lists,width", [(6, 300), (6, 1000), (300, 5001), (6, 70001)])
def test_given_entries_of_every_kind(backend, lists, width, given):  # noqa: F811
    """More given entries than a CTA has threads; masked ones and indices outside the list, in lists with a NaN or +inf
    (all of their log probabilities are NaN), in empty ones and in others."""
    rng = np.random.RandomState(width + given)
    z = rng.randn(lists, width) * 3
    z[:, : width // 3] = -np.inf
    z[0, -1] = np.nan
    z[1, width // 2] = np.inf
    z[2] = -np.inf
    scores = torch.from_numpy(z).float().cuda()
    ids = rng.randint(0, width, (lists, given)).astype(np.int32)
    ids[:, 0], ids[:, 1], ids[:, 2] = 0, -1, width  # masked; outside
    got = backend.log_probs(scores, given=torch.from_numpy(ids).cuda(), top=4)
    check_log_probs(scores[:6], rows_of(scores[:6]), ids, 4, 1.0,
                    type(got)(*[v[:6] for v in (got.given, got.entropy, got.log_sum, got.top_ids, got.top)]))
    assert torch.isnan(got.given[:2, 0]).all() and (got.given[:, 1:3] == -np.inf).all() and (got.given[2] == -np.inf).all()


# ---- a teacher's logits far from 0 ---------------------------------------------------------------------------------


@pytest.mark.parametrize("sizes", [[300] * 9, [1000] * 9, [5000] * 9, [40001] * 2, [9001] * 300, [5, 700, 90, 5000]])
def test_a_constant_on_a_teacher_s_logits_changes_nothing(backend, sizes):  # noqa: F811
    """Without a log sum: logits that are multiples of 1/8 about 0 and about 2^20 have the same differences in f32."""
    rng = np.random.RandomState(sizes[0])
    uneven = len(set(sizes)) > 1
    teacher = random_teacher(rng, sizes, 40, t=1.7)
    logits = torch.round(teacher.logits * 8) / 8
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    if uneven:
        scores, boundaries = torch.from_numpy(rng.randn(bounds[-1])).float().cuda(), torch.from_numpy(bounds.astype(np.int32)).cuda()
    else:
        scores, boundaries = torch.from_numpy(rng.randn(len(sizes), sizes[0])).float().cuda(), None
    for gradient in (False, True):
        near, far = [backend.distill(scores, TeacherTop(teacher.ids, logits + c, None, 1.7), boundaries=boundaries, gradient=gradient)
                     for c in (0.0, 2.0 ** 20)]
        assert torch.equal(near.loss, far.loss) and (not gradient or torch.equal(near.gradient, far.gradient))
    if not uneven:
        near = type(near)(near.loss[:9], near.gradient[:9])
        check_distill(scores[:9], TeacherTop(teacher.ids[:9], logits[:9], None, 1.7), near)


# ---- every entry once ----------------------------------------------------------------------------------------------


def borders(n, per, rng, count):
    """Entries at which a list is cut between CTAs, threads and batches of their loads (`per` entries a 16-byte vector, the
    first of them at any of the list's first entries), and those beside them; `count` of them."""
    at = {0, 1, n - 1, n - 2, n // 2}
    for head in range(per):
        vectors = max(0, (n - head) // per)
        at.add(head)
        at.add(head + vectors * per)
        for shares in (2, 4, 8):
            at.update(head + vectors * k // shares * per for k in range(1, shares))
        for threads in (128, 256, 512):
            at.update(range(head, n, threads * per))
            at.update(range(head, n, threads * per * 4))
    at = sorted({k for a in at for k in (a - 1, a, a + 1) if 0 <= k < n})
    return rng.choice(at, min(count, len(at)), replace=False)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("type_,lists,width,pad", [
    ("f32", 8, 600, 1), ("bf16", 8, 1001, 0), ("f32", 40, 3001, 3), ("bf16", 170, 5000, 1), ("f16", 160, 9003, 5),
    ("bf16", 40, 33000, 0), ("f32", 6, 40001, 2), ("bf16", 160, 40003, 1), ("f32", 170, 19000, 1), ("bf16", 4, 150_000, 3),
    ("f32", 2, 300_007, 1), ("bf16", 160, 140_001, 0)])
def test_every_entry_counts_once(backend, type_, lists, width, pad, rest):  # noqa: F811
    """All of a list's mass on 24 entries at the cuts between CTAs, threads and batches: one that is left out, or counted
    twice, changes the sums by a twenty-fourth. Runs of the same lengths too."""
    rng = np.random.RandomState(width + rest)
    per = 4 if type_ == "f32" else 8
    z = np.full((lists, width), -60.0)
    top = np.zeros((lists, 6), np.int32)
    for i in range(lists):
        at = borders(width, per, rng, 24)
        z[i, at] = rng.randint(-4, 5, len(at)) / 4
        top[i] = rng.choice(at, 6, replace=False)  # named by the teacher; with the rest, left out of the sum outside
    flat = torch.zeros(lists * (width + pad) + 1, dtype=TYPES[type_], device="cuda")
    scores = flat[1:].view(lists, width + pad)[:, :width]
    scores.copy_(torch.from_numpy(z))
    given = torch.from_numpy(top).cuda()
    logits = torch.from_numpy(rng.randn(lists, 6)).float().cuda()
    log_sum = torch.logsumexp(logits.double(), 1).float() + 0.5 if rest else None
    teacher = TeacherTop(given, logits, log_sum)
    boundaries = torch.from_numpy((np.arange(lists + 1) * width).astype(np.int32)).cuda()
    for s, b in ((scores, None), (scores.contiguous().flatten(), boundaries)):
        few = slice(0, 6)
        lp = backend.log_probs(s, given=given, top=8, boundaries=b)
        check_log_probs(scores[few], rows_of(scores[few]), top[few], 8, 1.0,
                        type(lp)(*[v[few] for v in (lp.given, lp.entropy, lp.log_sum, lp.top_ids, lp.top)]))
        some = TeacherTop(given[few], logits[few], None if log_sum is None else log_sum[few])
        for gradient in (False, True):
            got = backend.distill(s, teacher, boundaries=b, gradient=gradient, hessian=gradient)
            parts = [None if v is None else v.view(lists, -1)[few] for v in (got.gradient, got.hessian)]
            check_distill(scores[few], some, type(got)(got.loss[few], *parts), None, None, type_)


# ---- runs of 16-bit scores, and the longest lists ------------------------------------------------------------------


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("type_", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", [[0, 1, 0, 3, 0], [5] * 40, [1, 32, 33, 512, 513, 1024, 1025, 0, 7, 2000, 65, 4097, 1],
                                   [20000, 3, 9000, 1, 1], [700] * 200, [6001] * 160])
def test_runs_of_16_bit_scores(backend, sizes, type_, rest):  # noqa: F811
    rng = np.random.RandomState(len(sizes) + rest)
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    scores = torch.from_numpy(rng.randn(bounds[-1]) * 3).to(TYPES[type_]).cuda()
    boundaries = torch.from_numpy(bounds.astype(np.int32)).cuda()
    teacher = random_teacher(rng, sizes, 40, type_, rest, 0.9)
    few = 14
    ids = np.stack([[max(n - 1, 0), n] for n in sizes]).astype(np.int32)
    lp = backend.log_probs(scores, given=torch.from_numpy(ids).cuda(), top=40, temperature=0.9, boundaries=boundaries)
    check_log_probs(scores, rows_of(scores, bounds[: few + 1]), ids, 40, 0.9, lp)
    got = backend.distill(scores, teacher, boundaries=boundaries, hessian=True)
    some = TeacherTop(teacher.ids[:few], teacher.logits[:few], None if teacher.log_sum is None else teacher.log_sum[:few], 0.9)
    check_distill(scores, some, got, None, bounds[: few + 1], type_)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("type_,lists,width,uneven", [
    ("f32", 3, 500_003, False), ("bf16", 2, 1_000_001, False), ("f32", 150, 80_001, True), ("f32", 2, 700_000, True),
    ("f32", 150, 80_001, False)])
def test_the_longest_lists(backend, type_, lists, width, uneven, rest):  # noqa: F811
    """Lists that shared memory does not hold, shares of more than 65,536 entries, and a teacher whose indices lie 65,536
    and its multiples apart; the rest beside them counts."""
    rng = np.random.RandomState(width + rest)
    scores = torch.from_numpy((rng.randn(lists, width) * 2).astype(np.float32)).to(TYPES[type_]).cuda()
    base = np.array([5, 65_536 + 5, 17, 65_536 + 6, 2 * 65_536 + 5, 65_536 + 17, 70_000, 4_464])
    ids = np.stack([np.where(base + i < width, base + i, i) for i in range(lists)]).astype(np.int32)
    ids[1, 3] = ids[1, 0]
    logits = torch.from_numpy(rng.randn(lists, 8)).float().cuda()
    log_sum = torch.logsumexp(logits.double(), 1).float() + 0.6 if rest else None
    teacher = TeacherTop(torch.from_numpy(ids).cuda(), logits, log_sum)
    boundaries = torch.from_numpy((np.arange(lists + 1) * width).astype(np.int32)).cuda() if uneven else None
    s = scores.flatten() if uneven else scores
    few = slice(0, 2)
    some = TeacherTop(teacher.ids[few], logits[few], None if log_sum is None else log_sum[few])
    for gradient in (False, True):
        got = backend.distill(s, teacher, boundaries=boundaries, gradient=gradient, hessian=gradient)
        parts = [None if v is None else v.view(lists, -1)[few] for v in (got.gradient, got.hessian)]
        check_distill(scores[few], some, type(got)(got.loss[few], *parts), None, None, type_)


# ---- graphs over every way of working ------------------------------------------------------------------------------


@pytest.mark.parametrize("type_,lists,width,uneven", [
    ("f32", 40, 300, False), ("bf16", 40, 900, False), ("f32", 300, 20_011, False), ("bf16", 3, 150_001, False),
    ("bf16", 160, 33_000, False), ("f32", 2, 500_003, False), ("f32", 40, 200, True), ("f32", 30, 5_000, True),
    ("bf16", 2, 60_000, True)])
def test_graphs_replay_every_way_of_working(backend, type_, lists, width, uneven):  # noqa: F811
    """A graph captured on ordinary scores is replayed on a confident student's, on masked lists and on far scores, beside
    eager calls on the same inputs."""
    rng = np.random.RandomState(width)
    x = torch.randn(lists, width, device="cuda").to(TYPES[type_])
    teacher = random_teacher(rng, [width] * lists, 20, "f32", True)
    given = teacher.ids[:, :3].contiguous()
    boundaries = (torch.arange(lists + 1, device="cuda") * width).int() if uneven else None
    s = x.flatten() if uneven else x
    assert s.data_ptr() == x.data_ptr()

    def calls():
        lp = backend.log_probs(s, given=given, top=30, boundaries=boundaries)
        return [lp.given, lp.entropy, lp.log_sum, lp.top_ids, lp.top,
                *[v for gradient in (False, True)
                  for d in [backend.distill(s, teacher, boundaries=boundaries, gradient=gradient, hessian=gradient)]
                  for v in (d.loss, d.gradient, d.hessian) if v is not None]]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for turn in range(4):
        x.copy_(torch.randn(lists, width, device="cuda"))
        if turn == 1:
            x.scatter_(1, teacher.ids.long(), 200.0)
        if turn == 2:
            x[:, : width // 2] = -np.inf
            x[0] = -np.inf
        if turn == 3:
            x.mul_(3.0e6)
        graph.replay()
        for got, want in zip(out, calls()):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


# ---- a teacher's entries that the student masks by the type's lowest value -------------------------------------------


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("t", [1.0, 0.3, 0.05])
@pytest.mark.parametrize("type_,lists,width,uneven", [
    ("f32", 9, 40, False), ("bf16", 9, 900, False), ("f32", 300, 5_001, False), ("bf16", 3, 40_001, False),
    ("f32", 9, 300, True), ("bf16", 160, 1_501, True)])
def test_the_loss_of_entries_masked_by_the_lowest_value(backend, type_, lists, width, uneven, t, rest):  # noqa: F811
    """Losses of up to f32's largest, from terms beyond it; past it, infinite."""
    rng = np.random.RandomState(width)
    z = rng.randn(lists, width) * 3
    z[rng.rand(lists, width) < 0.5] = torch.finfo(TYPES[type_]).min
    z[:, :3] = 2.0
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    ids = np.stack([rng.choice(width, 5, replace=False) for _ in range(lists)]).astype(np.int32)
    logits = rng.randn(lists, 5) * t
    for i in range(lists):  # masked ones with 2^-1 to 2^-40 of the teacher's mass, the first with most of it
        z[i, ids[i, 0]] = 1.0
        masked = [k for k in range(1, 5) if z[i, ids[i, k]] < -1e30]
        logits[i, masked] -= rng.choice([0.5, 5.0, 28.0]) * t
    scores = torch.from_numpy(z).to(TYPES[type_]).cuda()
    logits = torch.from_numpy(logits).float()
    log_sum = torch.logsumexp(logits.double() / t, 1).float() + 0.4 if rest else None
    teacher = TeacherTop(torch.from_numpy(ids).cuda(), logits.cuda(), None if log_sum is None else log_sum.cuda(), t)
    boundaries = (torch.arange(lists + 1, device="cuda") * width).int() if uneven else None
    finite = 0
    for weight, gradient in ((1.0, False), (1.0, True), (0.125, False), (0.125, True)):
        got = backend.distill(scores.flatten() if uneven else scores, teacher, boundaries=boundaries, gradient=gradient,
                              weight=torch.full((lists,), weight, device="cuda"))
        for i in range(9 if lists > 9 else lists):
            want = ref.distill(rows_of(scores[i: i + 1])[0], ids[i], logits[i].numpy(), t,
                               None if log_sum is None else float(log_sum[i]), weight)
            loss = float(got.loss[i])
            if want["loss"] > 3.5e38:
                assert loss == np.inf
            elif want["loss"] < 3.3e38:
                # q is off by 4 U and by its argument's rounding, a term by three roundings more, a sum of five by three
                arg = np.abs(logits[i].numpy()).max() / t + (0.0 if log_sum is None else abs(float(log_sum[i])))
                tol = 2 * (16 + 4 * arg) * ref.U * want["terms"] + 4 * ref.slack(width) * want["terms"]
                assert abs(loss - want["loss"]) <= tol, (loss, want["loss"])
                finite += want["loss"] > 1e20
    assert finite > 0 or lists < 9


@pytest.mark.parametrize("weight", [2.0 ** -110, 2.0 ** -60, 2.0 ** 60, 2.0 ** 110])
@pytest.mark.parametrize("lists,width,uneven", [(9, 300, False), (5, 5_000, False), (300, 5_001, False), (9, 300, True)])
def test_a_weight_scales_the_loss_exactly(backend, lists, width, uneven, weight):  # noqa: F811
    """A power of two, however small or large."""
    rng = np.random.RandomState(width)
    scores = torch.from_numpy(rng.randn(lists, width) * 2).float().cuda()
    teacher = random_teacher(rng, [width] * lists, 7, "f32", True)
    boundaries = (torch.arange(lists + 1, device="cuda") * width).int() if uneven else None
    s = scores.flatten() if uneven else scores
    for gradient in (False, True):
        one, many = [backend.distill(s, teacher, boundaries=boundaries, gradient=gradient,
                                     weight=torch.full((lists,), w, device="cuda")) for w in (1.0, weight)]
        assert (one.loss.abs() > 1e-3).all() and torch.equal(many.loss, one.loss * weight)
