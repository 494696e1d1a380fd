"""The softmax operators over lists in 64 bits, list by list from their definitions (numpy), and how far f32 kernels may
be from them.

U = 2^-24 is half a step of f32. A sum of n non-negative terms, cut over 32 threads or more and joined by a tree, is
off by (n / 32 + 16) U of itself at most. A term exp((z - m) / T) is off by the function's 4 U and by its argument's
rounding (3 roundings of (z - m) log2(e) / T): 3 U |z - m| / T, whose mean under the softmax is 3 U ln n at most, since
the mean of (m - z) / T is the entropy less ln S <= ln n. So the sum S, and ln S, is off by

    slack(n) = (n / 32 + 24 + 3 ln n) U.
"""

from __future__ import annotations

import math

import numpy as np

U = 2.0 ** -24


def slack(n: int) -> float:
    return (n / 32 + 24 + 3 * math.log(max(n, 2))) * U


def softmax(z: np.ndarray, t: float):
    """(p, log p, ln sum exp(z / t)) of one list; an empty list has ln sum -inf."""
    x = z.astype(np.float64) / t
    if np.isnan(x).any() or (x == np.inf).any():
        nan = np.full_like(x, np.nan)
        return nan, nan, math.nan
    m = x.max() if len(x) else -np.inf
    if m == -np.inf:
        return np.zeros_like(x), np.full_like(x, -np.inf), -math.inf
    log_s = math.log(np.exp(x - m).sum())  # apart from m, which can be too large to hold it (the type's lowest value)
    return np.exp(x - m - log_s), x - m - log_s, m + log_s


def log_probs(z: np.ndarray, t: float, given, top: int) -> dict:
    p, lp, total = softmax(z, t)
    ent = 0.0 if total == -math.inf else math.nan if total != total else -float((p[p > 0] * lp[p > 0]).sum())
    order = np.argsort(-z.astype(np.float64), kind="stable")[:top]
    ids = np.full(top, -1, np.int64)
    out = np.full(top, -np.inf)
    ids[: len(order)], out[: len(order)] = order, lp[order]
    ids[out == -np.inf] = -1
    got = np.array([lp[g] if 0 <= g < len(z) else -np.inf for g in given], dtype=np.float64)
    return dict(given=got, entropy=ent, log_sum=total, top_ids=ids, top=out)


def teach(n: int, ids, logits, t: float, log_sum=None):
    """(q per entry of the list, whether it is in the top, the teacher's mass there, whether it has any entry)."""
    q, inside = np.zeros(n), np.zeros(n, bool)
    keep = [(int(i), float(v) / t) for i, v in zip(ids, logits) if 0 <= int(i) < n]
    y = np.array([v for _, v in keep], dtype=np.float64)
    if not keep:
        return q, inside, 0.0, False
    base = log_sum if log_sum is not None else (
        -math.inf if y.max() == -np.inf else y.max() + math.log(np.exp(y - y.max()).sum()))
    for (i, _), v in zip(keep, y):
        inside[i] = True
        q[i] += math.exp(v - base) if v > -math.inf else 0.0
    return q, inside, q.sum(), True


def distill(z: np.ndarray, ids, logits, t: float, log_sum=None, w: float = 1.0) -> dict:
    """The loss counts an entry that the teacher names twice with each of its logits."""
    n = len(z)
    p, lp, total = softmax(z, t)
    q, inside, held, any_entry = teach(n, ids, logits, t, log_sum)
    zero = np.zeros(n)
    if total == -math.inf or not any_entry:
        return dict(loss=0.0, grad=zero, hess=zero, scale=zero, terms=0.0)
    if total != total:
        nan = np.full(n, np.nan)
        return dict(loss=math.nan, grad=nan, hess=nan, scale=zero, terms=0.0)
    rest_p = float(p[~inside].sum())
    rest_q = max(0.0, 1.0 - held) if log_sum is not None and rest_p > 0 else 0.0
    keep = [(int(i), float(v) / t) for i, v in zip(ids, logits) if 0 <= int(i) < n and float(v) > -math.inf]
    base = log_sum if log_sum is not None else (math.log(sum(math.exp(v - max(u for _, u in keep)) for _, v in keep))
                                               + max(u for _, u in keep) if keep else 0.0)
    loss = terms = 0.0
    for i, v in keep:
        part = math.exp(v - base)
        if part > 0:
            loss += part * (v - base - lp[i])
            terms += part * (1 + abs(v - base) + abs(lp[i]) + abs(v) + abs(base))
    if rest_q > 0:
        loss += rest_q * math.log(rest_q / rest_p)
        terms += (1 + abs(math.log(rest_q / rest_p))) * (1 + held) + abs(math.log(rest_p))
    mass = held + rest_q
    pull = rest_q / rest_p if rest_q > 0 else 0.0
    grad = w / t * (mass * p - q - np.where(inside, 0.0, pull * p))
    hess = w / t ** 2 * mass * p * (1 - p)
    return dict(loss=w * loss, grad=grad, hess=hess, scale=w / t * (mass * p + q + pull * p), terms=w * terms)


def check_log_probs(z, t, given, top, got: dict):
    """`got` (one list's outputs) against the definition. A log probability (z - m) / T - ln S is off by slack(n), by
    3 U of |z - m| / T and by U of itself; the log sum m / T + ln S by slack(n) and 3 U of |m| / T + ln S; the entropy
    ln S - U1 / (T S), U1 / (T S) <= ln n, by slack(n) (1 + 2 ln n) and a step of either."""
    want = log_probs(z, t, given, top)
    n = len(z)
    s = slack(n)

    def near(a, b, tol):
        a, b = np.atleast_1d(np.asarray(a, np.float64)), np.atleast_1d(np.asarray(b, np.float64))
        fine = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~fine & ~np.isnan(b)], b[~fine & ~np.isnan(b)]), (a, b)
        assert (np.abs(a[fine] - b[fine]) <= np.broadcast_to(tol, b.shape)[fine]).all(), (a, b, tol)

    def of(v):
        v = np.abs(np.where(np.isfinite(v), v, 0.0))
        return s + 4 * U * (v + math.log(max(n, 2))) + 2 * U

    if abs(want["log_sum"]) > np.finfo(np.float32).max * (1 + U):  # past f32, whose rounding of it is infinite
        want["log_sum"] = math.copysign(math.inf, want["log_sum"])
    near(got["log_sum"], want["log_sum"], of(np.float64(want["log_sum"])) + 4 * U * (np.abs(z[np.isfinite(z)]).max(initial=0) / t))
    near(got["entropy"], want["entropy"], s * (1 + 2 * math.log(max(n, 2))) + 4 * U * math.log(max(n, 2)))
    if got.get("given") is not None:
        near(got["given"], want["given"], of(want["given"]))
    if got.get("top") is not None and not np.isnan(z).any():
        assert np.array_equal(got["top_ids"], want["top_ids"]), (got["top_ids"], want["top_ids"])
        near(got["top"], want["top"], of(want["top"]))


def check_distill(z, ids, logits, t, log_sum, w, got: dict, step: float, least: float = 0.0):
    """`step`: half a step of the gradient's type, relative (`least`: half its smallest). p = e / S is off by 2 slack(n)
    and 3 U |z - m| / T of itself, q alike over the top's k entries (and by U of its argument, |t| / T + |log sum|), the
    rest 1 - sum q by k steps of U: each term of the gradient by `relative` of itself. The loss's terms q (ln q - ln p)
    by `relative` of the sum of their absolute parts."""
    want = distill(z, ids, logits, t, log_sum, w)
    n, k = len(z), len(ids)
    if got.get("loss") is not None and np.isnan(want["loss"]):
        assert np.isnan(got["loss"])
        return
    fine = z[np.isfinite(z)].astype(np.float64)
    x = np.where(np.isfinite(z), (fine.max(initial=-1e30) - z.astype(np.float64)) / t, 0.0) if len(fine) else np.zeros(n)
    live = [abs(float(v)) / t for i, v in zip(ids, logits) if 0 <= int(i) < n and np.isfinite(v)]
    arg = max(live, default=0.0) + abs(log_sum or 0.0)
    relative = 4 * slack(n) + (k + 32 + 4 * arg) * U
    if got.get("loss") is not None:
        if np.isinf(want["loss"]):
            assert got["loss"] == want["loss"], (got["loss"], want["loss"])
        else:
            assert abs(got["loss"] - want["loss"]) <= relative * 2 * want["terms"] + 1e-37, (got["loss"], want["loss"])
    # the rest r = 1 - sum q loses relative precision where it is small; P, the mass outside the top, does not
    held = teach(n, ids, logits, t, log_sum)[2]
    rest_slack = 0.0
    if log_sum is not None and 1 - held > 0:
        rest_slack = (k + 32 + 4 * arg) * U * max(1.0, held)
    if got.get("grad") is not None:
        outside = ~teach(n, ids, logits, t, log_sum)[1]
        p = softmax(z, t)[0]
        rest_p = p[outside].sum()
        # a term exp((z - m) / T) below 2^-126 is 0: p is off by 2^-126 (S >= 1), its multiples by as much of theirs
        tiny = 2.0 ** -125 * abs(w) / t * (1 + held + (1 / rest_p if rest_p > 0 else 0.0))
        tol = want["scale"] * (relative + 4 * U * x) + step * np.abs(want["grad"]) * 1.001 + least + tiny
        if rest_p > 0:
            tol = tol + np.where(outside, abs(w) / t * p / rest_p * rest_slack, 0.0) + abs(w) / t * p * rest_slack
        bad = ~(np.abs(got["grad"] - want["grad"]) <= tol)
        assert not bad.any(), (np.nonzero(bad)[0][:5], got["grad"][bad][:5], want["grad"][bad][:5], tol[bad][:5])
    if got.get("hess") is not None:
        p = softmax(z, t)[0]
        # 1 - p is off by p (2 slack + 3 U x) + U, whatever it is itself
        tol = (want["hess"] + abs(w) / t ** 2 * p * p) * (relative + 4 * U * x) + abs(w) / t ** 2 * p * (rest_slack + 4 * U)
        tol = tol + step * np.abs(want["hess"]) * 1.001 + least + 2.0 ** -125 * abs(w) / t ** 2 * (1 + held)
        bad = ~(np.abs(got["hess"] - want["hess"]) <= tol)
        assert not bad.any(), (np.nonzero(bad)[0][:5], got["hess"][bad][:5], want["hess"][bad][:5], tol[bad][:5])
