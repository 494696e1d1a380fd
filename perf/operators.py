"""Cases of the softmax operators over lists of candidates: `log_probs` (log probabilities of given entries, entropy,
top alternatives) and `distill` (distillation from a teacher's top logits, forward and backward).

A list is a row of a dense matrix (a position's logits over a vocabulary) or a run of a flat array between two
boundaries (a query's documents), as a query of a ranking dataset is.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One generated token's logits over a large vocabulary, with the alternatives an API returns.
        dict(name="logprob_token", op="log_probs", lists=1, width=131072, pad=0, type="bf16", given=1, top=20,
             temperature=1.0, masked=0.0),
        # A decoding batch over an odd vocabulary in f32: rows that start on no vector boundary.
        dict(name="logprob_batch_odd", op="log_probs", lists=64, width=50257, pad=0, type="f32", given=1, top=5,
             temperature=0.7, masked=0.0),
        # A teacher asked for a grade per prompt: log probabilities of the five grades' tokens, a few alternatives.
        dict(name="logprob_grades", op="log_probs", lists=2048, width=32000, pad=0, type="bf16", given=5, top=8,
             temperature=1.0, masked=0.0),
        # Half of a large vocabulary masked (constrained answers), padded rows, the longest usual list of alternatives.
        dict(name="logprob_masked", op="log_probs", lists=512, width=65537, pad=7, type="f16", given=2, top=64,
             temperature=1.0, masked=0.5),
        # Whole prompts scored at once, the top alternatives kept as a teacher.
        dict(name="logprob_prompts", op="log_probs", lists=4096, width=131072, pad=0, type="bf16", given=1, top=20,
             temperature=1.0, masked=0.0),
        # The ranking configuration's queries (2M documents, Poisson(120) a query): a trained ranker's answers.
        dict(name="logprob_queries", op="log_probs", lists=16700, mean=120, longest=1000, type="f32", given=1, top=10,
             temperature=1.0, masked=0.0),
        # A small ranking set, a boosting iteration's gradients and hessians: the call's latency counts.
        dict(name="distill_queries_few", op="distill", lists=400, mean=5, longest=1000, type="f32", top=3, tail=False,
             temperature=1.0, weight=False, grad=True, hess=True),
        # The ranking configuration's queries: one boosting iteration of a ranker that learns a teacher's top 30.
        dict(name="distill_queries", op="distill", lists=16700, mean=120, longest=1000, type="f32", top=30, tail=False,
             temperature=1.0, weight=False, grad=True, hess=True),
        # Long candidate lists of uneven lengths, a teacher's log probabilities with the mass of the rest.
        dict(name="distill_candidates", op="distill", lists=700, mean=4000, longest=16000, type="f32", top=50, tail=True,
             temperature=1.0, weight=True, grad=True, hess=True),
        # A student's training step over a vocabulary, the teacher's rest kept as one more class.
        dict(name="distill_step", op="distill", lists=4096, width=32000, pad=0, type="bf16", top=64, tail=True,
             temperature=1.0, weight=False, grad=True, hess=False),
        # The same over a large vocabulary, softened, over the teacher's top alone: the largest.
        dict(name="distill_wide", op="distill", lists=2048, width=131072, pad=0, type="bf16", top=100, tail=False,
             temperature=2.0, weight=True, grad=True, hess=False),
        # The loss alone (evaluation) over an odd f16 vocabulary with padded rows.
        dict(name="distill_loss", op="distill", lists=1500, width=50257, pad=3, type="f16", top=20, tail=True,
             temperature=1.5, weight=False, grad=False, hess=False),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["log_probs", "distill"])
    c = dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), temperature=rng.choice([1.0, 1.0, 0.7, 2.0]))
    most = (1 << 28) if c["type"] == "f32" else (1 << 29)  # entries that no draw exceeds
    if op == "distill":
        most //= 2
    if rng.random() < 0.35:
        c["mean"] = _log_uniform(rng, 2, 4000)
        c["longest"] = rng.choice([4, 8]) * c["mean"]
        c["lists"] = _log_uniform(rng, 1, max(1, min(40000, most // 32 // c["mean"])))
        c["type"] = "f32"
    else:
        c["width"] = _log_uniform(rng, 100, 140000)
        c["pad"] = rng.choice([0, 0, 0, rng.randint(1, 9), 64])
        c["lists"] = _log_uniform(rng, 1, max(1, min(8192, most // (c["width"] + c["pad"]))))
    if op == "log_probs":
        c.update(given=rng.choice([1, 1, 2, 5, 8]), top=rng.choice([0, 1, 5, 8, 20, 64, 128]),
                 masked=rng.choice([0.0, 0.0, 0.5, 0.9]))
    else:
        c.update(top=_log_uniform(rng, 1, 128), tail=rng.random() < 0.5, weight=rng.random() < 0.5,
                 grad=rng.random() < 0.8)
        c["hess"] = c["grad"] and "mean" in c
    return c


def _sizes(case, seed):
    """The lists' lengths, Poisson for short lists (queries), log-normal for long ones, one at least; the seed orders
    them, so every seed has the same number of entries."""
    r = np.random.RandomState(case["lists"] + case["mean"])
    if case["mean"] <= 500:
        n = r.poisson(case["mean"], case["lists"])
    else:
        n = np.exp(r.normal(math.log(case["mean"]) - 0.32, 0.8, case["lists"])).astype(np.int64)
    return np.random.RandomState(seed % (1 << 31)).permutation(np.clip(n, 1, case["longest"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev, dtype, lists = "cuda", TYPES[case["type"]], case["lists"]
    s = dict(case=case, temperature=case["temperature"], boundaries=None)
    if "mean" in case:
        sizes = _sizes(case, seed)
        ends = np.cumsum(sizes)
        total = int(ends[-1])
        s["boundaries"] = torch.from_numpy(np.concatenate([[0], ends]).astype(np.uint32)).to(dev)
        s["sizes"] = torch.from_numpy(sizes).to(dev)
        # A ranker's scores: sums of a few trees' leaves, so documents tie.
        z = torch.round(torch.randn(total, generator=gen, device=dev) * 48.0) / 32.0
        s["scores"] = z.to(dtype)
        length = s["sizes"][:, None]
    else:
        whole = torch.randn(lists, case["width"] + case["pad"], generator=gen, device=dev).mul_(2.5)
        length = torch.full((lists, 1), case["width"], device=dev)
        s["whole"] = whole
    if case["op"] == "log_probs":
        near = torch.rand(lists, case["given"], generator=gen, device=dev)
        ids = (near * length).long().clamp(max=length - 1)
    else:
        # The teacher's top: distinct entries of each list, -1 behind the last of a short list.
        k = case["top"]
        first = (torch.rand(lists, 1, generator=gen, device=dev) * length).long().clamp(max=length - 1)
        j = torch.arange(k, device=dev)[None, :]
        step = (length // k).clamp(min=1)
        ids = torch.where(j < length, (first + j * step) % length, -1)
    if "mean" not in case:
        # A few likely entries in each list, among them the given ones and the teacher's.
        lift = torch.rand(ids.shape, generator=gen, device=dev) * 9.0
        whole.scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, lift, 0.0))
        if case.get("masked"):
            hidden = torch.rand(whole.shape, generator=gen, device=dev) < case["masked"]
            hidden.scatter_(1, ids[:, :1], False)
            whole.masked_fill_(hidden, float("-inf"))
        s["scores"] = s.pop("whole").to(dtype)[:, : case["width"]]
    s["ids"] = ids.to(torch.int32)
    if case["op"] == "distill":
        t = torch.randn(lists, case["top"], generator=gen, device=dev) * 2.0 + 3.0
        t = torch.sort(t, dim=1, descending=True).values
        s["logits"] = t.to(dtype)
        s["log_sum"] = None
        if case["tail"]:
            # The teacher's log sum over its whole list: its top holds 60 to 95 percent of the mass.
            held = torch.rand(lists, generator=gen, device=dev) * 0.35 + 0.6
            x = torch.where(ids >= 0, s["logits"].float() / case["temperature"], float("-inf"))
            s["log_sum"] = torch.logsumexp(x, 1) - torch.log(held)
        s["weight"] = torch.rand(lists, generator=gen, device=dev) + 0.5 if case["weight"] else None
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _stats(x, s):
    """(max, sum of exp(x - max), entry -> list) of x's lists; dense: kept dims."""
    if s["boundaries"] is None:
        m = x.amax(1, keepdim=True)
        return m, torch.exp(x - m).sum(1, keepdim=True), None
    lists = s["sizes"].numel()
    of = torch.repeat_interleave(torch.arange(lists, device=x.device), s["sizes"], output_size=x.numel())
    m = torch.segment_reduce(x, "max", lengths=s["sizes"])
    total = torch.segment_reduce(torch.exp(x - m[of]), "sum", lengths=s["sizes"])
    return m, total, of


def _starts(s):
    return s["boundaries"][:-1].long()[:, None]


def _plain_log_probs(s):
    c, z = s["case"], s["scores"].float()
    x = z / s["temperature"]
    m, total, of = _stats(x, s)
    ids, k = s["ids"].long(), c["top"]
    if of is None:
        log_sum = m + torch.log(total)
        d = x - m
        e = torch.exp(d)
        entropy = (torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total)[:, 0]
        given = torch.gather(x, 1, ids) - log_sum
        # Order by value, ties by the lower index: the value's bits in ascending order above the index's complement.
        bits = (z + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        kk = min(k, z.shape[1])
        key = (order << 32) | (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
        top_ids = 0xFFFFFFFF - (torch.topk(key, kk, dim=1).values & 0xFFFFFFFF)
        top = torch.gather(x, 1, top_ids) - log_sum
        top_ids = torch.where(top == float("-inf"), -1, top_ids)
        if kk < k:
            top_ids = torch.nn.functional.pad(top_ids, (0, k - kk), value=-1)
            top = torch.nn.functional.pad(top, (0, k - kk), value=float("-inf"))
        log_sum = log_sum[:, 0]
    else:
        log_sum = m + torch.log(total)
        d = x - m[of]
        e = torch.exp(d)
        part = torch.segment_reduce(torch.where(e > 0, e * d, 0.0), "sum", lengths=s["sizes"])
        entropy = torch.log(total) - part / total
        given = x[_starts(s) + ids] - log_sum[:, None]
        by_value = torch.sort(z, descending=True, stable=True).indices
        order = by_value[torch.sort(of[by_value], stable=True).indices]
        j = torch.arange(k, device=z.device)[None, :]
        at = order[(_starts(s) + j).clamp(max=z.numel() - 1)]
        there = j < s["sizes"][:, None]
        top = torch.where(there, x[at] - log_sum[:, None], float("-inf"))
        top_ids = torch.where(there, at - _starts(s), -1)
    return dict(given=given, entropy=entropy, log_sum=log_sum, top_ids=top_ids.int(), top=top)


def _plain_distill(s):
    c, t = s["case"], s["temperature"]
    x = s["scores"].float() / t
    m, total, of = _stats(x, s)
    ids = s["ids"].long()
    there = ids >= 0
    y = torch.where(there, s["logits"].float() / t, float("-inf"))
    if s["log_sum"] is None:
        e = torch.exp(y - y.amax(1, keepdim=True))
        q = e / e.sum(1, keepdim=True)
    else:
        q = torch.exp(y - s["log_sum"][:, None])
    at = ids.clamp(min=0) if of is None else _starts(s) + ids.clamp(min=0)
    if of is None:
        p = torch.exp(x - m) / total
        log_p = torch.gather(x, 1, at) - m - torch.log(total)
        taught = torch.zeros_like(x).scatter_add_(1, at, q)
    else:
        p = torch.exp(x - m[of]) / total[of]
        log_p = x[at] - (m + torch.log(total))[:, None]
        taught = torch.zeros_like(x).index_put_((at.reshape(-1),), q.reshape(-1), accumulate=True)
    log_q = torch.log(q)
    loss = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    held = q.sum(1)
    if s["log_sum"] is not None:
        top = torch.zeros(x.shape, dtype=torch.int32, device=x.device)
        if of is None:
            top = top.scatter_add_(1, at, there.int()) > 0
            rest = torch.where(top, 0.0, p).sum(1)
        else:
            top = top.index_put_((at.reshape(-1),), there.int().reshape(-1), accumulate=True) > 0
            rest = torch.segment_reduce(torch.where(top, 0.0, p), "sum", lengths=s["sizes"])
        r = torch.where(rest > 0, (1.0 - held).clamp(min=0.0), 0.0)
        loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(rest)), 0.0)
        held = held + r
        pull = torch.where(r > 0, r / rest, 0.0)
    w = s["weight"] if s["weight"] is not None else torch.ones_like(loss)
    out = dict(loss=loss * w)
    spread = (lambda v: v[:, None]) if of is None else (lambda v: v[of])
    if c["grad"]:
        g = spread(held) * p - taught
        if s["log_sum"] is not None:
            g = g - torch.where(top, 0.0, spread(pull) * p)
        out["grad"] = (g * spread(w / t)).to(s["scores"].dtype)
    if c["hess"]:
        out["hess"] = (spread(held * w / (t * t)) * p * (1.0 - p)).to(s["scores"].dtype)
    return out


# ---- the framework's calls ----------------------------------------------------------------------------------------

_handles = {}


def _backend():
    """The process's handle on the current device, as a program keeps it."""
    from silvic_b200 import B200Backend

    device = torch.cuda.current_device()
    if device not in _handles:
        _handles[device] = B200Backend(device)
    return _handles[device]


def run(state):
    c = state["case"]
    if not own:
        return _plain_log_probs(state) if c["op"] == "log_probs" else _plain_distill(state)
    if c["op"] == "log_probs":
        r = _backend().log_probs(state["scores"], given=state["ids"], top=c["top"], temperature=state["temperature"],
                                 boundaries=state["boundaries"])
        if not c["top"]:  # no alternatives: the call gives None, the plain form tensors without columns
            none = state["ids"].new_empty((c["lists"], 0))
            return dict(given=r.given, entropy=r.entropy, log_sum=r.log_sum, top_ids=none, top=none.float())
        return dict(given=r.given, entropy=r.entropy, log_sum=r.log_sum, top_ids=r.top_ids, top=r.top)
    from silvic_b200 import TeacherTop

    teacher = TeacherTop(state["ids"], state["logits"], state["log_sum"], state["temperature"])
    r = _backend().distill(state["scores"], teacher, boundaries=state["boundaries"], weight=state["weight"],
                           gradient=c["grad"], hessian=c["hess"])
    out = dict(loss=r.loss)
    if c["grad"]:
        out["grad"] = r.gradient
    if c["hess"]:
        out["hess"] = r.hessian
    return out


# ---- what a pass cannot do without, and its value in 64 bits --------------------------------------------------------


def work(case):
    size = 4 if case["type"] == "f32" else 2
    entries = case["lists"] * (case["width"] if "width" in case else case["mean"])
    per_list = 4 if "mean" in case else 0
    if case["op"] == "log_probs":
        per_list += case["given"] * 8 + 8 + case["top"] * 8
        return {"bytes": entries * size + case["lists"] * per_list, "flops": entries * 6}
    per_list += case["top"] * (4 + size) + 4 + (4 if case["tail"] else 0) + (4 if case["weight"] else 0)
    written = (1 if case["grad"] else 0) + (1 if case["hess"] else 0)
    return {"bytes": entries * size * (1 + written) + case["lists"] * per_list, "flops": entries * (4 + 3 * written)}


def _matrix(s, low, high):
    """Lists low .. high as a matrix in 64 bits, -inf behind the end of a short one."""
    z = s["scores"]
    if s["boundaries"] is None:
        return z[low:high].double()
    b = s["boundaries"].long().tolist()
    rows = [z[b[i]:b[i + 1]].double() for i in range(low, high)]
    return torch.nn.utils.rnn.pad_sequence(rows, batch_first=True, padding_value=float("-inf"))


def exact(case, seed):
    s = prepare(case, seed)
    t, lists, k = case["temperature"], case["lists"], case["top"]
    widest = case.get("width") or int(s["sizes"].max())
    chunk = max(1, (1 << 26) // widest)
    got = []
    for low in range(0, lists, chunk):
        high = min(lists, low + chunk)
        z = _matrix(s, low, high)
        lp = torch.log_softmax(z / t, 1)
        ids = s["ids"][low:high].long()
        if case["op"] == "log_probs":
            p = lp.exp()
            entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
            n = min(k, z.shape[1])
            order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :n]
            top = torch.gather(lp, 1, order)
            order = torch.where(top == float("-inf"), -1, order)
            top = torch.nn.functional.pad(top, (0, k - n), value=float("-inf"))
            order = torch.nn.functional.pad(order, (0, k - n), value=-1)
            got.append(dict(given=torch.gather(lp, 1, ids), entropy=entropy, log_sum=torch.logsumexp(z / t, 1),
                            top_ids=order.int(), top=top))
            continue
        p = lp.exp()
        there = ids >= 0
        y = torch.where(there, s["logits"][low:high].double() / t, float("-inf"))
        base = torch.logsumexp(y, 1) if s["log_sum"] is None else s["log_sum"][low:high].double()
        q = (y - base[:, None]).exp()
        # The teacher as a distribution over the whole list; the rest, where it counts, as one more class.
        full = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), q)
        in_top = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), there.double()) > 0
        rest_p = torch.where(in_top, 0.0, p).sum(1)
        rest_q = torch.zeros_like(rest_p)
        if s["log_sum"] is not None:
            rest_q = torch.where(rest_p > 0, (1.0 - q.sum(1)).clamp(min=0.0), 0.0)
        loss = torch.where(full > 0, full * (full.log() - lp), 0.0).sum(1)
        loss = loss + torch.where(rest_q > 0, rest_q * (rest_q / rest_p).log(), 0.0)
        w = torch.ones_like(loss) if s["weight"] is None else s["weight"][low:high].double()
        mass = (full.sum(1) + rest_q)[:, None]
        g = mass * p - full - torch.where(in_top, 0.0, p) * torch.where(rest_q > 0, rest_q / rest_p, 0.0)[:, None]
        row = dict(loss=loss * w)
        if case["grad"]:
            row["grad"] = g * (w / t)[:, None]
        if case["hess"]:
            row["hess"] = mass * p * (1.0 - p) * (w / t ** 2)[:, None]
        if s["boundaries"] is not None:
            inside = torch.arange(z.shape[1], device=z.device)[None, :] < s["sizes"][low:high, None]
            row = {name: v if v.dim() == 1 else v[inside] for name, v in row.items()}
        got.append(row)
    return {name: torch.cat([g[name] for g in got]) for name in got[0]}
