"""Measured cases of the label-selection operators: the teacher's record of top labels, the distillation loss against it
with its gradient, and drawing labels from given random numbers.

A row is one distribution over C labels: a pixel of a label map (scores [B, C, H, W]) or a line of a score matrix
([N, C]).  With b = score / temperature:

  top       values and labels of the k largest scores of a row, descending, the lowest label first among equals, and
            rest = log sum exp(b) over all other labels
  distill   p = the teacher's shares over its top labels and (with rest) everything else as one more outcome,
            q = softmax(b) of the student;  loss = T^2 (sum_j p_j log(p_j / q_j) + p_rest log(p_rest / q_rest)),
            and the gradient of sum(weight * loss) with respect to the student's scores
  sample    keep the top_k largest, of those the shortest descending run that holds at least top_p of their mass, of
            those the ones with at least min_p of the largest's share; then the first kept label, in label order, whose
            running sum exceeds u times the kept mass, and the logarithm of its share of that mass
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the record of a segmentation teacher: a training batch of 21-label marginals
        dict(name="top_map_21", op="top", shape="8,21,512,512", dtype="f32", k=4, temperature=2.0),
        # the same for the large label set, where a full record would be 150 values a pixel
        dict(name="top_map_150", op="top", shape="4,150,512,512", dtype="f32", k=8, temperature=1.0),
        # score rows over a large vocabulary, half precision, odd row length (rows start at odd addresses)
        dict(name="top_rows_32k", op="top", shape="1024,32001", dtype="bf16", k=64, temperature=1.0),
        # a handful of rows: launches and latency
        dict(name="distill_rows_few", op="distill", shape="16,32000", dtype="f32", k=16, temperature=1.0, rest=True, void=0.0),
        # training batch of label maps with void pixels
        dict(name="distill_map_21", op="distill", shape="8,21,512,512", dtype="f32", k=4, temperature=2.0, rest=True, void=0.06),
        # large images in half precision, the teacher's top labels renormalised
        dict(name="distill_map_19", op="distill", shape="2,19,1024,2048", dtype="bf16", k=3, temperature=1.5, rest=False, void=0.06),
        # the largest: a training batch of rows over a large vocabulary
        dict(name="distill_rows_128k", op="distill", shape="2048,128000", dtype="bf16", k=64, temperature=1.0, rest=True, void=0.02),
        # drawing label maps from the marginals as they are
        dict(name="sample_map_21", op="sample", shape="8,21,512,512", dtype="f32", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, rowwise=False, masked=False),
        # pseudo-labels from the plausible labels only
        dict(name="sample_map_150", op="sample", shape="2,150,512,512", dtype="f32", temperature=1.0, top_k=5, top_p=0.95,
             min_p=0.02, rowwise=False, masked=False),
        # one row: the smallest call of a serving loop
        dict(name="sample_one", op="sample", shape="1,128000", dtype="bf16", temperature=0.8, top_k=50, top_p=0.95, min_p=0.0,
             rowwise=False, masked=False),
        # a serving batch in which every row has its own settings
        dict(name="sample_rows_mixed", op="sample", shape="256,128000", dtype="f32", temperature=0.9, top_k=0, top_p=0.92,
             min_p=0.0, rowwise=True, masked=False),
        # temperature only, some labels forbidden, odd row length
        dict(name="sample_rows_plain", op="sample", shape="64,50001", dtype="f16", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, rowwise=False, masked=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["top", "distill", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    limit = 1 << 26                                       # scores of a case, well under the largest listed one
    if rng.random() < 0.5:
        c = _log_int(rng, 2, 160)
        h, w = _log_int(rng, 8, 1024), _log_int(rng, 8, 2048)
        b = max(1, min(_log_int(rng, 1, 16), limit // (c * h * w)))
        while b * c * h * w > limit:
            h = max(1, h // 2)
        shape, kmax = (b, c, h, w), 16
    else:
        c = _log_int(rng, 16, 200000)
        n = max(1, min(_log_int(rng, 1, 4096), limit // c))
        shape, kmax = (n, c), 128
    case = dict(op=op, shape=",".join(str(s) for s in shape), dtype=dtype, temperature=rng.choice([0.5, 0.7, 1.0, 1.3, 2.0, 4.0]))
    if op != "sample":
        case["k"] = _log_int(rng, 1, min(kmax, c))
    if op == "distill":
        case.update(rest=rng.random() < 0.6, void=rng.choice([0.0, 0.05, 0.3]))
    if op == "sample":
        kind = rng.choice(["plain", "k", "p", "min_p", "k_p", "all"])
        case.update(top_k=_log_int(rng, 1, min(100, c)) if kind in ("k", "k_p", "all") else 0,
                    top_p=round(rng.uniform(0.3, 0.99), 3) if kind in ("p", "k_p", "all") else 1.0,
                    min_p=round(rng.uniform(0.005, 0.3), 3) if kind in ("min_p", "all") else 0.0,
                    rowwise=rng.random() < 0.3, masked=rng.random() < 0.3)
    return case


def _shape(case):
    return tuple(int(s) for s in case["shape"].split(","))


# ------------------------------------------------------------------ inputs

def _scores(shape, gen, offset=0):
    """Scores as the path meets them: maps are smooth scores around a piecewise constant labelling, rows a common
    long-tailed profile with noise and a few labels that stand out."""
    if len(shape) == 4:
        b, c, h, w = shape
        block = 16
        coarse = torch.randint(0, c, (b, 1, (h + block - 1) // block, (w + block - 1) // block), generator=gen, device="cuda")
        labels = coarse.repeat_interleave(block, 2).repeat_interleave(block, 3)[:, :, :h, :w]
        z = torch.randn(shape, generator=gen, device="cuda")
        return z.scatter_add_(1, labels, 1.5 + 4.0 * torch.rand(labels.shape, generator=gen, device="cuda"))
    n, c = shape
    profile = -1.1 * torch.log1p(torch.randperm(c, generator=gen, device="cuda").float())
    z = profile + 1.5 * torch.randn(shape, generator=gen, device="cuda")
    lead = torch.rand(shape, generator=gen, device="cuda")
    return z + torch.where(lead < 6.0 / c, (9.0 * c / 6.0) * lead, torch.zeros_like(lead))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    shape, dtype = _shape(case), _DTYPES[case["dtype"]]
    n, c = shape[0], shape[1]
    rows = (n,) + shape[2:]
    z = _scores(shape, gen)
    state = dict(case)
    if case["op"] == "top":
        if len(shape) == 4:                               # marginals, as the mean-field loop returns them
            z = z - torch.logsumexp(z, 1, keepdim=True)
        state["scores"] = z.to(dtype)
    elif case["op"] == "distill":
        k = case["k"]
        teacher = z + 0.7 * torch.randn(shape, generator=gen, device="cuda")
        values, labels = torch.topk(teacher, k, 1)
        state["values"], state["labels"] = values.to(dtype).contiguous(), labels.to(torch.int32).contiguous()
        others = teacher.scatter(1, labels, float("-inf")) / case["temperature"]
        # (where the top labels are all there are, the rest is -inf)
        state["rest"] = torch.logsumexp(others, 1) if case["rest"] else None
        state["valid"] = torch.rand(rows, generator=gen, device="cuda") >= case["void"] if case["void"] > 0 else None
        state["weight"] = 0.5 + torch.rand(rows, generator=gen, device="cuda")
        state["scores"] = z.to(dtype).requires_grad_(True)
        del teacher, others
    else:
        if case["masked"]:                                # forbidden labels; label 0 is always allowed
            ban = torch.rand(c, generator=gen, device="cuda") < 0.3
            ban[0] = False
            z.masked_fill_(ban.reshape((1, c) + (1,) * (len(shape) - 2)), float("-inf"))
        state["scores"] = z.to(dtype)
        state["u"] = torch.rand(rows, generator=gen, device="cuda")
        if case["rowwise"]:                               # settings of every request (first dimension) of its own
            def spread(lo, hi):
                return lo + (hi - lo) * torch.rand(n, generator=gen, device="cuda")
            state["temperature"] = case["temperature"] * spread(0.8, 1.25)
            on = torch.rand(n, generator=gen, device="cuda")
            if case["top_k"]:
                state["top_k"] = torch.where(on < 0.5, torch.full_like(on, case["top_k"]), torch.zeros_like(on)).to(torch.int32)
            if case["top_p"] < 1:
                state["top_p"] = case["top_p"] * spread(0.8, 1.0)
            if case["min_p"]:
                state["min_p"] = case["min_p"] * spread(0.0, 1.0)
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    if own:
        return _run_own(state)
    return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[state["op"]](state)


def _run_own(state):
    import semantic_segmentation_amd as S
    if state["op"] == "top":
        values, labels, rest = S.ops.top_labels(state["scores"], state["k"], temperature=state["temperature"])
        return {"values": values, "labels": labels, "rest": rest}
    if state["op"] == "distill":
        loss = S.training.distillation_loss(state["scores"], state["values"], state["labels"], rest=state["rest"],
                                            temperature=state["temperature"], valid=state["valid"])
        grad, = torch.autograd.grad(loss, state["scores"], state["weight"])
        return {"loss": loss.detach(), "grad": grad}
    labels, logprob = S.ops.sample_labels(state["scores"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                          top_p=state["top_p"], min_p=state["min_p"], want_logprob=True)
    return {"labels": labels, "logprob": logprob}


def _plain_top(state):
    z, k, t = state["scores"], state["k"], state["temperature"]
    ordered, index = torch.sort(z.float(), dim=1, descending=True, stable=True)
    others = ordered[:, k:] / t
    if others.shape[1] == 0:
        rest = torch.full_like(ordered[:, 0], float("-inf"))
    else:
        top = others[:, :1]
        shift = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        rest = shift[:, 0] + torch.log(torch.exp(others - shift).sum(1))
    return {"values": ordered[:, :k].to(z.dtype).contiguous(), "labels": index[:, :k].to(torch.int32).contiguous(), "rest": rest}


def _plain_distill(state):
    scores, t = state["scores"].detach(), state["temperature"]
    b = scores.float() / t
    index = state["labels"].long()
    a = state["values"].float() / t
    ainf = torch.full_like(a[:, :1], float("-inf"))
    arest = ainf if state["rest"] is None else state["rest"].float()[:, None]
    everything = torch.cat([a, arest], 1)
    peak = everything.max(1, keepdim=True).values
    e = torch.exp(everything - peak)
    norm = e.sum(1, keepdim=True)
    p = e / norm
    logp = everything - peak - torch.log(norm)
    top = torch.zeros_like(b, dtype=torch.bool).scatter(1, index, True)
    bpeak = b.max(1, keepdim=True).values
    w = torch.exp(b - bpeak)
    sum_all = w.sum(1, keepdim=True)
    tail = torch.where(top, torch.full_like(b, float("-inf")), b)
    tpeak = tail.max(1, keepdim=True).values
    tpeak = torch.where(torch.isinf(tpeak), torch.zeros_like(tpeak), tpeak)
    wtail = torch.exp(tail - tpeak)
    sum_tail = wtail.sum(1, keepdim=True)
    lse = bpeak + torch.log(sum_all)
    logq = torch.cat([torch.gather(b, 1, index) - lse, tpeak + torch.log(sum_tail) - lse], 1)
    terms = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))
    loss = t * t * terms.sum(1)
    grad = w / sum_all
    grad = grad.scatter_add(1, index, -p[:, :-1])
    if state["rest"] is not None:
        grad = grad - torch.where(sum_tail > 0, p[:, -1:] * wtail / sum_tail, torch.zeros_like(wtail))
    weight = state["weight"]
    grad = grad * (t * weight[:, None])
    if state["valid"] is not None:
        loss = torch.where(state["valid"], loss, torch.zeros_like(loss))
        grad = torch.where(state["valid"][:, None], grad, torch.zeros_like(grad))
    return {"loss": loss, "grad": grad.to(scores.dtype)}


def _per_row(value, like):
    """A setting as a tensor that broadcasts over [N, C, ...]."""
    if torch.is_tensor(value):
        return value.double().reshape((-1,) + (1,) * (like.dim() - 1))
    return torch.full((1,) * like.dim(), float(value), dtype=torch.float64, device=like.device)


def _plain_sample(state):
    z = state["scores"].double()                          # 64 bits: the running sum is compared with u
    c = z.shape[1]
    t, p, low = (_per_row(state[key], z) for key in ("temperature", "top_p", "min_p"))
    k = _per_row(state["top_k"], z)
    kept = None
    if torch.is_tensor(state["top_k"]) or state["top_k"] > 0 or \
            torch.is_tensor(state["top_p"]) or state["top_p"] < 1:
        ordered, index = torch.sort(z, dim=1, descending=True, stable=True)
        w = torch.exp((ordered - ordered[:, :1]) / t)
        rank = torch.arange(c, device=z.device).reshape((1, c) + (1,) * (z.dim() - 2))
        keep = (rank < k) | (k <= 0)
        w = torch.where(keep, w, torch.zeros_like(w))
        running = torch.cumsum(w, 1)
        before = torch.cat([torch.zeros_like(running[:, :1]), running[:, :-1]], 1)
        keep = keep & ((before < p * running[:, -1:]) | (p >= 1) | (rank == 0))
        kept = torch.zeros_like(keep).scatter(1, index, keep)
        del ordered, index, running, before, keep
    peak = z.max(1, keepdim=True).values
    w = torch.exp((z - peak) / t)
    allowed = w >= low
    if kept is not None:
        allowed = allowed & kept
    w = torch.where(allowed, w, torch.zeros_like(w))
    running = torch.cumsum(w, 1)
    target = state["u"].double()[:, None] * running[:, -1:]
    labels = (running <= target).sum(1, keepdim=True)
    logprob = torch.log(torch.gather(w, 1, labels) / running[:, -1:])
    return {"labels": labels.squeeze(1), "logprob": logprob.squeeze(1).float()}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "sample": _exact_sample}[case["op"]](state)


def _as_rows(x):
    """[N, C, ...] -> [N * ..., C]"""
    return x.movedim(1, -1).reshape(-1, x.shape[1])


def _as_map(flat, shape):
    """[rows, j] -> [N, j, ...]"""
    return flat.reshape((shape[0],) + tuple(shape[2:]) + (flat.shape[1],)).movedim(-1, 1).contiguous()


def _exact_top(state):
    z = state["scores"].detach()
    k, t = state["k"], state["temperature"]
    rows = _as_rows(z).double()
    left = rows.clone()
    taken = torch.zeros(rows.shape, dtype=torch.bool, device=rows.device)
    line = torch.arange(rows.shape[0], device=rows.device)
    labels, values = [], []
    for _ in range(k):                                    # one label after the other: the first of the largest left
        best = left.max(1, keepdim=True).values
        first = ((left == best) & ~taken).to(torch.uint8).argmax(1)
        labels.append(first)
        values.append(rows[line, first])
        left[line, first] = -math.inf
        taken[line, first] = True
    rest = torch.logsumexp(torch.where(taken, torch.full_like(rows, -math.inf), rows) / t, 1)
    labels, values = torch.stack(labels, 1), torch.stack(values, 1)
    return {"values": _as_map(values, z.shape), "labels": _as_map(labels, z.shape).to(torch.int32),
            "rest": rest.reshape((z.shape[0],) + tuple(z.shape[2:]))}


def _exact_distill(state):
    """Row blocks; the loss through log-softmax terms, the gradient as softmax minus the target written out in full."""
    z, t = state["scores"].detach(), state["temperature"]
    shape = z.shape
    rows, index, values = _as_rows(z), _as_rows(state["labels"]).long(), _as_rows(state["values"])
    n = rows.shape[0]
    rest = None if state["rest"] is None else state["rest"].reshape(-1)
    weight = state["weight"].reshape(-1).double()
    valid = torch.ones(n, dtype=torch.bool, device=z.device) if state["valid"] is None else state["valid"].reshape(-1)
    loss = torch.empty(n, dtype=torch.float64, device=z.device)
    grad = torch.empty(rows.shape, dtype=torch.float64, device=z.device)
    step = max(1, (1 << 26) // rows.shape[1])
    for i in range(0, n, step):
        s = slice(i, min(n, i + step))
        b = rows[s].double() / t
        logq = torch.log_softmax(b, 1)
        target = values[s].double() / t
        if rest is not None:
            target = torch.cat([target, rest[s].double()[:, None]], 1)
        target = torch.log_softmax(target, 1)
        outside = torch.ones(b.shape, dtype=torch.bool, device=z.device)
        outside[torch.arange(b.shape[0], device=z.device)[:, None], index[s]] = False
        want = torch.zeros_like(b)
        want.scatter_add_(1, index[s], torch.exp(target[:, :index.shape[1]]))
        student = torch.gather(logq, 1, index[s])
        if rest is not None:
            hidden = torch.where(outside, logq, torch.full_like(logq, -math.inf))
            tail = torch.logsumexp(hidden, 1, keepdim=True)
            share = torch.exp(hidden - torch.where(torch.isinf(tail), torch.zeros_like(tail), tail))
            want += torch.exp(target[:, -1:]) * share
            student = torch.cat([student, tail], 1)
        ratio = torch.where(torch.isinf(target), torch.zeros_like(target), target - student)
        loss[s] = t * t * (torch.exp(target) * ratio).sum(1) * valid[s]
        grad[s] = t * (weight[s] * valid[s])[:, None] * (torch.exp(logq) - want)
    return {"loss": loss.reshape((shape[0],) + tuple(shape[2:])), "grad": _as_map(grad, shape)}


def _exact_sample(state):
    """Row blocks.  Few labels: a label's rank and the mass in front of it by comparing every pair.  Many: the rows in
    order of (score, label), packed into one sort key."""
    z = state["scores"]
    shape, c, device = z.shape, z.shape[1], z.device
    inner = 1
    for s in shape[2:]:
        inner *= s
    rows, u = _as_rows(z), state["u"].reshape(-1).double()
    n = rows.shape[0]

    def setting(key):
        v = state[key]
        if torch.is_tensor(v):
            return v.double().repeat_interleave(inner)[:, None]
        return torch.full((n, 1), float(v), dtype=torch.float64, device=device)

    temperature, top_k, top_p, min_p = (setting(key) for key in ("temperature", "top_k", "top_p", "min_p"))
    out = torch.empty(n, dtype=torch.int64, device=device)
    logprob = torch.empty(n, dtype=torch.float64, device=device)
    step = max(1, (1 << 25) // c)
    number = torch.arange(c, device=device)
    for i in range(0, n, step):
        s = slice(i, min(n, i + step))
        x = rows[s].double()
        w = torch.exp((x - x.max(1, keepdim=True).values) / temperature[s])
        k = torch.where(top_k[s] > 0, top_k[s], torch.full_like(top_k[s], float(c)))
        if c <= 160:
            rank = torch.zeros_like(x)
            for j in range(c):
                rank += (x[:, j:j + 1] > x) | ((x[:, j:j + 1] == x) & (j < number))
            w = w * (rank < k)
            front = torch.zeros_like(x)
            for j in range(c):
                front += w[:, j:j + 1] * (rank[:, j:j + 1] < rank)
        else:
            # descending by score, then ascending by label: sort the labels by score with equal scores kept in order
            order = torch.argsort(-x, dim=1, stable=True)
            rank = torch.empty_like(order).scatter_(1, order, number.expand_as(order))
            w = w * (rank < k)
            line = torch.gather(w, 1, order)
            front = torch.empty_like(x).scatter_(1, order, torch.cumsum(line, 1) - line)
            # (the sum in front of a label, taken after it was added: the first label's own is exactly zero)
        total = w.sum(1, keepdim=True)
        keep = (rank < k) & (w >= min_p[s]) & ((rank == 0) | (front < top_p[s] * total) | (top_p[s] >= 1))
        w = w * keep
        reach = torch.cumsum(w, 1)
        hit = reach > u[s][:, None] * reach[:, -1:]
        out[s] = torch.where(hit.any(1), hit.to(torch.uint8).argmax(1), (w > 0).long().cumsum(1).argmax(1))
        drawn = torch.gather(x, 1, out[s][:, None]) - x.max(1, keepdim=True).values
        logprob[s] = (drawn / temperature[s] - torch.log(reach[:, -1:]))[:, 0]
    grid = (shape[0],) + tuple(shape[2:])
    return {"labels": out.reshape(grid), "logprob": logprob.reshape(grid)}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    shape, size = _shape(case), _BYTES[case["dtype"]]
    scores = 1
    for s in shape:
        scores *= s
    rows = scores // shape[1]
    if case["op"] == "top":
        # every score read, the record written; a compare and an exponential's share of the sum per score
        return {"bytes": scores * size + rows * (case["k"] * (size + 4) + 4), "flops": 4 * scores}
    if case["op"] == "distill":
        # the scores read, the gradient written, the record read, loss and weight; the softmax of a row has to be known
        # before the first element of its gradient is: two exponentials' worth per score
        record = case["k"] * (size + 4) + (4 if case["rest"] else 0) + (1 if case["void"] > 0 else 0)
        return {"bytes": 2 * scores * size + rows * (record + 8), "flops": 8 * scores}
    return {"bytes": scores * size + rows * (4 + 8 + 4), "flops": 4 * scores}
