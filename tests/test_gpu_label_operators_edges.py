"""GPU tests of the label-selection operators where fp32 runs out: rows that are not numbers, gaps near the ends of the
fp32 exponent, masses far below the largest, bins of the cut that overflow their list, calls of very many rows.  The plain
64-bit restatements, the tolerances and their derivation are those of test_gpu_label_operators.py."""
import numpy as np
import pytest
import torch

import label_reference as R
import test_gpu_label_operators as G

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def S():
    import semantic_segmentation_amd as S
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return S


def lay(x, planes):
    """[rows, C] as a matrix, or as class planes of two images"""
    return x if not planes else x.reshape(2, x.shape[0] // 2, x.shape[1]).movedim(2, 1).contiguous()


def lay_rows(x, planes):
    return x if not planes else x.reshape(2, -1)


# ------------------------------------------------------------------ distillation

GAPS = [80.0, 86.9, 87.2, 87.4, 88.0, 88.4, 88.6, 88.75, 89.0, 95.0, 104.0]


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("C", [12, 24, 60, 900])
def test_distillation_of_gaps_near_the_end_of_the_exponent(C, planes, S):
    """Record and rest exp(gap) apart, on the student's side, on the teacher's, and on both: ratios around 2^126 and 2^128."""
    k = 3
    pairs = [(s, t) for s in [0.5, -1.0] + GAPS + [-g for g in GAPS] for t in [0.7] + GAPS + [-g for g in GAPS]]
    pairs += pairs[:len(pairs) % 2]                        # (an even number of rows)
    x = G.scores_of((len(pairs), C), torch.float32, 201, 0.5)
    labels = torch.rand(x.shape, generator=G.gen(202), device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    own = torch.gather(x, 1, labels.long())
    others = torch.logsumexp(x.scatter(1, labels.long(), -INF), 1, keepdim=True)
    student = torch.tensor([s for s, _ in pairs], device="cuda").unsqueeze(1)
    x.scatter_(1, labels.long(), own - torch.logsumexp(own, 1, keepdim=True) + others + student)
    values = G.scores_of((len(pairs), k), torch.float32, 203, 0.5)
    rest = torch.logsumexp(values, 1) - torch.tensor([t for _, t in pairs], device="cuda")
    G.check_distill(S, lay(x, planes), lay(values, planes), lay(labels, planes), lay_rows(rest, planes), 1.0)


@pytest.mark.parametrize("dtype", G.DTYPES)
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("C", [3, 21, 60, 900])
def test_distillation_of_rows_that_are_no_numbers(C, planes, dtype, S):
    """A NaN among a valid row's scores makes its loss and its whole gradient NaN, whatever else stands there: a student that
    has diverged must not look like one that has nothing to learn."""
    x = G.scores_of((8, C), torch.float32, 211)
    values = G.scores_of((8, 2), torch.float32, 212).to(dtype)
    labels = torch.tensor([[0, 2]] * 8, dtype=torch.int32, device="cuda")
    rest = torch.zeros(8, device="cuda")
    x[0] = NAN
    x[1] = -INF
    x[1, 1] = NAN                                          # outside the record
    x[2] = -INF
    x[2, 2] = NAN                                          # in it
    x[3, 1:] = NAN
    x[4, 0] = NAN
    x[5] = -INF                                            # nothing, but nothing wrong: 0
    x = x.to(dtype)
    for r in (rest, None):
        G.check_distill(S, lay(x, planes), lay(values, planes), lay(labels, planes), None if r is None else lay_rows(r, planes), 1.5)
        loss, _ = S.ops.distillation_forward(lay(x, planes), lay(values, planes), lay(labels, planes), None if r is None else lay_rows(r, planes), 1.5)
        assert torch.isnan(loss.reshape(-1)).tolist() == [True] * 5 + [False] * 3 and float(loss.reshape(-1)[5]) == 0


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("C", [3, 21, 60, 900])
def test_distillation_of_records_that_are_no_numbers(C, planes, S):
    """A NaN among the teacher's values, or a rest that is one, reaches every label whose gradient it enters: the record's
    labels, and with rest all others."""
    x = G.scores_of((6, C), torch.float32, 221)
    values = G.scores_of((6, 3), torch.float32, 222)
    labels = torch.tensor([[0, 2, 1]] * 6, dtype=torch.int32, device="cuda")
    rest = torch.zeros(6, device="cuda")
    values[0, 1] = NAN
    values[1] = NAN
    values[2], values[2, 0] = -INF, NAN
    values[3, 2], labels[3, 2] = NAN, -1                   # of no class: passed over
    labels[4, 1], values[4, 1] = 0, NAN                    # a label named twice
    for r in (rest, torch.full_like(rest, -INF), None):
        G.check_distill(S, lay(x, planes), lay(values, planes), lay(labels, planes), None if r is None else lay_rows(r, planes), 1.5)
    values = G.scores_of((6, 3), torch.float32, 223)
    rest[1::2] = NAN
    G.check_distill(S, lay(x, planes), lay(values, planes), lay(labels, planes), lay_rows(rest, planes), 1.5)


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("C", [3, 24, 60, 900])
def test_distillation_of_the_lowest_scores_at_low_temperatures(C, planes, S):
    """A student's mask of the type's lowest number, on labels that the teacher wants a little, in the record or outside it: a
    huge loss, but a number, where the score over T is none."""
    low = torch.finfo(torch.float32).min
    x = G.scores_of((6, C), torch.float32, 301)
    values = torch.tensor([[9.0, 4.0], [9.0, -2.0], [0.0, 0.0]] * 2, device="cuda")
    labels = torch.tensor([[0, 1]] * 6, dtype=torch.int32, device="cuda")
    rest = torch.tensor([-20.0, -1.0, 0.0] * 2, device="cuda")
    x[:3, 1] = low
    x[3:, 2:] = low
    for t in (0.5, 0.1):
        for r in (rest, None):
            G.check_distill(S, lay(x, planes), lay(values, planes), lay(labels, planes), None if r is None else lay_rows(r, planes), t)
            loss, _ = S.ops.distillation_forward(lay(x, planes), lay(values, planes), lay(labels, planes), None if r is None else lay_rows(r, planes), t)
            assert torch.isfinite(loss).all() and float(loss.max()) > 1e30


@pytest.mark.parametrize("C", [21, 600])
def test_distillation_of_forbidden_labels_that_the_teacher_hardly_wants(C, S):
    """A share below 2^-126 is 0 next to a student's -inf, a larger one makes the loss infinite; the gradients are finite."""
    x = torch.zeros(2, C, device="cuda")
    x[:, 1] = -INF
    values = torch.tensor([[0.0, -100.0], [0.0, -70.0]], device="cuda")
    labels = torch.tensor([[0, 1]] * 2, dtype=torch.int32, device="cuda")
    loss, stats = S.ops.distillation_forward(x, values, labels)
    assert abs(float(loss[0]) - np.log(C - 1.0)) <= (G.CHAIN(C) * 2.0 ** -23 + 2.0 ** -21) * (1 + 2 * np.log(C)) and float(loss[1]) == INF
    assert torch.isfinite(S.ops.distillation_backward(x, values, labels, stats, torch.ones_like(loss))).all()


@pytest.mark.parametrize("C", [21, 600])
def test_distillation_temperatures(C, S):
    """T^2 has to be an ordinary fp32 number; at the ends of the range results stay finite."""
    x = G.scores_of((3, C), torch.float32, 231)
    values, labels, rest = G.record_of(x, 3, 1.0, 232)
    for t in (1e-30, 1e-19, 1e19, 1e30):
        with pytest.raises(ValueError):
            S.ops.distillation_forward(x, values, labels, rest, t)
        loss = torch.ones(3, device="cuda")
        with pytest.raises(ValueError):
            S.ops.distillation_backward(x, values, labels, S.ops.distillation_forward(x, values, labels, rest)[1], loss, rest, t)
    for t in (1e-18, 1e18):
        loss, stats = S.ops.distillation_forward(x, values, labels, None, t)
        assert torch.isfinite(loss).all()
        assert torch.isfinite(S.ops.distillation_backward(x, values, labels, stats, torch.ones_like(loss), None, t)).all()


def test_distillation_statistics(S):
    """What forward hands to backward: five numbers a row, written in full, or nothing where backward needs nothing."""
    for C, n in [(2, 0), (24, 0), (25, 5), (300, 5)]:
        x = G.scores_of((2, C, 7, 9), torch.float32, 241)
        values, labels, rest = G.record_of(x, 2, 1.0, 242)
        loss, stats = S.ops.distillation_forward(x, values, labels, rest)
        assert tuple(stats.shape) == (n, 2, 7, 9) and torch.isfinite(stats).all()
        if n:
            z = torch.logsumexp(x.double(), 1) - x.max(1).values.double()
            assert torch.equal(stats[0], x.max(1).values) and float((stats[1].double() - z).abs().max()) <= G.CHAIN(C) * 2.0 ** -24 + 2.0 ** -20
        leaf = x.clone().requires_grad_(True)
        grad, = torch.autograd.grad(S.training.distillation_loss(leaf, values, labels, rest).sum(), leaf)
        assert torch.equal(grad, S.ops.distillation_backward(x, values, labels, stats, torch.ones_like(loss), rest))
        with pytest.raises(RuntimeError):
            S.ops.distillation_backward(x, values, labels, torch.zeros((5 - n, 2, 7, 9), device="cuda"), torch.ones_like(loss), rest)


def test_per_image_distillation_of_a_matrix(S):
    """[N, C] scores: every row an image of one pixel."""
    x = G.scores_of((6, 40), torch.float32, 251)
    values, labels, rest = G.record_of(x, 4, 1.0, 252)
    valid = torch.tensor([1, 0, 1, 1, 0, 1], dtype=torch.bool, device="cuda")
    as_map = lambda a: a.unsqueeze(-1).unsqueeze(-1)
    for v in (valid, None):
        got = S.training.per_image_distillation(x, values, labels, rest, 1.0, v)
        want = S.training.per_image_distillation(as_map(x), as_map(values), as_map(labels), as_map(rest), 1.0, None if v is None else as_map(v))
        rows = S.training.distillation_loss(x, values, labels, rest, 1.0, v).double()
        assert got.shape == () and abs(float(got) - float(rows.mean())) <= 8 * 2.0 ** -24 * float(rows.mean())
        assert abs(float(got) - float(want)) <= 16 * 2.0 ** -24 * float(rows.mean())


@pytest.mark.parametrize("by_rows", [True, False])
def test_distillation_gradient_past_32_bits(by_rows, S):
    """2^31 + scores whose last rows lie past 32-bit element offsets, against a teacher that differs from the student there:
    a gradient far from zero."""
    if by_rows:
        n, c = 33000, 65600
        x = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
        rows = G.scores_of((3, c), torch.bfloat16, 261)
        x[n - 3:] = rows
        tail = lambda t: t[n - 3:]
    else:
        c, h, w = 33, 8192, 8192
        x = torch.zeros(1, c, h, w, dtype=torch.bfloat16, device="cuda")
        rows = G.scores_of((3, c), torch.bfloat16, 262)
        x[0, :, h - 1, w - 3:] = rows.t()
        tail = lambda t: t[0, ..., h - 1, w - 3:].t() if t.dim() == 4 else t[0, h - 1, w - 3:]
    k = 3
    values, labels, rest = G.record_of(rows, k, 1.0, 263)
    outer = (x.shape[0],) + tuple(x.shape[2:])
    full = lambda shape, dtype, value, part: (lambda t: (tail(t).copy_(part), t)[1])(torch.full(shape, value, dtype=dtype, device="cuda"))
    wide = (x.shape[0], k) + tuple(x.shape[2:])
    values_all, labels_all, rest_all = full(wide, values.dtype, 1.0, values), full(wide, torch.int32, 0, labels), full(outer, torch.float32, 0.5, rest)
    loss, stats = S.ops.distillation_forward(x, values_all, labels_all, rest_all)
    # (so that memory of an earlier gradient does not pass for this one)
    torch.full_like(x, 7.0)
    grad = S.ops.distillation_backward(x, values_all, labels_all, stats, torch.ones_like(loss), rest_all)
    got_l, got_g, half = tail(loss).cpu().numpy(), tail(grad).float().cpu().numpy(), 2.0 ** -8
    unit = G.CHAIN(c) * 2.0 ** -23 + 2.0 ** -21
    for i in range(3):
        wl, wg, (bl, bg) = R.distill(rows[i].double().cpu().numpy(), values[i].float().cpu().numpy(), labels[i].cpu().numpy(), float(rest[i]), 1.0)
        assert wl > 0.01 and abs(got_l[i] - wl) <= unit * bl
        assert np.abs(wg).max() > 0.01
        assert (np.abs(got_g[i] - wg) <= unit * bg * (1 + half) + half * np.abs(wg) + 2.0 ** -125).all()


# ------------------------------------------------------------------ top labels

@pytest.mark.parametrize("C,k", [(40, 3), (300, 3), (700, 20), (9000, 3), (9000, 100)])
def test_rest_of_rows_that_are_no_numbers(C, k, S):
    """More NaN than the record holds, next to infinities: the rest is no number either."""
    x = G.scores_of((6, C), torch.float32, 271)
    x[0, : k + 2] = NAN
    x[0, k + 2:k + 4] = INF
    x[1, C - k - 5:] = NAN
    x[1, 0] = INF
    x[2] = NAN
    x[3], x[3, ::2] = -INF, NAN
    x[4, : k + 1], x[4, k + 1] = INF, -INF                 # infinities alone: an infinite rest
    for y in (x, x.reshape(2, 3, C).movedim(2, 1)):
        G.check_top(S, y, k, 1.0)


# ------------------------------------------------------------------ drawn labels

def long_draw(z, us, top_k, top_p):
    """R.sample for many draws of one row, in 80-bit arithmetic: next to a largest weight of 1 the sum of 10^5 weights of
    2^-44 is lost in the steps of 64 bits."""
    z = np.asarray(z, np.longdouble)
    w = np.exp(z - z.max())
    order = R.order_of(z)[: top_k or z.size]
    front = np.concatenate([[np.longdouble(0)], np.cumsum(w[order])])
    n = max(1, int((front[:-1] < np.longdouble(top_p) * front[-1]).sum())) if top_p < 1 else order.size
    keep = np.sort(order[:n])
    run = np.cumsum(w[keep])
    at = [min(int(np.searchsorted(run, np.longdouble(u) * run[-1], side="right")), n - 1) for u in us]
    return keep[at], np.array([np.log(w[keep[i]] / run[-1]) for i in at], np.float64), n


@pytest.mark.parametrize("rows,C,low,high,top_k", [(5, 1 << 20, 30.2, 30.2, 0), (5, 1 << 19, 28.5, 31.9, 0), (130, 1 << 19, 28.5, 31.9, 0),
                                                   (5, 1 << 19, 28.5, 36.0, 1 << 18), (5, 1 << 20, 30.2, 30.2, 1 << 19)])
def test_a_cut_deep_in_the_tail(rows, C, low, high, top_k, S):
    """One peak and a tail of labels 2^-41 to 2^-52 of it, which top_p cuts in the middle: every label of the tail keeps the
    mass it has.  The draws fall into the tail, whose labels stand in front of the peak."""
    gen = np.random.default_rng(7)
    z = -gen.permutation(np.linspace(low, high, C)).astype(np.float32)
    z[C - 1] = 0
    kept = np.sort(np.exp(z.astype(np.longdouble)))[::-1][: top_k or C]
    mass = float(kept[1:].sum())
    top_p = 1.0 - 0.5 * mass
    us = np.float32(mass * np.linspace(0.0, 0.45, 5)).tolist()
    want, logprob, n = long_draw(z, us, top_k, top_p)
    assert 2048 < n < C - 2048 and len(set(want.tolist())) == 5
    x = torch.from_numpy(z).cuda().expand(rows, C).contiguous()
    u = torch.tensor(us, dtype=torch.float32, device="cuda").repeat(rows // 5)
    got, lp = S.ops.sample_labels(x, u, top_k=top_k, top_p=top_p, want_logprob=True)
    assert got.cpu().numpy().tolist() == want.tolist() * (rows // 5)
    assert (np.abs(lp.cpu().numpy()[:5] - logprob) <= 2.0 ** -24 * np.abs(logprob) + 1e-9).all()


@pytest.mark.parametrize("shape,scale", [((3, 4096), 0.01), ((140, 9000), 0.004), ((4, 60000), 0.05), ((2, 200000), 0.1)])
def test_cuts_within_a_bin_of_many_different_scores(shape, scale, S):
    """Rows so flat that the part of the row the cut falls into holds more labels than its list, of different scores."""
    x = G.scores_of(shape, torch.float32, 281, scale)
    if shape[0] > 100:
        x[3:] = x[:1]                                      # (the restatement walks three rows; the others repeat the first)
    u = torch.rand(shape[0], generator=G.gen(282), device="cuda")
    if shape[0] > 100:
        u[3:] = u[0]
    C = shape[1]
    for kw in (dict(top_p=0.8), dict(top_p=0.5, min_p=0.9), dict(top_k=C // 3), dict(top_k=C // 2, top_p=0.7)):
        labels, logprob = S.ops.sample_labels(x, u, want_logprob=True, **kw)
        for i in range(min(3, shape[0])):
            want, lp = R.sample(x[i].cpu().numpy(), float(u[i]), **kw)
            assert int(labels[i]) == want and abs(float(logprob[i]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (i, kw)
        if shape[0] > 100:
            assert (labels[3:] == labels[0]).all()


def test_drawing_for_very_many_rows_of_a_few_hundred_labels(S):
    """2^22 and more rows that a workgroup each draws for (all of them one row of memory, seen with stride 0)."""
    n, C = (1 << 22) + 8, 256
    z = G.scores_of((1, C), torch.bfloat16, 291, 2.0)
    u = torch.rand(n, generator=G.gen(292), device="cuda")
    labels = S.ops.sample_labels(z.expand(n, C), u, top_p=0.9, dtype=torch.int32)
    for i in (0, 1, n // 2, n - 9, n - 8, n - 1):
        assert int(labels[i]) == R.sample(z[0].float().cpu().numpy(), float(u[i]), top_p=0.9)[0]
    assert torch.equal(labels[-8:], S.ops.sample_labels(z.expand(8, C), u[-8:], top_p=0.9, dtype=torch.int32))
