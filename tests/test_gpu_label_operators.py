"""GPU parity of the label-selection operators (top labels, distillation loss and gradient, drawn labels) with plain
64-bit restatements (label_reference.py), at the sizes, layouts and masks where they can go wrong.

Tolerances.  A sum of n positive fp32 terms added one after the other is off by at most n 2^-24 of itself; CHAIN(C) bounds
the longest chain of the kernels.  An exponent x is off by at most 2^-22 (1 + |x|): a difference of scores, its product
with log2(e) / T (itself rounded) and the exponential's own error, half a step each, with room for one more.  So the rest
is off by CHAIN 2^-24 + 2^-22 (1 + |m / T|), and losses and gradients by (CHAIN 2^-23 + 2^-21) of `bound`, the sum of the
absolute terms they are made of, each times 1 + its exponent.  Stored gradients add half a step of their type.  An exponential
below 2^-126 is flushed to zero: off by 2^-126, times the gradient's factor weight * T."""
import numpy as np
import pytest
import torch

import label_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
INF = float("inf")


def CHAIN(C):
    return C + 32 if C < 4096 else C // 64 + 128


@pytest.fixture(scope="module")
def S():
    import semantic_segmentation_amd as S
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return S


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def scores_of(shape, dtype, seed, scale=3.0):
    return (scale * torch.randn(shape, generator=gen(seed), device="cuda")).to(dtype)


def layouts(x):
    """The same scores in memory orders a caller may have."""
    yield "plain", x.contiguous()
    if x.dim() == 4:
        yield "channels_last", x.contiguous(memory_format=torch.channels_last)
        yield "turned", x.transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.full((x.shape[0], x.shape[1] + 3) + tuple(x.shape[2:]), float("nan"), dtype=x.dtype, device=x.device)
    wide[:, 1:-2] = x
    yield "slice", wide[:, 1:-2]
    back = x.movedim(1, -1).contiguous().movedim(-1, 1)
    yield "labels_last", back


def rows_np(t):
    return R.rows_of(t.detach().float().cpu().numpy()) if t.dtype.is_floating_point else R.rows_of(t.detach().cpu().numpy())


# ------------------------------------------------------------------ top labels

def check_top(S, x, k, t):
    values, labels, rest = S.ops.top_labels(x, k, temperature=t)
    assert values.dtype == x.dtype and labels.dtype == torch.int32 and rest.dtype == torch.float32
    assert tuple(values.shape) == (x.shape[0], k) + tuple(x.shape[2:]) == tuple(labels.shape)
    assert tuple(rest.shape) == (x.shape[0],) + tuple(x.shape[2:])
    z, v, l, r = rows_np(x), rows_np(values), rows_np(labels), rest.cpu().numpy().reshape(-1)
    for i in range(z.shape[0]):
        wv, wl, wr = R.top(z[i].astype(np.float64), k, t)
        assert np.array_equal(l[i], wl), (i, l[i], wl)
        assert np.array_equal(v[i], wv.astype(np.float32), equal_nan=True)
        if np.isfinite(wr):
            m = np.abs(z[i][np.isfinite(z[i])]).max() / t
            assert abs(r[i] - wr) <= CHAIN(z.shape[1]) * 2.0 ** -24 + 2.0 ** -22 * (1 + m), (i, r[i], wr)
        else:
            assert np.array_equal(r[i], wr, equal_nan=True), (i, r[i], wr)


TOP_SHAPES = [((1, 1), 1), ((3, 2), 2), ((2, 5, 3, 7), 3), ((1, 21, 9, 31), 4), ((2, 33, 4, 65), 8), ((1, 150, 5, 13), 16),
              ((2, 40, 3), 32), ((1, 40, 7), 40), ((3, 127), 127), ((2, 129), 128), ((5, 511), 8), ((3, 512), 1), ((4, 513), 65),
              ((2, 4097), 128), ((1, 70001), 50), ((70, 1030), 7), ((300, 600), 20), ((2, 1100, 3), 20), ((1, 20000), 128), ((5000, 70), 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,k", TOP_SHAPES)
def test_top_labels(shape, k, dtype, S):
    for i, (name, x) in enumerate(layouts(scores_of(shape, dtype, 10 + k))):
        if np.prod(shape) > 50000 and i > 1:
            continue
        check_top(S, x, k, 1.7)


@pytest.mark.parametrize("C,k", [(6, 3), (40, 12), (700, 20), (9000, 100)])
def test_top_labels_of_equal_masked_and_unusual_scores(C, k, S):
    x = torch.zeros(12, C, device="cuda")
    x[1] = -INF                                            # a mask that leaves nothing
    x[2, 1:] = -INF
    x[3] = torch.finfo(torch.float32).min
    x[4, C // 2:] = torch.finfo(torch.float32).min
    x[5, ::3] = -0.0
    x[6, C - 1] = float("nan")
    x[7, C // 3] = INF
    x[8] = torch.arange(C, device="cuda")                  # every label better than all before it
    x[9] = -torch.arange(C, device="cuda").float()
    x[10] = torch.arange(C, device="cuda") % 3             # long runs of equals
    x[11, : C // 2] = float("nan")
    for y in (x, x.reshape(3, 4, C).movedim(2, 1)):
        check_top(S, y, k, 1.0)


def test_top_labels_agree_with_argmax_labels(S):
    x = scores_of((2, 21, 33, 70), torch.float32, 4)
    assert torch.equal(S.ops.top_labels(x, 1)[1][:, 0].to(torch.uint8), S.ops.argmax_labels(x))


# ------------------------------------------------------------------ distillation

def record_of(x, k, t, seed, dtype=None):
    """A teacher near the student: values and labels of its k best, rest of the others, in plain torch."""
    teacher = x.detach().float() + torch.randn(x.shape, generator=gen(seed), device="cuda")
    teacher = torch.where(torch.isfinite(teacher), teacher, torch.zeros_like(teacher))
    values, labels = torch.topk(teacher, k, 1)
    rest = torch.logsumexp(teacher.scatter(1, labels, -INF) / t, 1)
    return values.to(dtype or x.dtype).contiguous(), labels.to(torch.int32).contiguous(), rest.contiguous()


def check_distill(S, x, values, labels, rest, t, valid=None, weight=None):
    weight = torch.rand((x.shape[0],) + tuple(x.shape[2:]), device="cuda", generator=gen(99)) + 0.5 if weight is None else weight
    leaf = x.detach().requires_grad_(True)
    loss = S.training.distillation_loss(leaf, values, labels, rest=rest, temperature=t, valid=valid)
    grad, = torch.autograd.grad(loss, leaf, weight)
    assert grad.dtype == x.dtype and grad.shape == x.shape and loss.dtype == torch.float32
    z, v, l = rows_np(x), rows_np(values), rows_np(labels)
    rr = None if rest is None else rest.cpu().numpy().reshape(-1)
    ok = np.ones(z.shape[0], bool) if valid is None else valid.cpu().numpy().reshape(-1) != 0
    w = weight.cpu().numpy().reshape(-1).astype(np.float64)
    got_l, got_g = loss.detach().cpu().numpy().reshape(-1), rows_np(grad)
    unit = CHAIN(z.shape[1]) * 2.0 ** -23 + 2.0 ** -21
    half = torch.finfo(x.dtype).eps / 2
    for i in range(z.shape[0]):
        wl, wg, (bl, bg) = R.distill(z[i].astype(np.float64), v[i], l[i], None if rr is None else rr[i], t, ok[i])
        if np.isfinite(wl):
            assert abs(got_l[i] - wl) <= unit * bl, (i, got_l[i], wl)
        else:
            assert np.array_equal(got_l[i], wl, equal_nan=True), (i, got_l[i], wl)
        wg = wg * w[i]
        tol = unit * bg * w[i] * (1 + half) + half * np.abs(wg) + TINY[x.dtype] + 2.0 ** -126 * w[i] * t
        assert np.array_equal(np.isnan(got_g[i]), np.isnan(wg))
        bad = np.abs(got_g[i] - wg) > tol
        assert not bad.any(), (i, int(bad.sum()), np.abs(got_g[i] - wg)[bad].max(), tol[bad].min())


DISTILL_SHAPES = [((1, 1), 1), ((3, 2), 1), ((2, 5, 3, 7), 5), ((1, 21, 9, 31), 4), ((2, 33, 4, 65), 8), ((1, 150, 5, 13), 16),
                  ((2, 300, 9), 40), ((3, 127), 127), ((5, 511), 8), ((3, 512), 128), ((4, 513), 3), ((2, 4097), 64), ((1, 70001), 50),
                  ((70, 1030), 7), ((2, 1100, 3), 20), ((1, 12, 7, 9), 2), ((1, 17, 7, 9), 9), ((1, 64, 130, 127), 20)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,k", DISTILL_SHAPES)
def test_distillation(shape, k, dtype, S):
    for i, (name, x) in enumerate(layouts(scores_of(shape, dtype, 20 + k))):
        if np.prod(shape) > 50000 and i > 1:
            continue
        t = (1.0, 2.5, 0.5)[i % 3]
        values, labels, rest = record_of(x, k, t, 3)
        check_distill(S, x, values, labels, rest if i % 2 == 0 else None, t)


@pytest.mark.parametrize("shape", [(40, 21), (2, 21, 4, 5), (6, 2000)])
def test_distillation_of_padded_records_and_void_rows(shape, S):
    x = scores_of(shape, torch.float32, 31)
    k, C = 6, shape[1]
    values, labels, rest = record_of(x, k, 1.5, 5, torch.bfloat16)
    rows = (shape[0],) + tuple(shape[2:])
    pick = torch.rand(labels.shape, generator=gen(6), device="cuda")
    labels[pick < 0.2] = -1                                # entries of no class
    labels[pick > 0.9] = C + 7
    labels[:, 4] = labels[:, 3]                            # one label named twice
    values[:, 5] = -INF                                    # no mass, still a label of the record
    labels[0] = -1                                         # nothing left of a record
    rest[1] = -INF
    valid = torch.rand(rows, generator=gen(7), device="cuda") > 0.3
    bad = ~valid
    x = torch.where(bad.unsqueeze(1), torch.full_like(x, float("nan")), x)      # what stands in void rows does not matter
    values = torch.where(bad.unsqueeze(1), torch.full_like(values, float("nan")), values)
    rest = torch.where(bad, torch.full_like(rest, INF), rest)
    weight = torch.where(bad, torch.full(rows, float("nan"), device="cuda"), torch.ones(rows, device="cuda"))
    for with_rest in (rest, None):
        loss = S.training.distillation_loss(x.requires_grad_(True), values, labels, rest=with_rest, temperature=1.5, valid=valid)
        assert (loss[bad] == 0).all() and torch.isfinite(loss[valid]).all()
        grad, = torch.autograd.grad(loss, x, weight)
        assert (grad.movedim(1, -1)[bad] == 0).all()
        keep = torch.where(bad, torch.zeros_like(weight), weight)
        clean = torch.where(bad.unsqueeze(1), torch.zeros_like(x), x).detach()
        check_distill(S, clean, torch.nan_to_num(values), labels, None if with_rest is None else torch.nan_to_num(with_rest, posinf=0.0),
                      1.5, valid, keep)
        x = x.detach()


@pytest.mark.parametrize("C", [9, 50, 900])
def test_distillation_of_masked_and_extreme_scores(C, S):
    low = torch.finfo(torch.float32).min
    x = scores_of((8, C), torch.float32, 41)
    values, labels, rest = record_of(x, 4, 1.0, 8)
    x[0, :] = -INF                                          # a row whose mask leaves nothing
    x[1, 5:] = -INF
    labels[1] = torch.tensor([0, 1, 2, 3], device="cuda")
    x[2] = low
    x[3, 4:] = low
    labels[3] = torch.tensor([0, 1, 2, 3], device="cuda")
    rest[3] = -INF
    x[4] *= 30                                              # a tail that would vanish next to the record
    x[5, labels[5].long()] += 60.0
    x[6] += 1000.0
    x[7, :] = 2.0
    for r in (rest, None):
        check_distill(S, x, values, labels, r, 1.0)
    # the student forbids a label that the teacher wants: an infinite loss, a finite gradient
    y = torch.zeros(1, C, device="cuda")
    y[0, 2] = -INF
    check_distill(S, y, torch.zeros(1, 2, device="cuda"), torch.tensor([[1, 2]], dtype=torch.int32, device="cuda"), None, 1.0)
    # a NaN stays in its row
    z = torch.zeros(2, C, device="cuda")
    z[0, 1] = float("nan")
    rec = (torch.zeros(2, 2, device="cuda"), torch.tensor([[1, 2], [1, 2]], dtype=torch.int32, device="cuda"))
    loss, _ = S.ops.distillation_forward(z, *rec)
    assert torch.isnan(loss[0]) and torch.isfinite(loss[1])


@pytest.mark.parametrize("C", [12, 600])
def test_distillation_gradient_against_differences(C, S):
    """Central differences of the loss itself: (L(z + h) - L(z - h)) / 2h is off by h^2 / 6 of the third derivative (at most
    1 / T for a softmax) and by the two losses' own errors over 2h."""
    t, h, k = 1.3, 0.05, 4
    x = scores_of((1, C), torch.float32, 51, 1.0)
    values, labels, rest = record_of(x, k, t, 9)
    loss, stats = S.ops.distillation_forward(x, values, labels, rest, t)
    grad = S.ops.distillation_backward(x, values, labels, stats, torch.ones_like(loss), rest, t)[0].cpu().numpy()
    pick = list(labels[0].tolist()) + [c for c in range(C) if c not in labels[0].tolist()][:8]
    step = torch.zeros(2 * len(pick), C, device="cuda")
    for i, c in enumerate(pick):
        step[2 * i, c], step[2 * i + 1, c] = h, -h
    many = (x + step).contiguous()
    rep = lambda a: a.expand((len(step),) + tuple(a.shape[1:])).contiguous()
    l = S.ops.distillation_forward(many, rep(values), rep(labels), rep(rest), t)[0].double().cpu().numpy()
    bound = R.distill(x[0].cpu().numpy().astype(np.float64), values[0].cpu().numpy(), labels[0].cpu().numpy(), float(rest[0]), t)[2][0]
    tol = h * h / 6 / t + 2 * (CHAIN(C) * 2.0 ** -23 + 2.0 ** -21) * bound / (2 * h)
    for i, c in enumerate(pick):
        assert abs((l[2 * i] - l[2 * i + 1]) / (2 * h) - grad[c]) <= tol, (c, grad[c], tol)


def test_per_image_distillation_is_the_mean_of_image_means(S):
    x = scores_of((3, 7, 6, 10), torch.float32, 61)
    values, labels, rest = record_of(x, 3, 1.0, 10)
    valid = torch.rand(3, 6, 10, generator=gen(11), device="cuda") > 0.4
    valid[1] = False
    rows = S.training.distillation_loss(x, values, labels, rest, 1.0, valid).cpu().double()
    v = valid.cpu()
    want = sum(float(rows[b][v[b]].mean()) if v[b].any() else 0.0 for b in range(3)) / 3
    got = float(S.training.per_image_distillation(x, values, labels, rest, 1.0, valid))
    assert abs(got - want) <= 64 * 2.0 ** -24 * abs(want)
    plain = float(S.training.per_image_distillation(x, values, labels, rest))
    full = S.training.distillation_loss(x, values, labels, rest).double().mean()
    assert abs(plain - float(full)) <= 64 * 2.0 ** -24 * float(full)


# ------------------------------------------------------------------ drawn labels

def check_sample(S, x, u, **kw):
    """Labels equal; logprob is one fp32 rounding of a 64-bit value."""
    labels, logprob = S.ops.sample_labels(x, u, want_logprob=True, **kw)
    assert labels.shape == u.shape == logprob.shape and labels.dtype == torch.int64
    inner = u[0].numel()
    per = {k: (v.double().cpu().numpy() if torch.is_tensor(v) else None) for k, v in kw.items()}
    z, uu = rows_np(x), u.cpu().numpy().reshape(-1).astype(np.float64)
    got, lp = labels.cpu().numpy().reshape(-1), logprob.cpu().numpy().reshape(-1)
    for i in range(z.shape[0]):
        s = {k: (float(per[k][i // inner]) if per[k] is not None else v) for k, v in kw.items()}
        if "temperature" in s:
            s["t"] = s.pop("temperature")
        if "top_k" in s:
            s["top_k"] = int(s["top_k"])
        want, wlp = R.sample(z[i].astype(np.float64), uu[i], **s)
        assert got[i] == want, (i, got[i], want, s)
        assert lp[i] == wlp or abs(lp[i] - wlp) <= 2.0 ** -24 * abs(wlp) + 1e-12, (i, lp[i], wlp)


SAMPLE_SHAPES = [(1, 1), (5, 2), (2, 5, 3, 7), (1, 21, 9, 31), (2, 33, 4, 65), (1, 150, 5, 13), (2, 300, 9), (3, 127), (5, 511), (3, 512),
                 (4, 513), (2, 4097), (1, 70001), (70, 1030)]
SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.6, min_p=0.05), dict(top_k=1), dict(temperature=1.4, top_k=7),
            dict(top_p=0.8), dict(temperature=2.0, top_p=0.97), dict(top_k=40, top_p=0.9, min_p=0.02), dict(top_k=300, top_p=0.6)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SAMPLE_SHAPES)
def test_sample_labels(shape, dtype, S):
    x = scores_of(shape, dtype, 71, 2.0)
    u = torch.rand((shape[0],) + tuple(shape[2:]), generator=gen(72), device="cuda")
    for kw in SETTINGS:
        check_sample(S, x, u, **kw)
    for name, y in list(layouts(x))[1:]:
        check_sample(S, y, u, top_k=12, top_p=0.9, temperature=1.1)
        check_sample(S, y, u, min_p=0.01)


@pytest.mark.parametrize("scale", [0.1, 2.0])
@pytest.mark.parametrize("shape,dtype", [((1, 70, 50, 60), torch.float32), ((2, 150, 33, 40), torch.bfloat16), ((1, 30, 60, 50), torch.float16),
                                         ((2, 1500, 3), torch.float32)])
def test_sample_labels_of_maps_with_flat_and_peaked_rows(shape, dtype, scale, S):
    """Enough pixels for one lane each; flat rows keep far more labels than a lane's list holds."""
    x = scores_of(shape, dtype, 70, scale)
    u = torch.rand((shape[0],) + tuple(shape[2:]), generator=gen(71), device="cuda")
    for kw in (dict(top_p=0.9), dict(top_p=0.55, min_p=0.02), dict(top_k=45), dict(top_k=60, top_p=0.7), dict(top_k=20, top_p=0.8)):
        check_sample(S, x, u, **kw)
    f = lambda *v: torch.tensor(v[:shape[0]], dtype=torch.float32, device="cuda")
    check_sample(S, x, u, temperature=f(0.7, 1.5), top_p=f(0.8, 0.95), min_p=f(0.0, 0.01),
                 top_k=torch.tensor([0, 50][:shape[0]], dtype=torch.int32, device="cuda"))
    check_sample(S, x, u, temperature=f(1.3, 0.0))


@pytest.mark.parametrize("shape", [(9, 40), (9, 30, 2, 3), (9, 1500), (9, 9000)])
def test_sample_labels_with_settings_of_every_row(shape, S):
    x = scores_of(shape, torch.float32, 73, 2.0)
    u = torch.rand((shape[0],) + tuple(shape[2:]), generator=gen(74), device="cuda")
    f = lambda *v: torch.tensor(v, dtype=torch.float32, device="cuda")
    t = f(0.0, 0.5, 1.0, 2.0, 1.0, -1.0, 1.0, 3.0, 0.7)
    k = torch.tensor([0, 5, -3, 1000000, 1, 4, 20, 200, 0], dtype=torch.int32, device="cuda")
    p = f(0.9, 1.0, 0.5, 2.0, 0.3, 0.9, 0.0, 0.95, 0.99)
    m = f(0.0, 0.1, -1.0, 0.0, 0.5, 0.0, 0.0, 0.01, 2.0)
    check_sample(S, x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check_sample(S, x, u, temperature=t, top_p=0.85)
    check_sample(S, x, u, top_k=k)


@pytest.mark.parametrize("C", [8, 100, 600, 5000, 30000])
def test_sample_labels_of_equal_masked_and_unusual_scores(C, S):
    low = torch.finfo(torch.float32).min
    x = torch.zeros(10, C, device="cuda")
    x[1] = -INF
    x[2, : C - 1] = -INF
    x[3] = low
    x[4, ::2] = low
    x[5, C // 2] = float("nan")
    x[6, C // 2] = INF
    x[7, ::2] = -INF
    x[8] = torch.arange(C, device="cuda") % 2
    x[9] = -900.0
    x[9, C - 1] = 0.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.3, 0.3, 0.0, 0.99, 0.99], device="cuda")
    for kw in (dict(), dict(top_k=4), dict(top_p=0.3), dict(top_p=0.5, top_k=6), dict(min_p=1.0), dict(temperature=0.0),
               dict(min_p=0.3, temperature=0.5)):
        check_sample(S, x, u, **kw)
        check_sample(S, x.reshape(5, 2, C).movedim(2, 1), u.reshape(5, 2), **kw)
    # a long run of one score that the cut falls into, in front of and behind others
    z = torch.zeros(4, C, device="cuda")
    z[0, : C // 5] = 1.0
    z[1, C // 3:] = -2.0
    z[2, ::3] = 0.5
    z[3, 1::7] = -INF
    for kw in (dict(top_p=0.7), dict(top_k=C // 2), dict(top_k=max(2, C // 2), top_p=0.9), dict(top_p=0.95, min_p=0.3), dict(top_k=C // 5 + 1)):
        check_sample(S, z, u[1:5].contiguous(), **kw)
    # numbers outside [0, 1): the first and the last kept label
    odd = torch.tensor([-1.0, 1.0, 2.0, float("nan")], device="cuda")
    y = torch.zeros(4, C, device="cuda")
    y[:, -1] = -INF
    assert S.ops.sample_labels(y, odd).tolist() == [0, C - 2, C - 2, 0]


def test_sample_labels_types_and_void(S):
    x = scores_of((2, 21, 8, 9), torch.float32, 75)
    x[0, :, 0, 0] = -INF
    u = torch.rand((2, 8, 9), generator=gen(76), device="cuda")
    a, b, c = (S.ops.sample_labels(x, u, top_k=3, dtype=d) for d in (torch.int64, torch.int32, torch.uint8))
    assert int(a[0, 0, 0]) == -1 and int(b[0, 0, 0]) == -1 and int(c[0, 0, 0]) == 255
    assert torch.equal(a.to(torch.int32), b) and torch.equal(a.to(torch.uint8), c)
    # greedy draws are argmax_labels, and the void pixel counts for no class
    greedy = S.ops.sample_labels(x, u, temperature=0.0, dtype=torch.uint8)
    keep = torch.ones_like(greedy, dtype=torch.bool)
    keep[0, 0, 0] = False
    assert torch.equal(greedy[keep], S.ops.argmax_labels(x)[keep])
    assert int(S.ops.iou_counts(greedy, greedy, 21)[1].sum()) == greedy.numel() - 1


def test_refusals_and_numbers_of_other_types(S):
    """Wrong companions are refused before a launch; numpy's numbers serve like Python's."""
    x = scores_of((4, 30, 5), torch.float32, 78)
    u = torch.rand(4, 5, generator=gen(79), device="cuda")
    values, labels, rest = S.ops.top_labels(x, np.int64(3), temperature=np.float32(1.5))
    assert all(torch.equal(a, b) for a, b in zip((values, labels, rest), S.ops.top_labels(x, 3, 1.5)))
    assert torch.equal(S.ops.sample_labels(x, u, top_k=np.int32(4), top_p=np.float32(0.5)), S.ops.sample_labels(x, u, top_k=4, top_p=0.5))
    assert torch.equal(S.ops.sample_labels(x, u, top_k=1 << 40), S.ops.sample_labels(x, u))
    for call, kind in [(lambda: S.ops.top_labels(x, 0), ValueError), (lambda: S.ops.top_labels(x, 31), ValueError),
                       (lambda: S.ops.top_labels(x, 3, 0.0), ValueError), (lambda: S.ops.top_labels(x.double(), 3), RuntimeError),
                       (lambda: S.ops.top_labels(x[0, 0], 1), RuntimeError), (lambda: S.ops.top_labels(x[:0], 1), RuntimeError),
                       (lambda: S.ops.sample_labels(x, u[:, :4]), RuntimeError), (lambda: S.ops.sample_labels(x, u.double()), RuntimeError),
                       (lambda: S.ops.sample_labels(x, u.cpu()), RuntimeError), (lambda: S.ops.sample_labels(x, u, top_k=-1), ValueError),
                       (lambda: S.ops.sample_labels(x, u, top_p=0.0), ValueError), (lambda: S.ops.sample_labels(x, u, min_p=1.5), ValueError),
                       (lambda: S.ops.sample_labels(x, u, temperature=-1.0), ValueError), (lambda: S.ops.sample_labels(x, u, dtype=torch.int16), TypeError),
                       (lambda: S.ops.sample_labels(x, u, temperature=torch.ones(3, device="cuda")), RuntimeError),
                       (lambda: S.ops.sample_labels(x, u, top_k=torch.ones(4, device="cuda")), RuntimeError),
                       (lambda: S.ops.distillation_forward(x, values, labels.long(), rest), RuntimeError),
                       (lambda: S.ops.distillation_forward(x, values[:, :2], labels, rest), RuntimeError),
                       (lambda: S.ops.distillation_forward(x, values, labels, rest[:2]), RuntimeError),
                       (lambda: S.ops.distillation_forward(x, values, labels, rest, valid=rest), RuntimeError),
                       (lambda: S.ops.distillation_forward(x, values[..., 0], labels, rest), RuntimeError),
                       (lambda: S.training.distillation_loss(x, values.requires_grad_(True), labels), RuntimeError)]:
        with pytest.raises(kind):
            call()


def test_sampled_shares_follow_the_distribution(S):
    """An even grid of draws: every label gets its share of it, to within the two ends of its interval."""
    n, C = 4096, 37
    z = scores_of((1, C), torch.float32, 77, 1.5)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    labels = S.ops.sample_labels(z.expand(n, C), u)
    share = torch.softmax(z[0].double(), 0).cpu().numpy()
    count = torch.bincount(labels, minlength=C).cpu().numpy()
    assert (np.abs(count - n * share) <= 2).all()


# ------------------------------------------------------------------ streams, graphs, offsets, the operators together

def test_on_another_stream(S):
    x = scores_of((2, 21, 40, 70), torch.float32, 81)
    u = torch.rand(2, 40, 70, generator=gen(82), device="cuda")
    want = S.ops.top_labels(x, 4), S.ops.sample_labels(x, u, top_k=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = S.ops.top_labels(x, 4), S.ops.sample_labels(x, u, top_k=5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want[0], got[0])) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("shape", [(2, 21, 24, 40), (6, 9001), (1, 40000)])
def test_captured_and_replayed(shape, S):
    """All four calls in one graph, replayed on new inputs between eager calls of the same sizes; each replay against the
    eager results, bit for bit."""
    t, k = 1.5, 5
    rows = (shape[0],) + tuple(shape[2:])
    x = scores_of(shape, torch.float32, 83)
    values, labels, rest = (a.clone() for a in record_of(x, k, t, 84))
    u, w = torch.rand(rows, generator=gen(85), device="cuda"), torch.rand(rows, generator=gen(86), device="cuda")

    def calls():
        loss, stats = S.ops.distillation_forward(x, values, labels, rest, t)
        return (*S.ops.top_labels(x, k, t), loss, S.ops.distillation_backward(x, values, labels, stats, w, rest, t),
                S.ops.sample_labels(x, u, top_k=9, top_p=0.9), S.ops.sample_labels(x, u), S.ops.sample_labels(x, u, top_p=0.9))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for seed in range(90, 94):
        x.copy_(scores_of(shape, torch.float32, seed))
        u.copy_(torch.rand(rows, generator=gen(seed), device="cuda"))
        graph.replay()
        want = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_two_graphs_do_not_share_memory(S):
    """Captured one after the other, replayed in turn on two streams."""
    xs = [scores_of((1, 30000), torch.float32, 95 + i) for i in range(2)]
    us = [torch.rand(1, generator=gen(97 + i), device="cuda") for i in range(2)]
    f = lambda i: (S.ops.top_labels(xs[i], 20), S.ops.sample_labels(xs[i], us[i], top_k=20), S.ops.sample_labels(xs[i], us[i]))
    flat = lambda o: [*o[0], o[1], o[2]]
    want = [[a.clone() for a in flat(f(i))] for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(flat(f(i)))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


@pytest.mark.parametrize("by_rows", [True, False])
def test_offsets_past_32_bits(by_rows, S):
    """2^31 + scores in half precision: the last rows (or the last classes) lie past 32-bit element offsets."""
    if by_rows:
        n, c = 33000, 65600
        big = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
        view, tail = big, slice(n - 3, n)
        tail_rows = scores_of((3, c), torch.bfloat16, 98)
        big[tail] = tail_rows
    else:
        c, h, w = 33, 8192, 8192
        big = torch.zeros(1, c, h, w, dtype=torch.bfloat16, device="cuda")
        tail_rows = scores_of((3, c), torch.bfloat16, 99)
        big[0, :, h - 1, w - 3:] = tail_rows.t()
        view = big
    pick = (lambda t: t[tail]) if by_rows else (lambda t: t[0, ..., h - 1, w - 3:].t() if t.dim() == 4 else t[0, h - 1, w - 3:])
    k = 3
    values, labels, rest = S.ops.top_labels(view, k)
    small = S.ops.top_labels(tail_rows, k)
    assert torch.equal(pick(values), small[0]) and torch.equal(pick(labels), small[1])
    loss, stats = S.ops.distillation_forward(view, values, labels, rest)
    grad = S.ops.distillation_backward(view, values, labels, stats, torch.ones_like(loss), rest)
    sl, ss = S.ops.distillation_forward(tail_rows, *small)
    sg = S.ops.distillation_backward(tail_rows, *small[:2], ss, torch.ones_like(sl), small[2])
    # the record is the scores' own: loss and gradient are what rounding leaves
    assert float((pick(loss) - sl).abs().max()) <= 1e-5 and float((pick(grad).float() - sg.float()).abs().max()) <= 1e-5
    u = torch.full(loss.shape, 0.5, device="cuda")
    assert torch.equal(pick(S.ops.sample_labels(view, u)), S.ops.sample_labels(tail_rows, pick(u).contiguous()))
    assert torch.equal(pick(S.ops.sample_labels(view, u, top_k=3)), S.ops.sample_labels(tail_rows, pick(u).contiguous(), top_k=3))


def test_teacher_to_student_on_the_mean_field_modules(S):
    """As they are used: a teacher's marginals become records and drawn pseudo-labels, a student trains on the records
    through the fused loop, its answers are compared with the draws."""
    B, L, H, W, k = 2, 8, 24, 72, 5
    torch.manual_seed(5)
    unary, image = scores_of((B, L, H, W), torch.float32, 101), scores_of((B, 3, H, W), torch.float32, 102, 1.0)
    teacher = S.MeanFieldLocal(H, W, L, k, iters=2, compat=True).cuda()
    student = S.MeanFieldLocal(H, W, L, k, iters=1, compat=True, affine=True).cuda()
    with torch.no_grad():
        marginals = teacher(unary, image)
    values, labels, rest = S.ops.top_labels(marginals, 3, temperature=2.0)
    u = torch.rand(B, H, W, generator=gen(103), device="cuda")
    drawn = S.ops.sample_labels(marginals, u, top_k=3, dtype=torch.uint8)
    assert ((labels == drawn.unsqueeze(1)).any(1)).all()
    valid = drawn != 0
    loss = S.training.per_image_distillation(student(unary, image), values, labels, rest, 2.0, valid)
    loss.backward()
    # the same step with the loss written out in torch
    got = {n: p.grad.clone() for n, p in student.named_parameters()}
    student.zero_grad()
    b = torch.log_softmax(student(unary, image) / 2.0, 1)
    a = torch.log_softmax(torch.cat([values / 2.0, rest.unsqueeze(1)], 1), 1)
    named = torch.zeros_like(b, dtype=torch.bool).scatter(1, labels.long(), True)
    q = torch.cat([torch.gather(b, 1, labels.long()), torch.logsumexp(b.masked_fill(named, -INF), 1, keepdim=True)], 1)
    rows = 4.0 * (a.exp() * (a - q)).sum(1) * valid
    want = (rows.flatten(1).sum(1) / valid.flatten(1).sum(1)).mean()
    want.backward()
    loss, want = float(loss.detach()), float(want.detach())
    assert abs(loss - want) <= 1e-5 * abs(want)
    for name, p in student.named_parameters():
        scale = float(p.grad.abs().max())
        assert float((got[name] - p.grad).abs().max()) <= 1e-4 * scale, name
    assert 0.0 <= S.ops.mean_intersection_over_union(S.ops.argmax_labels(student(unary, image).detach()), drawn, L) <= 1.0
