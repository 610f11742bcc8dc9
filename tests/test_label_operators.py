"""Refusals of the label-selection operators: the C ABI's checks come before any launch, and the Python wrappers' before
any call into the library, so both run without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import label_reference as R

one = ctypes.c_void_p(16)            # never dereferenced: the argument checks fail first
F32 = 0


@pytest.fixture(scope="module")
def L():
    from semantic_segmentation_amd import _lib
    return _lib.lib


def view(N=2, C=5, S=3, dtype=F32, strides=None, p=one):
    return (p, dtype, N, C, S) + tuple(strides or (C * S, S, 1))


def top(L, v, t=1.0, k=2, outs=(one, one, one)):
    return L.mfl_top_labels(*v, t, k, *outs, None, 0, None)


def test_views_are_checked(L):
    for v, want in [(view(p=None), -1), (view(N=0), -1), (view(C=0), -1), (view(S=-1), -1), (view(dtype=3), -1),
                    (view(strides=(-1, 1, 1)), -1), (view(N=1 << 16, S=1 << 16), -3), (view(C=(1 << 30) + 1), -3)]:
        assert top(L, v) == want
        assert L.mfl_distillation_forward(*v, one, F32, one, None, None, 2, 1.0, one, one, None, 0, None) == want
        assert L.mfl_distillation_backward(*v, one, F32, one, None, None, 2, 1.0, one, one, one, 15, 3, 1, None) == want
        assert L.mfl_sample_labels(*v, one, 1.0, None, 0, None, 1.0, None, 0.0, None, one, 8, None, None, 0, None) == want


def test_top_labels_refuses(L):
    for kw in (dict(k=0), dict(k=6), dict(t=0.0), dict(t=-1.0), dict(t=float("inf")), dict(t=float("nan")), dict(outs=(None, one, one)),
               dict(outs=(one, None, one)), dict(outs=(one, one, None))):
        assert top(L, view(), **kw) == -1
    assert top(L, view(C=200), k=129) == -1


def test_distillation_refuses(L):
    def fwd(values=one, vd=F32, labels=one, k=2, t=1.0, loss=one, stats=one):
        return L.mfl_distillation_forward(*view(), values, vd, labels, None, None, k, t, loss, stats, None, 0, None)

    for kw in (dict(values=None), dict(vd=7), dict(labels=None), dict(k=0), dict(k=129), dict(t=0.0), dict(loss=None), dict(stats=None)):
        assert fwd(**kw) == -1

    def bwd(stats=one, grad_loss=one, d=one, strides=(15, 3, 1)):
        return L.mfl_distillation_backward(*view(), one, F32, one, None, None, 2, 1.0, stats, grad_loss, d, *strides, None)

    for kw in (dict(stats=None), dict(grad_loss=None), dict(d=None), dict(strides=(15, -3, 1))):
        assert bwd(**kw) == -1


def test_sample_labels_refuses(L):
    def call(u=one, t=1.0, k=0, p=1.0, m=0.0, labels=one, size=8, C=5):
        return L.mfl_sample_labels(*view(C=C), u, t, None, k, None, p, None, m, None, labels, size, None, None, 0, None)

    for kw in (dict(u=None), dict(labels=None), dict(size=2), dict(t=-0.5), dict(t=float("nan")), dict(k=-1), dict(p=0.0), dict(p=1.5),
               dict(p=float("nan")), dict(m=-0.1), dict(m=1.1), dict(size=1, C=256)):
        assert call(**kw) == -1


def test_launches_past_32_bits_of_threads_are_refused(L):
    """2^25 rows of 300 labels would take one wave or workgroup each: more threads than a launch counts."""
    v = view(N=1 << 25, C=300, S=1, strides=(300, 1, 1))
    assert top(L, v) == -3
    assert L.mfl_distillation_forward(*view(N=1 << 25, C=600, S=1, strides=(600, 1, 1)), one, F32, one, None, None, 2, 1.0, one, one, one,
                                      1 << 40, None) == -3
    assert L.mfl_sample_labels(*v, one, 1.0, None, 0, None, 0.5, None, 0.0, None, one, 8, None, None, 0, None) == -3


def test_workspaces(L):
    """Small calls take none; a missing or short one is refused before any launch."""
    assert L.mfl_top_labels_workspace_bytes(8, 21, 4096, F32, 4) == 0
    n = L.mfl_top_labels_workspace_bytes(1, 128000, 1, F32, 50)
    assert n > 0
    v = view(N=1, C=128000, S=1, strides=(128000, 1, 1))
    assert L.mfl_top_labels(*v, 1.0, 50, one, one, one, None, 0, None) == -2
    assert L.mfl_top_labels(*v, 1.0, 50, one, one, one, one, n - 1, None) == -2
    m = L.mfl_distillation_workspace_bytes(1, 128000, 1, F32, 50)
    assert m > 0 and L.mfl_distillation_forward(*v, one, F32, one, None, None, 2, 1.0, one, one, one, m - 1, None) == -2
    q = L.mfl_sample_labels_workspace_bytes(1, 128000, 1, F32)
    assert q > 0 and L.mfl_sample_labels(*v, one, 1.0, None, 0, None, 1.0, None, 0.0, None, one, 8, None, None, 0, None) == -2


def test_wrappers_refuse_host_tensors_and_wrong_types():
    import semantic_segmentation_amd as S
    x, u = torch.zeros(2, 5, 4), torch.zeros(2, 4)
    record = (torch.zeros(2, 3, 4), torch.zeros(2, 3, 4, dtype=torch.int32))
    for call in (lambda z: S.ops.top_labels(z, 2), lambda z: S.ops.sample_labels(z, u), lambda z: S.ops.distillation_forward(z, *record)):
        with pytest.raises(RuntimeError, match="ROCm GPU only"):
            call(x)
    with pytest.raises(RuntimeError, match="no gradient for the teacher"):
        S.training.distillation_loss(x, record[0].requires_grad_(True), record[1])


def test_reference_against_brute_force():
    """The 64-bit restatement itself: softmax arithmetic on a row written out by hand."""
    z = np.array([0.0, np.log(2.0), np.log(4.0), 0.0])                      # shares 1/8, 2/8, 4/8, 1/8
    v, l, r = R.top(z, 2, 1.0)
    assert list(l) == [2, 1] and abs(r - np.log(2.0)) < 1e-15
    loss, grad, _ = R.distill(z, np.zeros(2), np.array([0, 3]), None, 1.0)  # teacher: 1/2 on labels 0 and 3
    assert abs(loss - np.log(4.0)) < 1e-15 and np.allclose(grad, [-0.375, 0.25, 0.5, -0.375], atol=1e-15)
    loss, grad, _ = R.distill(z, np.zeros(2), np.array([0, 3]), np.log(2.0), 1.0)       # 1/4, 1/4 and 1/2 elsewhere
    assert abs(loss - (0.5 * np.log(2.0) + 0.5 * np.log(2.0 / 3.0))) < 1e-15
    assert np.allclose(grad, [-0.125, 0.25 / 3, 0.5 / 3, -0.125], atol=1e-15)
    assert [R.sample(z, u)[0] for u in (0.0, 0.124, 0.126, 0.374, 0.376, 0.874, 0.876)] == [0, 0, 1, 1, 2, 2, 3]
    assert [R.sample(z, u, top_p=0.6)[0] for u in (0.0, 0.3, 0.34, 0.99)] == [1, 1, 2, 2]
    assert R.sample(z, 0.99, top_k=3)[0] == 2 and R.sample(z, 0.0, min_p=0.5)[0] == 1
