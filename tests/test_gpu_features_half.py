"""binary16 where it has a way of its own: reduced losses (their gradients are formed in 32 bits and rounded once), lengths, and small
gradients."""
import pytest
import torch

import features_reference as R
from test_gpu_attend import _check, _grads as _attend_grads, _inputs as _attend_inputs
from test_gpu_labels import _grads, _inputs

pytestmark = pytest.mark.gpu
HALF = torch.float16


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("N,D,V", [(1, 8, 2), (130, 17, 65), (2049, 8, 256), (5000, 40, 33), (300, 16, 90), (70, 256, 700)])
def test_reduced_loss(N, D, V, reduction):
    x, w, b, t, _ = _inputs(N, D, V, HALF)
    t[0] = V - 1
    got = _grads(x, w, t, b, torch.tensor(1.7, device="cuda"), reduction=reduction)
    n = int((t != -100).sum()) if reduction == "mean" else 1
    ref = R.labels(x, w, t, b, torch.full((N,), 1.7 / n, device="cuda", dtype=torch.float64))
    value, bound = ref["loss"]
    R.check(got[0], (value.sum() / n, bound.sum() / n + R.U * value.sum().abs() / n), "loss")
    for v, name in zip(got[1:], ("dx", "dw", "db")):
        value, bound = ref[name]
        R.check(v, (value, bound * (1 + 4 * R.U) + 4 * R.U * value.abs()), name)
    assert got[1].dtype == HALF and got[2].dtype == HALF


def test_small_gradients_are_rounded_once():
    """Upstream gradients of 1e-6: what binary16 cannot hold is lost when the sum is written, not in its terms."""
    x, w, b, t, up = _inputs(4000, 40, 90, HALF)
    up = 1e-6 * (up + 1.0)
    got, ref = _grads(x, w, t, b, up, reduction="none"), R.labels(x, w, t, b, up)
    for v, name in zip(got[2:], ("dw", "db")):
        R.check(v, ref[name], name)
    assert float(got[2].double().abs().max()) > 0


@pytest.mark.parametrize("size", [(7, 33, 200, 4, 2, 48, 48), (7, 3, 900, 8, 2, 128, 100), (7, 700, 70, 2, 2, 20, 8)])
def test_lengths(size):
    q, k, v, up = _attend_inputs(*size, HALF)
    n = size[2]
    lengths = [n, 0, 1, 64, 65, n - 1, 16]
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = _attend_grads(q, k, v, up, ln)
    _check(want, R.attend(q, k, v, lengths, up=up))
    assert (want[0][1] == 0).all() and all((g[1] == 0).all() for g in want[1:])
    for i, m in enumerate(lengths):
        assert (want[2][i, m:] == 0).all() and (want[3][i, m:] == 0).all()
    kk, vv = k.clone(), v.clone()
    for i, m in enumerate(lengths):
        kk[i, m:], vv[i, m:] = float("nan"), float("inf")
    for p, r in zip(want, _attend_grads(q, kk, vv, up, ln)):
        assert torch.equal(p, r)


def test_one_memory_row_gives_its_value_and_no_gradient_of_scores():
    q, k, v, up = _attend_inputs(2, 50, 1, 4, 2, 64, 64, HALF)
    out, dq, dk, dv = _attend_grads(q, k, v, up)
    assert torch.equal(out, v.repeat_interleave(2, 2).expand(2, 50, 4, 64))
    assert (dq == 0).all() and (dk == 0).all()


def test_a_table_without_channels_is_the_biases():
    import diff_surfel_tracing as dst
    x, w = torch.zeros(70, 24, device="cuda", dtype=HALF), torch.zeros(90, 24, device="cuda", dtype=HALF)
    b = torch.linspace(-3, 3, 90, device="cuda")
    label, log_prob = dst.label_rays(x, w, b)
    true = b.double()[-1] - torch.logsumexp(b.double(), 0)
    assert (label == 89).all() and float((log_prob.double() - true).abs().max()) <= 40 * R.U
