"""Rays that are all but sure of their label: the loss and its gradients keep digits of 1 - p, not of the logits.

Bounds. With R = sum over the other labels of exp(s_v - s_t): loss = log(1 + R), 1 - p_t = R / (1 + R). What is wrong in a logit
enters R by a factor (`rel`). What is rounded near 1 enters as it is: the label's own exponential (U: one unit in the last place), three
additions of it in pairs (U/2 each), the compensated running sum (U), its end (U/2), two of the four lanes' (U/2 each), that of the parts
(U/2): 5.5 U of the sum, times ln 2 below 4 U in the loss. 6 U are taken, U = 2^-23.
"""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu
U, NEAR_ONE = R.U, 6.0

#        rays, channels, labels, dtype
SIZES = [(257, 8, 150, torch.float32), (70000, 8, 200, torch.float32), (200, 16, 333, torch.float32), (300, 64, 4096, torch.float32),
         (3, 64, 20000, torch.float32), (100, 256, 5001, torch.bfloat16), (4000, 24, 90, torch.bfloat16), (100, 40, 700, torch.float16)]


def _sure_rays(N, D, V, dtype, shift=0.0, seed=0):
    """Rays along the row of their own label, as long as makes R what it is drawn as: 1e-6 to 1e-2."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, D, generator=g, device="cuda")
    w = (w / w.norm(dim=1, keepdim=True) * D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    along = w[t].double() / (w[t].double() ** 2).sum(1, keepdim=True)
    gap = (along @ w.double().T) - 1.0
    gap.scatter_(1, t[:, None], -float("inf"))
    want = 10.0 ** (-2.0 - 4.0 * torch.rand(N, generator=g, device="cuda").double())
    lo, hi = torch.zeros_like(want), torch.full_like(want, 1e5)
    for _ in range(60):
        mid = 0.5 * (lo + hi)
        more = (mid[:, None] * gap).exp().sum(1) > want
        lo, hi = torch.where(more, mid, lo), torch.where(more, hi, mid)
    x = (hi.clamp(max=3e4)[:, None] * along).to(dtype)
    b = torch.full((V,), shift, device="cuda") + 0.01 * torch.randn(V, generator=g, device="cuda")
    up = torch.rand(N, generator=g, device="cuda") + 0.5
    return x, w, b, t, up


def _reference(x, w, b, t, up):
    half, tiny, N, D, V = R.HALF[x.dtype], R.TINY[x.dtype], x.size(0), x.size(1), w.size(0)
    x, w, b, g = x.double(), w.double(), b.double(), up.double()[:, None]
    s = x @ w.T + b
    s_t = s.gather(1, t[:, None])
    others = (s - s_t).exp().scatter_(1, t[:, None], 0.0)
    r = others.sum(1)
    loss, q = torch.log1p(r), r / (1 + r)
    size = (x.abs() @ w.abs().T + b.abs()).amax(1)
    rel = 2 * (D + 4) * U * size + 2 * U * (2 * s.abs().amax(1) + 2) + (V / 32 + 16) * U
    ds = g * (others / (1 + r[:, None])).scatter_(1, t[:, None], -q[:, None])
    e = g * ((ds.abs() / g) * rel[:, None]).scatter_add_(1, t[:, None], torch.full_like(s_t, NEAR_ONE * U))
    e16 = e + half * ds.abs()
    dx, dw, db = ds @ w, ds.T @ x, ds.sum(0)
    return dict(loss=(loss, q * rel + NEAR_ONE * U + U * loss),
                dx=(dx, e16 @ w.abs() + (V / 16 + 8) * U * (ds.abs() @ w.abs()) + (half + 2 * U) * dx.abs() + tiny),
                dw=(dw, e16.T @ x.abs() + (N / 16 + 8) * U * (ds.abs().T @ x.abs()) + (half + 2 * U) * dw.abs() + tiny),
                db=(db, e.sum(0) + (N + 8) * U * ds.abs().sum(0)))


def _check(x, w, b, t, up):
    import diff_surfel_tracing as dst
    ref = _reference(x, w, b, t, up)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    loss = dst.label_loss(leaves[0], leaves[1], t, leaves[2], reduction="none")
    assert float(loss.detach().min()) >= 0.0
    got = [loss.detach()] + list(torch.autograd.grad(loss, leaves, up))
    for value, name in zip(got, ("loss", "dx", "dw", "db")):
        R.check(value, ref[name], name)


@pytest.mark.parametrize("N,D,V,dtype", SIZES, ids=str)
def test_rays_sure_of_their_label(N, D, V, dtype):
    _check(*_sure_rays(N, D, V, dtype))


@pytest.mark.parametrize("N,D,V", [(257, 8, 150), (300, 64, 4096), (3, 64, 20000)])
def test_rays_sure_of_their_label_far_from_zero(N, D, V):
    """All logits about 1000: what they are does not matter, only how far apart."""
    for shift in (1000.0, -1000.0):
        _check(*_sure_rays(N, D, V, torch.float32, shift))


def test_a_long_tail_is_not_lost():
    """A label with 32,000 others of 1e-8 each behind it, in the order in which a running sum near 1 would lose them."""
    import diff_surfel_tracing as dst
    V = 32001
    b = torch.full((V,), -18.4, device="cuda")
    b[0] = 0.0
    x, w, t = torch.zeros(70, 8, device="cuda"), torch.zeros(V, 8, device="cuda"), torch.zeros(70, dtype=torch.int64, device="cuda")
    others = float((b[1:].double().exp()).sum())
    loss = dst.label_loss(x, w, t, b, reduction="none").double()
    true = torch.log1p(torch.tensor(others, dtype=torch.float64))
    # (a bias is exact; exponent and sum of the others: 30 U of them)
    assert float((loss - true).abs().max()) <= NEAR_ONE * U + others * 60 * U


def test_mean_of_sure_rays():
    import diff_surfel_tracing as dst
    x, w, b, t, _ = _sure_rays(3000, 16, 90, torch.float32)
    up = torch.full((3000,), 1.0 / 3000, device="cuda")
    ref = _reference(x, w, b, t, up)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    got = torch.autograd.grad(dst.label_loss(leaves[0], leaves[1], t, leaves[2]), leaves)
    for value, name in zip(got, ("dx", "dw", "db")):
        v, bound = ref[name]
        R.check(value, (v, bound * (1 + 4 * U) + 4 * U * v.abs()), name)


def test_a_label_masked_by_the_lowest_value_as_target():
    """Its loss is what its logit lacks, and its gradient that of a weight of 0; a ray whose labels are all switched off has no loss."""
    import diff_surfel_tracing as dst
    low = torch.finfo(torch.float32).min
    for dtype in (torch.float32, torch.bfloat16):
        x, w = torch.ones(5, 24, device="cuda", dtype=dtype), torch.zeros(40, 24, device="cuda", dtype=dtype)
        b = torch.zeros(40, device="cuda")
        b[3] = low
        t = torch.full((5,), 3, device="cuda")
        loss = dst.label_loss(x.requires_grad_(True), w, t, b, reduction="none")
        assert (loss == -low).all()
        dx, = torch.autograd.grad(loss.sum(), x)
        assert torch.isfinite(dx).all()
        b[3] = float("-inf")
        assert (dst.label_loss(x, w, t, b, reduction="none") == float("inf")).all()
        assert torch.isnan(dst.label_loss(x, w, t, torch.full((40,), float("-inf"), device="cuda"), reduction="none")).all()


@pytest.mark.parametrize("N,V", [(70, 40), (3, 20000), (70000, 333)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_best_label_where_every_label_is_masked(N, V, dtype):
    """No label has a probability: NaN, not the most certain of all."""
    import diff_surfel_tracing as dst
    for D in (8, 40):
        x, w = torch.ones(N, D, device="cuda", dtype=dtype), torch.ones(V, D, device="cuda", dtype=dtype)
        b = torch.full((V,), float("-inf"), device="cuda")
        label, log_prob = dst.label_rays(x, w, b)
        assert torch.isnan(log_prob).all() and (label >= 0).all() and (label < V).all()
        b[V // 2] = 0.0      # one that is not
        label, log_prob = dst.label_rays(x, w, b)
        assert (label == V // 2).all() and (log_prob == 0).all()


@pytest.mark.parametrize("N,D,V,dtype", SIZES, ids=str)
def test_best_label_of_sure_rays(N, D, V, dtype):
    import diff_surfel_tracing as dst
    for shift in (0.0, 1000.0):
        x, w, b, t, up = _sure_rays(N, D, V, dtype, shift)
        label, log_prob = dst.label_rays(x, w, b)
        loss, bound = _reference(x, w, b, t, up)["loss"]
        assert torch.equal(label, t) and float(log_prob.max()) <= 0.0
        R.check(log_prob, (-loss, bound), "log_prob")


def test_a_long_tail_behind_the_best_label_is_not_lost():
    import diff_surfel_tracing as dst
    V = 32001
    b = torch.full((V,), -18.4, device="cuda")
    b[0] = 0.0
    label, log_prob = dst.label_rays(torch.zeros(70, 8, device="cuda"), torch.zeros(V, 8, device="cuda"), b)
    others = float((b[1:].double().exp()).sum())
    true = -torch.log1p(torch.tensor(others, dtype=torch.float64))
    assert (label == 0).all()
    assert float((log_prob.double() - true).abs().max()) <= NEAR_ONE * U + others * 60 * U
