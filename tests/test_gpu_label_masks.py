"""Labels masked by large negative biases of any size, so many that a lane, a tile or a part of the table has none but such."""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu
LOWS = [-1e9, -1e10, -3e10, -1e20, -1e30, -2e38, torch.finfo(torch.float32).min, float("-inf")]


def _inputs(N, D, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, D, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") * (4.0 / D ** 0.5)).to(dtype)
    b = 0.5 * torch.randn(V, generator=g, device="cuda")
    return x, w, b, torch.rand(N, generator=g, device="cuda") - 0.3, g


@pytest.mark.parametrize("low", LOWS)
@pytest.mark.parametrize("N,D,V,dtype", [(70, 8, 150, torch.float32), (300, 40, 700, torch.float32), (3, 24, 9000, torch.float32),
                                         (200, 64, 300, torch.bfloat16), (3, 16, 9000, torch.float16), (70000, 8, 130, torch.float32)], ids=str)
def test_whole_stretches_of_masked_labels(N, D, V, dtype, low):
    import diff_surfel_tracing as dst
    for there in (slice(V - 5, V), slice(0, 5), slice(V // 2, V // 2 + 40)):
        x, w, b, up, g = _inputs(N, D, V, dtype)
        kept = torch.zeros(V, dtype=torch.bool, device="cuda")
        kept[there] = True
        b[~kept] = low
        index = kept.nonzero()[:, 0]
        at = torch.randint(0, len(index), (N,), generator=g, device="cuda")
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        loss = dst.label_loss(leaves[0], leaves[1], index[at], leaves[2], reduction="none")
        dx, dw, db = torch.autograd.grad(loss, leaves, up)
        ref = R.labels(x, w[kept], at, b[kept], up)
        for got, name in ((loss.detach(), "loss"), (dx, "dx"), (dw[kept], "dw"), (db[kept], "db")):
            R.check(got, ref[name], name)
        assert (dw[~kept] == 0).all() and (db[~kept] == 0).all()
        label, log_prob = dst.label_rays(x, w, b)
        s = x.double() @ w[kept].double().T + b[kept].double()
        best = torch.where(s == s.amax(1, keepdim=True), index, V).amin(1)
        assert torch.equal(label, best)
        bound = R.labels(x, w[kept], torch.zeros(N, dtype=torch.int64, device="cuda"), b[kept])["loss"][1]
        R.check(log_prob, (s.amax(1) - torch.logsumexp(s, 1), bound), "log_prob")


@pytest.mark.parametrize("low", [v for v in LOWS if v != float("-inf")] + [1e9, 1e20, 2e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_every_label_masked_alike_is_no_mask(low, dtype):
    """All logits the same number, however large: all labels have the same weight."""
    import diff_surfel_tracing as dst
    for N, D, V in ((70, 8, 150), (3, 24, 9000), (300, 40, 90)):
        x, w = torch.zeros(N, D, device="cuda", dtype=dtype), torch.randn(V, D, device="cuda").to(dtype)
        b = torch.full((V,), low, device="cuda")
        t = torch.arange(N, device="cuda") % V
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        loss = dst.label_loss(leaves[0], leaves[1], t, leaves[2], reduction="none")
        dx, dw, db = torch.autograd.grad(loss.sum(), leaves)
        ref = R.labels(x, w, t, torch.zeros_like(b), torch.ones(N, device="cuda"))   # (what all logits have in common has no say)
        for got, name in ((loss.detach(), "loss"), (dx, "dx"), (dw, "dw"), (db, "db")):
            R.check(got, ref[name], name)
        label, log_prob = dst.label_rays(x, w, b)
        assert (label == 0).all()
        assert float((log_prob.double() + torch.log(torch.tensor(float(V), dtype=torch.float64))).abs().max()) <= (V / 32 + 16) * R.U


def test_a_masked_label_as_target():
    import diff_surfel_tracing as dst
    for low in (-1e10, -1e20, -2e38, torch.finfo(torch.float32).min):
        x, w = torch.ones(5, 24, device="cuda"), torch.zeros(40, 24, device="cuda")
        b = torch.zeros(40, device="cuda")
        b[3] = low
        t = torch.full((5,), 3, device="cuda")
        loss = dst.label_loss(x, w, t, b, reduction="none")
        assert float((loss.double() + torch.tensor(low, dtype=torch.float32).double().cuda()).abs().max()) <= abs(low) * 4 * R.U
