"""Attention of binary16 rows in which one weight leaves the others a long, thin tail."""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu
# The weights that the second product takes in binary16 start at 2^7: what their fixed steps below 2^-14 round away is at most
# 2^-25 2^-7 of the largest weight, a row of the memory.
STEP = 2.0 ** -32


def _thin_tail(queries, memory, weight, dtype, heads=1):
    """One row of the memory whose score lies -log2(weight) above all others', which are equal; its value is 0, theirs 1 or so."""
    q = torch.ones(1, queries, heads, 8, device="cuda", dtype=dtype)
    k = torch.zeros(1, memory, 1, 8, device="cuda", dtype=dtype)
    k[0, 1, 0, 0] = 16.0
    scale = float(-torch.log(torch.tensor(weight, dtype=torch.float64)) / 16.0)
    g = torch.Generator(device="cuda").manual_seed(1)
    v = (1.0 + torch.rand(1, memory, 1, 16, generator=g, device="cuda")).to(dtype)
    v[0, 1] = 0.0
    return q, k, v, scale


@pytest.mark.parametrize("weight", [2.0 ** -15.5, 2.0 ** -20.5, 2.0 ** -25.5, 2.0 ** -27.5])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("queries,memory", [(70000, 4096), (70000, 100), (3, 40000)])
def test_a_thin_tail_is_not_dropped(queries, memory, weight, grad):
    import diff_surfel_tracing as dst
    q, k, v, scale = _thin_tail(queries, memory, weight, torch.float16)
    # (the scale is rounded to 32 bits, once as it is and once by log2 e: the weights by 3 U of their logarithm)
    p = float(torch.exp(torch.tensor(-16.0, dtype=torch.float64) * torch.tensor(scale, dtype=torch.float32).double()))
    tail = v[0, :, 0].double().sum(0)
    true = p * tail / (1 + (memory - 1) * p)
    rel = 3 * R.U * 20 + (memory / 32 + 16) * R.U
    bound = STEP * tail + (R.HALF[torch.float16] + rel) * true * 2 + R.TINY[torch.float16]
    with torch.set_grad_enabled(grad):
        out = dst.attend_memory(q.requires_grad_(grad), k, v, scale=scale).detach()
    R.check(out[0, :, 0], (true.expand(queries, 16), bound.expand(queries, 16)), "out")
    assert float((out.double() - true).abs().max()) < 0.25 * float(true.max())


def test_gradients_of_a_thin_tail():
    """delta is formed of out: where out drops the tail, every score's gradient is off by what it dropped."""
    import diff_surfel_tracing as dst
    q, k, v, scale = _thin_tail(4096, 4096, 2.0 ** -24.5, torch.float16)
    up = torch.full((1, 4096, 1, 16), 64.0, device="cuda", dtype=torch.float16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = dst.attend_memory(*leaves, scale=scale)
    got = torch.autograd.grad(out, leaves, up)
    K, V = k.detach()[0, :, 0].double(), v.detach()[0, :, 0].double()
    Q, dO = q.detach()[0, :1, 0].double(), up[0, :1, 0].double()
    p = torch.softmax(scale * (Q @ K.T), 1)
    ds = scale * p * (dO @ V.T - (dO @ (p @ V).T))
    dq = ds @ K
    # (out's tail is off by the steps above, and twice by half a step of binary16 of its rounded rest: 2^-22 of it)
    off = scale * float((dO.abs() @ V.sum(0)[:, None]).max()) * STEP * 16.0
    assert float((got[0][0, :, 0].double() - dq).abs().max()) <= off + (R.HALF[torch.float16] + 2.0 ** -11) * float(dq.abs().max()) + R.TINY[torch.float16]


def test_the_lift_cancels():
    """Weights up to 2^8 above the running maximum, a lift of 2^7, values near binary16's largest: nothing overflows."""
    import diff_surfel_tracing as dst
    for memory in (64, 500, 5000):
        q = torch.ones(1, 300, 2, 8, device="cuda", dtype=torch.float16)
        # scores that rise by almost 8 in units of log 2 from one block to the next
        k = torch.zeros(1, memory, 2, 8, device="cuda", dtype=torch.float16)
        k[0, :, :, 0] = (torch.arange(memory, device="cuda") // 32 * 5.5)[:, None].half()
        g = torch.Generator(device="cuda").manual_seed(3)
        v = (60000 * (2 * torch.rand(1, memory, 2, 8, generator=g, device="cuda") - 1)).half()
        ref = R.attend(q, k, v, scale=1.0)["out"]
        R.check(dst.attend_memory(q, k, v, scale=1.0), ref, "out")
        R.check(dst.attend_memory(q.requires_grad_(True), k, v, scale=1.0).detach(), ref, "out, gradients wanted")
        one = dst.attend_memory(q, k[:, :1], v[:, :1], scale=1.0)
        assert torch.equal(one, v[:, :1].expand(1, 300, 2, 8))
