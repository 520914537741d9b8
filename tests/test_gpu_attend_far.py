"""Scores of any size: what counts is how far apart they are."""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("score", [1e5, 2.0 ** 24, 1e8, 1e10, 1.5e12, 1e20])
@pytest.mark.parametrize("queries,memory,D", [(3, 700, 8), (300, 90, 24), (200, 1000, 64)])
def test_a_row_far_above_the_others_is_taken_alone(queries, memory, D, score, dtype):
    """Scores are -1.7 score but for one row's, a third of it, at a place that moves with the query: its value is the answer, and no
    score has a gradient."""
    import diff_surfel_tracing as dst
    for sign in (1.0, -1.0):
        g = torch.Generator(device="cuda").manual_seed(0)
        q = torch.zeros(1, queries, 2, D, device="cuda", dtype=dtype)
        k = torch.zeros(1, memory, 2, D, device="cuda", dtype=dtype)
        at = torch.randint(0, memory, (4,), generator=g, device="cuda")
        which = torch.arange(queries, device="cuda") % 4
        # query: +1 at its own one of four channels; memory: `sign` everywhere, less (or more) at the row of a channel
        q[0, torch.arange(queries, device="cuda"), :, which] = 1.0
        k[0, :, :, :4] = -1.7 if sign > 0 else 0.55   # (not a power of two: a product with the scale rounds)
        for c in range(4):
            k[0, at[c], :, c] = -0.55 if sign > 0 else 1.7
        v = torch.randn(1, memory, 2, 16, generator=g, device="cuda").to(dtype)
        up = torch.randn(1, queries, 2, 16, generator=g, device="cuda").to(dtype)
        want = v[0, at[which]][None]
        assert torch.equal(dst.attend_memory(q, k, v, scale=score), want)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = dst.attend_memory(*leaves, scale=score)
        assert torch.equal(out.detach(), want)
        dq, dk, dv = torch.autograd.grad(out, leaves, up)
        assert (dq == 0).all() and (dk == 0).all()
        ref = torch.zeros(1, memory, 2, 16, dtype=torch.float64, device="cuda").index_add_(1, at[which], up.double())
        size = torch.zeros_like(ref).index_add_(1, at[which], up.double().abs())
        R.check(dv, (ref, (queries / 16 + 8) * R.U * size + (R.HALF[dtype] + 2 * R.U) * ref.abs()), "dv")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_equal_scores_of_any_size(dtype):
    import diff_surfel_tracing as dst
    for score in (1e3, 3e4, 1e7, 1.7e9, 1e10, 1e20):
        for sign in (1.0, -1.0):
            q, k = torch.ones(1, 200, 1, 8, device="cuda", dtype=dtype), torch.zeros(1, 64, 1, 8, device="cuda", dtype=dtype)
            k[..., 0] = 1.7 * sign
            v = torch.randn(1, 64, 1, 8, device="cuda").to(dtype)
            out = dst.attend_memory(q, k, v, scale=score)
            ref = v.double().mean(1, keepdim=True).expand(1, 200, 1, 8)
            bound = (R.HALF[dtype] * 2 + 64 * R.U) * (ref.abs() + v.double().abs().mean())
            R.check(out, (ref, bound), "out")
