"""attend_memory against its formulas in 64 bits, at the sizes, lengths and layouts where such kernels go wrong."""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu

#        B, Lq, Lk, H, Hkv, D, Dv
SIZES = [(1, 1, 1, 1, 1, 8, 8), (1, 1, 5000, 8, 8, 128, 128), (2, 3, 700, 4, 2, 64, 64), (1, 65, 63, 1, 1, 16, 16),
         (3, 17, 130, 6, 2, 40, 24), (1, 300, 33, 2, 2, 32, 32), (1, 130, 257, 2, 1, 256, 256), (2, 70, 64, 1, 1, 100, 7),
         (1, 2, 65, 3, 1, 1, 1), (1, 9, 70, 16, 1, 32, 32), (1, 5, 40, 32, 1, 130, 64), (2, 21, 90, 8, 2, 8, 4), (1, 600, 600, 1, 1, 16, 8),
        (1, 1000, 20, 1, 1, 3, 5), (1, 40, 2100, 2, 2, 96, 128)]


def _inputs(B, Lq, Lk, H, Hkv, D, Dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(B, Lq, H, D), r(B, Lk, Hkv, D), r(B, Lk, Hkv, Dv), r(B, Lq, H, Dv)


def _grads(q, k, v, up, lengths=None, **more):
    import diff_surfel_tracing as dst
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = dst.attend_memory(*leaves, lengths, **more)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, up))


def _check(got, ref):
    for value, name in zip(got, ("out", "dq", "dk", "dv")):
        R.check(value, ref[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(size, dtype):
    import diff_surfel_tracing as dst
    q, k, v, up = _inputs(*size, dtype)
    for lengths in [None] + ([[0, 1, 7][:size[0]]] if size[0] > 1 else []):
        ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
        ref = R.attend(q, k, v, lengths, up=up)
        R.check(dst.attend_memory(q, k, v, ln), ref["out"], "out, no gradients wanted")
        got = _grads(q, k, v, up, ln)
        assert all(t.dtype == dtype for t in got)
        _check(got, ref)


def test_lengths():
    import diff_surfel_tracing as dst
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, up = _inputs(7, 33, 200, 4, 2, 48, 48, dtype)
        lengths = [200, 0, 1, 64, 65, 127, 16]
        ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want = _grads(q, k, v, up, ln)
        _check(want, R.attend(q, k, v, lengths, up=up))
        assert (want[0][1] == 0).all() and all((g[1] == 0).all() for g in want[1:])
        # what lies behind a length may hold anything
        kk, vv = k.clone(), v.clone()
        for i, n in enumerate(lengths):
            kk[i, n:], vv[i, n:] = float("nan"), float("inf")
        for p, r in zip(want, _grads(q, kk, vv, up, ln)):
            assert torch.equal(p, r)
        # clamped, and of other whole types
        far = torch.tensor([2 ** 40, -5, 1, 64, 65, 127, 16], device="cuda")
        for p, r in zip(want, _grads(q, k, v, up, far)):
            assert torch.equal(p, r)
        assert torch.equal(dst.attend_memory(q, k, v, ln.clamp(max=127).to(torch.int8)), dst.attend_memory(q, k, v, ln.clamp(max=127)))


def test_no_queries_no_memory_no_batch():
    import diff_surfel_tracing as dst
    for B, Lq, Lk in ((1, 5, 0), (2, 0, 9), (0, 4, 6), (1, 0, 0)):
        q, k, v, up = _inputs(B, Lq, Lk, 2, 2, 16, 16, torch.float32)
        out, dq, dk, dv = _grads(q, k, v, up)
        assert out.shape == (B, Lq, 2, 16) and (out == 0).all() and (dq == 0).all() and (dk == 0).all() and (dv == 0).all()
        assert dst.attend_memory(q, k, v).shape == out.shape


def test_one_memory_row_gives_its_value_and_no_gradient_of_scores():
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, up = _inputs(2, 50, 1, 4, 2, 64, 64, dtype)
        out, dq, dk, dv = _grads(q, k, v, up)
        assert torch.equal(out, v.repeat_interleave(2, 2).expand(2, 50, 4, 64))
        assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-3])
def test_scales(scale):
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, up = _inputs(2, 70, 90, 2, 1, 24, 24, dtype)
        _check(_grads(q, k, v, up, scale=scale), R.attend(q, k, v, None, scale, up))


def test_far_scores_and_peaked_weights():
    for factor in (30.0, 300.0):
        q, k, v, up = _inputs(1, 100, 333, 2, 2, 32, 32, torch.float32)
        _check(_grads(factor * q, k, v, up), R.attend(factor * q, k, v, up=up))
    # scores that rise along the memory: the running maximum moves with every tile
    q, k, v, up = _inputs(1, 100, 500, 1, 1, 32, 32, torch.bfloat16)
    k = k + torch.linspace(0, 40, 500, device="cuda")[None, :, None, None].to(k.dtype) * q.mean(1, keepdim=True).sign()
    _check(_grads(q, k, v, up), R.attend(q, k, v, up=up))


def test_strides_and_broadcasts():
    import diff_surfel_tracing as dst
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, up = _inputs(2, 40, 90, 4, 2, 24, 20, dtype)
        want = _grads(q, k, v, up)
        ref = R.attend(q, k, v, up=up)
        packed = torch.full((2, 90, 2, 51), float("nan"), device="cuda", dtype=dtype)
        packed[..., 3:27], packed[..., 27:47] = k, v
        by_head = q.transpose(1, 2).contiguous().transpose(1, 2)
        for args in ((by_head, k, v), (q, packed[..., 3:27], packed[..., 27:47]),
                     (q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0), k, v)):
            _check(_grads(*args, up), ref)
        _check(_grads(q, k, v, up.transpose(1, 2).contiguous().transpose(1, 2)), ref)
        assert all(torch.equal(a, b) for a, b in zip(want, _grads(by_head, k, v, up)))
        # one memory for all batches: its gradient is the sum over them
        one_k, one_v = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
        out = dst.attend_memory(q, one_k.expand(2, -1, -1, -1), one_v.expand(2, -1, -1, -1))
        ref = R.attend(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), up=up)
        R.check(out.detach(), ref["out"], "out")
        for got, name in zip(torch.autograd.grad(out, [one_k, one_v], up), ("dk", "dv")):
            value, bound = ref[name]
            half = R.HALF[dtype] or R.U
            R.check(got, (value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + half * value.sum(0, keepdim=True).abs()), name)
        # keys and values the same tensor
        both = k.clone().requires_grad_(True)
        out = dst.attend_memory(q, both, both)
        ref = R.attend(q, k, k, up=torch.ones_like(out))
        got, = torch.autograd.grad(out, both, torch.ones_like(out))
        R.check(got, (ref["dk"][0] + ref["dv"][0], ref["dk"][1] + ref["dv"][1] + (R.HALF[dtype] or R.U) * (ref["dk"][0] + ref["dv"][0]).abs()), "both")


def test_gradients_that_are_not_asked_for():
    import diff_surfel_tracing as dst
    q, k, v, up = _inputs(2, 100, 300, 2, 2, 32, 32, torch.float32)
    want = _grads(q, k, v, up)
    for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
        args = [t.clone().requires_grad_(i in pick) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(dst.attend_memory(*args), [args[i] for i in pick], up)
        for i, g in zip(pick, got):
            assert torch.equal(g, want[1 + i])


def test_gradient_agrees_with_differences():
    import diff_surfel_tracing as dst
    q, k, v, up = _inputs(1, 30, 50, 2, 1, 12, 12, torch.float32)
    grads = _grads(q, k, v, up)
    g = torch.Generator(device="cuda").manual_seed(7)
    for i in range(3):
        args = [q, k, v]
        d = torch.randn(args[i].shape, generator=g, device="cuda")
        d /= d.norm()
        h = 2.0 ** -4

        def at(step):
            moved = list(args)
            moved[i] = args[i] + step * d
            return (dst.attend_memory(*moved).double() * up.double()).sum()
        slope = float((at(h) - at(-h)) / (2 * h))
        mine = float((grads[1 + i].double() * d.double()).sum())
        # 720 outputs, each off by 2^-19 at most (fp32, values below 4) and weighted by N(0,1): their sum is off by less than
        # sqrt(720) * 4 * 2^-19 as random errors; third derivatives along a unit direction: below 6 |up| |v| (|row| / sqrt(12))^3,
        # with rows of norm below 6 about 6 * 30 * 5.2, times h^2 / 6, of which a unit direction over all rows moves a small part
        assert abs(slope - mine) <= 27 * 4 * 2.0 ** -19 / h + 30 * 5.2 * h * h


def test_deterministic():
    q, k, v, up = _inputs(2, 500, 700, 4, 2, 64, 64, torch.bfloat16)
    first = _grads(q, k, v, up)
    for _ in range(3):
        for a, b in zip(first, _grads(q, k, v, up)):
            assert torch.equal(a, b)


def test_graph_replays_with_eager_work_between():
    import diff_surfel_tracing as dst
    sets = [_inputs(2, 20, 900, 4, 2, 64, 64, torch.bfloat16, seed=s) for s in range(3)]
    lens = [torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([900, 3], [0, 899], [64, 65])]
    want = [_grads(*s, n) for s, n in zip(sets, lens)]
    q, k, v, up = (t.clone() for t in sets[0])
    ln = lens[0].clone()
    for t in (q, k, v):
        t.requires_grad_(True)

    def step():
        out = dst.attend_memory(q, k, v, ln)
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v], up))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            for to, src in zip((q, k, v, up, ln), sets[i] + (lens[i],)):
                to.copy_(src)
        graph.replay()
        eager = _grads(*sets[i], lens[i])
        torch.cuda.synchronize()
        for a, b, c in zip(want[i], out, eager):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_side_streams_and_overlapping_calls():
    sets = [_inputs(1, 200, 3000, 2, 2, 64, 64, torch.bfloat16, seed=s) for s in range(3)]
    want = [_grads(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(_grads(*s))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_a_row_far_into_a_large_memory():
    """Offsets beyond 32 bits: the last batch of a strided memory starts 5 * 2^30 values into its storage."""
    import diff_surfel_tracing as dst
    big = torch.zeros(5 * 2 ** 30 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    k = big.as_strided((2, 100, 1, 64), (5 * 2 ** 30, 64, 64, 1))
    v = big.as_strided((2, 100, 1, 64), (5 * 2 ** 30, 64, 64, 1), 100 * 64)
    q, kk, vv, _ = _inputs(2, 9, 100, 1, 1, 64, 64, torch.bfloat16)
    k.copy_(kk), v.copy_(vv)
    R.check(dst.attend_memory(q, k, v), R.attend(q, kk, vv)["out"], "out")


def test_rows_far_apart_in_memory():
    import diff_surfel_tracing as dst
    pitch = 2 ** 24
    big = torch.empty(100 * pitch + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    q, kk, vv, up = _inputs(1, 9, 100, 2, 2, 64, 64, torch.bfloat16)
    k = big.as_strided((1, 100, 2, 64), (0, pitch, 2 ** 12, 1))
    v = big.as_strided((1, 100, 2, 64), (0, pitch, 2 ** 12, 1), 2 ** 10)
    k.copy_(kk), v.copy_(vv)
    for a, b in zip(_grads(q, k, v, up), _grads(q, kk, vv, up)):
        assert torch.equal(a, b)


def test_many_own_tiles_and_a_rest_that_is_cut():
    """512 own tiles of 128 rows, two rounds or one of the device's places, and one more, against enough rows that cutting it pays: queries for
    the forward kernel and that of dq, memory for that of dk and dv."""
    for size in ((1, 128 * 513, 1500, 1, 1, 64, 64), (1, 1500, 128 * 513, 1, 1, 64, 64)):
        q, k, v, up = _inputs(*size, torch.bfloat16)
        _check(_grads(q, k, v, up), R.attend(q, k, v, up=up))


def test_a_graph_walked_twice():
    import diff_surfel_tracing as dst
    q, k, v, up = (t.requires_grad_(True) for t in _inputs(1, 70, 90, 2, 1, 40, 40, torch.bfloat16))
    out = dst.attend_memory(q, k, v)
    first = torch.autograd.grad(out, [q, k, v], up.detach(), retain_graph=True)
    second = torch.autograd.grad(out, [q, k, v], up.detach())
    assert all(torch.equal(a, b) for a, b in zip(first, second))
