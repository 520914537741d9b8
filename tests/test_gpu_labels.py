"""label_loss and label_rays against their formulas in 64 bits, at the sizes and inputs where such kernels go wrong."""
import pytest
import torch

import features_reference as R

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (1, 8, 2), (5, 3, 7), (64, 8, 150), (65, 16, 64), (130, 17, 65), (200, 64, 1000), (33, 100, 333),
         (70, 256, 129), (2049, 8, 256), (3, 256, 5001), (300, 33, 1), (257, 128, 63)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(N, D, V, dtype, bias=True, seed=0, spread=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, D, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") * (spread / D ** 0.5)).to(dtype)
    b = 0.5 * torch.randn(V, generator=g, device="cuda") if bias else None
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[torch.rand(N, generator=g, device="cuda") < 0.2] = -100
    up = torch.rand(N, generator=g, device="cuda") - 0.3
    return x, w, b, t, up


def _grads(x, w, t, b, up, **more):
    import diff_surfel_tracing as dst
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b) if v is not None]
    out = dst.label_loss(leaves[0], leaves[1], t, leaves[2] if b is not None else None, **more)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, up))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_loss_of_every_ray_and_its_gradients(N, D, V, dtype):
    for bias in (False, True):
        x, w, b, t, up = _inputs(N, D, V, dtype, bias)
        got = _grads(x, w, t, b, up, reduction="none")
        ref = R.labels(x, w, t, b, up)
        assert got[0].dtype == torch.float32 and got[1].dtype == dtype and got[2].dtype == dtype
        for value, name in zip(got, ("loss", "dx", "dw", "db")):
            R.check(value, ref[name], name)
        assert (got[1][t == -100] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("N,D,V", [(1, 8, 2), (130, 17, 65), (2049, 8, 256), (5000, 40, 33)])
def test_reduced_loss(N, D, V, dtype, reduction):
    x, w, b, t, _ = _inputs(N, D, V, dtype)
    t[0] = V - 1
    up = torch.tensor(1.7, device="cuda")
    got = _grads(x, w, t, b, up, reduction=reduction)
    per_ray = 1.7 / float((t != -100).sum()) if reduction == "mean" else 1.7
    ref = R.labels(x, w, t, b, torch.full((N,), per_ray, device="cuda", dtype=torch.float64))
    value, bound = ref["loss"]
    n = (t != -100).sum() if reduction == "mean" else 1
    # (the sum over rays is in 64 bits, rounded once)
    R.check(got[0], (value.sum() / n, bound.sum() / n + R.U * value.sum().abs() / n), "loss")
    for v, name in zip(got[1:], ("dx", "dw", "db")):
        value, bound = ref[name]   # (1 / n and its product with the upstream gradient are rounded once each)
        R.check(v, (value, bound * (1 + 4 * R.U) + 4 * R.U * value.abs()), name)


def test_loss_is_deterministic():
    x, w, b, t, up = _inputs(3000, 24, 700, torch.float32)
    first = _grads(x, w, t, b, up, reduction="none")
    for _ in range(3):
        for p, q in zip(first, _grads(x, w, t, b, up, reduction="none")):
            assert torch.equal(p, q)


def test_nothing_counted():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(77, 8, 30, torch.float32)
    t.fill_(-100)
    x[3] = float("nan")
    x[4] = float("inf")
    out = _grads(x, w, t, b, up, reduction="none")
    assert all((o == 0).all() for o in out)
    out = _grads(x, w, t, b, torch.tensor(1.0, device="cuda"), reduction="sum")
    assert all((o == 0).all() for o in out)
    assert torch.isnan(dst.label_loss(x, w, t, b))                 # the mean of nothing, as torch's
    # no rays at all
    e = torch.empty(0, 8, device="cuda")
    t0 = torch.empty(0, dtype=torch.int64, device="cuda")
    out = _grads(e, w, t0, b, torch.empty(0, device="cuda"), reduction="none")
    assert out[0].shape == (0,) and out[1].shape == (0, 8) and (out[2] == 0).all() and (out[3] == 0).all()
    assert float(dst.label_loss(e, w, t0, b, reduction="sum")) == 0.0
    labels, logp = dst.label_rays(e, w, b)
    assert labels.shape == (0,) and logp.shape == (0,)


def test_ignored_rays_may_hold_anything():
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, t, up = _inputs(300, 20, 90, dtype)
        clean = _grads(x, w, t, b, up, reduction="none")
        dirty = x.clone()
        dirty[t == -100] = float("nan")
        dirty[(t == -100).nonzero()[0, 0]] = float("inf")
        for p, q in zip(clean, _grads(dirty, w, t, b, up, reduction="none")):
            assert torch.equal(p, q)
        other = torch.where(t == -100, 7, t)      # another number that stands for it
        keep = other != 7
        ref = R.labels(x, w, other, b, up, ignore=7)
        got = _grads(x, w, other, b, up, reduction="none", ignore_index=7)
        for v, name in zip(got, ("loss", "dx", "dw", "db")):
            R.check(v, ref[name], name)
        assert (got[0][~keep] == 0).all()


def test_a_label_that_is_none_is_not_passed_over():
    for bad in (-1, 90, 2 ** 40, -2 ** 62):
        x, w, b, t, up = _inputs(100, 20, 90, torch.float32)
        t[17] = bad
        loss, dx, dw, db = _grads(x, w, t, b, up, reduction="none")
        assert torch.isnan(loss[17]) and torch.isnan(dx[17]).all() and torch.isnan(dw).all() and torch.isnan(db).all()
        rest = torch.arange(100, device="cuda") != 17
        assert torch.isfinite(loss[rest]).all() and torch.isfinite(dx[rest]).all()


def test_labels_switched_off_and_far_logits():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(200, 16, 100, torch.float32)
    b[::3] = float("-inf")
    t = torch.where((t >= 0) & (t % 3 == 0), (t + 1) % 99, t)
    t = torch.where((t >= 0) & (t % 3 == 0), torch.ones_like(t), t)
    got, ref = _grads(x, w, t, b, up, reduction="none"), R.labels(x, w, t, b, up)
    for v, name in zip(got, ("loss", "dx", "dw", "db")):
        R.check(v, ref[name], name)
    labels, _ = dst.label_rays(x, w, b)
    assert (labels % 3 != 0).all()
    # logits of thousands, either sign: the running maximum carries them
    x, w, b, t, up = _inputs(200, 16, 100, torch.float32, spread=4000.0)
    got, ref = _grads(x, w, t, b, up, reduction="none"), R.labels(x, w, t, b, up)
    for v, name in zip(got, ("loss", "dx", "dw", "db")):
        R.check(v, ref[name], name)
    for shift in (-30000.0, 30000.0):   # all of them far from zero
        b = torch.full((100,), shift, device="cuda")
        x, w, _, t, up = _inputs(200, 16, 100, torch.float32)
        got, ref = _grads(x, w, t, b, up, reduction="none"), R.labels(x, w, t, b, up)
        for v, name in zip(got, ("loss", "dx", "dw", "db")):
            R.check(v, ref[name], name)


def test_strides_alignment_shapes_and_types_of_arguments():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(24 * 10, 12, 50, torch.float32)
    want = _grads(x, w, t, b, up, reduction="none")
    wide = torch.full((240, 31), float("nan"), device="cuda")
    wide[:, 5:17] = x                                            # rows at an odd pitch and offset
    tall = torch.full((50, 13), float("nan"), device="cuda")
    tall[:, 1:] = w
    for xx, ww in ((wide[:, 5:17], w), (x, tall[:, 1:]), (x.t().contiguous().t(), w.t().contiguous().t()),
                   (wide[:, 5:17].reshape(24, 10, 12), tall[:, 1:])):
        tt, uu = (t.reshape(24, 10), up.reshape(24, 10)) if xx.dim() == 3 else (t, up)
        got = _grads(xx, ww, tt, b, uu, reduction="none")
        for p, q in zip(want, got):
            assert torch.equal(p, q.reshape(p.shape))             # (however the rows are read, the same values)
    assert torch.equal(dst.label_loss(x, w, t.int(), b, reduction="none"), want[0])
    row = x[:1].expand(240, 12)                                  # broadcast rows
    assert torch.equal(dst.label_loss(row, w, t, b, reduction="none"), dst.label_loss(row.contiguous(), w, t, b, reduction="none"))
    loss = dst.label_loss(x, w, t, b.bfloat16().float(), reduction="none")
    xb, wb = x.bfloat16(), w.bfloat16()
    assert torch.equal(dst.label_loss(xb, wb, t, b.bfloat16()), dst.label_loss(xb, wb, t, b.bfloat16().float()))
    assert loss.shape == (240,)


def test_gradients_that_are_not_asked_for():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(500, 24, 300, torch.float32)
    want = _grads(x, w, t, b, up, reduction="none")
    for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
        args = [v.clone().requires_grad_(i in pick) for i, v in enumerate((x, w, b))]
        out = dst.label_loss(args[0], args[1], t, args[2], reduction="none")
        got = torch.autograd.grad(out, [args[i] for i in pick], up)
        for i, g in zip(pick, got):
            assert torch.equal(g, want[1 + i])
    with torch.no_grad():
        assert torch.equal(dst.label_loss(x.requires_grad_(True), w, t, b, reduction="none"), want[0])


def test_gradient_agrees_with_differences():
    import diff_surfel_tracing as dst
    x, w, b, t, _ = _inputs(60, 10, 40, torch.float32, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(5)
    for i, v in enumerate((x, w, b)):
        d = torch.randn(v.shape, generator=g, device="cuda")
        d /= d.norm()
        h = 2.0 ** -5
        args = [x, w, b]

        def at(step):
            args[i] = v + step * d
            return dst.label_loss(args[0], args[1], t, args[2], reduction="none").double().sum()
        slope = (at(h) - at(-h)) / (2 * h)
        grads = _grads(x, w, t, b, torch.ones(60, device="cuda"), reduction="none")
        mine = float((grads[1 + i].double() * d.double()).sum())
        # 60 losses below 8, each off by less than 2^-18 (fp32 sums of 40 exponentials), over 2 h; the third derivative of
        # a ray's loss along a unit direction is below 2 (3 max|row|)^3 ~ 2 * 5^3, times h^2 / 6 and 60 rays at most, of which a
        # direction of length one moves few: sum of the rows' cubes is below one
        assert abs(float(slope) - mine) <= 60 * 2.0 ** -18 / h + 2 * 125 * h * h / 6


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,D,V", SIZES + [(6000, 64, 2000)])
def test_best_label(N, D, V, dtype):
    import diff_surfel_tracing as dst
    for bias in (False, True):
        x, w, b, _, _ = _inputs(N, D, V, dtype, bias, seed=3)
        x[::7] = 0                                                # rays that met nothing
        label, logp = dst.label_rays(x, w, b)
        s = x.double() @ w.double().T + (0 if b is None else b.double())
        top = s.amax(1, keepdim=True)
        index = torch.arange(V, device="cuda").expand_as(s)
        assert label.dtype == torch.int64 and logp.dtype == torch.float32
        assert torch.equal(label, torch.where(s == top, index, V).amin(1))
        zero = torch.zeros(N, dtype=torch.int64, device="cuda")
        bound = R.labels(x, w, zero, b)["loss"][1]
        R.check(logp, (top[:, 0] - torch.logsumexp(s, 1), bound), "log_prob")


def test_best_label_of_equal_and_nearly_equal_ones():
    import diff_surfel_tracing as dst
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, _, _ = _inputs(500, 40, 300, dtype, False, seed=9)
        w = torch.cat([w, w, w])                                  # every label three times
        label, _ = dst.label_rays(x, w)
        s = x.double() @ w.double().T
        assert torch.equal(label, torch.where(s == s.amax(1, keepdim=True), torch.arange(900, device="cuda"), 900).amin(1))
        assert (label < 300).all()
    # two labels apart by one part in 2^23 of one channel: only the exact products tell them apart
    x = torch.ones(64, 33, device="cuda") * torch.linspace(0.5, 2.0, 64, device="cuda")[:, None]
    w = torch.rand(9, 33, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    w[5] = w[2] + 0.5
    w[2] = w[5]
    w[5, 7] = torch.nextafter(w[5, 7], torch.tensor(9.0, device="cuda"))
    label, _ = dst.label_rays(x, w)
    assert (label == 5).all()
    same, _ = dst.label_rays(torch.zeros(70, 33, device="cuda"), w)
    assert (same == 0).all()
    b = torch.zeros(9, device="cuda")
    b[4] = b[6] = 1.0
    same, logp = dst.label_rays(torch.zeros(70, 33, device="cuda"), w, b)
    assert (same == 4).all()


def test_graph_replays_with_eager_work_between():
    import diff_surfel_tracing as dst
    sets = [_inputs(700, 24, 500, torch.float32, seed=s) for s in range(3)]
    for s in sets:
        s[3][0] = 1
    want = [_grads(x, w, t, b, torch.tensor(1.0, device="cuda")) + list(dst.label_rays(x, w, b)) for x, w, b, t, _ in sets]
    x, w, b, t, _ = (v.clone() for v in sets[0])
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    one = torch.tensor(1.0, device="cuda")

    def step():
        out = dst.label_loss(x, w, t, b)
        return [out.detach()] + list(torch.autograd.grad(out, [x, w, b], one)) + list(dst.label_rays(x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in (1, 0, 2, 1):
        with torch.no_grad():
            for dst_t, src in zip((x, w, b, t), (sets[i][0], sets[i][1], sets[i][2], sets[i][3])):
                dst_t.copy_(src)
        graph.replay()
        eager = _grads(*(sets[i][k] for k in (0, 1, 3, 2)), torch.tensor(1.0, device="cuda"))   # between the replays
        torch.cuda.synchronize()
        for p, q in zip(want[i], out):
            assert torch.equal(p, q)
        for p, q in zip(want[i], eager):
            assert torch.equal(p, q)


def test_side_streams_and_overlapping_calls():
    sets = [_inputs(4000, 32, 900, torch.float32, seed=s) for s in range(3)]
    want = [_grads(x, w, t, b, up, reduction="none") for x, w, b, t, up in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for s, (x, w, b, t, up) in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append(_grads(x, w, t, b, up, reduction="none"))
    torch.cuda.synchronize()
    for p, q in zip(want, got):
        for u, v in zip(p, q):
            assert torch.equal(u, v)


def test_second_derivatives_are_refused():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(10, 4, 5, torch.float32)
    x.requires_grad_(True)
    g, = torch.autograd.grad(dst.label_loss(x, w, t, b, reduction="sum"), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("channels,dtype", [(8, torch.float32), (64, torch.float32), (64, torch.bfloat16), (64, torch.float16)])
def test_the_mean_of_nothing_has_no_gradient(channels, dtype):
    x, w, b, t, _ = _inputs(70, channels, 90, dtype)
    out = _grads(x, w, torch.full_like(t, -100), b, torch.tensor(1.0, device="cuda"))
    assert torch.isnan(out[0]) and all((o == 0).all() for o in out[1:])


def test_a_graph_walked_twice():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(300, 40, 70, torch.float32)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    out = dst.label_loss(x, w, t, b, reduction="none")
    first = torch.autograd.grad(out, leaves, up, retain_graph=True)
    second = torch.autograd.grad(out, leaves, up)
    assert all(torch.equal(a, c) for a, c in zip(first, second))
    t[0] = 3   # what the backward pass would need is no longer what the forward pass saw
    out = dst.label_loss(x, w, t, b, reduction="none")
    t[1] = 4
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, up)


def test_many_own_tiles_and_a_rest_that_is_cut():
    """512 own tiles, two rounds or one of the device's places, and two more: whole tiles and cut ones in one launch. Rays for the forward
    kernel, the best label's and that of dx (128 rows a tile), labels for that of dw (64)."""
    import diff_surfel_tracing as dst
    for N, V in ((128 * 513 + 5, 700), (700, 64 * 513 + 3)):
        x, w, b, t, up = _inputs(N, 129, V, torch.bfloat16)
        got, ref = _grads(x, w, t, b, up, reduction="none"), R.labels(x, w, t, b, up)
        for v, name in zip(got, ("loss", "dx", "dw", "db")):
            R.check(v, ref[name], name)
        label, _ = dst.label_rays(x, w, b)
        s = x.double() @ w.double().T + b.double()
        assert torch.equal(label, torch.where(s == s.amax(1, keepdim=True), torch.arange(V, device="cuda"), V).amin(1))


def test_a_table_and_rays_far_apart_in_memory():
    import diff_surfel_tracing as dst
    x, w, b, t, up = _inputs(300, 24, 90, torch.float32)
    want = _grads(x, w, t, b, up, reduction="none")
    for pitch in (2 ** 23, 2 ** 23 + 1):    # 257 rows of them are more than 2^31 bytes: read from copies
        big = torch.empty(300 * pitch, dtype=torch.float32, device="cuda")
        far_x, far_w = big.as_strided((300, 24), (pitch, 1)), big.as_strided((90, 24), (pitch, 1), 1000)
        far_x.copy_(x), far_w.copy_(w)
        for p, q in zip(want, _grads(far_x, far_w, t, b, up, reduction="none")):
            assert torch.equal(p, q)
        del big, far_x, far_w


def _best(x, w, b):
    s = x.double() @ w.double().T + (0.0 if b is None else b.double())
    return torch.where(s == s.amax(1, keepdim=True), torch.arange(len(w), device="cuda"), len(w)).amin(1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("channels", [8, 16, 64, 256])
def test_best_label_under_a_large_bias(channels, dtype):
    """Products that a bias of 4096 (values apart by 2^-11) rounds away, or up to a whole step, at every addition."""
    import diff_surfel_tracing as dst
    step = 2.0 ** -11
    w = torch.zeros(4, channels, device="cuda")
    w[0], w[1, :-1] = 0.49 * step, 0.51 * step       # (as each product is added by itself)
    w[2, ::4], w[3, :-4:4] = 0.49 * step, 0.51 * step   # (as four are)
    w = w.to(dtype)
    b = torch.full((4,), 4096.0, device="cuda")
    x = torch.ones(70, channels, device="cuda").to(dtype)
    for rows in ([0, 1], [1, 0], [2, 3], [3, 2], [0, 1, 2, 3]):
        label, _ = dst.label_rays(x, w[rows], b[rows])
        assert torch.equal(label, _best(x, w[rows], b[rows]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("channels", [8, 40])
def test_best_label_of_channels_whose_squares_vanish(channels, dtype):
    """A ray of 1e-24, whose square is 0 in 32 bits, against rows apart by their last bit."""
    import diff_surfel_tracing as dst
    x = torch.full((70, channels), 1e-24, device="cuda").to(dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    w = (torch.rand(1, channels, generator=g, device="cuda") + 1.0).to(dtype).repeat(9, 1)
    w[6, 3] += torch.finfo(dtype).eps
    label, _ = dst.label_rays(x, w)
    assert torch.equal(label, _best(x, w, None))
    label, _ = dst.label_rays(x * 0, w)
    assert (label == 0).all()


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_labels_masked_by_a_low_bias(low, dtype):
    x, w, b, t, up = _inputs(900, 40, 130, dtype)
    b[::3] = low
    t = torch.where(t % 3 == 0, t + 1, t)
    t[t >= 130] = 1
    import diff_surfel_tracing as dst
    label, logp = dst.label_rays(x, w, b)
    assert torch.equal(label, _best(x, w, b)) and (label % 3 != 0).all() and torch.isfinite(logp).all()
    there = torch.arange(130, device="cuda") % 3 != 0
    at = torch.cumsum(there, 0) - 1
    got = _grads(x, w, t, b, up, reduction="none")
    ref = R.labels(x, w[there], torch.where(t < 0, t, at[t.clamp(min=0)]), b[there], up)
    R.check(got[0], ref["loss"], "loss")
    R.check(got[1], ref["dx"], "dx")
    R.check(got[2][there], ref["dw"], "dw")
    R.check(got[3][there], ref["db"], "db")
    assert (got[2][~there] == 0).all() and (got[3][~there] == 0).all()
