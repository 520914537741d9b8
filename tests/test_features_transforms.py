"""The label and attention operators under forward-mode differentiation, functorch's transforms and recorded traces, on the CPU with
the launchers replaced: refused, or launched again, never passed over."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


@pytest.fixture
def launches(monkeypatch):
    import diff_surfel_tracing.features as F
    calls = []

    def rows(t, name):
        pass

    def loss(x, w, targets, bias, ignore_index, reduction):
        calls.append("loss")
        return torch.zeros(x.size(0) if reduction == 0 else ()), torch.zeros(x.size(0)), None

    def best(x, w, bias):
        calls.append("best")
        return torch.zeros(x.size(0), dtype=torch.int64), torch.zeros(x.size(0))

    def attend(q, k, v, lengths, scale, for_backward):
        calls.append("attend")
        return torch.zeros(q.shape[:3] + v.shape[3:]), torch.zeros(1), None
    monkeypatch.setattr(F, "_rows", rows)
    monkeypatch.setattr(F, "_loss_forward", loss)
    monkeypatch.setattr(F, "_best_forward", best, raising=False)
    monkeypatch.setattr(F, "_attend_forward", attend)
    return calls


def _calls():
    import diff_surfel_tracing as dst
    t = torch.zeros(4, dtype=torch.int64)
    lengths = torch.ones(1, dtype=torch.int32)
    return {"loss": (lambda *a: dst.label_loss(a[0], a[1], t, a[2]), [torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(5)]),
            "best": (lambda *a: dst.label_rays(*a)[1], [torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(5)]),
            "attend": (lambda *a: dst.attend_memory(*a, lengths),
                       [torch.zeros(1, 3, 2, 8), torch.zeros(1, 6, 2, 8), torch.zeros(1, 6, 2, 4)])}


@pytest.mark.parametrize("name", ["loss", "best", "attend"])
def test_forward_mode_tangents_are_refused(launches, name):
    call, args = _calls()[name]
    for k in range(3):
        with fwad.dual_level():
            dual = list(args)
            dual[k] = fwad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(NotImplementedError):
                call(*dual)
    with fwad.dual_level():            # no tangent among the inputs: a plain call
        n = len(launches)
        assert isinstance(call(*args), torch.Tensor) and launches[n:] == [name]


@pytest.mark.parametrize("name", ["loss", "best", "attend"])
def test_functorch_transforms_are_refused(launches, name):
    call, args = _calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: call(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: call(x, *args[1:]))(torch.stack([args[0]] * 2))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: call(x, *args[1:]).sum())(args[0])


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", ["loss", "best", "attend"])
def test_a_recorded_trace_launches_again(launches, name):
    call, args = _calls()[name]
    traced = torch.jit.trace(lambda x: call(x, *args[1:]), (args[0],), check_trace=False)
    n = len(launches)
    traced(args[0])
    assert launches[n:] == [name]


def test_labels_have_no_gradient(launches):
    import diff_surfel_tracing as dst
    label, log_prob = dst.label_rays(*(t.requires_grad_(True) for t in _calls()["best"][1]))
    assert not label.requires_grad and not log_prob.requires_grad


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_recorded_traces_answer_for_new_inputs():
    import diff_surfel_tracing as dst
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    w, b, t = r(50, 24), r(50), torch.randint(0, 50, (70,), generator=g, device="cuda")
    k, v = r(1, 90, 2, 24), r(1, 90, 2, 16)
    for call, shape in ((lambda x: dst.label_loss(x, w, t, b), (70, 24)), (lambda x: dst.label_loss(x, w, t, reduction="none"), (70, 24)),
                        (lambda x: dst.label_rays(x, w, b), (70, 24)), (lambda q: dst.attend_memory(q, k, v), (1, 33, 4, 24))):
        traced = torch.jit.trace(call, (r(*shape),), check_trace=False)
        for _ in range(2):
            x = r(*shape)
            got, want = traced(x), call(x)
            for p, q in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(p, q)
