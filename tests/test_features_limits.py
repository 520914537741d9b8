"""Sizes that one launch cannot hold: refused before memory is taken, on the host. A launch counts its threads in 32 bits, so it has at
most 2^24 - 1 workgroups of 256."""
import ctypes as C

import pytest

F32, BF16 = 0, 1
FORWARD, BACKWARD, BEST = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    import diff_surfel_tracing._C as binding
    return binding.load_library()


def _attend(**more):
    import diff_surfel_tracing._C as binding
    p = binding.DstAttendParams()
    p.batch, p.queries, p.memory, p.heads, p.kv_heads, p.channels, p.value_channels = 1, 1, 1, 1, 1, 17, 17
    p.scale, p.dtype = 0.25, F32
    p.q = p.k = p.v = p.out = p.lse = p.out_low = p.upstream = p.grad_q = p.grad_k = p.grad_v = 4096   # (never read)
    for k, v in more.items():
        setattr(p, k, v)
    return p


def _label(**more):
    import diff_surfel_tracing._C as binding
    p = binding.DstLabelParams()
    p.rays, p.channels, p.labels, p.dtype, p.reduction = 1, 17, 1, F32, 0
    p.features, p.features_stride, p.weight, p.weight_stride = 4096, 256, 4096, 256
    p.targets = p.lse = p.stats = p.loss = p.inverse = p.upstream = p.best = p.log_prob = 4096
    p.grad_features = p.grad_weight = p.grad_bias = 4096
    for k, v in more.items():
        setattr(p, k, v)
    return p


def _refused(lib, call, size, p, what, word):
    assert size(C.byref(p), what) == 0
    assert call(C.byref(p), None) != 0
    assert word in lib.dst_op_error(), lib.dst_op_error()


def _admitted(lib, call, size, p, what):
    """Past the sizes: refused only for the workspace that it lacks."""
    assert size(C.byref(p), what) > 0
    assert call(C.byref(p), None) == 1
    assert b"workspace" in lib.dst_op_error(), lib.dst_op_error()


@pytest.mark.parametrize("what", [FORWARD, BACKWARD])
def test_attention_with_a_workgroup_for_each_batch_and_head(lib, what):
    call = (lib.dst_attend_forward, lib.dst_attend_backward)[what]
    size = lib.dst_attend_workspace_bytes
    _refused(lib, call, size, _attend(batch=2 ** 24), what, b"too many rows")
    _refused(lib, call, size, _attend(batch=2 ** 23, heads=2, kv_heads=2), what, b"too many rows")
    _refused(lib, call, size, _attend(batch=8294400, heads=4, kv_heads=4, channels=8, value_channels=8, dtype=BF16), what, b"too many rows")
    _admitted(lib, call, size, _attend(batch=2 ** 24 - 1), what)


def test_attention_to_a_memory_too_long_for_its_gradient(lib):
    # (64 rows of memory a workgroup; 16-bit rows are read as they lie)
    big = dict(memory=2 ** 30 - 1, dtype=BF16, channels=256, value_channels=256)
    _refused(lib, lib.dst_attend_backward, lib.dst_attend_workspace_bytes, _attend(**big), BACKWARD, b"too many rows")


@pytest.mark.parametrize("what", [FORWARD, BACKWARD])
def test_attention_whose_copies_do_not_fit_a_launch(lib, what):
    call = (lib.dst_attend_forward, lib.dst_attend_backward)[what]
    size = lib.dst_attend_workspace_bytes
    wide = dict(channels=256, value_channels=256)
    _refused(lib, call, size, _attend(queries=2 ** 27, **wide), what, b"too many rows")
    _refused(lib, call, size, _attend(memory=2 ** 27, **wide), what, b"too many rows")
    _admitted(lib, call, size, _attend(queries=2 ** 24, memory=2 ** 20, **wide), what)


def test_labels(lib):
    size = lib.dst_label_workspace_bytes
    calls = (lib.dst_label_loss_forward, lib.dst_label_loss_backward, lib.dst_label_best)
    for what, call in enumerate(calls):   # copies into planes: 32 words of 16 bytes a row
        _refused(lib, call, size, _label(rays=2 ** 27, channels=256), what, b"too many rays")
        _admitted(lib, call, size, _label(rays=2 ** 25, channels=256), what)
    # 128 rays a workgroup, 64 labels a workgroup
    _refused(lib, calls[BACKWARD], size, _label(rays=2 ** 31 - 1, channels=8, dtype=BF16), BACKWARD, b"too many rays")
    _refused(lib, calls[BACKWARD], size, _label(labels=2 ** 30 - 1, channels=256, dtype=BF16, grad_features=None), BACKWARD, b"too many rays")
    _admitted(lib, calls[BEST], size, _label(rays=2 ** 31 - 1, channels=8, dtype=BF16), BEST)


@pytest.mark.parametrize("name", ["q_strides", "k_strides", "v_strides"])
@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("stride", [-1, -2 ** 62, 2 ** 44 + 1, 2 ** 62])
def test_strides_that_offsets_are_not_made_for(lib, name, at, stride):
    p = _attend()
    getattr(p, name)[at] = stride
    for what, call in ((FORWARD, lib.dst_attend_forward), (BACKWARD, lib.dst_attend_backward)):
        _refused(lib, call, lib.dst_attend_workspace_bytes, p, what, b"strides")


def test_label_strides_that_offsets_are_not_made_for(lib):
    for what, call in enumerate((lib.dst_label_loss_forward, lib.dst_label_loss_backward, lib.dst_label_best)):
        for name in ("features_stride", "weight_stride"):
            _refused(lib, call, lib.dst_label_workspace_bytes, _label(**{name: 2 ** 62}), what, b"stride")


@pytest.mark.parametrize("number", [2 ** 64 - 100, 2 ** 63, -2 ** 63 - 1])
def test_an_ignore_index_beyond_64_bits_does_not_become_another(monkeypatch, number):
    import torch

    import diff_surfel_tracing as dst
    import diff_surfel_tracing.features as F
    monkeypatch.setattr(F, "_rows", lambda t, name: None)
    monkeypatch.setattr(F, "_loss_forward", lambda x, *a: (torch.zeros(x.size(0)), None, None))
    args = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ignore_index"):
        dst.label_loss(*args, ignore_index=number, reduction="none")
    assert dst.label_loss(*args, ignore_index=-2 ** 63, reduction="none").shape == (4,)
