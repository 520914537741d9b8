"""Host-side checks of the label and attention operators that need no GPU: layouts, refusals at both boundaries."""
import ctypes as C
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def binding():
    import diff_surfel_tracing._C as binding
    binding.load_library()
    return binding


@pytest.mark.parametrize("block", ["DstLabelParams", "DstAttendParams"])
def test_parameter_blocks_have_the_header_s_fields_and_size(binding, block):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "dst_api.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (block, block), text, flags=re.S).group(1)
    fields = [re.findall(r"[A-Za-z_]\w*", part.split("[")[0])[-1] for decl in body.split(";") if decl.strip()
              for part in decl.split(",")]
    mirror = getattr(binding, block)
    assert fields == [f[0] for f in mirror._fields_]
    name = "dst_sizeof_label_params" if "Label" in block else "dst_sizeof_attend_params"
    assert getattr(binding.load_library(), name)() == C.sizeof(mirror)


def _label(binding, **more):
    p = binding.DstLabelParams()
    p.rays, p.channels, p.labels = 10, 8, 5
    p.features, p.features_stride, p.weight, p.weight_stride = 4096, 8, 4096, 8   # (never read: every call below is refused)
    p.targets = p.lse = p.loss = p.inverse = p.upstream = p.best = p.log_prob = 4096
    for k, v in more.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("more,word", [
    (dict(rays=-1), b"rays"), (dict(rays=2 ** 31), b"rays"), (dict(labels=0), b"labels"), (dict(labels=2 ** 30), b"labels"),
    (dict(channels=0), b"channels"), (dict(channels=257), b"channels"), (dict(dtype=3), b"dtype"), (dict(reduction=5), b"reduction"),
    (dict(features_stride=7), b"overlap"), (dict(weight_stride=0), b"overlap"), (dict(features=None), b"features"),
    (dict(weight=None), b"weight")])
def test_label_calls_are_refused_with_a_message(binding, more, word):
    lib, p = binding.load_library(), _label(binding, **more)
    for call in (lib.dst_label_loss_forward, lib.dst_label_loss_backward, lib.dst_label_best):
        assert call(C.byref(p), None) != 0
        assert word in lib.dst_op_error()
    assert lib.dst_label_workspace_bytes(C.byref(p), 0) == 0


def test_label_calls_without_their_buffers(binding):
    lib = binding.load_library()
    for call, missing in ((lib.dst_label_loss_forward, "targets lse loss"), (lib.dst_label_loss_backward, "targets lse upstream"),
                          (lib.dst_label_best, "best log_prob")):
        assert call(None, None) == 1
        for name in missing.split():
            assert call(C.byref(_label(binding, **{name: None})), None) == 1, name
            assert name.encode() in lib.dst_op_error()
    for call in (lib.dst_label_loss_forward, lib.dst_label_loss_backward):
        assert call(C.byref(_label(binding, reduction=2, inverse=None)), None) == 1
    # a workspace that is missing, too small or askew
    p = _label(binding, rays=100000, reduction=2)
    need = lib.dst_label_workspace_bytes(C.byref(p), 0)
    assert need > 0
    for at, size in ((None, need), (4096, need - 1), (4097, need)):
        p.workspace, p.workspace_bytes = at, size
        assert lib.dst_label_loss_forward(C.byref(p), None) == 1 and b"workspace" in lib.dst_op_error()
    p = _label(binding, grad_features=4100)
    assert lib.dst_label_loss_backward(C.byref(p), None) == 1 and b"aligned" in lib.dst_op_error()


def _attend(binding, **more):
    p = binding.DstAttendParams()
    p.batch, p.queries, p.memory, p.heads, p.kv_heads, p.channels, p.value_channels = 1, 100, 100, 2, 1, 16, 16
    p.scale = 0.25
    p.q = p.k = p.v = p.out = p.lse = p.upstream = p.grad_q = 4096
    for k, v in more.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("more,word", [
    (dict(batch=-1), b"negative"), (dict(queries=-1), b"negative"), (dict(memory=-1), b"negative"), (dict(heads=0), b"heads"),
    (dict(heads=3, kv_heads=2), b"heads"), (dict(kv_heads=0), b"heads"), (dict(channels=0), b"channels"),
    (dict(channels=257), b"channels"), (dict(value_channels=300), b"channels"), (dict(dtype=-1), b"dtype"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(queries=2 ** 30), b"rows"),
    (dict(memory=2 ** 31 - 1), b"rows"), (dict(batch=2 ** 20, queries=2 ** 20), b"rows"), (dict(q=None), b"q, k"),
    (dict(v=None), b"q, k"), (dict(out=None), b"q, k")])
def test_attention_calls_are_refused_with_a_message(binding, more, word):
    lib, p = binding.load_library(), _attend(binding, **more)
    for call in (lib.dst_attend_forward, lib.dst_attend_backward):
        assert call(C.byref(p), None) != 0
        assert word in lib.dst_op_error()
    assert lib.dst_attend_workspace_bytes(C.byref(p), 0) == 0 and lib.dst_attend_workspace_bytes(C.byref(p), 1) == 0


def test_attention_calls_without_their_buffers(binding):
    lib = binding.load_library()
    assert lib.dst_attend_forward(None, None) == 1 and lib.dst_attend_backward(None, None) == 1
    for name in ("lse", "upstream"):
        assert lib.dst_attend_backward(C.byref(_attend(binding, **{name: None})), None) == 1
        assert name.encode() in lib.dst_op_error()
    for dtype in (1, 2):   # (16-bit rows: what the rounding of out left)
        assert lib.dst_attend_backward(C.byref(_attend(binding, dtype=dtype)), None) == 1
        assert b"out_low" in lib.dst_op_error()
    assert lib.dst_attend_backward(C.byref(_attend(binding, grad_q=4104)), None) == 1
    for queries, memory in ((1, 65536), (100, 100)):
        p = _attend(binding, queries=queries, memory=memory)
        need = lib.dst_attend_workspace_bytes(C.byref(p), 1)
        assert need > 0
        for at, size in ((None, need), (4096, need - 1), (4097, need)):
            p.workspace, p.workspace_bytes = at, size
            assert lib.dst_attend_backward(C.byref(p), None) == 1 and b"workspace" in lib.dst_op_error()
    # nothing to do is done without a device
    assert lib.dst_attend_forward(C.byref(_attend(binding, batch=0)), None) == 0
    assert lib.dst_attend_backward(C.byref(_attend(binding, grad_q=None)), None) == 0


def test_python_refusals():
    import diff_surfel_tracing as dst
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    for bad, word in (((x.double(), w, t), "float32, bfloat16 or float16"), ((None, w, t), "tensor"), ((x, w, t), "CUDA"),
                      ((x.int(), w, t), "float32")):
        with pytest.raises(RuntimeError, match=word):
            dst.label_loss(*bad)
        with pytest.raises(RuntimeError, match=word):
            dst.label_rays(*bad[:2])
    q = torch.zeros(1, 2, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        dst.attend_memory(q, q, q)
    with pytest.raises(RuntimeError, match="float32"):
        dst.attend_memory(q.long(), q, q)


@pytest.fixture
def anywhere(monkeypatch):
    """The argument checks behind the one for a GPU, on CPU tensors: nothing is launched, every call below is refused."""
    import diff_surfel_tracing.features as F
    real = F._rows

    def rows(t, name):
        try:
            real(t, name)
        except RuntimeError as e:
            if "CUDA" not in str(e):
                raise
    monkeypatch.setattr(F, "_rows", rows)


def test_python_refusals_of_shapes_and_types(anywhere):
    import diff_surfel_tracing as dst
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    for args, more, word in (
            ((x, w.bfloat16(), t), {}, "dtype|float32"), ((x, torch.zeros(5, 7), t), {}, "weight"),
            ((x, torch.zeros(0, 8), t), {}, "weight"), ((x, w[0], t), {}, "weight"), ((x, w, t.float()), {}, "targets"),
            ((x, w, t[:3]), {}, "targets"), ((x, w, t > 0), {}, "targets"), ((x, w, None), {}, "targets"),
            ((x, w, t, torch.zeros(4)), {}, "bias"), ((x, w, t, torch.zeros(5).double()), {}, "bias"),
            ((x, w, t), {"reduction": "max"}, "reduction"), ((x, w.to("meta"), t), {}, "weight")):
        with pytest.raises(RuntimeError, match=word):
            dst.label_loss(*args, **more)
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 9, 2, 8)
    for args, word in (((q[0], k, k), "queries"), ((q, k[0], k), "keys"), ((q, k, k[:, :8]), "memory"), ((q, k[:1], k[:1]), "batch"),
                       ((q, k[..., :7], k), "channels"), ((q, k[:, :, :0], k[:, :, :0]), "heads"),
                       ((q[:, :, :3], k, k), "multiple"), ((q, k.half(), k), "float32"),
                       ((q, k, k, torch.zeros(2)), "lengths"), ((q, k, k, torch.zeros(3, dtype=torch.int32)), "lengths"),
                       ((q, k, k, [1, 2]), "lengths"), ((q, torch.zeros(2, 9, 2, 300), k), "channels")):
        with pytest.raises(RuntimeError, match=word):
            dst.attend_memory(*args)
