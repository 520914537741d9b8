"""Calls that the C boundary allows and the Python functions do not make."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


def _workspace(p, size, what):
    ws = torch.empty(max(256, size(C.byref(p), what)), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    return ws


@pytest.mark.parametrize("channels", [8, 40, 64])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_gradients_of_a_memory_that_nobody_asked(dtype, channels):
    """No queries: the memory's gradients are zeros, and neither rows nor memory are read (or have to be there)."""
    import diff_surfel_tracing._C as binding
    lib = binding.load_library()
    element = (torch.float32, torch.bfloat16, torch.float16)[dtype]
    p = binding.DstAttendParams()
    p.batch, p.queries, p.memory, p.heads, p.kv_heads, p.channels, p.value_channels = 2, 0, 300, 4, 2, channels, channels
    p.dtype, p.scale = dtype, 0.5
    p.k_strides = p.v_strides = (C.c_int64 * 3)(600 * channels, 2 * channels, channels)
    dk, dv = (torch.full((2, 300, 2, channels), float("nan"), device="cuda", dtype=element) for _ in range(2))
    p.grad_k, p.grad_v = dk.data_ptr(), dv.data_ptr()
    ws = _workspace(p, lib.dst_attend_workspace_bytes, 1)
    assert lib.dst_attend_backward(C.byref(p), binding._stream()) == 0, lib.dst_op_error()
    torch.cuda.synchronize()
    assert (dk == 0).all() and (dv == 0).all() and ws.numel() > 0


def test_gradients_of_a_table_that_no_ray_asked():
    import diff_surfel_tracing._C as binding
    lib = binding.load_library()
    for dtype, element in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        for channels in (8, 40, 64):
            w = torch.ones(90, channels, device="cuda", dtype=element)
            p = binding.DstLabelParams()
            p.rays, p.channels, p.labels, p.dtype, p.reduction = 0, channels, 90, dtype, 0
            p.features_stride, p.weight, p.weight_stride = channels, w.data_ptr(), channels
            dw, db = torch.full_like(w, float("nan")), torch.full((90,), float("nan"), device="cuda")
            p.grad_weight, p.grad_bias = dw.data_ptr(), db.data_ptr()
            ws = _workspace(p, lib.dst_label_workspace_bytes, 1)
            assert lib.dst_label_loss_backward(C.byref(p), binding._stream()) == 0, lib.dst_op_error()
            torch.cuda.synchronize()
            assert (dw == 0).all() and (db == 0).all() and ws.numel() > 0
