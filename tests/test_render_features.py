"""What render.py reads off a model's auxiliary channels: its files on the host, and on the GPU a rendered path's labels and
features against their formulas."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import dst_scenes as S
import render as RH

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _head(path, V=7, C=4, bias=True, seed=0):
    g = np.random.RandomState(seed)
    arrays = {"weight": g.randn(V, C).astype(np.float64)}
    if bias:
        arrays["bias"] = g.randn(V)
    np.savez(path, **arrays)
    return arrays


def _bank(path, C=4, heads=2, kv=1, d=6, M=30, dv=5, seed=0):
    g = np.random.RandomState(seed)
    arrays = {"query": g.randn(C, heads, d), "keys": g.randn(M, kv, d), "values": g.randn(M, kv, dv)}
    np.savez(path, **arrays)
    return arrays


def test_files_are_read_and_checked(tmp_path):
    arrays = _head(tmp_path / "h.npz")
    head = RH.load_label_head(str(tmp_path / "h.npz"))
    assert head["weight"].dtype == torch.float32
    np.testing.assert_array_equal(head["weight"].numpy(), arrays["weight"].astype(np.float32))
    _head(tmp_path / "n.npz", bias=False)
    assert set(RH.load_label_head(str(tmp_path / "n.npz"))) == {"weight"}
    np.savez(tmp_path / "b.npz", weight=np.zeros((3, 2)), bias=np.zeros(4))
    with pytest.raises(ValueError, match="bias"):
        RH.load_label_head(str(tmp_path / "b.npz"))
    np.savez(tmp_path / "w.npz", bias=np.zeros(4))
    with pytest.raises(ValueError, match="lacks weight"):
        RH.load_label_head(str(tmp_path / "w.npz"))
    np.savez(tmp_path / "d.npz", weight=np.zeros(4))
    with pytest.raises(ValueError, match="dimensions"):
        RH.load_label_head(str(tmp_path / "d.npz"))
    _bank(tmp_path / "m.npz")
    assert set(RH.load_memory_bank(str(tmp_path / "m.npz"))) == {"query", "keys", "values"}
    _bank(tmp_path / "k.npz", heads=3, kv=2)
    with pytest.raises(ValueError, match="fit"):
        RH.load_memory_bank(str(tmp_path / "k.npz"))
    with pytest.raises(ValueError, match="lacks"):
        RH.load_memory_bank(str(tmp_path / "h.npz"))


def test_model_channels_are_read_in_their_order(tmp_path):
    names = ["x", "y", "z", "f_dc_0", "f_dc_1", "f_dc_2"] + ["opacity", "scale_0", "scale_1", "rot_0", "rot_1", "rot_2", "rot_3"] + \
        ["aux_%d" % k for k in (2, 0, 1)]
    data = np.random.RandomState(0).randn(9, len(names)).astype("<f4")
    with open(tmp_path / "m.ply", "wb") as fh:
        fh.write(b"ply\nformat binary_little_endian 1.0\nelement vertex 9\n")
        fh.write("".join("property float %s\n" % n for n in names).encode() + b"end_header\n" + data.tobytes())
    m = RH.load_surfel_model(str(tmp_path / "m.ply"), 0)
    np.testing.assert_array_equal(m["others_precomp"].numpy(), data[:, [names.index("aux_%d" % k) for k in range(3)]])


def test_every_label_has_one_color():
    labels = torch.arange(4000).reshape(40, 100)
    colors = RH.label_colors(labels)
    assert colors.shape == (40, 100, 3) and float(colors.min()) >= 0 and float(colors.max()) <= 1
    assert torch.equal(colors, RH.label_colors(labels.to(torch.int32)))
    assert len(torch.unique(colors.reshape(-1, 3), dim=0)) > 3900


@pytest.mark.gpu
def test_rendered_labels_and_features(tmp_path, tracer):
    head, bank = _head(tmp_path / "h.npz"), _bank(tmp_path / "m.npz")
    head, bank = RH.load_label_head(str(tmp_path / "h.npz")), RH.load_memory_bank(str(tmp_path / "m.npz"))
    model = S.scene_cube(P=3000, aux=4)
    cameras = RH.orbit_cameras(2, 40, 56, 60.0, 3.0, 0.6)
    plain = RH.render_path(tracer, model, cameras)
    outs = RH.render_path(tracer, model, cameras, str(tmp_path / "out"), label_head=head, memory_bank=bank)
    for i, (out, ref) in enumerate(zip(outs, plain)):
        assert len(ref) == 4 and len(out) == 6
        for a, b in zip(out, ref):
            assert torch.equal(a, b)
        labels, features = out[4], out[5]
        assert labels.shape == (40, 56) and features.shape == (40, 56, 10)
        assert os.path.exists(tmp_path / "out" / "LABEL" / ("%04d.png" % i))
        np.testing.assert_array_equal(np.load(tmp_path / "out" / "LABEL" / ("%04d.npy" % i)), labels.cpu().numpy())
        np.testing.assert_array_equal(np.load(tmp_path / "out" / "FEATURE" / ("%04d.npy" % i)), features.cpu().numpy())
    with pytest.raises(ValueError, match="channels"):
        RH.render_path(tracer, S.scene_cube(P=100), cameras, label_head=head)


@pytest.mark.gpu
def test_the_command_writes_labels_and_features(tmp_path):
    _head(tmp_path / "h.npz", C=3)
    _bank(tmp_path / "m.npz", C=3)
    subprocess.check_call([sys.executable, os.path.join(ROOT, "diff-surfel-tracing_amd", "render.py"), "--scene", "cube", "--surfels",
                           "2000", "--frames", "1", "--height", "32", "--width", "40", "--result_dir", str(tmp_path / "out"),
                           "--labels", str(tmp_path / "h.npz"), "--memory", str(tmp_path / "m.npz")], timeout=100)
    assert np.load(tmp_path / "out" / "LABEL" / "0000.npy").shape == (32, 40)
    assert np.load(tmp_path / "out" / "FEATURE" / "0000.npy").shape == (32, 40, 10)
