"""Auxiliary channels of a model that nobody asked render.py to read: they change nothing, whatever they are called and however many."""
import numpy as np
import pytest
import torch

import dst_scenes as S
import render as RH

BASE = ["x", "y", "z", "f_dc_0", "f_dc_1", "f_dc_2", "opacity", "scale_0", "scale_1", "rot_0", "rot_1", "rot_2", "rot_3"]


def _ply(path, more):
    names = BASE + more
    data = np.random.RandomState(0).randn(9, len(names)).astype("<f4")
    with open(path, "wb") as fh:
        fh.write(b"ply\nformat binary_little_endian 1.0\nelement vertex 9\n")
        fh.write("".join("property float %s\n" % n for n in names).encode() + b"end_header\n" + data.tobytes())
    return names, data


def test_properties_that_only_begin_like_channels(tmp_path):
    names, data = _ply(tmp_path / "m.ply", ["aux_mask", "aux_1", "aux_0", "aux_", "aux_view_2"])
    m = RH.load_surfel_model(str(tmp_path / "m.ply"), 0)
    np.testing.assert_array_equal(m["others_precomp"].numpy(), data[:, [names.index("aux_0"), names.index("aux_1")]])
    _ply(tmp_path / "n.ply", ["aux_mask"])
    assert "others_precomp" not in RH.load_surfel_model(str(tmp_path / "n.ply"), 0)


class _Tracer:
    """Keeps what channels it was given."""

    def __init__(self):
        self.given = []

    def build_acceleration_structure(self, *a, **k):
        pass

    def __call__(self, ray_o, ray_d, vertices, others_precomp=None, **k):
        self.given.append(others_precomp)
        z = lambda c: torch.zeros(*ray_o.shape[:2], c)  # noqa: E731
        return z(3), z(1), z(1), z(3), z(1), z(2 if others_precomp is None else others_precomp.shape[1]), None, None


def test_channels_are_traced_only_where_something_reads_them(tmp_path, monkeypatch):
    _ply(tmp_path / "m.ply", ["aux_%d" % k for k in range(9)])   # (more than a trace takes)
    model, cameras = RH.load_surfel_model(str(tmp_path / "m.ply"), 0), RH.orbit_cameras(2, 4, 6, 60.0, 3.0, 0.6)
    tracer = _Tracer()
    RH.render_path(tracer, model, cameras, dev="cpu")
    assert tracer.given == [None, None]
    monkeypatch.setattr(RH, "pixel_labels", lambda aux, head: (torch.zeros(aux.shape[:2], dtype=torch.int64), None))
    head = {"weight": torch.zeros(3, 4)}
    tracer, model = _Tracer(), S.scene_cube(P=20, aux=4)
    RH.render_path(tracer, model, cameras, dev="cpu", label_head=head)
    assert [t.shape for t in tracer.given] == [(20, 4)] * 2
    with pytest.raises(ValueError, match="channels"):
        RH.render_path(tracer, model, cameras, dev="cpu", label_head={"weight": torch.zeros(3, 5)})
