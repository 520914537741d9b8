"""The operators as they are used together: channels traced through the scene, a label loss on them with gradients down to the
surfels, their labels, and what they read out of a memory."""
import pytest
import torch

import dst_scenes as S
import features_reference as R

pytestmark = pytest.mark.gpu


def _trace(tracer, g, others, ray_o, ray_d):
    import diff_surfel_tracing as dst
    eye = torch.eye(4, device="cuda")
    settings = dst.SurfelTracingSettings(image_height=ray_o.size(0), image_width=ray_o.size(1), tanfovx=1.0, tanfovy=1.0,
                                         bg=torch.zeros(3, device="cuda"), scale_modifier=1.0, viewmatrix=eye, projmatrix=eye,
                                         sh_degree=3, campos=torch.zeros(3, device="cuda"), prefiltered=False, debug=False)
    return tracer(ray_o, ray_d, g["vertices"], means3D=g["means3D"], grads3D=torch.zeros_like(g["means3D"]), shs=g["shs"],
                  others_precomp=others, opacities=g["opacities"], scales=g["scales"], rotations=g["rotations"],
                  tracer_settings=settings)[5]


def test_a_training_step_through_the_tracer(tracer):
    import diff_surfel_tracing as dst
    scene = S.scene_cube(P=4000, aux=8)
    g = {k: v.cuda() for k, v in scene.items()}
    tracer.build_acceleration_structure(g["vertices"], g["faces"], rebuild=True)
    ray_o, ray_d = (t.cuda() for t in S.rays_cube(48, 64))
    gen = torch.Generator(device="cuda").manual_seed(1)
    weight = torch.randn(21, 8, generator=gen, device="cuda").requires_grad_(True)
    bias = torch.randn(21, generator=gen, device="cuda").requires_grad_(True)
    targets = torch.randint(0, 21, (48, 64), generator=gen, device="cuda")
    targets[::5] = -100
    tracer.optix_context.deterministic = True
    try:
        others = g["others_precomp"].clone().requires_grad_(True)
        aux = _trace(tracer, g, others, ray_o, ray_d)
        loss = dst.label_loss(aux, weight, targets, bias)
        d_others, d_aux, d_weight, d_bias = torch.autograd.grad(loss, [others, aux, weight, bias])
        # the loss's own gradients against the formula, at the channels that the tracer gave
        n = int((targets != -100).sum())
        ref = R.labels(aux.detach().reshape(-1, 8), weight.detach(), targets.reshape(-1), bias.detach(),
                       torch.full((48 * 64,), 1.0 / n, dtype=torch.float64, device="cuda"))
        value, bound = ref["loss"]
        R.check(loss.detach(), (value.sum() / n, bound.sum() / n + R.U * value.sum() / n), "loss")
        for got, name in ((d_aux.reshape(-1, 8), "dx"), (d_weight, "dw"), (d_bias, "db")):
            R.check(got, (ref[name][0], ref[name][1] * (1 + 4 * R.U) + 4 * R.U * ref[name][0].abs()), name)
        # and the surfels' gradient is the tracer's for that gradient of its channels
        again = g["others_precomp"].clone().requires_grad_(True)
        want, = torch.autograd.grad(_trace(tracer, g, again, ray_o, ray_d), again, d_aux)
        assert torch.equal(d_others, want) and float(want.abs().max()) > 0
    finally:
        tracer.optix_context.deterministic = False


def test_labels_and_memory_features_of_a_view(tracer):
    import diff_surfel_tracing as dst
    scene = S.scene_room(P=20000, aux=8)
    g = {k: v.cuda() for k, v in scene.items()}
    tracer.build_acceleration_structure(g["vertices"], g["faces"], rebuild=True)
    ray_o, ray_d = (t.cuda() for t in S.rays_room(45, 80))
    with torch.no_grad():
        aux = _trace(tracer, g, g["others_precomp"], ray_o, ray_d)
        gen = torch.Generator(device="cuda").manual_seed(2)
        weight = torch.randn(151, 8, generator=gen, device="cuda")
        labels, log_prob = dst.label_rays(aux, weight)
        s = aux.reshape(-1, 8).double() @ weight.double().T
        top = s.amax(1, keepdim=True)
        assert torch.equal(labels.reshape(-1), torch.where(s == top, torch.arange(151, device="cuda"), 151).amin(1))
        assert labels.shape == (45, 80) and float(log_prob.max()) <= 0
        # the loss at the best label is its log probability
        at_best = dst.label_loss(aux, weight, labels, reduction="none")
        bound = R.labels(aux.reshape(-1, 8), weight, labels.reshape(-1))["loss"][1]
        assert ((at_best + log_prob).abs().reshape(-1) <= 2 * bound).all()
        # queries of the channels against a bank, as many as there are pixels
        proj, keys, values = (torch.randn(*n, generator=gen, device="cuda") for n in ((8, 2 * 16), (200, 2, 16), (200, 2, 12)))
        q = (aux.reshape(-1, 8) @ proj).reshape(1, -1, 2, 16)
        R.check(dst.attend_memory(q, keys[None], values[None]), R.attend(q, keys[None], values[None])["out"], "out")
