"""The renderer's own uses of the layer operators: the background network at shapes its kernels are not compiled for (layers.linear) and
repeatable gradients of the per-view pose / light deltas (layers.embedding)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import nrhints_amd as na
from nrhints_amd import _lib
from nrhints_amd.outside import OutsideNeRF
from nrhints_amd.pipeline import CameraModel
from nrhints_amd.ray_generator import RayGenerator, RayGeneratorConfig
from nrhints_amd.synthetic import make_rays

pytestmark = pytest.mark.gpu
T = torch.from_numpy
cu = lambda a: (T(a) if isinstance(a, np.ndarray) else a).float().contiguous().cuda()


def _encode(x, n):
    s = (x[..., None] * 2.0 ** torch.arange(n, dtype=x.dtype, device=x.device)).reshape(x.shape[0], -1)
    return torch.cat([x, torch.sin(torch.cat([s, s + np.pi / 2.0], dim=-1))], dim=-1)


def _nerf64(net, p, pts4, views, pls, ppr):
    """fields/nerf_density_field.py:66-89 at any shape, float64; also the smallest |argument of a ReLU| of every point."""
    x, v = _encode(pts4, net.multi_res), _encode(torch.cat([views, pls], -1), net.multi_res_view).repeat_interleave(ppr, 0)
    h, near = x, torch.full((pts4.shape[0],), 1e9, dtype=torch.float64, device=pts4.device)
    for i in range(len(net.pts_linears)):
        z = F.linear(h, p[f"pts_linears.{i}.weight"], p[f"pts_linears.{i}.bias"])
        near = torch.minimum(near, z.abs().min(1)[0])
        h = torch.relu(z)
        if i in net.skips:
            h = torch.cat([x, h], -1)
    z = F.linear(torch.cat([F.linear(h, p["feature_linear.weight"], p["feature_linear.bias"]), v], -1), p["views_linears.0.weight"], p["views_linears.0.bias"])
    near = torch.minimum(near, z.abs().min(1)[0])
    return F.linear(h, p["alpha_linear.weight"], p["alpha_linear.bias"]), F.linear(torch.relu(z), p["rgb_linear.weight"], p["rgb_linear.bias"]), near


@pytest.mark.parametrize("shape", [dict(), dict(d_hidden=320, n_layers=5, multi_res=6, multi_res_view=2, skips=(1,)),
                                   dict(d_hidden=258, n_layers=3, multi_res=1, multi_res_view=1, skips=()),
                                   dict(d_hidden=256, n_layers=9, skips=(2, 5))], ids=["default", "320x5", "258x3", "256x9"])
def test_background_network_layer_by_layer(shape):
    """Values and every gradient against float64, on points none of whose ReLU arguments is nearer to zero than float32 can tell.  Ten
    layers of float32 sums of at most 424 terms: each is off by at most (424 + 8) 2^-24 of its sum of magnitudes, 2.6e-4 of the largest
    over all layers if every one is off by its bound in the same direction."""
    torch.manual_seed(1)
    net = OutsideNeRF(4, 6, **shape).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    ppr, rays = 4, 600
    pts, views, pls = 0.5 * rnd(rays * ppr, 4), F.normalize(rnd(rays, 3), dim=-1), rnd(rays, 3)
    p64 = {k: v.detach().double() for k, v in net.named_parameters()}
    near = _nerf64(net, p64, pts.double(), views.double(), pls.double(), ppr)[2].reshape(rays, ppr).min(1)[0]
    keep = (near > 2e-6).nonzero()[:64, 0]
    assert keep.numel() >= 16
    keep = keep[:keep.numel() // 16 * 16]
    pts, views, pls = pts.reshape(rays, ppr, 4)[keep].reshape(-1, 4), views[keep], pls[keep]
    net.compiled = False                                   # the default shape, too, through the layers
    leaves = [t.clone().requires_grad_(True) for t in (pts, views, pls)]
    dens, rgb = net(*leaves, pts_per_ray=ppr)
    sd, sr = rnd(*dens.shape), rnd(*rgb.shape)
    grads = torch.autograd.grad([dens, rgb], leaves + list(net.parameters()), [sd, sr])
    l64 = [t.double().requires_grad_(True) for t in (pts, views, pls)]
    p64 = {k: v.requires_grad_(True) for k, v in p64.items()}
    want_d, want_c, _ = _nerf64(net, p64, *l64, ppr)
    want = torch.autograd.grad([want_d, want_c], l64 + list(p64.values()), [sd.double(), sr.double()])
    tol = 10 * 432 * 2.0 ** -24
    for got, exact in [(dens, want_d), (rgb, want_c)] + list(zip(grads, want)):
        assert got.dtype == torch.float32 and got.shape == exact.shape
        assert float((got.detach().double() - exact.detach()).abs().max()) <= tol * float(exact.detach().abs().max())
    if not shape:                                          # ... and the compiled kernels agree with the layers
        net.compiled, net.precision = True, "f32"
        d2, c2 = net(pts, views, pls, pts_per_ray=ppr)
        assert float((d2 - dens).abs().max()) <= tol * float(want_d.detach().abs().max()) and float((c2 - rgb).abs().max()) <= tol * float(want_c.detach().abs().max())


def test_renderer_with_a_wider_background_network():
    """use_outside_nerf with a 320 x 5 network (refused before the layers): the fused step equals forward() + backward() on the same batch
    and jitter in every gradient tensor, the captured step runs and moves the background's weights, an evaluation renders."""
    from nrhints_amd import train_fused
    from nrhints_amd.training import GraphedTrainStep, train_loss_dict
    cfg = na.NeuSModelConfig(renderer=na.NeuSRendererConfig(use_outside_nerf=True),
                             outside_nerf=na.NeRFConfig(d_hidden=320, n_layers=5, multi_res=6, multi_res_view=2, skips=[1]))
    torch.manual_seed(3)
    sd = na.NeuSHintRenderer(cfg).state_dict()
    sd["outside_nerf.alpha_linear.bias"] = sd["outside_nerf.alpha_linear.bias"] + 1.5          # a visible background

    def build():
        m = na.NeuSHintRenderer(cfg)
        m.load_state_dict(sd)
        return m.cuda().train()

    rays = make_rays(32, seed=31, spread=0.1)
    rb = lambda: na.RayBundle(**{k: cu(v) for k, v in zip(("origins", "directions", "pl_positions", "nears", "fars"), rays)})
    bg, gt = torch.ones(1, 3).cuda(), torch.full((32, 3), 0.5).cuda()
    rs = np.random.RandomState(4)
    tp, ts, to = (cu(rs.rand(32, k).astype(np.float32)) for k in (1, 64, 32))
    ref, fused = build(), build()
    assert not ref.outside_nerf.compiled
    out = ref(rb(), is_training=True, background_rgb=bg, global_step=20000, _t_rand_primary=tp, _t_rand_shadow=ts, _t_rand_outside=to)
    assert out.weights.shape == (32, 160) and float(out.weights[:, 128:].sum(-1).mean()) > 0.01
    ld = train_loss_dict(out, gt, 0.1)
    ld["loss"].backward()
    l8 = train_fused.train_step_backward(fused, rb(), gt, bg, 20000, t_rand_primary=tp, t_rand_shadow=ts, t_rand_outside=to)
    np.testing.assert_allclose(float(l8[0]), float(ld["loss"].detach()), rtol=2e-5)
    for (name, pa), (_, pf) in zip(ref.named_parameters(), fused.named_parameters()):
        assert pf.grad is not None and pf.grad.shape == pa.shape, name
        scale = float(pa.grad.abs().max()) + 1e-30
        # the tolerance of the compiled background's own fused-against-autograd test
        assert float((pa.grad - pf.grad).abs().max()) < 1e-4 * scale + 5e-6, (name, float((pa.grad - pf.grad).abs().max()), scale)
    cap = build()
    step = GraphedTrainStep(cap, 32, bg, lr=5e-4, warm_up_end=20, global_step=20000)
    assert step._use_fused
    before = {k: v.detach().clone() for k, v in cap.outside_nerf.named_parameters()}
    losses = [step(rb(), gt, global_step=20000 + i)["loss"] for i in range(4)]
    assert all(np.isfinite(losses)) and abs(losses[0] - float(ld["loss"].detach())) < 0.05 * abs(float(ld["loss"].detach()))
    assert all(float((p.detach() - before[k]).abs().max()) > 0.0 for k, p in cap.outside_nerf.named_parameters() if k.endswith("weight"))
    step.release()
    with torch.no_grad():
        img = ref.eval()(rb(), background_rgb=bg).rgb
    assert torch.isfinite(img).all() and img.shape == (32, 3)


@pytest.mark.parametrize("mode,pl", [("SO3xR3", True), ("SE3", False), ("off", True)])
def test_ray_generator_deterministic_gradients(mode, pl):
    """The same rays bit for bit, gradients equal to the scattered ones up to the order of float32 sums of c terms, and equal to
    themselves on every run; a view index outside the tables refines nothing and receives nothing."""
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    views, n = 7, 5000
    cam = CameraModel(H=64, W=64, cx=32.0, cy=32.0, fx=70.0, fy=70.0)
    cfg = RayGeneratorConfig(cam_opt_mode=mode, pl_opt=pl)
    gens = [RayGenerator(cam, views, cfg).cuda(), RayGenerator(cam, views, cfg, deterministic=True).cuda()]
    for name, p in gens[0].named_parameters():
        p.data.copy_(0.05 * rnd(*p.shape))
        getattr(gens[1], name).data.copy_(p.data)
    poses = torch.eye(4, device="cuda").repeat(n, 1, 1)
    poses[:, :3, 3] = rnd(n, 3)
    idx = torch.randint(0, views, (n, 1), generator=g, device="cuda")
    pb = na.RawPixelBundle(img_indices=idx, h_indices=torch.randint(0, 64, (n, 1), generator=g, device="cuda").float(),
                           w_indices=torch.randint(0, 64, (n, 1), generator=g, device="cuda").float(), poses=poses, pls=rnd(n, 3))
    probe = [rnd(n, 3), rnd(n, 3), rnd(n, 3)]

    def run(rg, bundle):
        rb = rg(bundle)
        rays = (rb.origins, rb.directions, rb.pl_positions)
        grads = torch.autograd.grad(sum((r * p).sum() for r, p in zip(rays, probe)), list(rg.parameters()), retain_graph=False)
        return [r.detach() for r in rays] + [rb.nears.detach(), rb.fars.detach()], grads

    (ra, ga), (rb_, gb) = run(gens[0], pb), run(gens[1], pb)
    assert all(torch.equal(x, y) for x, y in zip(ra, rb_))
    count = int(torch.bincount(idx.reshape(-1)).max())
    for x, y in zip(ga, gb):
        assert x.abs().max() > 0 and float((x - y).abs().max()) <= 2 * count * 2.0 ** -24 * float(12 * sum(p.abs().max() for p in probe) * count)
        assert float((x - y).abs().max()) <= 1e-4 * float(x.abs().max())
    for _ in range(3):
        again = run(gens[1], pb)[1]
        assert all(torch.equal(x, y) for x, y in zip(gb, again))
    bad = na.RawPixelBundle(img_indices=torch.where(torch.arange(n, device="cuda")[:, None] % 3 == 0, torch.full_like(idx, views + 2), idx),
                            h_indices=pb.h_indices, w_indices=pb.w_indices, poses=pb.poses, pls=pb.pls)
    (ra, ga), (rb_, gb) = run(gens[0], bad), run(gens[1], bad)
    assert all(torch.equal(x, y) for x, y in zip(ra, rb_)) and all(float((x - y).abs().max()) <= 1e-4 * float(x.abs().max()) for x, y in zip(ga, gb))
