"""GPU: the paths that call gs_sample, gs_relocate and gs_tile_balance — Trainer(strategy="relocate"),
Trainer(balance_weight=...) — and the C++ operators over them."""
import numpy as np
import pytest
import torch

from opensplat_amd import cabi, scenes
from tests import population_oracle as orc

pytestmark = pytest.mark.gpu


def setup(N=6000, W=256, H=160, K=4, ncam=3, **kw):
    from opensplat_amd.train import Trainer

    s = scenes.camera_scene(N, W, H, K=K, seed=5, sigma_px=(0.6, 5.0), znear=1.0, zfar=100.0)
    T = Trainer(*scenes.raw_parameters(s), device="cuda:0", sh_degree_interval=1, **kw)
    cams, gts = [], []
    for j, yaw in enumerate((-6.0, 1.0, 7.0)[:ncam]):
        vm, pm = scenes.yaw_camera(W, H, yaw, 1.0, 100.0)
        cams.append(dict(viewmat=vm, projmat=pm, fx=s.fx, fy=s.fy, cx=s.cx, cy=s.cy, W=W, H=H))
        gts.append(torch.from_numpy(np.random.RandomState(40 + j).uniform(0, 1, (H, W, 3)).astype(np.float32)).cuda())
    return T, cams, gts, torch.zeros(3, device="cuda")


def kill(T, share, seed=0):
    dead = torch.from_numpy(np.random.default_rng(seed).random(T.N) < share).cuda()
    T.params.v_opacity[dead] = -7.0
    return dead


def test_relocation_moves_the_dead_onto_drawn_sources():
    T, cams, gts, bg = setup(strategy="relocate", refine_every=10, warmup_length=5, max_steps=1000)
    T.exp_avg.flat.normal_()
    kill(T, 0.1)
    dead = T.opacity_logits <= float(np.log(0.005 / 0.995))      # (some of the scene were there already)
    before = [t.clone() for t in T._param_list(T.params)]
    T.render(cams[0], bg, 1)
    assert T.after_train(7) is None and T.after_train(500) is None
    c = T.after_train(10)
    n = int(dead.sum())
    assert c == dict(relocated=n, added=0) and T.N == 6000
    # every dead row holds a living row's features, at its share of the opacity; living rows kept theirs
    dc, old = T.features_dc, before[4]
    assert torch.equal(dc[~dead], old[~dead])
    key = {tuple(r): i for i, r in enumerate(old.cpu().numpy().tolist())}
    src = torch.tensor([key[tuple(r)] for r in dc[dead].cpu().numpy().tolist()], device="cuda")
    assert not dead[src].any()
    times = torch.bincount(src, minlength=T.N)
    logit, shrink = orc.shares(before[3].view(-1)[src].cpu().numpy(), times[src].cpu().numpy() + 1, 0.005)
    assert np.abs(T.opacity_logits[dead].cpu().numpy() - logit).max() < 1e-5
    assert torch.equal(T.opacity_logits[src], T.opacity_logits[dead])
    assert np.abs((T.log_scales[dead] - before[1][src]).cpu().numpy() - shrink[:, None]).max() < 1e-5
    assert torch.equal(T.means[~dead], before[0][~dead])
    far = (T.means[dead] - before[0][src]) / T.log_scales[dead].exp().amax(1, keepdim=True)
    assert 0 < float(far.abs().max()) < 2.5
    for i in (dead.nonzero().view(-1), src):
        assert all((t[i] == 0).all() for t in T._param_list(T.exp_avg))
    rest = ~dead & (times == 0)
    assert (T.exp_avg.v_means[rest] != 0).any()
    T.train_step(cams[0], gts[0], bg, 1)


def test_the_set_grows_to_its_budget_and_no_further():
    T, cams, gts, bg = setup(N=2000, strategy="relocate", refine_every=2, warmup_length=0, max_gaussians=2300)
    sizes = []
    for step in range(1, 13):
        T.train_step(cams[step % 3], gts[step % 3], bg, 1)
        c = T.after_train(step)
        if c is not None:
            sizes.append(T.N)
    assert sizes == [2100, 2205, 2300, 2300, 2300, 2300]
    assert all(torch.isfinite(t).all() for t in T._param_list(T.params))
    assert T.grads.N == 2300 and T.exp_avg.N == 2300


def test_equal_trainers_stay_equal():
    """Draws depend on the step and the parameters alone: what keeps ranks together."""
    out = []
    for _ in range(2):
        T, cams, gts, bg = setup(N=3000, strategy="relocate", refine_every=3, warmup_length=0, max_gaussians=3300,
                                 balance_weight=0.01, deterministic=True, source_temperature=0.8, source_top_p=0.95)
        for step in range(1, 10):
            T.train_step(cams[step % 3], gts[step % 3], bg, 1)
            if step == 2:
                kill(T, 0.05)
            T.after_train(step)
        out.append(T.params.flat.clone())
    assert torch.equal(*out)


def test_nothing_alive_and_nothing_dead():
    T, cams, gts, bg = setup(N=500, strategy="relocate", refine_every=1, warmup_length=0, max_gaussians=600)
    T.render(cams[0], bg, 1)
    kill(T, 1.1)
    was = T.params.flat.clone()
    assert T.after_train(1) == dict(relocated=0, added=0) and torch.equal(T.params.flat, was)
    T.params.v_opacity[:] = 1.0
    c = T.after_train(2)
    assert c["relocated"] == 0 and c["added"] == 25 and T.N == 525


@pytest.mark.parametrize("graph", [False, True])
def test_balance_gradient_joins_the_opacities(graph):
    """The step's opacity gradient is the image's plus the balance loss's on the frame's own lists: one float32 addition."""
    from tests.util import np_

    grads = []
    for w in (0.0, 0.5):
        T, cams, gts, bg = setup(balance_weight=w, deterministic=True, experimental_graph=graph)
        T.train_step(cams[0], gts[0], bg, 1)
        torch.cuda.synchronize()
        grads.append({k: t.clone() for k, t in T.grads.views.items()})
        b = T._ctx[4]
    loss, counts, v = cabi.tile_balance(256, 160, b.packed, b.tile_bins, 0.5, cabi.GS_FLAG_LOGIT_OPACITY)
    assert float(v.abs().max()) > 0
    assert torch.equal(grads[1]["v_opacity"], grads[0]["v_opacity"] + v)
    for k in grads[0]:
        if k != "v_opacity":
            assert torch.equal(grads[0][k], grads[1][k]), k
    assert torch.equal(T.balance_out[0], loss) and torch.equal(T.balance_out[1], counts)
    assert np.isfinite(np_(T.params.flat)).all()


def test_balance_of_a_camera_batch():
    """Two in flight equals the serial loop's bits; the sum over the cameras, each with its share of the weight."""
    T, cams, gts, bg = setup(balance_weight=0.3, deterministic=True)
    T0, _, _, _ = setup(deterministic=True)
    T.train_step_batch(cams, gts, bg, 1, step_optimizer=False, serial=True)
    a = T.grads.v_opacity.clone()
    T.train_step_batch(cams, gts, bg, 1, step_optimizer=False)
    torch.cuda.synchronize()
    assert torch.equal(a, T.grads.v_opacity)
    T0.train_step_batch(cams, gts, bg, 1, step_optimizer=False)
    want = T0.grads.v_opacity.double()
    parts = []
    for c in cams:
        T0.render(c, bg, 1)
        b = T0._ctx[4]
        parts.append(cabi.tile_balance(256, 160, b.packed, b.tile_bins, 0.3 / 3, cabi.GS_FLAG_LOGIT_OPACITY)[2].double())
    # (three image and three balance terms added in float32 in either order: five roundings of partial sums)
    size = sum(p.abs() for p in parts) + want.abs() + max(float(p.abs().max()) for p in parts)
    assert ((a.double() - want - sum(parts)).abs() <= 8 * 2.0 ** -24 * size + 2.0 ** -20 * want.abs().max()).all()


def test_balance_reaches_a_replaced_gradient_buffer():
    """A refinement that leaves the set's size as it was still replaces the gradient buffer."""
    from opensplat_amd import dist

    T, cams, gts, bg = setup(balance_weight=0.3, deterministic=True)
    T.train_step_batch(cams, gts, bg, 1, step_optimizer=False)
    want = T.grads.v_opacity.clone()
    T.grads = dist.GradBuffer(T.N, T.K, T.dev)
    T._shape = None
    T.train_step_batch(cams, gts, bg, 1, step_optimizer=False)
    torch.cuda.synchronize()
    assert torch.equal(T.grads.v_opacity, want)


def test_refused_arguments():
    for kw in (dict(strategy="other"), dict(min_opacity=0.0), dict(source_temperature=0.0), dict(source_top_p=0.0),
               dict(strategy="relocate", reference_alpha_reset=True)):
        with pytest.raises(ValueError):
            setup(N=50, **kw)


def test_operators_over_the_same_calls():
    from opensplat_amd import ops

    rng = np.random.default_rng(1)
    x = torch.randn((4, 900), device="cuda").bfloat16()[:, :777]
    u = torch.rand((4, 5), device="cuda")
    t, k = torch.rand(4, device="cuda") + 0.5, torch.tensor([5, 0, 100, 1], device="cuda", dtype=torch.int32)
    assert torch.equal(ops.sample_indices(x, u, t, k), cabi.sample(x, u, t, k))
    assert torch.equal(ops.sample_indices(x, u, opacity=True), cabi.sample(x, u, opacity=True))
    from tests.test_gpu_population import gaussian_set, records

    p, bins, _, _ = records(rng, 400, 200, 120)
    packed, bins = torch.from_numpy(p).cuda(), torch.from_numpy(bins).cuda()
    logits = torch.logit(packed[:, 5]).view(-1, 1).requires_grad_(True)
    loss = ops.tile_balance(logits, packed, bins, 120, 200, True)
    (3.0 * loss).backward()
    want = cabi.tile_balance(200, 120, packed, bins, 1.0, cabi.GS_FLAG_LOGIT_OPACITY)
    assert loss.shape == () and torch.equal(loss.detach().view(1), want[0])
    assert torch.equal(logits.grad.view(-1), 3.0 * want[2])
    sets = gaussian_set(rng, 100, 4)
    a, b = ([[torch.from_numpy(t).cuda() for t in s] for s in sets] for _ in range(2))
    i = torch.arange(20, device="cuda", dtype=torch.int32)
    ops.relocate(*a, i, i + 50)
    cabi.relocate(*b, i, i + 50)
    assert all(torch.equal(x, y) for s, r in zip(a, b) for x, y in zip(s, r))
    bad = [lambda: ops.sample_indices(x.double(), u), lambda: ops.sample_indices(x, u.cpu()),
           lambda: ops.sample_indices(x[:, ::2], u), lambda: ops.sample_indices(x, u, t[:2]),
           lambda: ops.tile_balance(logits, packed, bins, 160, 200), lambda: ops.relocate(*a, i.long(), i),
           lambda: ops.relocate(a[0][:5], [], [], i, i), lambda: cabi.sample(x, u, temperature=-1.0),
           lambda: cabi.sample(x, u, top_k=k.long()), lambda: cabi.tile_balance(200, 160, packed, bins),
           lambda: cabi.tile_balance(200, 120, packed, bins, flags=cabi.GS_FLAG_ACCUMULATE_GRADS),
           lambda: cabi.relocate(*a, i, i[:3]), lambda: cabi.relocate([t[:50] if t.dim() < 2 else t for t in a[0]], None, None, i, i.long())]
    for f in bad:
        with pytest.raises((RuntimeError, ValueError)):
            f()
