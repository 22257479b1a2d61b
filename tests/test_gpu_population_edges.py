"""GPU: gs_sample, gs_relocate and the bindings of both at the ends of their ranges."""
import numpy as np
import pytest
import torch

from opensplat_amd import cabi
from tests.test_gpu_population import check_relocate, check_sample, dev, gaussian_set, logits_of, records
from tests.test_gpu_train_population import setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [7, 600, 9001])
@pytest.mark.parametrize("top", [-600.0, -657.0, -660.0, -680.0, -690.0, -699.0, -701.0, -5000.0])
def test_sample_opacities_that_are_all_far_below(cols, top):
    """Opacity logits whose largest lies near the smallest powers of two that a weight is made of."""
    rng = np.random.default_rng(cols)
    x = np.full((1, cols), -1e6, np.float32)
    x[0, cols // 2], x[0, cols // 3] = top, top - 5.0
    x[0, 0] = top - 1.0
    u = dev(np.concatenate([rng.random(200), [0.0, 0.999]]).astype(np.float32)[None])
    for kw in (dict(), dict(temperature=0.5), dict(top_p=0.9), dict(top_k=2)):
        got = check_sample(dev(x), u, True, **kw)
        assert set(got[0]) <= {0, cols // 3, cols // 2}


@pytest.mark.parametrize("logit", [-38.0, -60.0, -100.0, -700.0, -744.0, -746.0, -800.0, -1e30, -np.inf])
@pytest.mark.parametrize("copies", [1, 2, 100])
def test_relocate_sources_of_next_to_no_opacity(logit, copies):
    """o' = o / m and the extent stays, to 2^-54 of it for o below e^-37: logit' = x - log m, the scales as they are."""
    rng = np.random.default_rng(copies)
    p, _, _ = gaussian_set(rng, copies + 3, 4, moments=False)
    p[3][1] = logit
    gpu = [dev(a) for a in p]
    cabi.relocate(gpu, None, None, dev(np.arange(2, copies + 2, dtype=np.int32)), dev(np.ones(copies, np.int32)), 1e-38)
    low = np.log(np.float64(np.float32(1e-38)))
    want = max(logit - np.log(copies + 1.0), low)
    got, scales = gpu[3].cpu().numpy().reshape(-1)[1:copies + 2], gpu[1].cpu().numpy()[1:copies + 2]
    assert (np.abs(got - want) <= 2.0 ** -24 * 1.001 * abs(want)).all(), (got, want)
    assert (scales == p[1][1]).all()


def test_relocate_does_not_hide_a_nan():
    """A source whose logit is NaN: it and its copies get NaN logits and scales, no other row does."""
    for pairs in (2, 3000):
        rng = np.random.default_rng(pairs)
        p, _, _ = gaussian_set(rng, 2 * pairs + 2, 1, moments=False)
        p[3][0] = np.nan
        gpu = [dev(a) if a is not None else None for a in p]
        t = np.arange(2, pairs + 2, dtype=np.int32)
        s = np.where(t % 2 == 0, 0, t + pairs).astype(np.int32)
        cabi.relocate(gpu, None, None, dev(t), dev(s))
        named = np.zeros(len(p[0]), bool)
        named[0] = named[t[s == 0]] = True
        assert np.array_equal(np.isnan(gpu[3].cpu().numpy().reshape(-1)), named)
        assert np.array_equal(np.isnan(gpu[1].cpu().numpy()).all(1), named)
        assert np.array_equal(gpu[0].cpu().numpy()[t], p[0][s])


@pytest.mark.parametrize("min_opacity", [0.005, 0.02, 0.1])
def test_growth_from_sources_that_the_copying_left_at_the_bound(min_opacity):
    """One living Gaussian, just above the bound, takes all the others: every share stands at the bound, as gs_relocate
    rounds it, and the set still grows by copies of it."""
    T, cams, gts, bg = setup(N=500, strategy="relocate", refine_every=1, warmup_length=0, max_gaussians=600,
                             min_opacity=min_opacity)
    T.params.v_opacity[:] = -12.0
    T.params.v_opacity[77] = float(np.log(min_opacity / (1 - min_opacity))) + 0.01
    T.render(cams[0], bg, 1)
    assert T.after_train(1) == dict(relocated=499, added=25) and T.N == 525
    for t in (T.features_dc, T.features_rest, T.quats):
        assert torch.equal(t[500:], t[77:78].expand_as(t[500:]))
    # (each source's own copies share its extent: near the one that all come from, which nothing else is)
    assert float((T.log_scales[500:] - T.log_scales[77]).abs().max()) < 0.1
    assert (T.opacity_logits == T.opacity_logits[77]).all()


def test_growth_without_a_source_adds_nothing_that_is_seen():
    """All that is alive is NaN: no source can be drawn."""
    T, cams, gts, bg = setup(N=400, strategy="relocate", refine_every=1, warmup_length=0, max_gaussians=500)
    T.params.v_opacity[:] = -9.0
    T.params.v_opacity[5] = float("nan")
    T.render(cams[0], bg, 1)
    assert T.after_train(1) == dict(relocated=399, added=20)
    new = slice(400, 420)
    assert (torch.sigmoid(T.opacity_logits[new]) < 1 / 255).all() and torch.isfinite(T.params.v_means[new]).all()
    assert torch.equal(T.quats[new].norm(dim=1), torch.ones(20, device="cuda"))


def test_bounds_that_are_none_in_float32_are_refused():
    for low in (1.0 - 1e-9, 1e-60, float("nan")):
        with pytest.raises(ValueError):
            setup(N=50, strategy="relocate", min_opacity=low)


@pytest.mark.parametrize("rows,draws", [(1, 4336), (1, 4337), (2, 4608), (2, 4609), (2, 120_000), (17, 73_729), (20, 9000)])
def test_sample_many_draws_behind_a_top_k_of_few(rows, draws):
    """Long rows whose candidates fit a list, with few draws and with many: one workgroup's, or the whole chip's."""
    rng = np.random.default_rng(draws)
    x = logits_of(rng, rows, 20_000, "f32")
    x[rows // 2] = -np.inf
    x[rows // 2, 3_000:3_040] = 0.5
    u = dev(rng.random((rows, draws), dtype=np.float32))
    check_sample(x, u, top_k=700)
    check_sample(x, u, top_k=dev(np.resize(np.array([30, 0, 4000], np.int32), rows)), temperature=0.7, top_p=0.8)


def test_second_derivative_of_the_balance_loss_is_refused():
    """The gradient's own derivative with respect to the opacities is not formed: asking for it is an error, not 0.  With
    respect to a factor of the loss it is the gradient."""
    from opensplat_amd import ops

    p, bins, _, _ = records(np.random.default_rng(1), 300, 200, 120)
    packed, bins = torch.from_numpy(p).cuda(), torch.from_numpy(bins).cuda()
    o = packed[:, 5].clone().requires_grad_(True)
    f = torch.tensor(2.0, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(f * ops.tile_balance(o, packed, bins, 120, 200), o, create_graph=True)
    want = cabi.tile_balance(200, 120, packed, bins)[2]
    assert torch.equal(g.detach(), 2.0 * want)
    d, = torch.autograd.grad(g.square().sum(), f, retain_graph=True)
    assert abs(float(d) - 4.0 * float(want.double().square().sum())) <= 1e-5 * abs(float(d))
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.sum(), o, retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    # an optimiser's step between the forward and the backward, as before
    loss = ops.tile_balance(o, packed, bins, 120, 200)
    with torch.no_grad():
        o.add_(1.0)
    loss.backward()
    assert torch.equal(o.grad, want)


def test_numbers_that_do_not_fit_the_c_abi_are_refused():
    """32-bit sizes and settings: a larger one is an error, not its low half."""
    x, u = torch.zeros((1, 20), device="cuda"), torch.rand((1, 8), device="cuda")
    for k in (2 ** 31, 2 ** 32 + 1, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            cabi.sample(x, u, top_k=k)
    assert cabi.sample(x, u, top_k=2 ** 31 - 1).shape == (1, 8)
    wide = torch.empty(2 ** 32 + 5, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        cabi.sample(wide, u[0])
    del wide
    many = torch.empty(2 ** 32, device="cuda", dtype=torch.float32)
    with pytest.raises(ValueError):
        cabi.sample(x[0], many)
    with pytest.raises(ValueError):
        cabi.sample(many.view(-1, 1), many.view(-1, 1))
    i = many.view(torch.int32)
    p = [torch.zeros(s, device="cuda") for s in ((9, 3), (9, 3), (9, 4), (9, 1), (9, 3))] + [None]
    with pytest.raises(ValueError):
        cabi.relocate(p, None, None, i, i)
    del many, i
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [511, 512, 513, 767, 768, 769, 1023, 1025, 2047, 2049])
def test_relocate_around_the_launch_forms(n):
    """One workgroup's phases and three launches give the same; among the pairs some that do not hold."""
    rng = np.random.default_rng(n)
    N = 3 * n
    order = rng.permutation(N)
    targets, sources = order[:n].astype(np.int64), order[n:][(rng.random(n) ** 3 * n).astype(int)]
    targets[5], targets[n - 1], sources[7], sources[n // 2] = targets[n - 2], -1, targets[3], N
    check_relocate(gaussian_set(rng, N, 4), targets.tolist(), sources.tolist())


def test_tile_balance_of_a_4k_frame_captured():
    """A table that takes most of the LDS, asked for inside a capture; replayed with eager calls between."""
    p, bins, lists, _ = records(np.random.default_rng(0), 4000, 3840, 2160)
    packed, bins = dev(p), dev(bins)
    want = [t.clone() for t in cabi.tile_balance(3840, 2160, packed, bins)]
    assert np.array_equal(want[1].cpu().numpy(), lists)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = cabi.tile_balance(3840, 2160, packed, bins)
    for turn in range(4):
        for t in out:
            t.zero_()
        packed[:, 5] = packed[:, 5].roll(turn)
        want = [t.clone() for t in cabi.tile_balance(3840, 2160, packed, bins)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_balance_through_the_factored_exchange():
    """The opacities' gradient is the flat exchange's to the bit; one camera and a batch."""
    grads = []
    for exchange in ("flat", "factored"):
        T, cams, gts, bg = setup(balance_weight=0.4, deterministic=True, exchange=exchange)
        T.factored = exchange == "factored"
        T.train_step(cams[0], gts[0], bg, 1)
        one = T.grads.v_opacity.clone()
        T2, _, _, _ = setup(balance_weight=0.4, deterministic=True, exchange=exchange)
        T2.train_step_batch(cams, gts, bg, 1, step_optimizer=False)
        torch.cuda.synchronize()
        grads.append((one, T2.grads.v_opacity.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*grads)) and (grads[0][0] != 0).any()


@pytest.mark.parametrize("K", [1, 9])
def test_a_budget_with_other_numbers_of_bases(K):
    T, cams, gts, bg = setup(N=1500, K=K, strategy="relocate", refine_every=2, warmup_length=0, max_gaussians=1700,
                             balance_weight=0.01)
    for step in range(1, 9):
        T.params.v_opacity[step::50] = -8.0
        T.train_step_batch(cams, gts, bg, 0 if K == 1 else 1, step=step)
        c = T.after_train(step)
        assert (c is None) == (step % 2 == 1)
    assert T.N == 1700 and all(torch.isfinite(t).all() for t in T._param_list(T.params) if t is not None)


def test_sample_in_a_workspace_of_the_callers():
    """One workspace for calls of other shapes, in stream order; one byte less is refused, as is one at an odd address."""
    rng = np.random.default_rng(3)
    need = max(cabi.lib().gs_sample_workspace_bytes(r, c) for r, c in ((3, 20_000), (1, 70_000), (5, 900)))
    ws = torch.full((need + 64,), 0xA5, device="cuda", dtype=torch.uint8)
    for r, c in ((3, 20_000), (1, 70_000), (5, 900), (3, 20_000)):
        x, u = logits_of(rng, r, c, "f32"), dev(rng.random((r, 20), dtype=np.float32))
        for kw in (dict(), dict(top_k=30, top_p=0.7), dict(top_p=0.7), dict(top_k=9000)):
            got = cabi.sample(x, u, workspace=ws[:need], **kw)
            assert torch.equal(got, cabi.sample(x, u, **kw))
            assert (ws[need:] == 0xA5).all()
    x, u = logits_of(rng, 1, 70_000, "f32"), dev(rng.random((1, 20), dtype=np.float32))
    with pytest.raises(ValueError):
        cabi.sample(x, u, workspace=ws[:cabi.lib().gs_sample_workspace_bytes(1, 70_000) - 1])
    with pytest.raises(RuntimeError):
        cabi.sample(x, u, workspace=ws[8:])


def test_sample_a_row_of_two_thousand_million():
    """Indices, chunks and places of a row that ends shortly before 2^31 entries."""
    n = 2_000_000_011
    x = torch.full((n,), -torch.inf, device="cuda", dtype=torch.float16)
    at = torch.tensor([7, 4096, 1_073_741_823, 1_073_741_824, 1_999_999_999, n - 1])
    x[at.cuda()] = torch.tensor([0.0, 1.0, 1.0, -1.0, 2.0, 1.0], dtype=torch.float16).cuda()
    u = torch.linspace(0, 1 - 2.0 ** -24, 301)
    w = torch.exp(x[at.cuda()].double().cpu() - 2.0)

    def want(keep):
        mass = (w * keep).cumsum(0)
        return at[torch.searchsorted(mass, u.double() * mass[-1], right=True)].int()

    every = torch.ones(6)
    for kw, keep in ((dict(), every), (dict(top_k=3), torch.tensor([0, 1, 1, 0, 1, 0])), (dict(min_p=0.2), w >= 0.2),
                     (dict(top_p=0.5), torch.tensor([0, 1, 0, 0, 1, 0]))):
        assert torch.equal(cabi.sample(x, u.cuda(), **kw).cpu(), want(keep)), kw
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(1, 28, 512), (1, 28, 513), (1, 400, 70_000), (3, 1500, 2049), (2, 8192, 8193),
                                   (1, 8160, 100_001), (600, 2100, 9000), (9000, 10, 600)])
def test_sample_many_draws_of_short_rows(shape):
    """A row's draws shared by several workgroups; where the rows fill the chip, by one each."""
    rows, cols, draws = shape
    rng = np.random.default_rng(draws)
    x = logits_of(rng, rows, cols, "f32", pad=1)
    x[rows // 2, cols // 2:] = -np.inf
    if rows > 2:
        x[1] = np.nan
    u = dev(rng.random((rows, draws), dtype=np.float32))
    # (the temperature as the call takes it: of five million draws, some lie closer to a border than 0.8 to its float32)
    check_sample(x, u, temperature=float(np.float32(0.8)), top_p=0.9)


def test_sample_long_rows_on_two_streams_at_once():
    rng = np.random.default_rng(8)
    calls = []
    for r, c, kw in ((3, 60_000, dict(top_p=0.9)), (2, 200_000, dict(top_k=20_000, top_p=0.7)), (1, 500_000, dict()),
                     (4, 30_000, dict(top_k=100))):
        calls.append((logits_of(rng, r, c, "f32"), dev(rng.random((r, 500), dtype=np.float32)), kw))
    want = [cabi.sample(x, u, **kw) for x, u, kw in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(6):
        for k, (x, u, kw) in enumerate(calls):
            with torch.cuda.stream(streams[(turn + k) % 2]):
                got.append((k, cabi.sample(x, u, **kw)))
    torch.cuda.synchronize()
    assert all(torch.equal(ids, want[k]) for k, ids in got)
