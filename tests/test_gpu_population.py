"""GPU: gs_sample, gs_tile_balance and gs_relocate against their definitions in 64 bits and more."""
import numpy as np
import pytest
import torch

from tests import population_oracle as orc

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t.to(dtype) if dtype is not None else t).cuda()


def host(t):
    return t.detach().float().cpu().numpy()


# ---- sample ---------------------------------------------------------------------------------------------------
# Ids are whole numbers and have to be equal: the kernels' weights carry a relative error of a few 2^-50 (64-bit exp of a
# product, log1p), their sums less than 2^-48; the draws of these tests lie further than that from every border but
# where weights and goals are exact in both (equal weights, u = 0).

def check_sample(x, u, opacity=False, **kw):
    """x: GPU logits [R, V], u: GPU uniforms [R, D]."""
    from opensplat_amd import cabi

    got = cabi.sample(x, u, opacity=opacity, **kw).cpu().numpy()
    ref = {k: (v.cpu().numpy() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    want = orc.sample(host(x), u.cpu().numpy(), opacity=opacity, **ref)
    assert np.array_equal(got, want), (np.argwhere(got != want)[:8].tolist(), got[got != want][:8], want[got != want][:8])
    return got


def logits_of(rng, rows, cols, dt, pad=0, spread=2.5):
    x = rng.standard_normal((rows, cols + pad)).astype(np.float32) * spread
    return dev(x, DT[dt])[:, :cols]


SIZES = [(1, 1, 1), (1, 2, 5), (3, 28, 1), (5, 63, 7), (2, 64, 64), (4, 65, 3), (1, 511, 100), (2, 513, 9), (7, 1025, 2),
         (1, 2047, 50), (3, 4097, 11), (2, 8160, 64), (1, 8193, 8), (5, 16385, 3), (2, 33000, 5), (1, 131072, 300),
         (1, 262147, 1000)]
SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=3), dict(top_p=0.8), dict(min_p=0.05),
            dict(temperature=1.3, top_k=40, top_p=0.9, min_p=0.01)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("opt", range(len(SETTINGS)))
def test_sample_sizes_and_settings(size, opt):
    rows, cols, draws = size
    rng = np.random.default_rng(1000 * opt + cols)
    dt = ("f32", "bf16", "f16")[(cols + opt) % 3]
    x = logits_of(rng, rows, cols, dt, pad=(0, 1, 8, 13)[(cols + opt) % 4])
    u = dev(rng.random((rows, draws), dtype=np.float32))
    check_sample(x, u, **SETTINGS[opt])


@pytest.mark.parametrize("cols", [5, 700, 9000, 70001])
@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("opacity", [False, True])
def test_sample_settings_per_row(cols, dt, opacity):
    rng = np.random.default_rng(cols)
    rows = 9
    x = logits_of(rng, rows, cols, dt, pad=5)
    lens = np.maximum(1, (cols * np.linspace(0.1, 1, rows)).astype(int))
    for r in range(rows):
        x[r, lens[r]:] = -np.inf
    x[4] = -np.inf                                             # a row that the mask leaves empty
    u = dev(rng.random((rows, 6), dtype=np.float32))
    f = lambda *v: dev(np.array(v, np.float32))  # noqa: E731
    kw = dict(temperature=f(1, 0.5, 0, 2, 1, 1e-3, 1, 0.9, 100), top_p=f(1, 0.9, 0.5, 0, 0.5, 1.5, 0.99, 0.3, 0.999),
              min_p=f(0, 0.01, 0, 0, 0.1, 0, 2.0, 1.0, -1), top_k=dev(np.array([0, 7, 3, 0, 1, 10**9, 50, -5, 2], np.int32)))
    got = check_sample(x, u, opacity, **kw)
    assert (got[4] == -1).all()


@pytest.mark.parametrize("cols", [300, 8192, 40000])
def test_sample_bad_settings_of_a_row_draw_nothing(cols):
    rng = np.random.default_rng(5)
    x, u = logits_of(rng, 5, cols, "f32"), dev(rng.random((5, 4), dtype=np.float32))
    nan = float("nan")
    f = lambda *v: dev(np.array(v, np.float32))  # noqa: E731
    got = check_sample(x, u, temperature=f(1, -1, nan, 1, 1), top_p=f(1, 1, 1, nan, 1), min_p=f(0, 0, 0, 0, nan))
    assert (got[1:] == -1).all() and (got[0] >= 0).all()


@pytest.mark.parametrize("cols", [33, 5000, 8193, 100003])
@pytest.mark.parametrize("opt", [dict(), dict(top_k=17), dict(top_p=0.5), dict(top_k=1000, top_p=0.25), dict(min_p=1.0)])
def test_sample_equal_values_and_masks(cols, opt):
    """All entries equal; all at the type's lowest value; two values only; infinities and NaN among them."""
    rng = np.random.default_rng(cols)
    rows = np.zeros((7, cols), np.float32)
    rows[1] = np.finfo(np.float32).min
    rows[2] = np.where(rng.random(cols) < 0.3, 1.0, 0.0)
    rows[3] = np.where(rng.random(cols) < 0.5, np.nan, np.where(rng.random(cols) < 0.5, -np.inf, -1.0))
    rows[4, ::3] = np.inf
    rows[5] = np.where(rng.random(cols) < 0.5, np.finfo(np.float32).min, 0.25)
    rows[6] = np.where(rng.random(cols) < 0.5, -0.0, 0.0)
    u = rng.random((7, 40), dtype=np.float32)
    u[:, 0], u[:, 1], u[:, 2], u[:, 3] = 0.0, 1.0 - 2.0 ** -24, 1.0, np.nan
    u[:, 4], u[:, 5] = -0.5, 7.0
    check_sample(dev(rows), dev(u), **opt)


@pytest.mark.parametrize("cols", [100, 60000])
@pytest.mark.parametrize("dt", sorted(DT))
def test_sample_top_k_cuts_among_equal_values(cols, dt):
    """Values on a coarse grid: every border lies among ties, the lowest indices stay."""
    rng = np.random.default_rng(3)
    x = dev(np.round(rng.standard_normal((6, cols)) * 2).astype(np.float32) / 2, DT[dt])
    u = dev(rng.random((6, 50), dtype=np.float32))
    k = dev(np.array([1, 2, 5, cols // 3, cols - 1, cols], np.int32))
    check_sample(x, u, top_k=k)
    check_sample(x, u, top_k=k, top_p=0.77, temperature=0.6)


def test_sample_opacity_extremes():
    x = np.array([[-1000, -88, -20, -1, 0, 1, 20, 40, 90, np.inf, -np.inf, np.nan, -3.4e38]], np.float32)
    u = dev(np.linspace(0, 0.999, 77, dtype=np.float32)[None])
    for kw in (dict(), dict(temperature=0.3), dict(top_k=4), dict(temperature=30.0)):
        check_sample(dev(x), u, True, **kw)
    check_sample(dev(x[:, [0, 1, 12]]), u, True)
    check_sample(dev(x[:, [0, 12]] * 1.0), u, True, temperature=200.0)


def test_sample_frequencies_follow_the_weights():
    """A grid of uniforms counts every index within one step of its share."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal(50).astype(np.float32)
    n = 1 << 16
    from opensplat_amd import cabi

    ids = cabi.sample(dev(x), (torch.arange(n, device="cuda", dtype=torch.float32) + 0.5) / n).cpu().numpy()
    w = np.exp(x.astype(np.float64)) / np.exp(x.astype(np.float64)).sum()
    assert np.abs(np.bincount(ids, minlength=50) - n * w).max() <= 1.0 + 1e-6


def test_sample_large_row_with_many_draws():
    rng = np.random.default_rng(11)
    x = np.minimum(rng.standard_normal((1, 1_200_000)).astype(np.float32) * 2, np.float32(np.log(0.25)))
    x[rng.random(x.shape) < 0.05] = -np.inf
    u = dev(rng.random((1, 60_000), dtype=np.float32))
    check_sample(dev(x), u, True)
    check_sample(dev(x), u, True, top_p=0.9)
    check_sample(dev(x), u, True, top_k=700_001, min_p=0.5)


@pytest.mark.parametrize("opt", [dict(), dict(top_k=9_000_000, min_p=0.2), dict(top_p=0.7, temperature=0.5)])
def test_sample_row_of_more_chunks_than_a_table_holds(opt):
    """17 M entries: the forms for rows whose chunks' maxima and running sums do not fit beside a workgroup."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1, 17_000_003), device="cuda", generator=g).bfloat16()
    x[0, 5_000_000:6_000_000] = -torch.inf
    for draws in (7, 20_000):
        check_sample(x, torch.rand((1, draws), device="cuda", generator=g), **opt)


@pytest.mark.parametrize("shape", [(3000, 28, 2), (700, 1500, 3), (300, 8000, 2), (300, 9000, 40)])
def test_sample_many_rows(shape):
    rows, cols, draws = shape
    rng = np.random.default_rng(rows)
    x, u = logits_of(rng, rows, cols, "f16", pad=3), dev(rng.random((rows, draws), dtype=np.float32))
    x[::7] = -np.inf
    p = dev((0.3 + 0.8 * rng.random(rows)).astype(np.float32))
    k = dev(rng.integers(0, 60, rows).astype(np.int32))
    check_sample(x, u, top_p=p, top_k=k, temperature=0.9)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("size", [(1, 2_097_152), (1, 2_097_153), (1, 4_194_305), (6, 8193), (6, 100_000)])
def test_sample_top_k_where_few_or_many_candidates_are_left(size, dt):
    """Top-k rows whose candidates behind the first digit fit one workgroup (8192 entries), just do not, are fewer than k,
    stand in one place or all over the row; greedy and unlimited rows beside them."""
    rows, cols = size
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32) * 0.1 - 3.0
    for r in range(rows):
        top = (8192, 8193, 100, 5000, 8191, 1)[r] if rows > 1 else 3000
        top = min(top, cols)
        at = rng.permutation(cols)[:top] if r % 2 == 0 else np.arange(cols - top, cols)
        x[r, at] = 1.0 + 0.9 * rng.random(top).astype(np.float32)
    if rows > 1:
        x[2, 5000:] = -np.inf
        x[4, :10] = np.nan
    u = dev(rng.random((rows, 9), dtype=np.float32))
    ks = np.array([40, 8000, 7000, 4999, 8191, 3][:rows], np.int32)
    check_sample(dev(x, DT[dt]), u, top_k=dev(ks))
    check_sample(dev(x, DT[dt]), u, True, top_k=dev(ks), top_p=0.6, temperature=0.4)
    check_sample(dev(x, DT[dt]), u, top_k=25, min_p=0.7)
    check_sample(dev(x, DT[dt]), u, top_k=8192)
    check_sample(dev(x, DT[dt]), u, top_k=8193, top_p=0.9)
    if rows > 1:
        t = dev(np.array([1, 0, 0.5, 0, 2, 1], np.float32))
        k = dev(np.array([0, 5, 1, 9000, 0, 20], np.int32))
        p = dev(np.array([0.5, 0.5, 0.5, 1, 1, 0], np.float32))
        check_sample(dev(x, DT[dt]), u, top_k=k, temperature=t, top_p=p)


def test_sample_replays_whose_rows_change_between_lists_and_passes():
    """One captured call of long rows; between its replays the settings and logits change so that the same row is listed in
    one and goes through all the passes in the next."""
    from opensplat_amd import cabi

    rng = np.random.default_rng(4)
    rows, cols = 4, 50_000
    x, u = logits_of(rng, rows, cols, "f32"), dev(rng.random((rows, 5), dtype=np.float32))
    k, t, p = (torch.zeros(rows, device="cuda", dtype=d) for d in (torch.int32, torch.float32, torch.float32))
    kw = dict(top_k=k, temperature=t, top_p=p)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cabi.sample(x, u, **kw)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ids = cabi.sample(x, u, **kw)
    for turn in range(5):
        x.copy_(torch.from_numpy((rng.standard_normal((rows, cols)) * (0.01, 3.0)[turn % 2]).astype(np.float32)))
        u.copy_(torch.from_numpy(rng.random((rows, 5), dtype=np.float32)))
        k.copy_(torch.from_numpy(np.roll(np.array([50, 30_000, 0, 1], np.int32), turn)))
        t.copy_(torch.from_numpy(np.roll(np.array([1, 0.5, 1, 0], np.float32), 2 * turn)))
        p.copy_(torch.from_numpy(np.roll(np.array([0.9, 1, 0.3, 0.7], np.float32), -turn)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = ids.clone()
        assert torch.equal(torch.from_numpy(check_sample(x, u, **kw)).cuda(), got), turn


def test_sample_rows_beyond_32_bit_offsets():
    """The last rows start more than 2^31 elements behind the first."""
    rows, cols, stride = 5, 1000, 600_000_000
    base = torch.empty(4 * stride + cols, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((rows, cols), (stride, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    x.copy_(torch.randn((rows, cols), device="cuda", generator=g))
    u = torch.rand((rows, 9), device="cuda", generator=g)
    check_sample(x, u, top_p=0.9)


def test_sample_empty_calls():
    from opensplat_amd import cabi

    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    assert cabi.sample(z(0, 5), z(0, 3)).shape == (0, 3)
    assert cabi.sample(z(4, 5), z(4, 0)).shape == (4, 0)
    assert (cabi.sample(z(2, 0), z(2, 3)) == -1).all()
    assert cabi.sample(z(5), z(3)).shape == (3,)


# ---- tile balance ---------------------------------------------------------------------------------------------
# The kernel's sums are 64-bit and each output is rounded once: half a step of float32 = 2^-24 relative, to which the
# 64-bit subtraction A - c Q / S adds 2^-50 of its operands.

def records(rng, N, W, H, reach=10.0, seen=0.8):
    c = rng.random((N, 2)) * [W, H]
    r = np.exp(rng.standard_normal((N, 2)) * 0.8 + np.log(reach))
    lo = np.maximum(np.floor(c - r), 0).astype(np.int64)
    hi = np.minimum(np.ceil(c + r) + 1, [W, H]).astype(np.int64)
    ok = (rng.random(N) < seen) & (hi > lo).all(1)
    lo[~ok], hi[~ok] = 0, 0
    p = rng.standard_normal((N, 12)).astype(np.float32)
    p[:, 5] = rng.random(N)
    p[:, 7] = (lo[:, 0] | hi[:, 0] << 16).astype(np.uint32).view(np.float32)
    p[:, 11] = (lo[:, 1] | hi[:, 1] << 16).astype(np.uint32).view(np.float32)
    tw, th = -(-W // 16), -(-H // 16)
    covers, lists = [], np.zeros(tw * th, np.int64)
    for a, b in zip(lo, hi):
        t = np.zeros(0, np.int64)
        if (b > a).all():
            x, y = np.arange(a[0] // 16, -(-b[0] // 16)), np.arange(a[1] // 16, -(-b[1] // 16))
            t = (y[:, None] * tw + x).reshape(-1)
        covers.append(t)
        lists[t] += 1
    ends = np.cumsum(lists)
    return p, np.stack([ends - lists, ends], 1).astype(np.int32), lists, covers


def close(got, want, operands):
    """Half a step of float32 on the value, 2^-48 of the operands of the difference it comes from."""
    assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) * 1.01 + 2.0 ** -48 * operands + 1e-45).all(), \
        np.abs(got - want).max()


@pytest.mark.parametrize("shape", [(1, 16, 16), (1, 1, 1), (7, 17, 33), (300, 100, 50), (2000, 640, 360), (500, 4111, 20),
                                   (500, 20, 4111), (3000, 1920, 1080), (2000, 9999, 1050), (700, 40000, 300)])
@pytest.mark.parametrize("logit", [False, True])
def test_tile_balance(shape, logit):
    from opensplat_amd import cabi

    N, W, H = shape
    rng = np.random.default_rng(N + W)
    p, bins, lists, covers = records(rng, N, W, H, seen=1.0 if N == 1 else 0.8)
    flags = cabi.GS_FLAG_LOGIT_OPACITY if logit else 0
    loss, counts, v = cabi.tile_balance(W, H, dev(p), dev(bins), scale=0.3, flags=flags)
    want, grad = orc.tile_balance(lists, covers, p[:, 5], float(np.float32(0.3)), logit)
    assert np.array_equal(counts.cpu().numpy(), lists)
    S, M = sum(len(t) * float(o) for t, o in zip(covers, p[:, 5])), lists.sum()
    top = 0.3 * len(lists) / max(M * S, 1e-30) * max([lists[t].sum() for t in covers] + [1])
    close(float(loss[0]), want, abs(want))
    close(v.cpu().numpy().astype(np.float64), grad, top)
    # again, added to what is there; and the value alone
    base = torch.randn(N, device="cuda")
    acc = base.clone()
    out = (torch.empty(1, device="cuda"), None, acc)
    cabi.tile_balance(W, H, dev(p), dev(bins), scale=0.3, flags=flags | cabi.GS_FLAG_ACCUMULATE_GRADS, out=out)
    assert torch.equal(acc, base + v) and torch.equal(out[0], loss)
    again = cabi.tile_balance(W, H, dev(p), dev(bins), scale=0.3, flags=flags, want_grad=False)
    assert again[2] is None and torch.equal(again[0], loss) and torch.equal(again[1], counts)


def test_tile_balance_against_differences():
    """d loss / d opacity of a few Gaussians from central differences of the loss itself (the counts do not depend on
    the opacity).  The loss is a ratio of linear functions of one opacity: over a step h the difference quotient is off
    by h^2 c^2 / S^2 of the slope, and by a rounding of each loss, 2^-24 loss / h."""
    from opensplat_amd import cabi

    rng = np.random.default_rng(4)
    p, bins, lists, covers = records(rng, 12, 96, 64, seen=1.0)
    _, _, v = cabi.tile_balance(96, 64, dev(p), dev(bins))
    h, S = 2.0 ** -6, sum(len(t) * float(o) for t, o in zip(covers, p[:, 5]))
    for g in range(12):
        side = []
        for sign in (1, -1):
            q = p.copy()
            q[g, 5] = np.float32(p[g, 5] + sign * h)
            side.append((float(q[g, 5]), float(cabi.tile_balance(96, 64, dev(q), dev(bins))[0][0])))
        (o1, l1), (o0, l0) = side
        slope = (l1 - l0) / (o1 - o0)
        assert abs(slope - float(v[g])) <= 2 * (h * len(covers[g]) / S) ** 2 * abs(slope) + 2.0 ** -23 * l1 / h


def test_tile_balance_of_nothing():
    from opensplat_amd import cabi

    for N in (0, 3):
        p = np.zeros((N, 12), np.float32)
        loss, counts, v = cabi.tile_balance(50, 40, dev(p), torch.zeros((12, 2), dtype=torch.int32, device="cuda"))
        assert float(loss[0]) == 0 and (counts == 0).all() and (v == 0).all() and v.shape == (N,)
    # lists, but no opacity in them
    p, bins, _, _ = records(np.random.default_rng(0), 20, 64, 64)
    p[:, 5] = 0
    loss, _, v = cabi.tile_balance(64, 64, dev(p), dev(bins))
    assert float(loss[0]) == 0 and (v == 0).all()
    # a NaN opacity is not swallowed
    p[3, 5] = np.nan
    covered = (p[3, 7].view(np.uint32) >> 16) > 0
    loss, _, v = cabi.tile_balance(64, 64, dev(p), dev(bins))
    assert bool(torch.isnan(loss[0])) == covered


def test_tile_balance_of_a_binned_frame():
    """On the records and lists of the framework's own binning: entries walked through the sorted ids."""
    from opensplat_amd import cabi, scenes
    from tests.util import hip_pipeline

    s = scenes.camera_scene(3000, 200, 136, K=4, seed=3)
    b = hip_pipeline(s, backward=False)["binned"]
    loss, counts, v = cabi.tile_balance(s.W, s.H, b.packed, b.tile_bins)
    bins, ids = b.tile_bins.cpu().numpy(), b.gaussian_ids_sorted.cpu().numpy()
    covers = [[] for _ in range(s.N)]
    for t, (lo, hi) in enumerate(bins):
        for g in ids[lo:hi]:
            covers[g].append(t)
    lists = bins[:, 1] - bins[:, 0]
    want, grad = orc.tile_balance(lists, [np.array(c, np.int64) for c in covers], b.packed[:, 5].cpu().numpy())
    assert lists.sum() > 1000 and np.array_equal(counts.cpu().numpy(), lists)
    close(float(loss[0]), want, want)
    close(v.cpu().numpy().astype(np.float64), grad, np.abs(grad).max() + want)


# ---- relocate -------------------------------------------------------------------------------------------------
# New logits and scales are 64-bit values rounded once: 2^-24 of the value; the scale's change is added to the old value
# in float32 after a rounding of its own: 2^-24 of the change and of the sum.  The alternating sum behind it has terms up
# to e^Y, Y = softplus(logit) <= 16 + 2^-23, each a product of up to forty factors of two roundings: 100 2^-53 e^Y.

def gaussian_set(rng, N, K, moments=True):
    shapes = [(N, 3), (N, 3), (N, 4), (N, 1), (N, 3), (N, K - 1, 3)]
    make = lambda: [rng.standard_normal(s).astype(np.float32) if np.prod(s) or N == 0 else None for s in shapes]  # noqa: E731
    p = make()
    p[3] *= 3
    return p, (make() if moments else None), (make() if moments else None)


def check_relocate(sets, targets, sources, low=0.005):
    from opensplat_amd import cabi

    gpu = [[dev(a) if a is not None else None for a in s] if s is not None else None for s in sets]
    cabi.relocate(*gpu, dev(np.asarray(targets, np.int32)), dev(np.asarray(sources, np.int32)), low)
    want = orc.relocate(*sets, list(targets), list(sources), low)
    for s, (g, w) in enumerate(zip(gpu, want)):
        for k in range(6):
            if g is None or g[k] is None:
                continue
            got, ref, old = g[k].cpu().numpy(), w[k], sets[s][k]
            if s == 0 and k in (1, 3):
                ref = ref.reshape(old.shape)
                tol = 2.0 ** -24 * 1.001 * np.abs(ref)
                if k == 1:
                    came = {t: s_ for t, s_ in zip(targets[::-1], sources[::-1])}      # (a row's old value: its source's)
                    was = old[[came[i] if i in came and 0 <= came[i] < len(old) else i for i in range(len(old))]]
                    top = np.exp(min(float(sets[0][3].max()), 16.0) + 0.1)
                    tol = tol + 2.0 ** -24 * 1.001 * np.abs(ref - was) + 2.0 ** -53 * 100 * top
                assert (np.abs(got - ref) <= tol).all(), (k, np.abs(got - ref).max())
                same = (ref == old).all(1)
                assert np.array_equal(got[same], old[same])
            else:
                assert np.array_equal(got, np.asarray(ref, np.float32)), (s, k)
    return gpu


@pytest.mark.parametrize("K", [1, 4, 16])
@pytest.mark.parametrize("size", [(2, 1), (50, 7), (1000, 200), (5000, 2111)])
def test_relocate(K, size):
    N, n = size
    rng = np.random.default_rng(N + K)
    order = rng.permutation(N)
    sources = order[n:][np.minimum((rng.random(n) ** 3 * (N - n)).astype(int), N - n - 1)]
    check_relocate(gaussian_set(rng, N, K), order[:n], sources)


@pytest.mark.parametrize("copies", [1, 2, 10, 63, 64, 65, 200, 3000])
def test_relocate_many_copies_of_one(copies):
    """One source, of every opacity up to the bound and beyond it."""
    for logit in (-12.0, -5.3, -1.0, 0.0, 2.5, 8.0, 16.0, 30.0):
        rng = np.random.default_rng(copies)
        sets = gaussian_set(rng, copies + 3, 1, moments=False)
        sets[0][3][1] = logit
        check_relocate(sets, [0] + list(range(3, copies + 2)), [1] * copies, 1e-5)


def test_relocate_pairs_that_do_not_hold():
    rng = np.random.default_rng(0)
    sets = gaussian_set(rng, 40, 4)
    #        twice the same target | out of range          | a source that is a target | itself | fine, same source
    targets = [5, 5, 6,              -1, 40, 7, 8, 2 ** 30,  9, 10,                      11,      12, 13, 5]
    sources = [20, 21, 21,           22, 22, -1, 40, -7,     10, 23,                     11,      20, 20, 24]
    check_relocate(sets, targets, sources)
    check_relocate(sets, [1, 2], [-1, -1])
    check_relocate(sets, [], [])


@pytest.mark.parametrize("which", [0, 1, 2])
def test_relocate_without_some_moments(which):
    rng = np.random.default_rng(which)
    p, m, v = gaussian_set(rng, 300, 9)
    m, v = (None if which == 0 else m), (None if which == 1 else v)
    if which == 2:
        m[5] = m[0] = v[3] = None
    check_relocate((p, m, v), np.arange(0, 60), np.arange(100, 160) // 2 * 2)


# ---- a run of them, streams, graphs ---------------------------------------------------------------------------

def run_all(s):
    """Sources for the dead drawn by opacity, relocation, the balance loss of the lists, on the current stream."""
    from opensplat_amd import cabi

    ids = cabi.sample(torch.where(s["dead"], -torch.inf, s["p"][3].view(-1)), s["u"], opacity=True, min_p=0.01)
    cabi.relocate(s["p"], s["m"], s["v"], s["targets"], ids)
    loss, counts, v = cabi.tile_balance(s["W"], s["H"], s["packed"], s["bins"])
    return ids, loss, counts, v


def state_for(seed, N=3000, n=150):
    rng = np.random.default_rng(seed)
    p, m, v = gaussian_set(rng, N, 4)
    packed, bins, _, _ = records(rng, N, 320, 200)
    targets = rng.permutation(N)[:n].astype(np.int32)
    dead = np.zeros(N, bool)
    dead[targets] = True
    return dict(p=[dev(a) for a in p], m=[dev(a) for a in m], v=[dev(a) for a in v], u=dev(rng.random(n, dtype=np.float32)),
                targets=dev(targets), dead=dev(dead), packed=dev(packed), bins=dev(bins), W=320, H=200,
                host=(p, m, v), th=targets, dh=dead)


def test_a_run_of_them():
    s = state_for(1)
    ids, loss, counts, v = run_all(s)
    p = s["host"][0]
    want = orc.sample_row(np.where(s["dh"], -np.inf, p[3].reshape(-1)), s["u"].cpu().numpy(), min_p=0.01, opacity=True)
    assert np.array_equal(ids.cpu().numpy(), want)
    ref, m, _ = orc.relocate(*s["host"], list(s["th"]), list(want), 0.005)
    assert np.abs(s["p"][3].cpu().numpy() - ref[3]).max() < 1e-5
    assert np.array_equal(s["p"][5].cpu().numpy(), ref[5].astype(np.float32))
    assert np.array_equal(s["m"][0].cpu().numpy(), m[0])


def test_two_streams_and_captured_replays_give_the_eager_bits():
    want = [[t.clone() for t in run_all(s) + tuple(s["p"]) + tuple(s["m"])] for s in (state_for(1), state_for(2))]
    torch.cuda.synchronize()
    # two streams at once
    states, outs = [state_for(1), state_for(2)], []
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            outs.append(run_all(s))
    torch.cuda.synchronize()
    for s, o, w in zip(states, outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o + tuple(s["p"]) + tuple(s["m"]), w))
    # one capture, replayed over refreshed inputs with eager work between
    s = state_for(1)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        run_all(state_for(3))
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = run_all(s)
    for seed in (1, 2, 1, 2):
        fresh = state_for(seed)
        for k in ("p", "m", "v"):
            for a, b in zip(s[k], fresh[k]):
                a.copy_(b)
        for k in ("u", "targets", "dead", "packed", "bins"):
            s[k].copy_(fresh[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out + tuple(s["p"]) + tuple(s["m"]), want[seed - 1])), seed
        run_all(state_for(7))


def test_calls_leave_what_is_behind_their_outputs():
    from opensplat_amd import cabi

    rng = np.random.default_rng(0)
    x, u = logits_of(rng, 3, 500, "f32"), dev(rng.random((3, 7), dtype=np.float32))
    whole = torch.full((40,), 77, device="cuda", dtype=torch.int32)
    cabi.sample(x, u, out=whole[4:25].view(3, 7))
    assert (whole[:4] == 77).all() and (whole[25:] == 77).all() and (whole[4:25] != 77).any()
    p, bins, lists, _ = records(rng, 33, 100, 50)
    buf = torch.full((1 + len(lists) + 33 + 30,), 5.0, device="cuda")
    ints = torch.full((len(lists) + 16,), 5, device="cuda", dtype=torch.int32)
    cabi.tile_balance(100, 50, dev(p), dev(bins), out=(buf[10:11], ints[8:8 + len(lists)], buf[20:53]))
    assert (buf[:10] == 5).all() and (buf[11:20] == 5).all() and (buf[53:] == 5).all()
    assert (ints[:8] == 5).all() and (ints[8 + len(lists):] == 5).all()
