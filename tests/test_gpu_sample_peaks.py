"""GPU: gs_sample against its definition with no weight rounded, on rows whose mass sits in a few entries: a tail of
millions that each weigh next to nothing is drawn where its running sums say.

Tolerances.  A weight is 2^y, y = (l - max l) log2(e) / T with five roundings behind it and a polynomial good to 2^-51:
relative to the weight 2^-51 + 5 |y| 2^-53, below 2^-44 for the |y| <= 64 of these rows.  It is rounded once to a multiple
of 2^-(124 - 2 ceil log2 cols) of the largest (rows of more than 8192 entries): n entries are off by n 2^-(125 - 2 c) at
most, 2^-59 at 4 M.  The largest weighs 1 exactly.  So a running sum is off by 2^-44 of the other entries' mass and 2^-58,
and so is the goal."""
import numpy as np
import pytest
import torch

from tests import population_oracle as orc

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check_borders(x, u, got, opacity=False, **kw):
    """Every id's running sum reaches past its goal, and the one before it does not, but for the tolerance above.  The one
    largest weight is left out of the sums here: with it a tail's sums would lose what this looks at to their own rounding
    (150 000 additions to 1 of up to 2^-64 each are 8e-15)."""
    kept, w = orc.kept_weights(x, opacity=opacity, **kw)
    peak = int(np.argmax(w))
    assert w[peak] == 1 and (np.delete(w, peak) < 1).all()
    sums = orc.running(np.where(np.arange(w.size) == peak, 0, w))
    tail = sums[-1]
    tol = 2 * (np.longdouble(2.0) ** -44 * tail + np.longdouble(2.0) ** -58)
    at = np.searchsorted(kept, got)
    assert np.array_equal(kept[np.minimum(at, kept.size - 1)], got)
    u = u.astype(np.longdouble)
    goal = lambda i: np.where(i >= peak, u * tail - (1 - u), u * tail + u)  # noqa: E731  (u (1 + tail), less the peak behind it)
    over = sums[at] > goal(at) - tol
    below = (at == 0) | (sums[np.maximum(at - 1, 0)] <= goal(at - 1) + tol)
    assert over.all() and below.all(), (int((~over).sum()), int((~below).sum()))


def peaked(cols, gap, dt, spread, seed=0):
    """One entry at 0, the rest `gap` lower; `spread`: by as much again up and down, in the type's own steps."""
    rng = np.random.default_rng(seed)
    x = np.full(cols, -float(gap), np.float32)
    if spread:
        x += rng.uniform(-spread, spread, cols).astype(np.float32)
    x[cols // 2] = 0.0
    return torch.from_numpy(x).to(DT[dt]).cuda()


@pytest.mark.parametrize("gap", [15, 20, 25, 29])
@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("shape", [(4_000_000, 0.0), (300_000, 2.0), (8200, 1.0)])
def test_sample_peak_over_a_tail(gap, dt, shape):
    from opensplat_amd import cabi

    cols, spread = shape
    x = peaked(cols, gap, dt, spread)
    rng = np.random.default_rng(gap)
    tail = min(1.0, 2 * cols * np.exp(spread - gap))         # most draws into the tail before the peak and behind it
    u = np.concatenate([rng.random(4000) * tail, 1 - rng.random(4000) * tail, rng.random(2000)])
    u = np.minimum(u.astype(np.float32), np.float32(1 - 2.0 ** -24))
    got = cabi.sample(x, torch.from_numpy(u).cuda()).cpu().numpy()
    check_borders(x.float().cpu().numpy(), u, got)


@pytest.mark.parametrize("logit", [-3.0, 2.0])
def test_sample_peak_over_a_tail_of_opacities(logit):
    from opensplat_amd import cabi

    rng = np.random.default_rng(1)
    x = np.full(2_000_000, logit - 18.0, np.float32)
    x[777_777] = logit
    u = np.minimum(rng.random(20_000, dtype=np.float32) * np.float32(0.02), np.float32(1 - 2.0 ** -24))
    for kw in (dict(), dict(temperature=0.8)):
        got = cabi.sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), opacity=True, **kw).cpu().numpy()
        check_borders(x, u, got, opacity=True, **kw)


@pytest.mark.parametrize("cols", [50_001, 4_000_000])
@pytest.mark.parametrize("opt", ["p", "k", "kp", "pm"])
def test_sample_cuts_among_the_ties_of_a_tail(cols, opt):
    """The last index that a cut keeps, drawn by u = 1: an integer, some of the tail's ties counted off by their mass.
    (2^-44 of the mass is 2^-44 of the ties' number, far from the distance that is checked here.)"""
    from opensplat_amd import cabi

    gap = 18.0
    x = peaked(cols, gap, "f32", 0.0)
    w, n = np.exp(-np.longdouble(gap)), cols - 1
    k = 0 if opt in ("p", "pm") else int(0.8 * cols)
    some = min(n, k - 1) if k else n
    # the shortest prefix is the peak and m of the tail
    total = 1 + w * some
    for share in (0.1, 0.37, 0.9):
        p = np.float32((1 + w * (share * some)) / total) if opt != "k" else np.float32(1.0)
        m = float((np.longdouble(p) * total - 1) / w)
        if opt != "k" and (p >= 1 or abs(m - round(m)) < 1e-3):
            continue
        keep = some if opt == "k" else int(np.ceil(m))
        kw = dict(top_p=float(p)) if opt != "k" else {}
        if k:
            kw["top_k"] = k
        if opt == "pm":
            kw["min_p"] = float(np.float32(w / 2))
        tail = np.delete(np.arange(cols), cols // 2)[:keep]
        last = max(int(tail[-1]), cols // 2)
        u = np.array([1.0, 0.0, -0.0, 7.0, -3.0, np.nan], np.float32)
        got = cabi.sample(x, torch.from_numpy(u).cuda(), **kw).cpu().numpy()
        assert got.tolist() == [last, 0, 0, last, 0, -1], (share, keep, got, last)
