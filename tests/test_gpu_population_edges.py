"""GPU: gs_sample, gs_relocate and the bindings of both at the ends of their ranges."""
import numpy as np
import pytest
import torch

from tests.test_gpu_population import check_sample, dev, gaussian_set

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
    from opensplat_amd import cabi

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
    from opensplat_amd import cabi

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
