"""GPU: gs_sample, gs_relocate and the bindings of both at the ends of their ranges."""
import numpy as np
import pytest
import torch

from tests.test_gpu_population import check_sample, dev

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
