"""CPU: what gs_sample, gs_tile_balance and gs_relocate refuse before any device work, and their oracles."""
import ctypes as C

import numpy as np
import pytest
import torch

from opensplat_amd import cabi
from tests import population_oracle as orc

NULL, ONE = C.c_void_p(0), C.c_void_p(64)
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
BIG = 1 << 40


def sample(rows=2, cols=5, logits=ONE, stride=5, draws=3, u=ONE, ids=ONE, ws=ONE, size=BIG, **cfg):
    c = cabi.GsSampleConfig(0, 0, 1.0, 0, 1.0, 0.0)
    for k, v in cfg.items():
        setattr(c, k, v)
    return cabi.lib().gs_sample(rows, cols, logits, stride, C.byref(c), draws, u, ids, ws, size, NULL)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=-1), dict(draws=-1), dict(logits=NULL), dict(u=NULL),
                                dict(ids=NULL), dict(ws=NULL), dict(stride=4), dict(dtype=3), dict(dtype=-1),
                                dict(flags=1), dict(temperature=-0.5), dict(temperature=float("nan")),
                                dict(top_p=float("nan")), dict(min_p=1.5), dict(min_p=float("nan")),
                                dict(logits=C.c_void_p(66)), dict(logits=C.c_void_p(65), dtype=1),
                                dict(ws=C.c_void_p(72)), dict(ids=C.c_void_p(66)), dict(u=C.c_void_p(66)),
                                ])
def test_sample_refuses(kw):
    assert sample(**kw) == INVALID


def test_sample_limits():
    """More threads than a launch can have."""
    assert sample(rows=1 << 27) == UNSUPPORTED and sample(rows=1 << 23, cols=8000, stride=8000) == UNSUPPORTED
    assert sample(rows=1 << 20, cols=1 << 20, stride=1 << 20) == UNSUPPORTED
    assert sample(rows=1 << 12, cols=9000, stride=9000, draws=1 << 21) == UNSUPPORTED


def test_sample_workspace_and_empty_calls():
    need = cabi.lib().gs_sample_workspace_bytes(2, 5)
    assert need > 0 and sample(size=need - 1) == WORKSPACE
    assert cabi.lib().gs_sample_workspace_bytes(-1, 5) == 0 and cabi.lib().gs_sample_workspace_bytes(3, -1) == 0
    assert sample(rows=0) == 0 and sample(draws=0) == 0
    assert cabi.lib().gs_sample(2, 5, ONE, 5, None, 3, ONE, ONE, ONE, BIG, NULL) == INVALID


def balance(W=64, H=64, N=4, packed=ONE, bins=ONE, scale=1.0, loss=ONE, counts=NULL, v=NULL, flags=0, ws=ONE, size=BIG):
    return cabi.lib().gs_tile_balance(W, H, N, packed, bins, scale, loss, counts, v, flags, ws, size, NULL)


@pytest.mark.parametrize("kw", [dict(W=0), dict(H=-3), dict(N=-1), dict(packed=NULL), dict(bins=NULL), dict(loss=NULL),
                                dict(ws=NULL), dict(flags=1), dict(flags=8), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(packed=C.c_void_p(68)), dict(bins=C.c_void_p(68)),
                                dict(ws=C.c_void_p(72)), dict(flags=32)])
def test_tile_balance_refuses(kw):
    assert balance(**kw) == INVALID


def test_tile_balance_limits():
    assert balance(W=65536) == UNSUPPORTED and balance(H=65536) == UNSUPPORTED
    need = cabi.lib().gs_tile_balance_workspace_bytes(64, 64, 4)
    assert need > 0 and balance(size=need - 1) == WORKSPACE
    assert cabi.lib().gs_tile_balance_workspace_bytes(0, 5, 4) == 0 and \
        cabi.lib().gs_tile_balance_workspace_bytes(64, 64, -1) == 0


def relocate(N=9, K=4, pairs=2, targets=ONE, sources=ONE, low=0.005, params=True, ws=ONE, size=BIG, drop=()):
    s = cabi.GsGaussianSet(*[0 if f[0] in drop else 64 for f in cabi.GsGaussianSet._fields_])
    return cabi.lib().gs_relocate(N, K, pairs, targets, sources, low, C.byref(s) if params else None, None, None, ws, size,
                                  NULL)


@pytest.mark.parametrize("kw", [dict(N=0), dict(N=-2), dict(K=0), dict(pairs=-1), dict(targets=NULL), dict(sources=NULL),
                                dict(low=0.0), dict(low=1.0), dict(low=float("nan")), dict(params=False), dict(ws=NULL),
                                dict(ws=C.c_void_p(72)), dict(drop=("means",)), dict(drop=("opacity_logits",)),
                                dict(drop=("features_rest",))])
def test_relocate_refuses(kw):
    assert relocate(**kw) == INVALID


def test_relocate_workspace_and_empty_calls():
    need = cabi.lib().gs_relocate_workspace_bytes(9, 2)
    assert need > 0 and relocate(size=need - 1) == WORKSPACE
    assert relocate(pairs=0) == 0
    assert relocate(pairs=1 << 29) == UNSUPPORTED


def test_host_tensors_are_refused():
    z = torch.zeros
    with pytest.raises((ValueError, AssertionError)):
        cabi.sample(z(2, 5), z(2, 3))
    with pytest.raises((ValueError, AssertionError, RuntimeError)):
        cabi.tile_balance(64, 64, z(4, 12), z((16, 2), dtype=torch.int32))
    with pytest.raises((ValueError, AssertionError, RuntimeError)):
        cabi.relocate([z(4, 3), z(4, 3), z(4, 4), z(4, 1), z(4, 3), None], None, None, z(1, dtype=torch.int32),
                      z(1, dtype=torch.int32))


def test_oracle_shares_keep_opacity_and_extent():
    """m equal shares laid over each other have the opacity and, as an integral over the line, the extent of the one."""
    logit, m = np.array([-3.0, 0.0, 4.0]), np.array([2, 7, 30])
    new, shrink = orc.shares(logit, m, 1e-6)
    o, p = 1 / (1 + np.exp(-logit)), 1 / (1 + np.exp(-new))
    assert np.allclose(np.asarray(1 - (1 - p) ** m, float), o, rtol=1e-12)
    t = np.linspace(-40, 40, 40001)
    for k in range(3):
        s = np.exp(float(shrink[k]))
        over = 1 - (1 - float(p[k]) * np.exp(-t ** 2 / (2 * s * s))) ** m[k]
        assert abs(np.trapezoid(over, t) - o[k] * np.sqrt(2 * np.pi)) < 1e-9


def test_oracle_sample_on_a_row_by_hand():
    x = np.log(np.array([4.0, 1.0, 4.0, 1.0]))
    u = np.array([0.0, 0.39, 0.41, 0.55, 0.95])
    assert orc.sample_row(x, u).tolist() == [0, 0, 1, 2, 3]
    assert orc.sample_row(x, u, top_k=1).tolist() == [0] * 5
    assert orc.sample_row(x, u, top_p=0.5).tolist() == [0, 0, 0, 2, 2]
    assert orc.sample_row(x, u, min_p=0.5).tolist() == [0, 0, 0, 2, 2]
    assert orc.sample_row([-np.inf, np.nan], u).tolist() == [-1] * 5
