"""Plain numpy forms, in 64 bits and more, of gs_sample, gs_tile_balance and gs_relocate (include/gsplat_densify.h,
include/gsplat_train.h), written from their definitions: what the tests compare the kernels with."""
import numpy as np

SETS = ("params", "exp_avg", "exp_avg_sq")


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, opacity=False):
    """x [V] float values, u [D] -> ids [D]."""
    x = np.asarray(x, np.float64)
    out = np.full(len(u), -1, np.int32)
    if not temperature >= 0 or np.isnan(top_p) or np.isnan(min_p):
        return out
    at = np.flatnonzero(x > -np.inf)
    if at.size == 0:
        return out
    v = x[at].astype(np.longdouble)
    if opacity:
        v = -np.logaddexp(np.longdouble(0), -v)
    with np.errstate(invalid="ignore"):
        d = np.where(v == v.max(), 0, v - v.max()) / np.longdouble(temperature if temperature > 0 else 1.0)
    w = np.exp(d)
    order = np.argsort(-x[at], kind="stable")
    n = order.size
    if top_k > 0:
        n = min(n, int(top_k))
    if top_p < 1.0:
        mass = np.cumsum(w[order[:n]])
        n = 1 if top_p <= 0 else min(n, 1 + int(np.searchsorted(mass, np.longdouble(np.float32(top_p)) * mass[-1])))
    if temperature == 0 or min_p > 1.0:
        n = 1
    kept = np.sort(order[:n])
    if n > 1:
        kept = kept[w[kept] >= np.longdouble(np.float32(min_p))]
    # (weights are rounded once, by definition)
    unit = np.longdouble(2.0) ** min(50, 62 - int(np.ceil(np.log2(max(x.size, 2)))))
    q = np.rint(w * unit)
    kept = kept[q[kept] > 0]
    mass = np.cumsum(q[kept])
    pick = np.searchsorted(mass, np.clip(np.nan_to_num(np.asarray(u, np.longdouble)), 0, 1) * mass[-1], side="right")
    return np.where(np.isnan(u), -1, at[kept[np.minimum(pick, kept.size - 1)]]).astype(np.int32)


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, opacity=False):
    rows = [np.broadcast_to(np.asarray(v), (len(x),)) for v in (temperature, top_k, top_p, min_p)]
    return np.stack([sample_row(x[r], u[r], *[v[r] for v in rows], opacity=opacity) for r in range(len(x))])


def tile_balance(lists, covers, opacity, scale=1.0, logit=False):
    """lists [T] entries per tile; covers: for every Gaussian the tiles whose lists hold it; -> loss, gradient [N]."""
    n = np.asarray(lists, np.float64)
    o = np.asarray(opacity, np.float64)
    S_t = np.zeros(len(n))
    for g, tiles in enumerate(covers):
        S_t[tiles] += o[g]
    T, M, S = len(n), n.sum(), S_t.sum()
    if M == 0 or not S > 0:
        return 0.0, np.zeros(len(o))
    loss = scale * T * (n / M * S_t / S).sum()
    grad = np.array([scale * T * (n[t].sum() / (M * S) - len(t) * (n * S_t).sum() / (M * S * S)) for t in covers])
    return loss, grad * (o * (1 - o) if logit else 1.0)


def shares(logit, m, min_opacity):
    """New logit and log(scale factor) of each of the m Gaussians that replace one (the scale factor from the integral of
    1 - (1 - o' exp(-t^2))^m over the line, trapezoid rule, whose error for this entire function is below 1e-14)."""
    x = np.minimum(np.asarray(logit, np.longdouble), 16)
    m = np.asarray(m, np.longdouble)
    y = np.logaddexp(np.longdouble(0), x) / m
    p = -np.expm1(-y)
    t = np.arange(-12, 12, 0.05, dtype=np.longdouble)
    f = -np.expm1(m[:, None] * np.log1p(-p[:, None] * np.exp(-t * t)))
    extent = f.sum(1) * 0.05 / np.sqrt(np.longdouble(np.pi))
    low = np.longdouble(np.float32(min_opacity))
    return np.maximum(np.log(np.expm1(y)), np.log(low / (1 - low))), -np.logaddexp(np.longdouble(0), -x) - np.log(extent)


def relocate(params, exp_avg, exp_avg_sq, targets, sources, min_opacity):
    """Lists of numpy arrays [N, ...] (moment lists may be None) -> new lists (params in longdouble)."""
    N = len(params[0])
    ok = [0 <= t < N and 0 <= s < N for t, s in zip(targets, sources)]
    named = {t for t, k in zip(targets, ok) if k}
    seen, pairs = set(), []
    for t, s, k in zip(targets, sources, ok):
        if not k or t in seen:
            continue
        seen.add(t)
        if s not in named:
            pairs.append((t, s))
    p = [a.astype(np.longdouble) if a is not None else None for a in params]
    moments = [[a.copy() if a is not None else None for a in s] if s is not None else None for s in (exp_avg, exp_avg_sq)]
    if pairs:
        drawn, times = np.unique([s for _, s in pairs], return_counts=True)
        logit, shrink = shares(params[3].reshape(-1)[drawn], times + 1, min_opacity)
        p[3].reshape(-1)[drawn] = logit
        p[1][drawn] += shrink[:, None]
        t, s = np.array(pairs).T
        for a in p:
            if a is not None:
                a[t] = a[s]
        for a in [a for m in moments if m is not None for a in m if a is not None]:
            a[t] = 0
            a[drawn] = 0
    return p, moments[0], moments[1]


def running(w):
    """Running sums in longdouble, a block's inside it and the blocks' before it: each has seen some 2 sqrt(n) roundings of
    2^-64, not n of them all the same way."""
    side = int(np.ceil(np.sqrt(max(len(w), 1))))
    a = np.zeros(side * side, np.longdouble)
    a[:len(w)] = w
    a = np.cumsum(a.reshape(side, side), 1)
    a[1:] += np.cumsum(a[:-1, -1])[:, None]
    return a.reshape(-1)[:len(w)]


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, opacity=False):
    """What sample_row draws from, no weight rounded: the kept indices of a row x [V] in ascending order and their weights
    (the largest is 1)."""
    x = np.asarray(x, np.float64)
    at = np.flatnonzero(x > -np.inf)
    v = x[at].astype(np.longdouble)
    if opacity:
        v = -np.logaddexp(np.longdouble(0), -v)
    w = np.exp((v - v.max()) / np.longdouble(np.float32(temperature)))   # (as the C ABI takes it)
    order = np.argsort(-x[at], kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        mass = running(w[order])
        order = order[:1 + int(np.searchsorted(mass, np.longdouble(np.float32(top_p)) * mass[-1]))]
    kept = np.sort(order)
    kept = kept[w[kept] >= np.longdouble(np.float32(min_p))]
    return at[kept], w[kept]
