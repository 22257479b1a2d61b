"""Three operators of a fixed budget of Gaussians, as calls that can be timed and compared: drawing indices
from given random numbers, the balance loss of the tile lists, and the relocation of drawn sources.

`own = False`: `run` is the plain form of an operator, elementary torch operations in the order of its
definition.  `own = True`: the call a program makes of `opensplat_amd.cabi`.

  sample        ids[r, j] = the lowest index whose running weight exceeds uniforms[r, j] * total, with weights
                softmax(logits / T) — or sigmoid(logit)^(1/T) for opacity logits — on the entries that top-k,
                top-p and min-p keep
  tile_balance  loss = T sum_t f_t P_t over the T tiles of a frame: f_t the share of the list entries that tile
                t holds, P_t the share of the opacity in its list; with the entries per tile and the gradient
                with respect to the opacity logits
  relocate      target rows become copies of source rows; a source and its copies together keep the source's
                opacity and extent; the Adam moments of the rows that changed are cleared
"""
import math

import numpy as np
import torch

own = False

TILE = 16        # pixels per tile side
RECORD = 12      # 4-byte words of a packed Gaussian record: [5] opacity, [7] x0 | x1 << 16, [11] y0 | y1 << 16
ROWS = (3, 3, 4, 1, 3, 45)   # floats per Gaussian of the six parameter tensors (SH degree 3)
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _sample(name, rows, cols, draws, dtype="float32", opacity=False, temperature=False, top_k=False, top_p=False,
            min_p=False, pad=0, reset=False):
    return dict(name=name, op="sample", rows=rows, cols=cols, draws=draws, dtype=dtype, opacity=opacity,
                temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, pad=pad, reset=reset)


def _balance(name, count, width, height, hot=False):
    return dict(name=name, op="tile_balance", count=count, width=width, height=height, hot=hot)


def _relocate(name, count, pairs):
    return dict(name=name, op="relocate", count=count, pairs=pairs)


def listed():
    return [
        # the next camera of a 28-image capture, drawn by the images' losses
        _sample("camera_pick", 1, 28, 1, temperature=True),
        # a hundred tiles of every image of the capture at 1080p, drawn by their error, the small ones left out
        _sample("tiles_28x8160", 28, 8160, 100, temperature=True, top_p=True),
        # sources for the dead twentieth of a million Gaussians, right behind an alpha reset (many equal logits)
        _sample("sources_1m", 1, 1_000_000, 50_000, opacity=True, reset=True),
        # the same at five million, sharpened, from the strongest that hold 95 % of the opacity
        _sample("sources_5m_top_p", 1, 5_000_000, 250_000, opacity=True, temperature=True, top_p=True),
        # a batch of long rows with settings of their own, padded rows of an odd stride, one entry per row
        _sample("rows_64x131072", 64, 131_072, 1, "bfloat16", temperature=True, top_k=True, top_p=True, min_p=True,
                pad=13),
        # ten thousand Gaussians in a 256 x 256 frame: the smallest training frame
        _balance("balance_10k_256", 10_000, 256, 256),
        # a million Gaussians at 1080p
        _balance("balance_1m_1080p", 1_000_000, 1920, 1080),
        # five million at 4K, a part of them in a small window
        _balance("balance_5m_4k", 5_000_000, 3840, 2160, hot=True),
        # a young set of 6000 Gaussians
        _relocate("relocate_6k", 6_000, 300),
        # the dead twentieth of 200 000 and of a million
        _relocate("relocate_200k", 200_000, 10_000),
        _relocate("relocate_1m", 1_000_000, 50_000),
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(("sample", "sample", "tile_balance", "relocate"))
    if op == "sample":
        opacity = rng.random() < 0.4
        cols = spread(28, 4_000_000)
        rows = 1 if opacity else min(spread(1, 256), max(1, 6_000_000 // cols))
        draws = max(1, cols // spread(15, 60)) if opacity else min(spread(1, 200), cols)
        flag = lambda: rng.random() < 0.5  # noqa: E731
        return _sample("", rows, cols, draws, "float32" if opacity else rng.choice(sorted(DTYPES)), opacity, flag(),
                       flag(), flag(), flag(), rng.choice((0, 0, 1, 8, 13)), opacity and flag())
    if op == "tile_balance":
        width = spread(64, 3840)
        height = max(48, min(2160, int(width * rng.uniform(0.5, 1.1))))
        return _balance("", spread(1_000, 4_500_000), width, height, rng.random() < 0.4)
    count = spread(1_000, 950_000)
    return _relocate("", count, max(1, int(count * rng.uniform(0.005, 0.05))))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_sample(case, g):
    rows, cols, draws = case["rows"], case["cols"], case["draws"]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    logits = normal(rows, cols + case["pad"]).mul_(1.5 if case["opacity"] else 2.5)
    if case["opacity"]:
        logits.sub_(0.5)
        if case["reset"]:
            logits.clamp_(max=math.log(0.2 / 0.8))
        logits.masked_fill_(uniform(rows, cols + case["pad"]) < 0.05, -math.inf)     # the dead
    elif rows > 1:
        # rows of different lengths: masked behind their ends, one of a longer batch masked as a whole
        ends = (uniform(rows, 1) * 0.5 + 0.5).mul_(cols).long().clamp_(min=1)
        if rows > 8:
            ends[rows // 2] = 0
        logits.masked_fill_(torch.arange(cols + case["pad"], device="cuda")[None] >= ends, -math.inf)
    logits = logits.to(DTYPES[case["dtype"]])[:, :cols]
    state = dict(case=case, logits=logits, uniforms=uniform(rows, draws), temperature=None, top_k=None, top_p=None,
                 min_p=None)
    if case["temperature"]:
        state["temperature"] = uniform(rows).mul_(0.8).add_(0.6)
    if case["top_k"]:
        state["top_k"] = (uniform(rows) * min(cols, 4000)).int().add_(1)
    if case["top_p"]:
        state["top_p"] = uniform(rows).mul_(0.4).add_(0.58)
    if case["min_p"]:
        state["min_p"] = uniform(rows).mul_(0.02)
    return state


def _prepare_balance(case, g):
    count, width, height = case["count"], case["width"], case["height"]
    uniform = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    size = torch.tensor([width, height], device="cuda")
    centre = uniform(count, 2) * size
    if case["hot"]:
        few = uniform(count, 1) < 0.02
        centre = torch.where(few, size * 0.4 + uniform(count, 2) * 48.0, centre)
    reach = torch.randn((count, 2), generator=g, device="cuda").mul_(0.6).add_(1.6).exp_()
    lo = (centre - reach).floor().long().clamp_(min=0)
    hi = torch.minimum((centre + reach).ceil().long() + 1, size)
    seen = (uniform(count) > 0.2) & (hi > lo).all(1)
    lo, hi = lo * seen[:, None], hi * seen[:, None]
    packed = torch.randn((count, RECORD), generator=g, device="cuda")
    packed[:, 5] = torch.sigmoid(torch.randn(count, generator=g, device="cuda").mul_(1.5).sub_(0.5))
    word = lambda k: (lo[:, k] | (hi[:, k] << 16)).int().view(torch.float32)  # noqa: E731
    packed[:, 7], packed[:, 11] = word(0), word(1)
    # the lists' extents, as the binning leaves them: corners of the covered tiles, summed over both axes
    tw, th = -(-width // TILE), -(-height // TILE)
    t0, t1 = lo // TILE, -(-hi // TILE)
    corner = torch.zeros((th + 1) * (tw + 1), dtype=torch.int64, device="cuda")
    one = seen.long()
    for y, x, sign in ((t0, t0, 1), (t0, t1, -1), (t1, t0, -1), (t1, t1, 1)):
        corner.index_add_(0, y[:, 1] * (tw + 1) + x[:, 0], one * sign)
    lists = corner.view(th + 1, tw + 1).cumsum(0).cumsum(1)[:th, :tw].reshape(-1)
    ends = lists.cumsum(0)
    return dict(case=case, packed=packed, tile_bins=torch.stack([ends - lists, ends], 1).int().contiguous())


def _prepare_relocate(case, g):
    count, pairs = case["count"], case["pairs"]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    shape = lambda k: (count, 15, 3) if k == 45 else (count, k)  # noqa: E731
    params = [normal(*shape(k)) for k in ROWS]
    params[1].sub_(4.0)
    params[3].mul_(1.5).sub_(0.5)
    order = torch.randperm(count, generator=g, device="cuda")
    targets, alive = order[:pairs].int(), order[pairs:]
    params[3][targets.long()] = -6.0
    # strong Gaussians are drawn several times
    pick = torch.rand(pairs, generator=g, device="cuda").pow_(3.0).mul_(alive.numel()).long()
    return dict(case=case, params=params, exp_avg=[normal(*shape(k)) for k in ROWS],
                exp_avg_sq=[normal(*shape(k)).square_() for k in ROWS], targets=targets,
                sources=alive[pick.clamp_(max=alive.numel() - 1)].int())


def prepare(case, seed):
    make = {"sample": _prepare_sample, "tile_balance": _prepare_balance, "relocate": _prepare_relocate}[case["op"]]
    return make(case, _generator(seed))


def _plain_sample(s):
    x, u = s["logits"].double(), s["uniforms"].double()
    if s["case"]["opacity"]:
        x = torch.where(x < 0, x - torch.log1p(torch.exp(x)), -torch.log1p(torch.exp(-x)))
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    row = lambda v: v.double()[:, None]  # noqa: E731
    scaled = (x - top) / row(s["temperature"]) if s["temperature"] is not None else x - top
    w = torch.where(x == -math.inf, 0.0, torch.where(x == top, 1.0, torch.exp(scaled)))
    if s["top_k"] is not None or s["top_p"] is not None:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        sorted_w = w.gather(1, order)
        keep = torch.ones_like(sorted_w, dtype=torch.bool)
        if s["top_k"] is not None:
            keep = torch.arange(x.shape[1], device=x.device)[None] < s["top_k"].long()[:, None]
        if s["top_p"] is not None:
            running = (sorted_w * keep).cumsum(1)
            before = torch.cat([torch.zeros_like(top), running[:, :-1]], 1)
            keep = keep & (before < row(s["top_p"]) * running[:, -1:])
        w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    if s["min_p"] is not None:
        w = torch.where(w >= row(s["min_p"]), w, 0.0)
    running = w.view(-1).cumsum(0)[None] if w.shape[0] == 1 else w.cumsum(1)
    total = running[:, -1:]
    ids = torch.searchsorted(running, u * total, right=True).clamp_(max=x.shape[1] - 1)
    return torch.where(total > 0, ids, -1).int()


def _corners(packed):
    """First and one-past-last tile of every record's rectangle, per axis (equal: the record is in no list)."""
    words = packed[:, [7, 11]].contiguous().view(torch.int32).long()
    lo, hi = words & 0xFFFF, (words >> 16) & 0xFFFF
    seen = (hi > lo).all(1, keepdim=True)
    return torch.where(seen, lo // TILE, 0), torch.where(seen, -(-hi // TILE), 0)


def _plain_balance(s):
    tw = -(-s["case"]["width"] // TILE)
    t0, t1 = _corners(s["packed"])
    lists = s["tile_bins"][:, 1] - s["tile_bins"][:, 0]
    across = t1[:, 0] - t0[:, 0]
    held = across * (t1[:, 1] - t0[:, 1])
    # every (Gaussian, tile) entry, one after the other
    who = torch.repeat_interleave(held)
    nth = torch.arange(who.numel(), device=who.device) - (held.cumsum(0) - held)[who]
    wide = across.clamp(min=1)[who]
    tile = (t0[who, 1] + nth // wide) * tw + t0[who, 0] + nth % wide
    crowd = torch.zeros_like(held).index_add_(0, who, lists[tile].long()).double()
    opacity = s["packed"][:, 5].double()
    entries, mass = held.sum().double(), (opacity * held).sum()
    mean = (opacity * crowd).sum() / mass
    scale = lists.numel() / entries
    slope = scale / mass * (crowd - held * mean)
    ok = (entries > 0) & (mass > 0)
    loss = torch.where(ok, scale * mean, 0.0)
    grad = torch.where(ok, slope * opacity * (1.0 - opacity), 0.0)
    return loss.float().reshape(1), lists, grad.float()


def _plain_relocate(s):
    targets, sources = s["targets"].long(), s["sources"].long()
    copies = torch.zeros(s["case"]["count"], dtype=torch.int64, device=targets.device)
    copies.index_add_(0, sources, torch.ones_like(sources))
    m = (copies[sources] + 1).double()[:, None]
    x = s["params"][3].view(-1)[sources].double().clamp(max=16.0)[:, None]
    y = torch.where(x > 0, x + torch.log1p(torch.exp(-x)), torch.log1p(torch.exp(x))) / m     # -log(1 - o) / m
    p = -torch.expm1(-y)
    # extent of m copies laid over each other: sum_j (-1)^(j-1) C(m, j) p^j / sqrt(j)
    j = torch.arange(1, 97, device=m.device, dtype=torch.float64)[None]
    terms = ((m - j + 1).clamp(min=0) / j * p).cumprod(1) / j.sqrt()
    extent = (terms[:, ::2] - terms[:, 1::2]).sum(1, keepdim=True)
    low = math.log(0.005 / 0.995)
    logit = torch.log(torch.expm1(y)).clamp(min=low).float()
    shrink = (torch.log(torch.sigmoid(x)) - torch.log(extent)).float()
    for k, t in enumerate(s["params"]):
        rows = t[sources]
        if k == 1:
            rows = rows + shrink
        elif k == 3:
            rows = logit
        t[targets] = rows
        t[sources] = rows
    for t in s["exp_avg"] + s["exp_avg_sq"]:
        t[targets] = 0.0
        t[sources] = 0.0
    return s["params"], s["exp_avg"], s["exp_avg_sq"]


def run(state):
    case = state["case"]
    if own:
        from opensplat_amd import cabi

        if case["op"] == "sample":
            return cabi.sample(state["logits"], state["uniforms"], temperature=state["temperature"],
                               top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"],
                               opacity=case["opacity"])
        if case["op"] == "tile_balance":
            return cabi.tile_balance(case["width"], case["height"], state["packed"], state["tile_bins"],
                                     flags=cabi.GS_FLAG_LOGIT_OPACITY)
        cabi.relocate(state["params"], state["exp_avg"], state["exp_avg_sq"], state["targets"], state["sources"],
                      min_opacity=0.005)
        return state["params"], state["exp_avg"], state["exp_avg_sq"]
    if case["op"] == "sample":
        return _plain_sample(state)
    return _plain_balance(state) if case["op"] == "tile_balance" else _plain_relocate(state)


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        n = case["rows"] * case["cols"]
        return {"bytes": n * size + case["rows"] * case["draws"] * 8, "flops": 4 * n}
    if case["op"] == "tile_balance":
        tiles = -(-case["width"] // TILE) * -(-case["height"] // TILE)
        return {"bytes": case["count"] * 16 + tiles * 12 + 4, "flops": 12 * case["count"]}
    # a row is read once and written once; both moments of the target, and of its source, are cleared
    return {"bytes": case["pairs"] * (8 + 4 * sum(ROWS) * 6), "flops": 200 * case["pairs"]}


def _exact_sample(s):
    ids = np.full((s["case"]["rows"], s["case"]["draws"]), -1, np.int32)
    every, uniforms = s["logits"].float().cpu().numpy().astype(np.float64), s["uniforms"].cpu().numpy()
    given = {k: s[k].cpu().numpy().astype(np.float64) if s[k] is not None else None
             for k in ("temperature", "top_k", "top_p", "min_p")}
    for r, x in enumerate(every):
        if s["case"]["opacity"]:
            x = -np.logaddexp(0.0, -x)
        at = np.flatnonzero(x > -np.inf)
        if not at.size:
            continue
        z = x[at] / (given["temperature"][r] if given["temperature"] is not None else 1.0)
        w = np.exp(z - z.max())
        order = np.argsort(-x[at], kind="stable")
        n = order.size
        if given["top_k"] is not None:
            n = min(n, int(given["top_k"][r]))
        mass = np.cumsum(w[order[:n]].astype(np.longdouble))
        if given["top_p"] is not None:
            n = min(n, 1 + int(np.searchsorted(mass, np.longdouble(given["top_p"][r]) * mass[-1], side="left")))
        kept = np.sort(order[:n])
        if given["min_p"] is not None:
            kept = kept[w[kept] >= given["min_p"][r]]
        mass = np.cumsum(w[kept].astype(np.longdouble))
        pick = np.searchsorted(mass, uniforms[r].astype(np.longdouble) * mass[-1], side="right")
        ids[r] = at[kept[np.minimum(pick, kept.size - 1)]]
    return torch.from_numpy(ids)


def _exact_balance(s):
    tw, th = -(-s["case"]["width"] // TILE), -(-s["case"]["height"] // TILE)
    words = s["packed"][:, [7, 11]].contiguous().view(torch.int32).cpu().numpy().view(np.uint32)
    lo, hi = (words & 0xFFFF).astype(np.int64), (words >> 16).astype(np.int64)
    seen = (hi > lo).all(1)
    (x0, y0), (x1, y1) = ((lo // TILE) * seen[:, None]).T, ((hi + TILE - 1) // TILE * seen[:, None]).T
    bins = s["tile_bins"].cpu().numpy().astype(np.int64)
    lists = bins[:, 1] - bins[:, 0]
    area = np.zeros((th + 1, tw + 1), np.int64)
    area[1:, 1:] = lists.reshape(th, tw).cumsum(0).cumsum(1)
    crowd = area[y1, x1] - area[y0, x1] - area[y1, x0] + area[y0, x0]
    held = (x1 - x0) * (y1 - y0)
    o = s["packed"][:, 5].cpu().numpy().astype(np.float64)
    share, mass = lists / lists.sum(), (o * held).sum()
    loss = lists.size * (o * crowd).sum() / lists.sum() / mass
    grad = (lists.size / lists.sum() * crowd / mass - loss * held / mass) * o * (1.0 - o)
    assert abs(share.sum() - 1.0) < 1e-9
    return torch.tensor([loss]), torch.from_numpy(lists.astype(np.int32)), torch.from_numpy(grad)


def _exact_relocate(s):
    targets, sources = s["targets"].cpu().numpy(), s["sources"].cpu().numpy()
    drawn, back, times = np.unique(sources, return_inverse=True, return_counts=True)
    x = np.minimum(s["params"][3].view(-1).cpu().numpy()[drawn].astype(np.float64), 16.0)
    m = times + 1.0
    y = np.logaddexp(0.0, x) / m
    # the extent as the integral it stands for: of 1 - (1 - p exp(-t^2))^m over the line, over sqrt(pi)
    t = np.arange(0.0, 8.0, 0.05)
    extent = np.zeros_like(x)
    for k, e in enumerate(np.exp(-t * t)):
        extent -= (1.0 if k else 0.5) * np.expm1(m * np.log1p(np.expm1(-y) * e))
    extent *= 2.0 * 0.05 / math.sqrt(math.pi)
    change = {1: -np.logaddexp(0.0, -x) - np.log(extent),
              3: np.maximum(np.log(np.expm1(y)), math.log(0.005 / 0.995))}
    out = []
    for k, p in enumerate(s["params"]):
        a = p.cpu().numpy().astype(np.float64)
        rows = a[drawn]
        if k == 1:
            rows = rows + change[1][:, None]
        elif k == 3:
            rows = change[3][:, None]
        a[drawn] = rows
        a[targets] = rows[back]
        out.append(torch.from_numpy(a))
    moments = []
    for t in s["exp_avg"] + s["exp_avg_sq"]:
        a = t.cpu().double()
        a[torch.from_numpy(targets).long()] = 0.0
        a[torch.from_numpy(drawn).long()] = 0.0
        moments.append(a)
    return out, moments[:6], moments[6:]


def exact(case, seed):
    what = {"sample": _exact_sample, "tile_balance": _exact_balance, "relocate": _exact_relocate}[case["op"]]
    return what(prepare(case, seed))
