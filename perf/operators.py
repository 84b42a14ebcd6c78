"""Cases of the operators around a mixture of forests: rows routed among several
models, sorted by model and gathered, the models' outputs combined, and a softmax
head over many classes trained on top.

With `own` false `run` computes each operator with elementary torch operations in
32 bits; with `own` true it calls this package (macboost_b200._core).  `exact`
gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
LAYOUTS = {"feature": 0, "row": 1}


# ---- cases ----------------------------------------------------------------

def _route(rows, experts, k, norm="chosen", masked=0.0, grad=False, **kw):
    return {"op": "route", "rows": rows, "experts": experts, "k": k, "norm": norm,
            "masked": masked, "grad": grad, **kw}


def _dispatch(rows, cols, experts, k, type="f32", source="row", target="feature", align=4,
              dropped=0.0, **kw):
    return {"op": "dispatch", "rows": rows, "cols": cols, "experts": experts, "k": k,
            "type": type, "source": source, "target": target, "align": align,
            "dropped": dropped, **kw}


def _combine(rows, cols, experts, k, type="f32", align=1, dropped=0.0, grad=False, **kw):
    return {"op": "combine", "rows": rows, "cols": cols, "experts": experts, "k": k,
            "type": type, "align": align, "dropped": dropped, "grad": grad, **kw}


def _head(rows, cols, classes, type="bf16", ignored=0.0, grad=False, **kw):
    return {"op": "head", "rows": rows, "cols": cols, "classes": classes, "type": type,
            "ignored": ignored, "grad": grad, **kw}


def listed():
    return [
        # A serving batch: 64 rows choose two of eight models. Latency counts.
        _route(64, 8, 2, name="route small"),
        # A ten-class gate forest over a million rows, with the gradient a trainer of
        # the gate needs (its pseudo-residuals).
        _route(1_000_000, 10, 2, grad=True, name="route 1M"),
        # Many small models, a share of them switched off row by row, some rows with
        # none left; weights of the full softmax.
        _route(65_537, 256, 8, norm="all", masked=0.3, grad=True, name="route wide masked"),
        # A serving batch of hard segments: 500 rows of 100 features, one of four models.
        _dispatch(500, 100, 4, 1, name="dispatch small"),
        # The 10M x 28 feature-major matrix split by segment among eight models.
        _dispatch(10_000_000, 28, 8, 1, source="feature", dropped=0.02, name="dispatch segments"),
        # Numpy rows of 100 features to two of 64 models each, laid out feature-major
        # for the forests.
        _dispatch(500_000, 100, 64, 2, name="dispatch transposed"),
        # Half-precision embeddings to eight of 128 experts, row to row.
        _dispatch(8_191, 2_048, 128, 8, type="bf16", target="row", align=1, dropped=0.05,
                  name="dispatch wide rows"),
        # Ten class margins of two models each, combined, with the gradient for margins
        # (the models' pseudo-residuals) and weights.
        _combine(1_000_000, 10, 64, 2, align=4, grad=True, name="combine margins"),
        # Wide half-precision outputs of eight experts, with the gradient.
        _combine(8_191, 2_048, 128, 8, type="bf16", dropped=0.05, grad=True,
                 name="combine wide rows"),
        # The log-probability of one answer among 131,072: a single row, the weights
        # are read once.
        _head(1, 1_024, 131_072, name="head one row"),
        # Calibration of ten class margins by a 10 x 10 softmax layer, one training step
        # over 500k held-out rows.
        _head(500_000, 10, 10, type="f32", grad=True, name="head calibration"),
        # A training step of a head over 131,072 classes, some rows without a label.
        _head(8_192, 1_024, 131_072, ignored=0.05, grad=True, name="head large"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("route", "dispatch", "combine", "head"))
    if op == "route":
        experts = _log(rng, 2, 256)
        return _route(_log(rng, 1, 16_000_000 // max(16, experts)), experts,
                      rng.randint(1, min(8, experts)), norm=rng.choice(("chosen", "all")),
                      masked=rng.choice((0.0, 0.3)), grad=rng.random() < 0.5)
    if op == "head":
        cols, classes = _log(rng, 8, 1_024), _log(rng, 10, 131_072)
        type = rng.choice(("f32", "bf16"))
        most = 10 ** 12 // (cols * classes * (8 if type == "f32" else 1))
        return _head(_log(rng, 1, max(1, min(8_192, most))), cols, classes, type=type,
                     ignored=rng.choice((0.0, 0.1)), grad=rng.random() < 0.6)
    experts = _log(rng, 2, 256)
    k = rng.randint(1, min(8, experts))
    cols = _log(rng, 1, 2_048)
    rows = _log(rng, 1, max(1, min(2_000_000, 128_000_000 // (k * cols), 256_000_000 // experts)))
    dropped = rng.choice((0.0, 0.1))
    if op == "combine":
        return _combine(rows, cols, experts, k, type=rng.choice(("f32", "bf16", "f16")),
                        align=rng.choice((1, 4)), dropped=dropped, grad=rng.random() < 0.6)
    source, target = rng.choice((("row", "row"), ("row", "feature"), ("feature", "feature")))
    type = rng.choice(("f32", "bf16", "f16")) if target == "row" else "f32"
    return _dispatch(rows, cols, experts, k, type=type, source=source, target=target,
                     align=rng.choice((1, 4)), dropped=dropped)


def _capacity(c):
    """Slots that k entries a row can take when each expert's segment starts at a
    multiple of `align`."""
    return c["rows"] * c["k"] + c["experts"] * (c["align"] - 1)


def work(c):
    n, size = c["rows"], 4 if c.get("type", "f32") == "f32" else 2
    if c["op"] == "route":
        e, k = c["experts"], c["k"]
        moved = n * e * 4 + n * k * 8
        if c["grad"]:
            moved += n * k * 4 + n * e * 4
        return {"bytes": moved, "flops": n * e * (8 if c["grad"] else 4)}
    if c["op"] == "dispatch":
        cap, cols = _capacity(c), c["cols"]
        return {"bytes": n * c["k"] * 8 + cap * 4 + n * cols * size + cap * cols * size,
                "flops": 0}
    if c["op"] == "combine":
        cap, cols, k = _capacity(c), c["cols"], c["k"]
        moved = n * k * 8 + n * k * cols * size + n * cols * size
        if c["grad"]:
            moved += n * cols * size + cap * cols * size + n * k * 4
        return {"bytes": moved, "flops": n * k * cols * (5 if c["grad"] else 2)}
    d, v = c["cols"], c["classes"]
    moved = (n + v) * d * size + n * 12
    if c["grad"]:
        moved += (n + v) * d * size + n * 4
    return {"bytes": moved, "flops": 2.0 * n * v * d * (3 if c["grad"] else 1)}


# ---- inputs ---------------------------------------------------------------

def _ids(c, g):
    """Distinct experts of each row, the first ones popular; a share of entries is -1."""
    n, e, k = c["rows"], c["experts"], c["k"]
    if k == 1:
        ids = (torch.rand((n, 1), device="cuda", generator=g) ** 1.5 * e).to(torch.int32)
        ids.clamp_(max=e - 1)
    else:
        score = torch.rand((n, e), device="cuda", generator=g)
        score -= torch.linspace(0, 0.5, e, device="cuda")
        ids = score.topk(k, dim=1).indices.to(torch.int32)
    if c["dropped"]:
        ids[torch.rand((n, k), device="cuda", generator=g) < c["dropped"]] = -1
    return ids


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, type=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(type)

    s = {"case": c, "kept": {}}
    n = c["rows"]
    if c["op"] == "route":
        s["logits"] = normal(n, c["experts"], scale=2.0)
        if c["masked"]:
            off = torch.rand((n, c["experts"]), device="cuda", generator=g) < c["masked"]
            off[96::97] = True
            s["logits"][off] = -math.inf
        if c["grad"]:
            s["dweights"] = normal(n, c["k"])
        return s
    if c["op"] == "head":
        t = TYPES[c["type"]]
        s["h"] = normal(n, c["cols"], type=t)
        s["w"] = normal(c["classes"], c["cols"], scale=2.0 / math.sqrt(c["cols"]), type=t)
        y = torch.randint(0, c["classes"], (n,), device="cuda", generator=g, dtype=torch.int32)
        if c["ignored"]:
            y[torch.rand(n, device="cuda", generator=g) < c["ignored"]] = -1
        s["labels"] = y
        if c["grad"]:
            # the mean over labelled rows, with a weight for each row
            wt = 0.5 + torch.rand(n, device="cuda", generator=g)
            s["dloss"] = wt / (y >= 0).sum().clamp(min=1)
        return s
    t = TYPES[c["type"]]
    ids = _ids(c, g)
    if c["op"] == "dispatch":
        s["ids"] = ids
        shape = (n, c["cols"]) if c["source"] == "row" else (c["cols"], n)
        s["x"] = normal(*shape, type=t)
        return s
    s["offsets"], s["counts"], s["order"], s["slots"] = _sorted(ids, c["experts"], c["align"])
    s["y"] = normal(_capacity(c), c["cols"], type=t)
    s["weights"] = normal(n, c["k"]).softmax(1)
    if c["grad"]:
        s["dout"] = normal(n, c["cols"], type=t)
    return s


# ---- the plain forms ------------------------------------------------------

def _sorted(ids, experts, align):
    """Entries (row-major over (rows, k)) stably sorted by expert: the segments'
    starts (the last: their end), their lengths, the entry in each slot (-1: none)
    and the slot of each entry (-1: not dispatched)."""
    n, k = ids.shape
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    by_expert = key.argsort(stable=True)
    counts = torch.bincount(key, minlength=experts + 1)
    before = counts.cumsum(0) - counts
    room = (counts[:experts] + align - 1) // align * align
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = room.cumsum(0)
    key_sorted = key[by_expert]
    place = torch.arange(n * k, device=ids.device) - before[key_sorted] + offsets[key_sorted]
    place = torch.where(key_sorted < experts, place, -1)
    slots = torch.empty(n * k, dtype=torch.int32, device=ids.device)
    slots[by_expert] = place.int()
    # one place more, which takes what is not dispatched
    capacity = n * k + experts * (align - 1)
    order = torch.full((capacity + 1,), -1, dtype=torch.int32, device=ids.device)
    order[torch.where(place >= 0, place, capacity)] = by_expert.int()
    return offsets, counts[:experts].int(), order[:capacity], slots.view(n, k)


def _plain_route(s, c):
    logits = s["logits"].float()
    top, ids = logits.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :c["k"]], ids[:, :c["k"]]
    found = top > -math.inf
    biggest = torch.where(found[:, :1], top[:, :1], 0.0)
    e = torch.exp(top - biggest)
    over = torch.exp(logits - biggest) if c["norm"] == "all" else e
    total = over.sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    weights = e / total
    out = {"ids": torch.where(found, ids, -1).int(), "weights": weights}
    if c["grad"]:
        dw = torch.where(found, s["dweights"], 0.0)
        mean = (weights * dw).sum(1, keepdim=True)
        if c["norm"] == "all":
            d = -(over / total) * mean
            d.scatter_add_(1, ids, weights * dw)
        else:
            d = torch.zeros_like(logits)
            d.scatter_(1, ids, weights * (dw - mean))
        out["dlogits"] = d
    return out


def _plain_dispatch(s, c):
    offsets, counts, order, slots = _sorted(s["ids"], c["experts"], c["align"])
    row = (order // c["k"]).clamp(min=0)
    if c["source"] == "row":
        picked = torch.where((order >= 0)[:, None], s["x"][row], 0.0)
        picked = picked.t() if c["target"] == "feature" else picked
    else:
        picked = torch.where((order >= 0)[None, :], s["x"][:, row], 0.0)
    return {"offsets": offsets, "counts": counts, "order": order, "slots": slots,
            "x": picked.contiguous()}


def _plain_combine(s, c):
    n, k, t = c["rows"], c["k"], s["y"].dtype
    there = s["slots"] >= 0
    at = s["slots"].clamp(min=0).long()
    picked = s["y"][at].float() * there[:, :, None]
    w = s["weights"] * there
    out = {"out": (picked * w[:, :, None]).sum(1).to(t)}
    if c["grad"]:
        dout = s["dout"].float()
        out["dweights"] = (picked * dout[:, None, :]).sum(2)
        # as in _sorted, one row more for what is not dispatched
        dy = torch.zeros((s["y"].shape[0] + 1, c["cols"]), dtype=t, device="cuda")
        to = torch.where(there, at, s["y"].shape[0])
        dy[to.view(-1)] = (w[:, :, None] * dout[:, None, :]).to(t).view(n * k, -1)
        out["dy"] = dy[:-1]
    return out


def _plain_head(s, c):
    h, w, y = s["h"].float(), s["w"].float(), s["labels"].long()
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    lse = torch.exp(logits - top).sum(1).log() + top[:, 0]
    known = y >= 0
    at = y.clamp(min=0)[:, None]
    loss = torch.where(known, lse - logits.gather(1, at)[:, 0], 0.0)
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        logits -= lse[:, None]
        g = logits.exp_()
        g.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
        g *= torch.where(known, s["dloss"], 0.0)[:, None]
        out["dh"] = (g @ w).to(s["h"].dtype)
        out["dw"] = (g.t() @ h).to(s["w"].dtype)
    return out


# ---- the package's calls --------------------------------------------------

def _kept(s, name, shape, type):
    """A buffer that the program keeps from pass to pass."""
    if name not in s["kept"]:
        s["kept"][name] = torch.empty(shape, dtype=type, device="cuda")
    return s["kept"][name]


def _own_route(s, c, core, stream):
    n, e, k = c["rows"], c["experts"], c["k"]
    ids = _kept(s, "ids", (n, k), torch.int32)
    weights = _kept(s, "weights", (n, k), torch.float32)
    norm = core.ROUTE_ALL if c["norm"] == "all" else core.ROUTE_CHOSEN
    core.route_device(0, s["logits"].data_ptr(), n, e, e, k, norm, ids.data_ptr(),
                      weights.data_ptr(), stream=stream)
    out = {"ids": ids, "weights": weights}
    if c["grad"]:
        d = _kept(s, "dlogits", (n, e), torch.float32)
        core.route_grad_device(0, s["logits"].data_ptr(), n, e, e, k, norm, ids.data_ptr(),
                               weights.data_ptr(), s["dweights"].data_ptr(), d.data_ptr(), e,
                               stream=stream)
        out["dlogits"] = d
    return out


def _own_dispatch(s, c, core, stream):
    n, e, k, cols = c["rows"], c["experts"], c["k"], c["cols"]
    cap = _capacity(c)
    offsets = _kept(s, "offsets", (e + 1,), torch.int64)
    counts = _kept(s, "counts", (e,), torch.int32)
    order = _kept(s, "order", (cap,), torch.int32)
    slots = _kept(s, "slots", (n, k), torch.int32)
    if "workspace" not in s["kept"]:
        s["room"] = core.sort_rows_workspace(n, k, e)
    room = _kept(s, "workspace", (max(1, s["room"]),), torch.uint8)
    core.sort_rows_device(0, s["ids"].data_ptr(), n, k, e, c["align"], offsets.data_ptr(),
                          counts.data_ptr(), order.data_ptr(), slots.data_ptr(),
                          room.data_ptr(), s["room"], stream=stream)
    shape = (cap, cols) if c["target"] == "row" else (cols, cap)
    x = _kept(s, "x", shape, s["x"].dtype)
    core.gather_rows_device(0, CODES[c["type"]], s["x"].data_ptr(), n, cols, s["x"].shape[1],
                            LAYOUTS[c["source"]], k, e, offsets.data_ptr(), order.data_ptr(),
                            slots.data_ptr(), cap, x.data_ptr(), shape[1],
                            LAYOUTS[c["target"]], stream=stream)
    return {"offsets": offsets, "counts": counts, "order": order, "slots": slots, "x": x}


def _own_combine(s, c, core, stream):
    n, k, cols = c["rows"], c["k"], c["cols"]
    cap, code = s["y"].shape[0], CODES[c["type"]]
    out = _kept(s, "out", (n, cols), s["y"].dtype)
    core.combine_rows_device(0, code, s["y"].data_ptr(), cap, cols, cols, s["slots"].data_ptr(),
                             s["weights"].data_ptr(), n, k, out.data_ptr(), cols, stream=stream)
    got = {"out": out}
    if c["grad"]:
        dy = _kept(s, "dy", (cap, cols), s["y"].dtype)
        dw = _kept(s, "dweights", (n, k), torch.float32)
        core.combine_rows_grad_device(0, code, s["y"].data_ptr(), cap, cols, cols,
                                      s["order"].data_ptr(), s["slots"].data_ptr(),
                                      s["weights"].data_ptr(), n, k, s["dout"].data_ptr(), cols,
                                      dy.data_ptr(), cols, dw.data_ptr(), stream=stream)
        got.update(dy=dy, dweights=dw)
    return got


def _own_head(s, c, core, stream):
    n, d, v = c["rows"], c["cols"], c["classes"]
    code = CODES[c["type"]]
    loss = _kept(s, "loss", (n,), torch.float32)
    lse = _kept(s, "lse", (n,), torch.float32)
    if "workspace" not in s["kept"]:
        s["room"] = core.head_workspace(code, n, d, v, grad=c["grad"])
    room = _kept(s, "workspace", (max(1, s["room"]),), torch.uint8)
    core.head_loss_device(0, code, s["h"].data_ptr(), n, d, d, s["w"].data_ptr(), v, d,
                          s["labels"].data_ptr(), loss.data_ptr(), lse.data_ptr(),
                          room.data_ptr(), s["room"], stream=stream)
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        dh = _kept(s, "dh", (n, d), s["h"].dtype)
        dw = _kept(s, "dw", (v, d), s["w"].dtype)
        core.head_grad_device(0, code, s["h"].data_ptr(), n, d, d, s["w"].data_ptr(), v, d,
                              s["labels"].data_ptr(), lse.data_ptr(), s["dloss"].data_ptr(),
                              dh.data_ptr(), d, dw.data_ptr(), d, room.data_ptr(), s["room"],
                              stream=stream)
        out.update(dh=dh, dw=dw)
    return out


def run(s):
    c = s["case"]
    if not own:
        return globals()["_plain_" + c["op"]](s, c)
    from macboost_b200 import _core
    return globals()["_own_" + c["op"]](s, c, _core, torch.cuda.current_stream().cuda_stream)


# ---- the definitions in 64 bits -------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    f64 = torch.float64
    if c["op"] == "route":
        x = s["logits"].to(f64)
        n, e = x.shape
        k = c["k"]
        # the k best by taking the largest k times; argmax of the reversed row picks
        # the last of equal values, so its mirror image is the lowest index
        left, ids = x.clone(), torch.empty((n, k), dtype=torch.int64, device=x.device)
        rows = torch.arange(n, device=x.device)
        for j in range(k):
            best = left.amax(1, keepdim=True)
            first = torch.where(left == best, torch.arange(e, device=x.device), e).amin(1)
            ids[:, j] = torch.where(best[:, 0] > -math.inf, first, -1)
            left[rows, first.clamp(max=e - 1)] = -math.inf
        chosen = torch.zeros((n, e + 1), dtype=torch.bool, device=x.device)
        chosen[rows[:, None], torch.where(ids >= 0, ids, e)] = True
        chosen = chosen[:, :e]
        among = x if c["norm"] == "all" else torch.where(chosen, x, -math.inf)
        p = torch.nan_to_num(torch.softmax(among, 1), nan=0.0)
        at = ids.clamp(min=0)
        weights = torch.where(ids >= 0, p.gather(1, at), 0.0)
        out = {"ids": ids, "weights": weights}
        if c["grad"]:
            up = torch.zeros((n, e + 1), dtype=f64, device=x.device)
            up[rows[:, None], torch.where(ids >= 0, ids, e)] = s["dweights"].to(f64)
            up = up[:, :e]
            up[~chosen] = 0.0
            out["dlogits"] = p * (up - (p * up).sum(1, keepdim=True))
        return out
    if c["op"] == "dispatch":
        x = s["x"] if c["source"] == "row" else s["x"].t()
        n, k, e, a = c["rows"], c["k"], c["experts"], c["align"]
        ids = s["ids"].view(-1)
        got = torch.zeros((_capacity(c), c["cols"]), dtype=f64, device=x.device)
        order = torch.full((_capacity(c),), -1, dtype=torch.int64, device=x.device)
        slots = torch.full((n * k,), -1, dtype=torch.int64, device=x.device)
        starts, counts = [0], []
        for i in range(e):
            mine = (ids == i).nonzero()[:, 0]
            at = slice(starts[-1], starts[-1] + len(mine))
            order[at] = mine
            slots[mine] = torch.arange(at.start, at.stop, device=x.device)
            got[at] = x[mine // k].to(f64)
            counts.append(len(mine))
            starts.append(starts[-1] + -(-len(mine) // a) * a)
        return {"offsets": torch.tensor(starts), "counts": torch.tensor(counts), "order": order,
                "slots": slots.view(n, k),
                "x": got if c["target"] == "row" else got.t().contiguous()}
    if c["op"] == "combine":
        n, k = c["rows"], c["k"]
        out = torch.zeros((n, c["cols"]), dtype=f64, device="cuda")
        dw = torch.zeros((n, k), dtype=f64, device="cuda")
        dy = torch.zeros((_capacity(c), c["cols"]), dtype=f64, device="cuda")
        for j in range(k):
            rows = (s["slots"][:, j] >= 0).nonzero()[:, 0]
            at = s["slots"][rows, j].long()
            w = s["weights"][rows, j].to(f64)[:, None]
            out[rows] += w * s["y"][at].to(f64)
            if c["grad"]:
                up = s["dout"][rows].to(f64)
                dy[at] = w * up
                dw[rows, j] = torch.einsum("nc,nc->n", up, s["y"][at].to(f64))
        return {"out": out, "dy": dy, "dweights": dw} if c["grad"] else {"out": out}
    h, w, y = s["h"].to(f64), s["w"].to(f64), s["labels"].long()
    n, v = c["rows"], c["classes"]
    loss, lse = (torch.zeros(n, dtype=f64, device="cuda") for _ in range(2))
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    step = max(1, min(n, 200_000_000 // v))
    for i in range(0, n, step):
        logp = torch.log_softmax(h[i:i + step] @ w.t(), 1)
        r = torch.arange(logp.shape[0], device="cuda")
        yi = y[i:i + step]
        first = h[i:i + step] @ w[0]
        lse[i:i + step] = first - logp[:, 0]
        has = yi >= 0
        loss[i:i + step] = torch.where(has, -logp[r, yi.clamp(min=0)], 0.0)
        if c["grad"]:
            g = logp.exp()
            g[r[has], yi[has]] -= 1.0
            g *= torch.where(has, s["dloss"][i:i + step].to(f64), 0.0)[:, None]
            dh[i:i + step] = g @ w
            dw += g.t() @ h[i:i + step]
    out = {"loss": loss, "lse": lse}
    return {**out, "dh": dh, "dw": dw} if c["grad"] else out
