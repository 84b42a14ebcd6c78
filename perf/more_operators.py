"""Cases of the operators of a network trained on top of forests: embeddings of the
leaves that rows reach (or of tokens and categories), a gated feed-forward block, and
the norm of all gradients with their clipping.

With `own` false `run` computes each operator with elementary torch operations in
32 bits; with `own` true it calls this package (macboost_b200._core).  `exact`
gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


# ---- cases ----------------------------------------------------------------

def _embed(rows, k, entries, cols, type="f32", scale=1.0, dropped=0.0, grad=False, **kw):
    """Rows of k ids; with k > 1 every id has entries / k of its own (a tree's nodes)."""
    return {"op": "embed", "rows": rows, "k": k, "entries": entries, "cols": cols, "type": type,
            "scale": scale, "dropped": dropped, "grad": grad, **kw}


def _ffn(rows, cols, width, outs, type="bf16", act="silu", grad=False, **kw):
    return {"op": "ffn", "rows": rows, "cols": cols, "width": width, "outs": outs, "type": type,
            "act": act, "grad": grad, **kw}


def _clip(tensors, most, type="f32", ratio=0.25, **kw):
    """Gradients of 1 to `most` values; the largest norm allowed is `ratio` of theirs."""
    return {"op": "clip", "tensors": tensors, "most": most, "type": type, "ratio": ratio, **kw}


def listed():
    return [
        # The next token of one sequence: a single row of the table. Latency counts.
        _embed(1, 1, 131_072, 1_024, type="bf16", scale=32.0, name="embed one token"),
        # Leaves of 100 depth-6 trees (127 nodes each) embedded and added up, one training step
        # over 65,537 rows: few ids, each of them met by thousands of rows.
        _embed(65_537, 100, 12_700, 64, grad=True, name="embed leaves"),
        # A training batch of tokens, a few of them very frequent, some padding.
        _embed(16_384, 1, 131_072, 2_048, type="bf16", scale=32.0, dropped=0.02, grad=True,
               name="embed tokens"),
        # One row through a block: reading the weights is the work.
        _ffn(1, 4_096, 16_384, 4_096, name="ffn one row"),
        # A serving batch of 48 rows.
        _ffn(48, 2_048, 8_192, 2_048, name="ffn serving"),
        # A block over 100 features to ten class margins in float32, odd sizes, one training
        # step.
        _ffn(10_007, 100, 403, 10, type="f32", act="gelu", grad=True, name="ffn features"),
        # A training step in float32.
        _ffn(2_048, 1_024, 4_096, 1_024, type="f32", act="gelu_tanh", grad=True, name="ffn float32"),
        # A prompt of 8,192 rows, no gradient.
        _ffn(8_192, 1_024, 4_096, 1_024, act="gelu", name="ffn prompt"),
        # A training step in half precision.
        _ffn(8_192, 2_048, 8_192, 2_048, grad=True, name="ffn training"),
        # The gradients of a small network. Latency counts.
        _clip(12, 20_000, name="clip small"),
        # Many small tensors of odd sizes, below the largest norm: copied as they are.
        _clip(1_500, 70_001, ratio=2.0, name="clip many"),
        # The gradients of a large network in half precision.
        _clip(300, 8_388_608, type="bf16", name="clip large"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("embed", "ffn", "clip"))
    if op == "embed":
        type = rng.choice(("f32", "bf16", "f16"))
        k = rng.choice((1, _log(rng, 2, 128)))
        cols = _log(rng, 1, 4_096)
        per = _log(rng, 2, max(2, min(262_144, 268_435_456 // cols) // k))
        rows = _log(rng, 1, max(1, min(1_000_000, 268_435_456 // (k * cols), 8_000_000 // k)))
        return _embed(rows, k, per * k, cols, type=type, scale=rng.choice((1.0, 0.125, 8.0)),
                      dropped=rng.choice((0.0, 0.1)), grad=rng.random() < 0.6)
    if op == "clip":
        tensors = _log(rng, 1, 2_000)
        return _clip(tensors, _log(rng, 1, 600_000_000 // max(tensors, 75)),
                     type=rng.choice(("f32", "bf16", "f16")), ratio=rng.choice((0.1, 0.5, 2.0)))
    type = rng.choice(("f32", "bf16", "bf16"))
    cols, width, outs = _log(rng, 8, 4_096), _log(rng, 8, 16_384), _log(rng, 1, 4_096)
    most = 2_400_000_000_000 // ((2 * cols + outs) * width * 6 * (8 if type == "f32" else 1))
    return _ffn(_log(rng, 1, max(1, min(16_384, most))), cols, width, outs, type=type,
                act=rng.choice(tuple(ACTIVATIONS)), grad=rng.random() < 0.6)


def _sizes(c):
    """Lengths of the gradients: spread over 1 ... most on a logarithmic scale, odd ones
    among them, the last one the largest."""
    n = c["tensors"]
    return [max(1, round(c["most"] ** ((i * 7919 % n + 1) / n))) for i in range(n - 1)] + [c["most"]]


def work(c):
    size = 2 if c.get("type") in ("bf16", "f16") else 4
    if c["op"] == "embed":
        n, k, d = c["rows"], c["k"], c["cols"]
        moved = n * k * 4 + min(n * k, c["entries"]) * d * size + n * d * size
        if c["grad"]:
            moved += n * d * size + c["entries"] * d * size
        return {"bytes": moved, "flops": n * k * d * (2 if c["grad"] else 1)}
    if c["op"] == "ffn":
        n, d, f, o = c["rows"], c["cols"], c["width"], c["outs"]
        weights = (2 * d + o) * f
        moved = (weights + n * (d + o)) * size
        if c["grad"]:
            moved += (weights + n * (d + o)) * size
        return {"bytes": moved, "flops": 2.0 * n * weights * (3 if c["grad"] else 1)}
    values = sum(_sizes(c))
    return {"bytes": 2 * values * size, "flops": 3 * values}


# ---- inputs ---------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, type=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(type)

    s = {"case": c, "kept": {}}
    t = TYPES[c["type"]]
    if c["op"] == "embed":
        n, k, entries = c["rows"], c["k"], c["entries"]
        u = torch.rand((n, k), device="cuda", generator=g)
        if k == 1:
            # frequent ids and rare ones, spread over the table
            ids = (u.double() * math.log(entries + 1)).exp().long().sub_(1).clamp_(0, entries - 1)
            ids = (ids * 7919 + seed) % entries
            s["starts"] = None
        else:
            # the leaves of a tree are the second half of its heap, some of them popular
            nodes = entries // k
            ids = nodes // 2 + (u * u * (nodes - nodes // 2)).long()
            ids.clamp_(max=nodes - 1)
            s["starts"] = torch.arange(k, dtype=torch.int32, device="cuda") * nodes
        ids = ids.to(torch.int32)
        if c["dropped"]:
            ids[torch.rand((n, k), device="cuda", generator=g) < c["dropped"]] = -1
        s["ids"] = ids
        s["table"] = normal(entries, c["cols"], scale=0.05, type=t)
        if c["grad"]:
            s["dout"] = normal(n, c["cols"], scale=0.01, type=t)
        return s
    if c["op"] == "ffn":
        n, d, f, o = c["rows"], c["cols"], c["width"], c["outs"]
        s["x"] = normal(n, d, type=t)
        s["w_in"] = normal(2 * f, d, scale=1.0 / math.sqrt(d), type=t)
        s["w_out"] = normal(o, f, scale=1.0 / math.sqrt(f), type=t)
        if c["grad"]:
            s["dy"] = normal(n, o, scale=0.01, type=t)
        return s
    sizes = _sizes(c)
    # as a training program keeps them: one stretch of memory, each tensor on 16 bytes
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += (n + 7) // 8 * 8
    flat = torch.empty(end, dtype=t, device="cuda")
    for at in range(0, end, 1 << 26):
        stop = min(end, at + (1 << 26))
        flat[at:stop] = normal(stop - at, scale=0.02, type=t)
    s["places"] = list(zip(starts, sizes))
    s["grads"] = [flat[at:at + n] for at, n in s["places"]]
    s["length"] = end
    s["max_norm"] = c["ratio"] * 0.02 * math.sqrt(sum(sizes))
    return s


# ---- the plain forms ------------------------------------------------------

def _entries_of(s, c, j):
    """Table rows of the j-th ids, the table's length for those that add nothing."""
    at = s["ids"][:, j].long()
    start = 0 if s["starts"] is None else s["starts"][j].long()
    inside = (at >= 0) & (at + start < c["entries"])
    return torch.where(inside, at + start, c["entries"])


def _plain_embed(s, c):
    t = s["table"].dtype
    n, entries = c["rows"], c["entries"]
    out = torch.zeros((n, c["cols"]), device="cuda")
    for j in range(c["k"]):
        at = _entries_of(s, c, j)
        row = s["table"][at.clamp(max=entries - 1)].float()
        out += torch.where((at < entries)[:, None], row, 0.0)
    got = {"out": (out * c["scale"]).to(t)}
    if c["grad"]:
        # a row more for what adds nothing
        d = torch.zeros((entries + 1, c["cols"]), device="cuda")
        dout = s["dout"].float()
        for j in range(c["k"]):
            d.index_add_(0, _entries_of(s, c, j), dout)
        got["dtable"] = (d[:entries] * c["scale"]).to(t)
    return got


def _activation(a, act):
    """act(a) and its derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-a))
        return a * p, p * (1.0 + a * (1.0 - p))
    if act == "gelu":
        p = 0.5 * (1.0 + torch.erf(a * math.sqrt(0.5)))
        return a * p, p + a * torch.exp(-0.5 * a * a) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (a + 0.044715 * a * a * a))
    return (0.5 * a * (1.0 + th),
            0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * a * a))


def _plain_ffn(s, c):
    t, f = s["x"].dtype, c["width"]
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    pre = x @ w_in.t()
    act, slope = _activation(pre[:, :f], c["act"])
    up = pre[:, f:]
    hidden = act * up
    out = {"y": (hidden @ w_out.t()).to(t)}
    if c["grad"]:
        dy = s["dy"].float()
        dhidden = dy @ w_out
        dpre = torch.cat((dhidden * up * slope, dhidden * act), 1)
        out["dx"] = (dpre @ w_in).to(t)
        out["dw_in"] = (dpre.t() @ x).to(t)
        out["dw_out"] = (dy.t() @ hidden).to(t)
    return out


def _plain_clip(s, c):
    squares = torch.stack([(g.float() * g.float()).sum() for g in s["grads"]])
    norm = squares.double().sum().sqrt()
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0).float()
    # laid out as the gradients are, zeros between them
    out = torch.zeros(s["length"], dtype=s["grads"][0].dtype, device="cuda")
    for g, (at, n) in zip(s["grads"], s["places"]):
        out[at:at + n] = g.float() * factor
    return {"norm": norm.float(), "grads": out}


# ---- the package's calls --------------------------------------------------

def _kept(s, name, shape, type):
    """A buffer that the program keeps from pass to pass."""
    if name not in s["kept"]:
        s["kept"][name] = torch.empty(shape, dtype=type, device="cuda")
    return s["kept"][name]


def _own_embed(s, c, core, stream):
    n, k, entries, cols = c["rows"], c["k"], c["entries"], c["cols"]
    code, t = CODES[c["type"]], s["table"].dtype
    starts = 0 if s["starts"] is None else s["starts"].data_ptr()
    out = _kept(s, "out", (n, cols), t)
    core.embed_device(0, code, s["table"].data_ptr(), entries, cols, cols, s["ids"].data_ptr(), n, k,
                      starts, c["scale"], out.data_ptr(), cols, stream=stream)
    got = {"out": out}
    if c["grad"]:
        if "workspace" not in s["kept"]:
            s["room"] = core.embed_workspace(entries, cols, n, k)
        room = _kept(s, "workspace", (max(1, s["room"]),), torch.uint8)
        d = _kept(s, "dtable", (entries, cols), t)
        core.embed_grad_device(0, code, s["dout"].data_ptr(), n, cols, cols, s["ids"].data_ptr(), k,
                               starts, c["scale"], d.data_ptr(), entries, cols, room.data_ptr(),
                               s["room"], stream=stream)
        got["dtable"] = d
    return got


def _own_ffn(s, c, core, stream):
    n, d, f, o = c["rows"], c["cols"], c["width"], c["outs"]
    code, t, act = CODES[c["type"]], s["x"].dtype, ACTIVATIONS[c["act"]]
    hidden = _kept(s, "hidden", (n, f), t)
    pre = _kept(s, "pre", (n, 2 * f), torch.float32).data_ptr() if c["grad"] else 0
    y = _kept(s, "y", (n, o), t)
    if "workspace" not in s["kept"]:
        s["room"] = core.ffn_workspace(code, n, d, f, o, grad=c["grad"])
    room = _kept(s, "workspace", (max(1, s["room"]),), torch.uint8)
    block = (s["x"].data_ptr(), n, d, d, s["w_in"].data_ptr(), f, d, s["w_out"].data_ptr(), o, f)
    core.ffn_device(0, code, act, *block, hidden.data_ptr(), f, pre, 2 * f, y.data_ptr(), o,
                    room.data_ptr(), s["room"], stream=stream)
    out = {"y": y}
    if c["grad"]:
        dx = _kept(s, "dx", (n, d), t)
        dw_in = _kept(s, "dw_in", (2 * f, d), t)
        dw_out = _kept(s, "dw_out", (o, f), t)
        core.ffn_grad_device(0, code, act, *block, hidden.data_ptr(), f, pre, 2 * f,
                             s["dy"].data_ptr(), o, dx.data_ptr(), d, dw_in.data_ptr(), d,
                             dw_out.data_ptr(), f, room.data_ptr(), s["room"], stream=stream)
        out.update(dx=dx, dw_in=dw_in, dw_out=dw_out)
    return out


def _own_clip(s, c, core, stream):
    kept = s["kept"]
    if "clipped" not in kept:
        grads = s["grads"]
        # laid out as the gradients are, zeros between them
        flat = torch.zeros(s["length"], dtype=grads[0].dtype, device="cuda")
        kept["clipped"] = flat
        kept["list"] = core.GradientList([CODES[c["type"]]] * len(grads),
                                         [g.data_ptr() for g in grads], [g.numel() for g in grads],
                                         [flat[at:].data_ptr() for at, _ in s["places"]])
        s["room"] = core.clip_workspace(kept["list"])
    norm = _kept(s, "norm", (), torch.float32)
    room = _kept(s, "workspace", (max(1, s["room"]),), torch.uint8)
    core.clip_device(0, kept["list"], s["max_norm"], norm.data_ptr(), room.data_ptr(), s["room"],
                     stream=stream)
    return {"norm": norm, "grads": kept["clipped"]}


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
    if c["op"] == "embed":
        n, k, entries, cols = c["rows"], c["k"], c["entries"], c["cols"]
        at = s["ids"].long()
        if s["starts"] is not None:
            at = torch.where(at >= 0, at + s["starts"].long(), -1)
        there = at >= 0
        out = torch.zeros((n, cols), dtype=f64, device="cuda")
        d = torch.zeros((entries, cols), dtype=f64, device="cuda") if c["grad"] else None
        for j in range(k):
            rows = there[:, j].nonzero()[:, 0]
            step = max(1, 100_000_000 // cols)
            for i in range(0, len(rows), step):
                r = rows[i:i + step]
                out[r] += c["scale"] * s["table"][at[r, j]].to(f64)
                if c["grad"]:
                    d.index_add_(0, at[r, j], s["dout"][r].to(f64), alpha=c["scale"])
        return {"out": out, "dtable": d} if c["grad"] else {"out": out}
    if c["op"] == "ffn":
        x, w_in, w_out = (s[name].to(f64).requires_grad_(c["grad"]) for name in ("x", "w_in", "w_out"))
        gate, up = (x @ w_in.t()).split(c["width"], 1)
        fn = torch.nn.functional
        act = (fn.silu(gate) if c["act"] == "silu"
               else fn.gelu(gate, approximate="none" if c["act"] == "gelu" else "tanh"))
        y = (act * up) @ w_out.t()
        out = {"y": y.detach()}
        if c["grad"]:
            out["dx"], out["dw_in"], out["dw_out"] = torch.autograd.grad(y, (x, w_in, w_out),
                                                                         s["dy"].to(f64))
        return out
    norm = sum(float((g.to(f64) ** 2).sum()) for g in s["grads"]) ** 0.5
    factor = min(1.0, s["max_norm"] / norm) if norm > 0 else 1.0
    out = torch.zeros(s["length"], dtype=f64, device="cuda")
    for g, (at, n) in zip(s["grads"], s["places"]):
        out[at:at + n] = g.to(f64) * factor
    return {"norm": torch.tensor(norm, dtype=f64), "grads": out}
