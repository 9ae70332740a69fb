"""Cases and plain forms of the library's operators for language-model training and serving:
embedding lookup and its gradient, tokens sorted by expert and back with the gradient, and the
clipping of gradients by their global norm.

`run` makes the library's calls where `own` is true and otherwise computes the same outputs
with elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8}
_EPS = 1e-6  # beside the norm in the clipping coefficient


def _dcopy():
    import sys
    if "data-copy_b200" not in sys.path:
        sys.path.insert(0, "data-copy_b200")
    import dcopy
    return dcopy


# ---- cases ------------------------------------------------------------------------------


def _embed(op, tokens, vocab, width, table, out, pad=0.0, scale=1.0, ids="int64"):
    return {"op": op, "tokens": tokens, "vocab": vocab, "width": width, "table": table, "out": out,
            "pad": pad, "scale": scale, "ids": ids}


def _experts(op, tokens, slots, experts, width, dtype, align=1, drop=0.0, weighted=True, ids="int64"):
    return {"op": op, "tokens": tokens, "slots": slots, "experts": experts, "width": width,
            "type": dtype, "align": align, "drop": drop, "weighted": weighted, "ids": ids}


def _clip(layers, width, vocab, dtype, out, ratio):
    return {"op": "clip", "layers": layers, "width": width, "vocab": vocab, "type": dtype, "out": out,
            "ratio": ratio}


def listed():
    bf, hf, f = "bfloat16", "float16", "float32"
    return [
        # One decoding step of a batch of 64 sequences: the next tokens' rows. Latency counts.
        {"name": "embed decode", **_embed("embed", 64, 32000, 2048, bf, bf)},
        # A packed training batch: 32 Ki tokens of a large vocabulary, scaled by sqrt(width), padding ids.
        {"name": "embed prompt", **_embed("embed", 32768, 131072, 4096, bf, bf, 0.02, 64.0)},
        # Gradient of a small model's embedding, ragged: odd tokens, vocabulary and width; half in, fp32 out.
        {"name": "embed_grad ragged", **_embed("embed_grad", 2047, 32003, 1031, hf, f, 0.1, 32.0, "int32")},
        # Gradient of a large embedding for a packed batch: every row of the table is written.
        {"name": "embed_grad batch", **_embed("embed_grad", 16384, 131072, 4096, bf, bf, 0.02)},
        # One decoding step of 32 sequences through a mixture of experts: sort, then rows to the experts.
        {"name": "to_experts decode", **_experts("to_experts", 32, 8, 64, 2048, bf)},
        # A prompt or training batch to its experts; segments start at multiples of 128 for tiled products.
        {"name": "to_experts batch", **_experts("to_experts", 16384, 8, 128, 4096, bf, 128)},
        # The way back of the decoding step: a weighted sum of 8 rows a token.
        {"name": "from_experts decode", **_experts("from_experts", 32, 8, 64, 2048, bf)},
        # The way back of a batch in half precision, some choices dropped for lack of capacity.
        {"name": "from_experts batch", **_experts("from_experts", 8191, 4, 64, 5120, hf, 16, 0.1, True, "int32")},
        # Training in fp32 on a small batch with a width that no wide vector divides.
        {"name": "from_experts_grad ragged", **_experts("from_experts_grad", 1501, 2, 8, 1002, f, 1, 0.05)},
        # Gradient of the weighted sum for a batch: row gradients and the weights' gradients.
        {"name": "from_experts_grad batch", **_experts("from_experts_grad", 16384, 8, 128, 2048, bf)},
        # A small model's fp32 gradients, some 50 tensors of odd sizes: two short passes. Latency counts.
        {"name": "clip small", **_clip(6, 131, 2003, f, f, 0.3)},
        # A large model's bf16 gradients, some 200 tensors, clipped into the buffer the optimiser reads.
        {"name": "clip large", **_clip(24, 1280, 50000, bf, bf, 0.37)},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, widths=(64, 128, 256, 384, 640, 896, 1280, 1536, 2048, 2560, 4096, 5120, 6400, 8192)):
    """Mostly a width as models have it; else any whole number of the same range."""
    return rng.choice(widths) if rng.random() < 0.65 else _log(rng, widths[0], widths[-1])


_MOST = 1.1e9  # bytes of a drawn case


def draw(rng):
    while True:
        op = rng.choice(["embed", "embed_grad", "to_experts", "from_experts", "from_experts_grad", "clip"])
        a, b = rng.choice(list(_TYPES)), rng.choice(list(_TYPES))
        ids = rng.choice(["int32", "int64"])
        if op in ("embed", "embed_grad"):
            c = _embed(op, _log(rng, 1, 65536), _log(rng, 1000, 262144), _width(rng), a, b,
                       rng.choice([0.0, 0.02, 0.3]), rng.choice([1.0, 0.125, 45.25]), ids)
        elif op == "clip":
            c = _clip(_log(rng, 1, 32), _width(rng, (64, 96, 160, 256, 320, 640, 1280, 1536)), _log(rng, 1000, 60000), a,
                      rng.choice([a, "float32"]), rng.choice([0.1, 0.9, 2.0]))
        else:
            c = _experts(op, _log(rng, 1, 32768), rng.choice([1, 2, 4, 6, 8]), _log(rng, 8, 384), _width(rng),
                         a, rng.choice([1, 1, 16, 128]), rng.choice([0.0, 0.0, 0.1]), rng.random() < 0.7, ids)
        if _bytes(c) <= _MOST:
            return c


def _rows(c):
    """Rows of the buffer in expert order: every entry and each expert's padding."""
    n = c["tokens"] * c["slots"]
    return n + min(c["experts"], n) * (c["align"] - 1)


def _shapes(c):
    """The weights of a plain decoder: an embedding, then per layer two gains, two biases and four matrices."""
    d = c["width"]
    layer = [(d,), (d, 3 * d), (3 * d,), (d, d), (d,), (d, 4 * d), (4 * d,), (4 * d, d)]
    return [(c["vocab"], d)] + layer * c["layers"] + [(d,)]


def _distinct(c):
    """Expected number of different table rows read (ids are log-uniform over the vocabulary)."""
    v = np.arange(1, c["vocab"] + 1, dtype=np.float64)
    p = np.log1p(1.0 / v) / math.log(c["vocab"] + 1.0)
    return float((1.0 - np.exp(-c["tokens"] * (1.0 - c["pad"]) * p)).sum())


def _bytes(c):
    if c["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(c))
        return n * (_BYTES[c["type"]] + _BYTES[c["out"]])
    if c["op"] == "embed":
        rows, s = c["tokens"] * c["width"], _BYTES[c["out"]]
        return rows * s + _distinct(c) * c["width"] * _BYTES[c["table"]] + c["tokens"] * _BYTES[c["ids"]]
    if c["op"] == "embed_grad":
        return (c["tokens"] * c["width"] * _BYTES[c["table"]] + c["vocab"] * c["width"] * _BYTES[c["out"]]
                + c["tokens"] * _BYTES[c["ids"]])
    n, s = c["tokens"] * c["slots"], c["width"] * _BYTES[c["type"]]
    kept = n * (1.0 - c["drop"])
    if c["op"] == "to_experts":
        return n * (_BYTES[c["ids"]] + 4) + _rows(c) * (4 + s) + c["tokens"] * s
    if c["op"] == "from_experts":
        return kept * s + c["tokens"] * s + n * 8
    return kept * s + c["tokens"] * s + _rows(c) * s + n * 12


def work(case):
    c = case
    if c["op"] == "clip":
        flops = 3.0 * sum(math.prod(s) for s in _shapes(c))
    elif c["op"] in ("embed", "embed_grad"):
        flops = 1.0 * c["tokens"] * c["width"]
    else:
        flops = {"to_experts": 0.0, "from_experts": 2.0, "from_experts_grad": 3.0}[c["op"]] \
            * c["tokens"] * c["slots"] * c["width"]
    return {"bytes": _bytes(c), "flops": flops}


# ---- inputs -----------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    """Normal values, made in pieces so that a large tensor needs no 32-bit copy of itself."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    for part in t.view(-1).split(1 << 26):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return t


def _token_ids(c, g):
    """Ids as text has them: the frequency falls with the rank; -1 where a sequence is padded."""
    u = torch.rand(c["tokens"], generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(c["vocab"] + 1.0)) - 1.0).long().clamp_(0, c["vocab"] - 1)
    padded = torch.rand(c["tokens"], generator=g, device="cuda") < c["pad"]
    return torch.where(padded, -1, ids).to(torch.int32 if c["ids"] == "int32" else torch.int64)


def _routes(c, g):
    """Each token's experts and weights: the highest of scores whose means differ from expert to
    expert, as an imbalanced router's do; -1 where a choice was dropped."""
    bias = torch.randn(c["experts"], generator=g, device="cuda") * 0.5
    score = torch.randn(c["tokens"], c["experts"], generator=g, device="cuda") + bias
    top, ids = score.topk(c["slots"], dim=1)
    gone = torch.rand(ids.shape, generator=g, device="cuda") < c["drop"]
    ids = torch.where(gone, -1, ids).to(torch.int32 if c["ids"] == "int32" else torch.int64)
    return ids.contiguous(), torch.softmax(top, dim=1).contiguous()


def prepare(case, seed):
    c, g = case, _gen(seed)
    st = {"case": c}
    if c["op"] == "clip":
        grads, outs, flats = [], [], []
        shapes = _shapes(c)
        for dtype in (c["type"], c["out"]):  # views of one buffer, as gradient buckets are
            flats.append(torch.empty(sum(math.prod(s) for s in shapes), dtype=_TYPES[dtype], device="cuda"))
        at = 0
        for s in shapes:
            n = math.prod(s)
            grads.append(flats[0][at:at + n].view(s))
            outs.append(flats[1][at:at + n].view(s))
            grads[-1].copy_(_normal(g, s, _TYPES[c["type"]], 1e-2 / math.sqrt(s[-1])))
            at += n
        # The bound lies at `ratio` times the norm that such gradients have.
        norm = 1e-2 * math.sqrt(sum(math.prod(s) / s[-1] for s in shapes))
        st.update(grads=grads, outs=outs, flat=flats[1], max_norm=c["ratio"] * norm,
                  norm=torch.empty(1, device="cuda"))
        if own:
            st["list"] = _dcopy().GradList(grads, outs)
        return st
    if c["op"] in ("embed", "embed_grad"):
        st["ids"] = _token_ids(c, g)
        t, o, shape = _TYPES[c["table"]], _TYPES[c["out"]], (c["tokens"], c["width"])
        if c["op"] == "embed":
            st["table"] = _normal(g, (c["vocab"], c["width"]), t, 0.02)
            st["out"] = torch.empty(shape, dtype=o, device="cuda")
        else:
            st["dout"] = _normal(g, shape, t, 1e-3 if t != torch.float16 else 1.0)
            st["grad"] = torch.empty((c["vocab"], c["width"]), dtype=o, device="cuda")
            if own:
                st["space"] = torch.empty(_dcopy().embedding_grad_workspace(c["tokens"], c["vocab"], c["width"]),
                                          dtype=torch.uint8, device="cuda")
        return st
    t, rows = _TYPES[c["type"]], _rows(c)
    ids, weights = _routes(c, g)
    shape = (c["tokens"], c["width"])
    whole = dict(dtype=torch.int32, device="cuda")
    if c["op"] == "to_experts":
        st.update(ids=ids, x=_normal(g, shape, t), out=torch.empty((rows, c["width"]), dtype=t, device="cuda"),
                  dest=torch.empty(ids.shape, **whole), source=torch.empty(rows, **whole),
                  offsets=torch.empty(c["experts"] + 1, **whole))
        if own:
            st["space"] = torch.empty(_dcopy().expert_sort_workspace(ids.numel(), c["experts"]),
                                      dtype=torch.uint8, device="cuda")
        return st
    dest, source, _ = _sort(ids, c["experts"], c["align"], rows)
    st.update(dest=dest, source=source, weights=weights if c["weighted"] or c["op"] != "from_experts" else None)
    st["y"] = _normal(g, (rows, c["width"]), t)
    if c["op"] == "from_experts":
        st["out"] = torch.empty(shape, dtype=t, device="cuda")
    else:
        st.update(dout=_normal(g, shape, t), dy=torch.empty((rows, c["width"]), dtype=t, device="cuda"),
                  dweights=torch.empty_like(weights))
    return st


# ---- the plain forms --------------------------------------------------------------------


def _sort(ids, experts, align, rows):
    """(dest, source, offsets) of the entries in expert order, the earlier entry first."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    by = key[order]
    count = torch.bincount(key, minlength=experts + 1)
    first = torch.cumsum(count, 0) - count
    padded = (count[:experts] + align - 1) // align * align
    offsets = torch.cat([padded.new_zeros(1), torch.cumsum(padded, 0)])
    row = torch.arange(flat.numel(), device=flat.device) - first[by] + offsets[by]
    row = torch.where(by < experts, row, rows)  # what belongs to no expert goes behind the end
    dest = torch.empty_like(flat)
    dest[order] = torch.where(by < experts, row, -1)
    source = flat.new_full((rows + 1,), -1)
    source[row] = torch.where(by < experts, order, -1)
    return dest.view(ids.shape).int(), source[:rows].int(), offsets.int()


def _plain(st):
    c = st["case"]
    if c["op"] == "clip":
        flat = torch.cat([g.reshape(-1) for g in st["grads"]]).float()
        norm = flat.square().sum().sqrt()
        factor = torch.clamp(st["max_norm"] / (norm + _EPS), max=1.0)
        return {"norm": norm.reshape(1), "out": (flat * factor).to(st["flat"].dtype)}
    if c["op"] == "embed":
        known = (st["ids"] >= 0) & (st["ids"] < c["vocab"])
        rows = st["table"][torch.where(known, st["ids"], 0)].float()
        return {"out": (rows * (known * c["scale"])[:, None]).to(st["out"].dtype)}
    if c["op"] == "embed_grad":
        known = (st["ids"] >= 0) & (st["ids"] < c["vocab"])
        rows = st["dout"].float() * known[:, None]
        total = torch.zeros((c["vocab"], c["width"]), device="cuda")
        total.index_add_(0, torch.where(known, st["ids"], 0), rows)
        return {"grad": (total * c["scale"]).to(st["grad"].dtype)}
    if c["op"] == "to_experts":
        dest, source, offsets = _sort(st["ids"], c["experts"], c["align"], st["out"].shape[0])
        rows = st["x"].float()[source.clamp(min=0) // c["slots"]] * (source >= 0)[:, None]
        return {"dest": dest, "source": source, "offsets": offsets, "out": rows.to(st["out"].dtype)}
    kept = st["dest"] >= 0
    rows = st["y"].float()[st["dest"].clamp(min=0)]
    if c["op"] == "from_experts":
        factor = kept if st["weights"] is None else kept * st["weights"]
        return {"out": (rows * factor[:, :, None]).sum(1).to(st["out"].dtype)}
    dout = st["dout"].float()
    dweights = (rows * dout[:, None, :]).sum(2) * kept
    token = st["source"].clamp(min=0)
    factor = st["weights"].reshape(-1)[token] * (st["source"] >= 0)
    dy = dout[token // c["slots"]] * factor[:, None]
    return {"dy": dy.to(st["dy"].dtype), "dweights": dweights}


def _calls(st):
    c, d = st["case"], _dcopy()
    if c["op"] == "clip":
        d.clip_grad_norm(st["list"], st["max_norm"], st["norm"], eps=_EPS)
        return {"norm": st["norm"], "out": st["flat"]}
    if c["op"] == "embed":
        d.embedding_lookup(st["out"], st["table"], st["ids"], scale=c["scale"])
        return {"out": st["out"]}
    if c["op"] == "embed_grad":
        d.embedding_grad(st["grad"], st["dout"], st["ids"], scale=c["scale"], workspace=st["space"])
        return {"grad": st["grad"]}
    if c["op"] == "to_experts":
        d.expert_sort(st["dest"], st["source"], st["offsets"], st["ids"], align=c["align"], workspace=st["space"])
        d.expert_dispatch(st["out"], st["x"], st["dest"], st["source"])
        return {"dest": st["dest"], "source": st["source"], "offsets": st["offsets"], "out": st["out"]}
    if c["op"] == "from_experts":
        d.expert_combine(st["out"], st["y"], st["dest"], st["weights"])
        return {"out": st["out"]}
    d.expert_combine_grad(st["dy"], st["dweights"], st["dout"], st["y"], st["dest"], st["weights"], st["source"])
    return {"dy": st["dy"], "dweights": st["dweights"]}


def run(state):
    return _calls(state) if own else _plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------------


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] == "clip":
        square = math.fsum(float((g.double() ** 2).sum()) for g in st["grads"])
        norm = math.sqrt(square)
        factor = min(1.0, st["max_norm"] / (norm + _EPS))
        return {"norm": torch.tensor([norm], dtype=torch.float64),
                "out": torch.cat([g.double().view(-1).mul_(factor) for g in st["grads"]])}
    if c["op"] == "embed":
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        at = torch.nonzero((st["ids"] >= 0) & (st["ids"] < c["vocab"]))[:, 0]
        out[at] = torch.index_select(st["table"], 0, st["ids"][at].long()).double() * c["scale"]
        return {"out": out}
    if c["op"] == "embed_grad":
        # Sums over the runs of equal ids as differences of a running sum.
        at = torch.nonzero((st["ids"] >= 0) & (st["ids"] < c["vocab"]))[:, 0]
        grad = torch.zeros(st["grad"].shape, dtype=torch.float64, device="cuda")
        if at.numel():
            value, order = torch.sort(st["ids"][at].long())
            run_sum = torch.cumsum(st["dout"][at[order]].double(), 0)
            last = torch.nonzero(torch.cat([value[1:] != value[:-1], value.new_ones(1, dtype=torch.bool)]))[:, 0]
            ends = run_sum[last]
            ends[1:] -= run_sum[last[:-1]]
            grad[value[last]] = ends * c["scale"]
        return {"grad": grad}
    if c["op"] == "to_experts":
        # The rows of each expert one after the other, by a sort on the host.
        flat = st["ids"].reshape(-1).cpu().numpy().astype(np.int64)
        entries = np.flatnonzero((flat >= 0) & (flat < c["experts"]))
        entries = entries[np.argsort(flat[entries], kind="stable")]
        count = np.bincount(flat[entries], minlength=c["experts"])
        lead = np.cumsum(-(-count // c["align"]) * c["align"] - count)
        row = np.arange(entries.size) + (lead - (-(-count // c["align"]) * c["align"] - count))[flat[entries]]
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        out[torch.from_numpy(row).cuda()] = st["x"].double()[torch.from_numpy(entries // c["slots"]).cuda()]
        return {"dest": None, "source": None, "offsets": None, "out": out}
    token, slot = torch.nonzero(st["dest"] >= 0, as_tuple=True)
    row = st["dest"][token, slot].long()
    w = None if st["weights"] is None else st["weights"].double()[token, slot]
    if c["op"] == "from_experts":
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        for j in range(c["slots"]):
            m = slot == j
            part = st["y"][row[m]].double()
            out[token[m]] += part if w is None else part * w[m, None]
        return {"out": out}
    dy = torch.zeros(st["dy"].shape, dtype=torch.float64, device="cuda")
    dweights = torch.zeros(st["dweights"].shape, dtype=torch.float64, device="cuda")
    for part in torch.arange(row.numel(), device="cuda").split(1 << 14):
        t, r, j = token[part], row[part], slot[part]
        d = st["dout"][t].double()
        dy[r] = d * w[part, None]
        dweights[t, j] = torch.linalg.vecdot(d, st["y"][r].double())
    return {"dy": dy, "dweights": dweights}
