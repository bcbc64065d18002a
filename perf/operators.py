"""Cases of the training-block operators: element embedding, gated feed-forward, irreps dropout.

``run`` makes one pass through an operator in its plain form (elementary torch operations in
32 bits, rounded once at the end) or, with ``own`` set, through this repository's entry
points. Rows are rank blocks l = 0..l_max of (2l+1, channels), components outer, channels
contiguous, as everywhere in this repository; l_max = 0 is a plain (rows, channels) matrix.
"""

import math

import numpy as np
import torch

own = False

F32, BF16 = "float32", "bfloat16"
TYPES = {F32: torch.float32, BF16: torch.bfloat16}
SIZE = {F32: 4, BF16: 2}


def listed():
    return [
        # the 192-atom water box: element features of the atoms, where launch latency counts
        {"name": "embed_atoms_192", "op": "embed", "rows": 192, "vocab": 2, "dim": 64, "dtype": F32, "train": False,
         "scale": 1.0, "offset": 0.0, "law": "few"},
        # element-dependent path weights 1 + delta[type] of a 128-channel (3,3)->3 product on 27,648 atoms
        {"name": "embed_path_weights", "op": "embed", "rows": 27648, "vocab": 2, "dim": 2944, "dtype": F32,
         "train": False, "scale": 1.0, "offset": 1.0, "law": "few"},
        # element features of the edges' senders (16 per edge) and their gradient: long runs of few types
        {"name": "embed_train_edges", "op": "embed", "rows": 1492998, "vocab": 4, "dim": 16, "dtype": F32,
         "train": True, "scale": 1.0, "offset": 0.0, "law": "few"},
        # a generic token table in 16 bits: many types, most of them rare, some frequent
        {"name": "embed_train_tokens_bf16", "op": "embed", "rows": 65537, "vocab": 50000, "dim": 512, "dtype": BF16,
         "train": True, "scale": 22.627417, "offset": 0.0, "law": "zipf"},
        # gate layer of the 192-atom run (64 channels, ranks <= 2), forward
        {"name": "gated_atoms_192", "op": "gated", "rows": 192, "l_max": 2, "c": 64, "h": 64, "act": "sigmoid",
         "bias": True, "dtype": F32, "train": False},
        # gate layer of the 27,648-atom water box (128 channels, ranks <= 3), forward
        {"name": "gated_water", "op": "gated", "rows": 27648, "l_max": 3, "c": 128, "h": 128, "act": "sigmoid",
         "bias": True, "dtype": F32, "train": False},
        # one training pass over 32 random-walk molecules (about 1,300 atoms, 64 channels, ranks <= 2)
        {"name": "gated_train_molecules", "op": "gated", "rows": 1283, "l_max": 2, "c": 64, "h": 64, "act": "silu",
         "bias": True, "dtype": F32, "train": True},
        # the same with the gradients of everything, for a large structure
        {"name": "gated_train_water", "op": "gated", "rows": 27648, "l_max": 3, "c": 128, "h": 128, "act": "sigmoid",
         "bias": True, "dtype": F32, "train": True},
        # scalars only, 16-bit, hidden width unlike the input's, odd row count
        {"name": "gated_train_rows_bf16", "op": "gated", "rows": 100003, "l_max": 0, "c": 96, "h": 200, "act": "silu",
         "bias": False, "dtype": BF16, "train": True},
        # whole-irrep dropout of the hidden features, forward and gradient: small, MD-sized, and odd 16-bit rows
        {"name": "dropout_atoms_192", "op": "dropout", "rows": 192, "l_max": 2, "c": 64, "p": 0.1, "dtype": F32},
        {"name": "dropout_water", "op": "dropout", "rows": 27648, "l_max": 3, "c": 128, "p": 0.1, "dtype": F32},
        {"name": "dropout_rows_bf16", "op": "dropout", "rows": 200003, "l_max": 0, "c": 100, "p": 0.25,
         "dtype": BF16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "gated", "dropout"])
    dtype = rng.choice([F32, F32, BF16])
    if op == "embed":
        dim = _log(rng, 5, 2944)
        rows = _log(rng, 150, min(1492998, 80_000_000 // dim))
        law = rng.choice(["few", "zipf"])
        vocab = _log(rng, 2, 118) if law == "few" else _log(rng, 300, 50000)
        return {"op": op, "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype, "train": rng.random() < 0.7,
                "scale": rng.choice([1.0, math.sqrt(dim)]), "offset": rng.choice([0.0, 1.0]), "law": law}
    if op == "gated":
        l_max = rng.choice([0, 1, 2, 3])
        c, h = _log(rng, 16, 256 if l_max == 0 else 128), _log(rng, 16, 256 if l_max == 0 else 128)
        if rng.random() < 0.7:  # channel counts are mostly multiples of 8, and at times anything
            c, h = (c + 7) // 8 * 8, (h + 7) // 8 * 8
        most = 27648 * 20 * 128 * 128 // (((l_max + 1) ** 2 + l_max + 1) * c * h)
        rows = _log(rng, 100, min(most, 200003 if l_max == 0 else 27648))
        return {"op": op, "rows": rows, "l_max": l_max, "c": c, "h": h, "act": rng.choice(["silu", "sigmoid"]),
                "bias": rng.random() < 0.5, "dtype": dtype, "train": rng.random() < 0.6}
    l_max = rng.choice([0, 1, 2, 3])
    c = _log(rng, 16, 256)
    rows = _log(rng, 150, min(200003, 27648 * 16 * 128 // ((l_max + 1) ** 2 * c)))
    return {"op": op, "rows": rows, "l_max": l_max, "c": c, "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "dtype": dtype}


def _types(case, gen):
    """Token of every row: a handful of elements of unequal share, or a long-tailed vocabulary."""
    rows, vocab = case["rows"], case["vocab"]
    u = torch.rand(rows, generator=gen, device="cuda")
    if case["law"] == "few":
        share = torch.rand(vocab, generator=gen, device="cuda") + 0.1
    else:
        share = 1.0 / torch.arange(2, vocab + 2, device="cuda", dtype=torch.float32)
    cdf = torch.cumsum(share.double(), 0)
    return torch.searchsorted((cdf / cdf[-1]).float(), u).clamp_(max=vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "embed":
        s["table"] = normal(case["vocab"], case["dim"], scale=0.05 if case["offset"] else 1.0)
        s["index"] = _types(case, gen)
        if case["train"]:
            s["grad"] = normal(case["rows"], case["dim"], scale=0.01)
            s["table"].requires_grad_(True)
        return s
    comps = (case["l_max"] + 1) ** 2
    spread = torch.exp(0.25 * torch.randn(case["rows"], 1, generator=gen, device="cuda"))
    s["x"] = (torch.randn(case["rows"], comps * case["c"], generator=gen, device="cuda") * spread).to(dtype)
    if case["op"] == "dropout":
        s["rng"] = torch.tensor([seed * 7919 + 3, seed % 1000], dtype=torch.int64, device="cuda")
        s["grad"] = normal(*s["x"].shape, scale=0.01)
        s["x"].requires_grad_(True)
        return s
    c, h, ranks = case["c"], case["h"], case["l_max"] + 1
    s["value_weights"] = [normal(h, c) for _ in range(ranks)]
    s["gate_weight"] = normal(ranks * h, c)
    s["gate_bias"] = normal(ranks * h, scale=0.1) if case["bias"] else None
    # one scale for each rank's value map, the gate map's, and the activation's
    s["scales"] = torch.tensor([c ** -0.5] * (ranks + 1) + [1.8462285 if case["act"] == "sigmoid" else 1.6765325],
                               device="cuda")
    if case["train"]:
        s["grad"] = normal(case["rows"], comps * h, scale=0.01)
        for t in _gated_inputs(s):
            t.requires_grad_(True)
    return s


def _gated_inputs(s):
    """What a training pass returns gradients of, in their order."""
    return [s["x"], *s["value_weights"], s["gate_weight"]] + ([s["gate_bias"]] if s["gate_bias"] is not None else [])


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {"embed": _plain_embed, "gated": _plain_gated, "dropout": _plain_dropout}[case["op"]](state, case)


# ------------------------------------------------------------------------------ this repository's operators


def _run_own(s, case):
    from flashcart_b200 import ops

    if case["op"] == "embed":
        y = ops.embedding(s["table"], s["index"], case["scale"], case["offset"])
        if not case["train"]:
            return {"out": y}
        return {"out": y.detach(), "grad_table": torch.autograd.grad(y, s["table"], s["grad"])[0]}
    if case["op"] == "dropout":
        y = ops.irreps_dropout(s["x"], s["rng"], case["p"], case["l_max"])
        return {"out": y.detach(), "grad_x": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    y = ops.gated_feed_forward(s["x"], s["value_weights"], s["gate_weight"], s["gate_bias"], s["scales"],
                               case["l_max"], case["act"])
    if not case["train"]:
        return {"out": y}
    return {"out": y.detach(), "grads": list(torch.autograd.grad(y, _gated_inputs(s), s["grad"]))}


# ------------------------------------------------------------------------------ plain forms


def _plain_embed(s, case):
    table, index = s["table"].float(), s["index"]
    out = (case["offset"] + case["scale"] * table[index]).to(s["table"].dtype)
    if not case["train"]:
        return {"out": out}
    g = torch.zeros_like(table).index_add_(0, index, s["grad"].float()) * case["scale"]
    return {"out": out, "grad_table": g.to(s["table"].dtype)}


def _rank_of_component(l_max, device="cuda"):
    k = torch.arange((l_max + 1) ** 2, device=device, dtype=torch.float64)
    return k.sqrt().floor().long()


def _plain_gated(s, case):
    n, c, h, ranks = case["rows"], case["c"], case["h"], case["l_max"] + 1
    comps = ranks * ranks
    of = _rank_of_component(case["l_max"])
    x = s["x"].float().view(n, comps, c).transpose(0, 1)
    sc = s["scales"]
    wv = torch.stack([w.float() for w in s["value_weights"]]) * sc[:ranks, None, None]
    wg = s["gate_weight"].float() * sc[ranks]
    pre = x[0] @ wg.t()
    if s["gate_bias"] is not None:
        pre = pre + s["gate_bias"].float()
    sig = 1.0 / (1.0 + torch.exp(-pre))
    gate = sc[ranks + 1] * (sig if case["act"] == "sigmoid" else pre * sig)
    per_comp = gate.view(n, ranks, h).transpose(0, 1)[of]
    values = x @ wv[of].transpose(1, 2)
    dtype = s["x"].dtype
    out = (values * per_comp).transpose(0, 1).reshape(n, comps * h).to(dtype)
    if not case["train"]:
        return {"out": out}
    g = s["grad"].float().view(n, comps, h).transpose(0, 1)
    d_values = g * per_comp
    d_gate = torch.zeros(ranks, n, h, device="cuda").index_add_(0, of, g * values)
    slope = sig * (1.0 - sig) if case["act"] == "sigmoid" else sig * (1.0 + pre * (1.0 - sig))
    d_pre = d_gate.transpose(0, 1).reshape(n, ranks * h) * (sc[ranks + 1] * slope)
    gx = d_values @ wv[of]
    gx[0] += d_pre @ wg
    gw = torch.zeros(ranks, h, c, device="cuda").index_add_(0, of, d_values.transpose(1, 2) @ x)
    gw = gw * sc[:ranks, None, None]
    grads = [gx.transpose(0, 1).reshape(n, comps * c), *gw.unbind(0), (d_pre.t() @ x[0]) * sc[ranks]]
    if s["gate_bias"] is not None:
        grads.append(d_pre.sum(0))
    return {"out": out, "grads": [t.to(dtype) for t in grads]}


def _threshold(p):
    """A channel of a rank is dropped where its 32 random bits are below this."""
    return int(p * 4294967296.0)


def _plain_dropout(s, case):
    n, c, ranks = case["rows"], case["c"], case["l_max"] + 1
    quads = (c + 3) // 4  # one 4-word block of the generator for four channels of a rank
    block = torch.arange(n * ranks * quads, device="cuda")
    seed, offset = s["rng"][0], s["rng"][1]
    low = 0xFFFFFFFF
    w = [block & low, block >> 32, (offset & low).expand_as(block), ((offset >> 32) & low).expand_as(block)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = w[0] * 0xD2511F53, w[2] * 0xCD9E8D57
        w = [((p1 >> 32) & low) ^ w[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ w[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    bits = torch.stack(w, -1).view(n, ranks, quads * 4)[:, :, :c]
    factor = (bits >= _threshold(case["p"])).float() * (1.0 / (1.0 - case["p"]))
    factor = factor[:, _rank_of_component(case["l_max"])].reshape(n, -1)
    dtype = s["x"].dtype
    return {"out": (s["x"].float() * factor).to(dtype), "grad_x": (s["grad"].float() * factor).to(dtype)}


# ------------------------------------------------------------------------------ work


def work(case):
    b, rows = SIZE[case["dtype"]], case["rows"]
    if case["op"] == "embed":
        moved, table = rows * case["dim"] * b, case["vocab"] * case["dim"] * b
        touched = min(table, moved)  # rows of the table that are looked up
        out = {"bytes": touched + rows * 8 + moved, "flops": 2 * rows * case["dim"]}
        if case["train"]:
            out["bytes"] += moved + table
            out["flops"] += rows * case["dim"]
        return out
    comps = (case["l_max"] + 1) ** 2
    if case["op"] == "dropout":
        n = rows * comps * case["c"]
        return {"bytes": 4 * n * b + 16, "flops": 2 * n}
    c, h, ranks = case["c"], case["h"], case["l_max"] + 1
    weights = 2 * ranks * c * h + (ranks * h if case["bias"] else 0)
    products = 2 * rows * (comps + ranks) * c * h
    out = {"bytes": (rows * comps * (c + h) + weights) * b, "flops": products}
    if case["train"]:  # input, output gradient and weights again, their gradients; three products for each map
        out["bytes"] += (rows * comps * (c + h) + weights) * b
        out["flops"] += 2 * products
    return out


# ------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embed":
            return _exact_embed(s, case)
        if case["op"] == "dropout":
            return _exact_dropout(s, case)
        return _exact_gated(s, case)


def _exact_embed(s, case):
    table = s["table"].detach().cpu().double().numpy()
    index = s["index"].cpu().numpy()
    out = torch.from_numpy(table.take(index, axis=0) * case["scale"] + case["offset"])
    if not case["train"]:
        return {"out": out}
    order = np.argsort(index, kind="stable")
    sums = np.zeros_like(table)
    present, first = np.unique(index[order], return_index=True)
    grad = s["grad"].cpu().double().numpy()
    sums[present] = np.add.reduceat(grad[order], first, axis=0)
    return {"out": out, "grad_table": torch.from_numpy(sums * case["scale"])}


def _exact_gated(s, case):
    n, c, h, ranks = case["rows"], case["c"], case["h"], case["l_max"] + 1
    x, sc = s["x"].detach().double(), s["scales"].double()
    wg = s["gate_weight"].detach().double().view(ranks, h, c)
    wv = [w.detach().double() for w in s["value_weights"]]
    bias = s["gate_bias"]
    bias = torch.zeros(ranks, h, device="cuda", dtype=torch.float64) if bias is None else bias.detach().double()
    bias = bias.view(ranks, h)
    outs, gxs, gws, ggs, gbs = [], [], [], [], []
    x0, g0 = x[:, :c], torch.zeros(n, c, device="cuda", dtype=torch.float64)
    for l in range(ranks):
        m = 2 * l + 1
        xl = x[:, l * l * c:(l + 1) ** 2 * c].view(n, m, c)
        z = sc[ranks] * torch.einsum("nc,hc->nh", x0, wg[l]) + bias[l]
        sg = torch.sigmoid(z)
        gate, slope = (sg, sg * (1 - sg)) if case["act"] == "sigmoid" else (z * sg, sg * (1 + z * (1 - sg)))
        gate, slope = gate * sc[ranks + 1], slope * sc[ranks + 1]
        v = sc[l] * torch.einsum("nmc,hc->nmh", xl, wv[l])
        outs.append((v * gate[:, None]).reshape(n, -1))
        if not case["train"]:
            continue
        g = s["grad"].double()[:, l * l * h:(l + 1) ** 2 * h].view(n, m, h)
        dv = g * gate[:, None] * sc[l]
        dz = (g * v).sum(1) * slope
        gxs.append(torch.einsum("nmh,hc->nmc", dv, wv[l]).reshape(n, -1))
        gws.append(torch.einsum("nmh,nmc->hc", dv, xl))
        ggs.append(torch.einsum("nh,nc->hc", dz, x0) * sc[ranks])
        gbs.append(dz.sum(0))
        g0 += torch.einsum("nh,hc->nc", dz, wg[l]) * sc[ranks]
    out = torch.cat(outs, 1)
    if not case["train"]:
        return {"out": out}
    gx = torch.cat(gxs, 1)
    gx[:, :c] += g0
    grads = [gx, *gws, torch.cat(ggs)]
    if case["bias"]:
        grads.append(torch.cat(gbs))
    return {"out": out, "grads": grads}


def _exact_dropout(s, case):
    """The counter-based generator (Philox 4x32, ten rounds) word by word in unsigned 64-bit integers."""
    n, c, ranks = case["rows"], case["c"], case["l_max"] + 1
    seed, offset = (int(v) & 0xFFFFFFFFFFFFFFFF for v in s["rng"].tolist())
    quads = -(-c // 4)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    a = np.arange(n * ranks * quads, dtype=np.uint64)
    b, a = a >> half, a & low
    d, e = np.full_like(a, offset & 0xFFFFFFFF), np.full_like(a, offset >> 32)
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        left, right = a * np.uint64(0xD2511F53), d * np.uint64(0xCD9E8D57)
        a, b, d, e = (right >> half) ^ b ^ np.uint64(key[0]), right & low, (left >> half) ^ e ^ np.uint64(key[1]), left & low
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack([a, b, d, e], axis=1).reshape(n, ranks, 4 * quads)[:, :, :c]
    kept = words >= np.uint64(_threshold(case["p"]))
    kept = np.repeat(kept, [2 * l + 1 for l in range(ranks)], axis=1).reshape(n, -1)
    kept = torch.from_numpy(kept).double() / (1.0 - case["p"])
    return {"out": s["x"].detach().cpu().double() * kept, "grad_x": s["grad"].cpu().double() * kept}
