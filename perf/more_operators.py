"""One attention sublayer of a latent-attention model for several sequences in a call, as cases that can be timed and compared: the rows of the latent cache
written to pages with their norm and rotation, the attention that reads them, and the products in front and behind with bias, activation and residual in
one call.

A case is a dict of plain values.  Where `own` is false, run() computes the operators with elementary torch operations; where it is true it makes the
calls that a program makes of this framework.  exact() is the same from the definitions, in 64 bits.

Definitions.  A cached row is [c | r]: c the first `rank` columns of what the projection gave, divided by their root mean square and multiplied by a weight;
r the next `rest` columns, pairs of neighbours turned by position x frequency; both rounded to 16 bits once.  A query head is [n | p], `dim` columns as they
come and `rest` turned ones, rounded to 16 bits.  Keys and values of a head are k = [U c | r] and v = V c; a token sees the positions of its sequence up to its
own, `window` of them where that is not 0; a sink adds exp(sink) to the sum of the weights.  A product is act(W x + bias) + residual, x rounded to the type of W."""
import math
import random

import numpy as np
import torch

own = False

LATENT = {"heads": 16, "dim": 128, "rest": 64, "vdim": 128, "rank": 512}
BASE, EPS = 10000.0, 1e-5
F = torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ------------------------------------------------------------------------------------------------------------------------
def _batch(name, kind, model, page, seqs, pos, new, mix, **more):
    """pos, new: what the sequences have in the cache and bring along, at least and at most"""
    case = dict(model, kind=kind, page=page, seqs=seqs, pos_lo=pos[0], pos_hi=pos[1], new_lo=new[0], new_hi=new[1], mix=mix, **more)
    return dict(case, name=name) if name else case


def _product(name, rows, m, k, w, x, out, bias, act, residual):
    case = {"kind": "product", "rows": rows, "m": m, "k": k, "w": w, "x": x, "out": out, "bias": bias, "act": act, "residual": residual}
    return dict(case, name=name) if name else case


def listed():
    plain = {"window": 0, "sink": False}
    return [
        # one token's heads back into the 32-bit residual stream of a 4096 wide layer: a call's latency
        _product("product token", 1, 4096, 4096, "bf16", "bf16", "f32", False, "none", True),
        # the next tokens of several sequences through an up projection of a 7B layer
        _product("product 13 rows", 13, 11008, 4096, "bf16", "bf16", "bf16", True, "silu", False),
        # a ragged portion of a prompt through a down projection into the residual stream
        _product("product ragged prompt", 509, 4096, 14336, "f16", "f16", "f32", True, "none", True),
        # a whole prompt through an up projection
        _product("product prompt", 2048, 14336, 4096, "bf16", "bf16", "bf16", True, "gelu", False),
        # one sequence's next token: a call's latency
        _batch("append token", "append", LATENT, 16, 1, (300, 300), (1, 1), 1, src="f32"),
        # the next tokens of a full batch
        _batch("append 64 sequences", "append", LATENT, 32, 64, (20, 4000), (1, 1), 2, src="f32"),
        # portions of three prompts, behind what the cache has
        _batch("append prompts", "append", LATENT, 64, 3, (0, 900), (200, 900), 3, src="bf16"),
        # one sequence's next token over a long cache
        _batch("attention long", "attention", LATENT, 64, 1, (32000, 32000), (1, 1), 4, **plain),
        # the next tokens of a full batch of sequences of all lengths
        _batch("attention 64 sequences", "attention", LATENT, 32, 64, (20, 4000), (1, 1), 5, **plain),
        # drafted tokens checked for several sequences, under a window and with a sink
        _batch("attention drafts", "attention", {"heads": 8, "dim": 64, "rest": 32, "vdim": 64, "rank": 256}, 64, 8, (500, 6000), (2, 6), 6, window=4096, sink=True),
        # portions of three prompts behind what the cache has
        _batch("attention prompts", "attention", LATENT, 64, 3, (0, 2000), (300, 1500), 7, **plain),
        # a whole prompt
        _batch("attention prompt", "attention", LATENT, 64, 1, (0, 0), (4000, 4000), 8, **plain),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["product", "append", "attention", "attention"])
    if kind == "product":
        w = rng.choice(["bf16", "bf16", "f16"])
        return _product("", _log(rng, 1, 2048), _log(rng, 200, 14336), rng.choice([16 * _log(rng, 8, 256), _log(rng, 100, 4096)]), w, rng.choice([w, "f32"]),
                        rng.choice([w, "f32"]), rng.random() < 0.5, rng.choice(["none", "none", "silu", "gelu", "relu2"]), rng.random() < 0.5)
    dim, rest, vdim, rank = rng.choice([(128, 64, 128, 512), (128, 64, 128, 512), (64, 32, 64, 256), (32, 16, 32, 64), (48, 16, 80, 160), (96, 32, 64, 384)])
    H, S, prompt = rng.choice([1, 3, 4, 8, 8, 12, 16, 24, 32]), _log(rng, 1, 64), rng.random() < 0.4
    S = min(S, 3) if prompt else S
    hi = _log(rng, 50, 4000 if kind == "append" else 2000 if prompt else 8000 if S < 16 else 4000)
    new = _log(rng, 20, 1200) if prompt else rng.choice([1, 1, 2, 6])
    while kind == "attention" and 4 * S * new * (hi + new) * H * (rank + rest) > 4.0e11:
        new = max(1, new * 2 // 3)
    return _batch("", kind, {"heads": H, "dim": dim, "rest": rest, "vdim": vdim, "rank": rank}, rng.choice([16, 32, 64, 128]), S, (rng.randint(0, hi), hi),
                  (rng.randint(1, new), new), rng.randint(0, 1 << 20),
                  **({"window": rng.choice([0, 0, _log(rng, 16, 4096)]), "sink": rng.random() < 0.3} if kind == "attention" else {"src": rng.choice(["f32", "bf16", "f16"])}))


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """(tokens in the cache, new tokens) of every sequence"""
    r = random.Random(c["mix"])
    return [(r.randint(c["pos_lo"], c["pos_hi"]), r.randint(c["new_lo"], c["new_hi"])) for _ in range(c["seqs"])]


class Inputs:
    """torch values made on the GPU from the seed alone, in a fixed order"""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, scale=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * scale

    def shuffled(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _product_inputs(c, seed):
    r = Inputs(seed)
    # activations with a few large channels and rows of different size
    x = r.normal(c["rows"], c["k"]) * torch.exp(0.7 * r.normal(c["k"])) * torch.exp(0.5 * r.normal(c["rows"], 1))
    t = {"x": x.to(TYPES[c["x"]]), "w": r.normal(c["m"], c["k"], scale=c["k"] ** -0.5).to(TYPES[c["w"]])}
    if c["bias"]:
        t["bias"] = r.normal(c["m"], scale=0.5)
    if c["residual"]:
        t["residual"] = r.normal(c["rows"], c["m"]).to(TYPES[c["out"]])
    return t


def _table(c, r):
    """pages of every sequence in no order, [sequences, pages of the longest], and how many there are"""
    need = [(p + n + c["page"] - 1) // c["page"] for p, n in _lengths(c)]
    order, table, at = r.shuffled(sum(need)).tolist(), np.zeros((c["seqs"], max(need)), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need)


def _pages(c, r, n_pages):
    """a layer whose sequences have their tokens so far: normed latents with channels of different size, and rotated columns"""
    rows = r.normal(n_pages, c["page"], c["rank"] + c["rest"])
    rows[..., :c["rank"]] *= torch.exp(0.3 * r.normal(c["rank"]))
    return rows.half()


def _append_inputs(c, seed):
    r = Inputs(seed)
    table, n_pages = _table(c, r)
    T = sum(n for _, n in _lengths(c))
    s = {"table": table, "n_pages": n_pages}
    # one stacked projection's result: the query heads, then the row of the cache
    s["src"] = (r.normal(T, c["heads"] * (c["dim"] + c["rest"]) + c["rank"] + c["rest"]) * torch.exp(0.5 * r.normal(T, 1))).to(TYPES[c["src"]])
    s["norm"] = 1.0 + 0.2 * r.normal(c["rank"])
    i = torch.arange(c["rest"] // 2, device="cuda", dtype=F)
    s["freq"] = (BASE ** (-2.0 * i / c["rest"])).float()
    s["pages"] = _pages(c, r, n_pages)
    return s


def _attention_inputs(c, seed):
    r = Inputs(seed)
    table, n_pages = _table(c, r)
    T, H = sum(n for _, n in _lengths(c)), c["heads"]
    s = {"table": table, "n_pages": n_pages, "pages": _pages(c, r, n_pages), "q": r.normal(T, H * (c["dim"] + c["rest"]), scale=1.5).half()}
    s["uk"], s["uv"] = (r.normal(H * d, c["rank"], scale=c["rank"] ** -0.5).half() for d in (c["dim"], c["vdim"]))
    if c["sink"]:
        s["sinks"] = r.normal(H)
    return s


def _indices(c, table):
    """what a step's program knows about its tokens, as index tensors: made once a step, for all layers"""
    P, lengths = c["page"], _lengths(c)
    to = lambda v: torch.tensor(v, device="cuda", dtype=torch.int64)  # noqa: E731
    rows = [(i, p + j) for i, (p, n) in enumerate(lengths) for j in range(n)]
    seq, pos = to([r[0] for r in rows]), to([r[1] for r in rows])
    ix = {"pos": pos, "table": to(table.astype(np.int64))}
    ix["row_page"], ix["row_off"] = ix["table"][seq, pos // P], pos % P
    # queries of every sequence side by side, padded to the longest
    lens, count = to([p + n for p, n in lengths]), to([n for _, n in lengths])
    first, most = to(np.cumsum([0] + [n for _, n in lengths])[:-1].tolist()), max(n for _, n in lengths)
    j = torch.arange(most, device="cuda")
    ix["pad_token"] = (first[:, None] + j).clamp(0, len(rows) - 1)
    ix["pad_pos"] = lens[:, None] - count[:, None] + j                  # positions of padded rows run past the end: their results are dropped
    ix["flat"] = seq * most + (pos - (lens - count)[seq])
    return ix


def prepare(case, seed):
    c = case
    s = {"case": c}
    s.update({"product": _product_inputs, "append": _append_inputs, "attention": _attention_inputs}[c["kind"]](c, seed))
    if c["kind"] != "product":
        s["ix"] = _indices(c, s["table"])
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------------------------------
_device = []


def _torch(t):
    """a tensor of the framework as one of torch, on the same memory"""
    from crabml_b200 import capi
    return torch.as_tensor(t.bits(), device="cuda").view(torch.bfloat16) if t.dtype() == capi.BF16 else torch.as_tensor(t, device="cuda")


def _prepare_own(s):
    """device tensors with the inputs, and the plan of the step"""
    from crabml_b200 import CudaTensor, CudaTensorDevice, capi, paged
    if not _device:
        _device.append(CudaTensorDevice(0))
    dev, c = _device[0], s["case"]
    types = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}

    def give(t):
        ct = CudaTensor.alloc(list(t.shape), types[t.dtype], dev)
        dev.synchronize()
        _torch(ct).copy_(t)
        return ct
    s["h"] = {n: give(t) for n, t in s.items() if torch.is_tensor(t)}
    if c["kind"] != "product":
        s["h"]["plan"] = paged.PagePlan(dev, page_size=c["page"], n_pages=s["n_pages"], table=s["table"], pos0=[p for p, _ in _lengths(c)], counts=[n for _, n in _lengths(c)])
        s["pages"] = _torch(s["h"]["pages"])                            # what the program sees of its cache: the same memory


def _run_own(s):
    from crabml_b200 import capi, paged, seqops
    c, h = s["case"], s["h"]
    if c["kind"] == "product":
        act = {"none": capi.ACT_NONE, "silu": capi.ACT_SILU, "gelu": capi.ACT_GELU_TANH, "relu2": capi.ACT_RELU_SQUARED}[c["act"]]
        out = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[c["out"]]
        return _torch(seqops.product(h["w"], h["x"], bias=h.get("bias"), act=act, residual=h.get("residual"), out_type=out))
    if c["kind"] == "attention":
        return _torch(paged.latent_attention(h["plan"], h["pages"], c["rank"], h["q"], c["heads"], h["uk"], h["uv"], (c["dim"] + c["rest"]) ** -0.5, window=c["window"],
                                             sink=h.get("sinks"), out_type=capi.BF16))
    q = paged.latent_append(h["plan"], h["pages"], c["rank"], h["src"], c["heads"] * (c["dim"] + c["rest"]), norm_w=h["norm"], eps=EPS, q_src=h["src"], q_col0=0,
                            n_heads=c["heads"], dim=c["dim"], freq=h["freq"])
    return {"q": _torch(q), "pages": s["pages"]}


# ---- their plain form ---------------------------------------------------------------------------------------------------------------------
def _turn(x, pos, freq):
    """x [T, ..., columns], neighbouring columns turned by their token's position: angles in 64 bits"""
    angle = pos.to(F)[:, None] * freq.to(F)
    angle = angle.reshape(angle.shape[0], *[1] * (x.ndim - 2), angle.shape[1])
    x = x.to(F)
    u, v = x[..., 0::2], x[..., 1::2]
    return torch.stack([u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()], -1).reshape(x.shape).float()


def _plain_append(s):
    c, ix, T = s["case"], s["ix"], s["src"].shape[0]
    H, dim, rank = c["heads"], c["dim"], c["rank"]
    src = s["src"].float()
    q, kv = src[:, :H * (dim + c["rest"])].reshape(T, H, -1), src[:, H * (dim + c["rest"]):]
    q = torch.cat([q[..., :dim], _turn(q[..., dim:], ix["pos"], s["freq"])], -1).reshape(T, -1).half()
    lat = kv[:, :rank]
    lat = lat / torch.sqrt(lat.square().mean(-1, keepdim=True) + EPS) * s["norm"]
    s["pages"][ix["row_page"], ix["row_off"]] = torch.cat([lat, _turn(kv[:, rank:], ix["pos"], s["freq"])], -1).half()
    return {"q": q, "pages": s["pages"]}


def _plain_attention(s):
    c, ix = s["case"], s["ix"]
    H, S, rank, dim, vdim = c["heads"], c["seqs"], c["rank"], c["dim"], c["vdim"]
    rows = s["pages"][ix["table"]].float().reshape(S, -1, rank + c["rest"])                                # [sequences, positions, columns]
    q = s["q"].float().reshape(-1, H, dim + c["rest"])[ix["pad_token"]].transpose(1, 2)                   # [sequences, heads, tokens, columns]
    q = torch.cat([torch.matmul(q[..., :dim], s["uk"].float().reshape(H, dim, rank)), q[..., dim:]], -1)   # against the cached rows themselves
    x = torch.matmul(q.reshape(S, -1, rank + c["rest"]), rows.transpose(1, 2)) * (dim + c["rest"]) ** -0.5
    back = ix["pad_pos"][:, :, None] - torch.arange(rows.shape[1], device="cuda")                       # [sequences, tokens, positions]
    seen = back >= 0
    if c["window"]:
        seen &= back < c["window"]
    x = x.reshape(S, H, -1, rows.shape[1]).masked_fill_(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-1e30)
    sink = s["sinks"][:, None, None] if c["sink"] else None
    top = top if sink is None else torch.maximum(top, sink)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - top)
    y = torch.matmul((x / total).reshape(S, -1, rows.shape[1]), rows[..., :rank]).reshape(S, H, -1, rank)
    y = torch.matmul(y, s["uv"].float().reshape(H, vdim, rank).transpose(1, 2)).transpose(1, 2).reshape(-1, H * vdim)
    return y[ix["flat"]].bfloat16()


def _activated(y, act):
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return torch.clamp_min(y, 0.0) ** 2 if act == "relu2" else y


def _plain_product(s):
    c = s["case"]
    y = torch.matmul(s["x"].to(TYPES[c["w"]]).float(), s["w"].float().T)
    if c["bias"]:
        y = y + s["bias"]
    y = _activated(y, c["act"])
    return (y + s["residual"].float() if c["residual"] else y).to(TYPES[c["out"]])


def run(s):
    if own:
        return _run_own(s)
    return {"product": _plain_product, "append": _plain_append, "attention": _plain_attention}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "product":
        n, m, k = c["rows"], c["m"], c["k"]
        return {"bytes": 2 * m * k + size[c["x"]] * n * k + 4 * m * c["bias"] + size[c["out"]] * n * m * (1 + c["residual"]), "flops": 2 * n * m * k}
    H, dim, rest, vdim, rank = c["heads"], c["dim"], c["rest"], c["vdim"], c["rank"]
    T, cols = sum(n for _, n in _lengths(c)), rank + rest
    if c["kind"] == "append":
        return {"bytes": T * (cols + H * (dim + rest)) * (size[c["src"]] + 2), "flops": T * (4 * rank + 3 * rest * (H + 1))}
    w, flops, seen = c["window"], 0, 0
    for p, n in _lengths(c):
        pairs = sum(min(i + 1, w) if w else i + 1 for i in range(p, p + n))
        rows = p + n - (max(0, p + 1 - w) if w else 0)
        # the cheaper of the two orders: queries and results carried over to the latents, or keys and values made of them
        flops += 2 * H * min(pairs * (2 * rank + rest) + n * rank * (dim + vdim), pairs * (dim + rest + vdim) + rows * rank * (dim + vdim))
        seen += rows
    return {"bytes": 2 * (seen * cols + T * H * (dim + rest + vdim) + H * (dim + vdim) * rank), "flops": flops}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------------------------
def _exact_product(c, seed):
    t = _product_inputs(c, seed)
    y = t["x"].to(TYPES[c["w"]]).to(F) @ t["w"].to(F).T
    if "bias" in t:
        y += t["bias"].to(F)
    if c["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif c["act"] == "gelu":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))      # (1 + tanh z) / 2 = sigmoid(2 z)
    elif c["act"] == "relu2":
        y = torch.where(y > 0, y * y, torch.zeros_like(y))
    return y + t["residual"].to(F) if "residual" in t else y


def _turned_exactly(x, pos, freq):
    a, out = pos.to(F)[:, None] * freq.to(F), x.to(F).clone()
    z = torch.polar(torch.ones_like(a), a) * torch.complex(x[:, 0::2].to(F), x[:, 1::2].to(F))
    out[:, 0::2], out[:, 1::2] = z.real, z.imag
    return out


def _exact_append(c, seed):
    t = _append_inputs(c, seed)
    H, dim, rest, rank, P = c["heads"], c["dim"], c["rest"], c["rank"], c["page"]
    pages, q = t["pages"].to(F), t["src"][:, :H * (dim + rest)].to(F)
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in _lengths(c)])
    for h in range(H):
        at = h * (dim + rest) + dim
        q[:, at:at + rest] = _turned_exactly(q[:, at:at + rest], pos, t["freq"])
    rows = t["src"][:, H * (dim + rest):].to(F)
    size = torch.sqrt((rows[:, :rank] ** 2).sum(1, keepdim=True) / rank + EPS)
    rows = torch.cat([rows[:, :rank] / size * t["norm"].to(F), _turned_exactly(rows[:, rank:], pos, t["freq"])], 1)
    at = 0
    for i, (p, n) in enumerate(_lengths(c)):
        for b in range(p // P, (p + n - 1) // P + 1):
            lo, hi = max(p, b * P), min(p + n, (b + 1) * P)
            pages[int(t["table"][i, b]), lo - b * P:hi - b * P] = rows[at + lo - p:at + hi - p]
        at += n
    return {"q": q, "pages": pages}


def _exact_attention(c, seed):
    t = _attention_inputs(c, seed)
    H, dim, rest, vdim, rank = c["heads"], c["dim"], c["rest"], c["vdim"], c["rank"]
    q, uk, uv = t["q"].to(F).reshape(-1, H, dim + rest), t["uk"].to(F).reshape(H, dim, rank), t["uv"].to(F).reshape(H, vdim, rank)
    out, at = torch.empty(q.shape[0], H, vdim, device="cuda", dtype=F), 0
    for i, (p, n) in enumerate(_lengths(c)):
        L = p + n
        pages = torch.tensor(t["table"][i, :(L + c["page"] - 1) // c["page"]].astype(np.int64), device="cuda")
        rows = t["pages"][pages].to(F).reshape(-1, rank + rest)[:L]
        mine, keys = torch.arange(p, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        hidden = keys > mine
        if c["window"]:
            hidden = hidden | (keys <= mine - c["window"])
        for h in range(H):
            k, v = torch.cat([rows[:, :rank] @ uk[h].T, rows[:, rank:]], 1), rows[:, :rank] @ uv[h].T
            z = (q[at:at + n, h] @ k.T / math.sqrt(dim + rest)).masked_fill(hidden, -math.inf)
            if c["sink"]:
                z = torch.cat([z, t["sinks"][h].to(F).expand(n, 1)], 1)
            z = torch.softmax(z, 1)
            out[at:at + n, h] = z[:, :L] @ v
        at += n
    return out.reshape(-1, H * vdim)


def exact(case, seed):
    return {"product": _exact_product, "append": _exact_append, "attention": _exact_attention}[case["kind"]](case, seed)
