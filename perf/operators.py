"""Serving several sequences in 8 bits, as cases that can be timed and compared: keys and values appended to the pages of a cache with the rotation
of their positions on the way, attention over such pages (16-bit numbers, or 8-bit numbers with a factor for each block of tokens and head), and the
product of a layer in 8-bit integers with a factor for each token and each output channel.

A case is a dict of plain values.  Where `own` is false, run() computes the operators with elementary torch operations; where it is true it makes the
calls that a program makes of this framework.  exact() is the same from the definitions, in 64 bits.

Definitions.  A token at position p has its queries and keys turned, column pairs i by the angle p * freq[i]; keys and values are rounded to 32 bits and
then to 16.  Pages of 16 bits hold them as they are.  Pages of 8 bits hold a block of `page` tokens once it is complete: per head the largest magnitude a
of the block's 16-bit numbers, the factor a / 127 and the codes round(x * 127 / a), ties to even; the tokens of a block that is not complete, and of the
one before it, lie in a sequence's two open blocks as 16-bit numbers (block b in half b mod 2).  A product's activations are coded the same way, row by row."""
import math
import random

import numpy as np
import torch

own = False

LLAMA_7B = {"heads": 32, "kv_heads": 32, "dim": 128}
MISTRAL_7B = {"heads": 32, "kv_heads": 8, "dim": 128}
BASE = 10000.0
F = torch.float64


# ---- the cases ------------------------------------------------------------------------------------------------------------------------
def _batch(name, kind, model, bits, page, seqs, pos, new, mix, **more):
    """pos, new: what the sequences have in the cache and bring along, at least and at most"""
    case = dict(model, kind=kind, bits=bits, page=page, seqs=seqs, pos_lo=pos[0], pos_hi=pos[1], new_lo=new[0], new_hi=new[1], mix=mix, **more)
    return dict(case, name=name) if name else case


def listed():
    plain = {"window": 0, "softcap": 0.0}
    return [
        # one token through a square projection of a 7B layer: a call's latency
        {"name": "product token", "kind": "product", "rows": 1, "m": 4096, "k": 4096},
        # the next tokens of several sequences against the up projection of a 7B layer
        {"name": "product 13 rows", "kind": "product", "rows": 13, "m": 11008, "k": 4096},
        # a ragged portion of a prompt through a down projection
        {"name": "product ragged prompt", "kind": "product", "rows": 509, "m": 4096, "k": 14336},
        # a whole prompt through an up projection
        {"name": "product prompt", "kind": "product", "rows": 2048, "m": 14336, "k": 4096},
        # one sequence's next token into 16-bit pages, every head with keys of its own: a call's latency
        _batch("append token", "append", LLAMA_7B, 16, 16, 1, (300, 300), (1, 1), 1),
        # the next tokens of a full batch into 8-bit pages
        _batch("append 64 sequences", "append", MISTRAL_7B, 8, 32, 64, (20, 400), (1, 1), 2),
        # portions of three prompts into 8-bit pages, behind what the cache has
        _batch("append prompts", "append", MISTRAL_7B, 8, 64, 3, (0, 900), (200, 900), 3),
        # one sequence's next token over a long cache
        _batch("attention long", "attention", MISTRAL_7B, 8, 64, 1, (32000, 32000), (1, 1), 4, **plain),
        # the next tokens of a full batch of sequences of all lengths
        _batch("attention 64 sequences", "attention", MISTRAL_7B, 8, 32, 64, (20, 4000), (1, 1), 5, **plain),
        # a batch over 16-bit pages, every head with keys of its own
        _batch("attention 16 bits", "attention", LLAMA_7B, 16, 16, 16, (100, 2000), (1, 1), 6, **plain),
        # drafted tokens checked for several sequences, under a window and with capped scores
        _batch("attention drafts", "attention", {"heads": 16, "kv_heads": 4, "dim": 64}, 8, 64, 8, (500, 6000), (2, 6), 7, window=4096, softcap=30.0),
        # portions of three prompts
        _batch("attention prompts", "attention", MISTRAL_7B, 8, 64, 3, (0, 2000), (300, 1500), 8, **plain),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["product", "append", "attention", "attention"])
    if kind == "product":
        return {"kind": kind, "rows": _log(rng, 1, 2048), "m": _log(rng, 200, 14336), "k": rng.choice([16 * _log(rng, 8, 256), _log(rng, 100, 4096)])}
    G, d, S, prompt = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 256]), _log(rng, 1, 64), rng.random() < 0.4
    H = G * rng.choice([1, 2, 4, 8])
    S = min(S, 3) if prompt else S
    hi = _log(rng, 50, 400 if kind == "append" else 2000 if prompt else 8000 if S < 16 else 4000)
    new = _log(rng, 20, 1200) if prompt else rng.choice([1, 1, 2, 6])
    while kind == "attention" and 4 * S * new * (hi + new) * H * d > 2.0e11:
        new = new * 2 // 3
    return _batch("", kind, {"heads": H, "kv_heads": G, "dim": d}, rng.choice([8, 8, 16]), rng.choice([16, 32, 64, 128]), S, (rng.randint(0, hi), hi),
                  (rng.randint(1, new), new), rng.randint(0, 1 << 20),
                  **({"window": rng.choice([0, 0, _log(rng, 16, 4096)]), "softcap": rng.choice([0.0, 0.0, 30.0])} if kind == "attention" else {}))


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

    def uniform(self, *shape, lo, hi):
        return torch.rand(shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def shuffled(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _product_inputs(c, seed):
    r = Inputs(seed)
    # activations with a few large channels and rows of different size, as they come out of a norm
    x = r.normal(c["rows"], c["k"]) * torch.exp(0.7 * r.normal(c["k"])) * torch.exp(0.5 * r.normal(c["rows"], 1))
    w = r.normal(c["m"], c["k"]).mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    return {"x": x, "w": w, "w_scale": r.uniform(c["m"], lo=0.5, hi=1.5) / (36.0 * math.sqrt(c["k"]))}


def _table(c, r):
    """pages of every sequence in no order, [sequences, pages of the longest], and how many there are"""
    need = [(p + n + c["page"] - 1) // c["page"] for p, n in _lengths(c)]
    order, table, at = r.shuffled(sum(need)).tolist(), np.zeros((c["seqs"], max(need)), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need)


def _blocks(x):
    """16-bit numbers [..., page, dim] as codes and factors [...]"""
    a = x.float().abs().amax((-2, -1))
    codes = torch.round(x.to(F) * 127.0 / a.to(F).clamp_min(1e-300)[..., None, None])
    return codes.to(torch.int8), a / 127.0


def _cache_inputs(c, r, n_pages):
    """the pages and open blocks of a layer whose sequences have their tokens so far"""
    d, G, P = c["dim"], c["kv_heads"], c["page"]
    out = {}
    for name, size in (("k", torch.exp(0.5 * r.normal(d))), ("v", torch.ones(d, device="cuda"))):
        x = (r.normal(n_pages, G, P, d) * size).half()
        if c["bits"] == 16:
            out[name] = x
            continue
        out[name], out[name + "_scale"] = _blocks(x)
        out[name + "_open"] = (r.normal(2 * c["seqs"], G, P, d) * size).half()
    return out


def _append_inputs(c, seed):
    r = Inputs(seed)
    table, n_pages = _table(c, r)
    T = sum(n for _, n in _lengths(c))
    s = {"table": table, "n_pages": n_pages, "qkv": r.normal(T, (c["heads"] + 2 * c["kv_heads"]) * c["dim"])}
    i = torch.arange(c["dim"] // 2, device="cuda", dtype=F)
    s["freq"] = (BASE ** (-2.0 * i / c["dim"])).float()
    s["cache"] = _cache_inputs(c, r, n_pages)
    return s


def _attention_inputs(c, seed):
    r = Inputs(seed)
    table, n_pages = _table(c, r)
    T = sum(n for _, n in _lengths(c))
    return {"table": table, "n_pages": n_pages, "q": r.normal(T, c["heads"] * c["dim"], scale=2.0), "cache": _cache_inputs(c, r, n_pages)}


def _indices(c, table):
    """what a step's program knows about its tokens and blocks, as index tensors: made once a step, for all layers"""
    P, rows = c["page"], []
    seg = {"seq": [], "block": [], "page": [], "first": [], "pos0": [], "end": []}
    t = 0
    for i, (p, n) in enumerate(_lengths(c)):
        rows += [(i, p + j) for j in range(n)]
        for b in range(p // P, (p + n - 1) // P + 1):
            for key, v in (("seq", i), ("block", b), ("page", int(table[i, b])), ("first", t), ("pos0", p), ("end", p + n)):
                seg[key].append(v)
        t += n
    to = lambda v: torch.tensor(v, device="cuda", dtype=torch.int64)  # noqa: E731
    seg = {k: to(v) for k, v in seg.items()}
    seq, pos = to([r[0] for r in rows]), to([r[1] for r in rows])
    row = torch.arange(P, device="cuda")
    p_of = seg["block"][:, None] * P + row                              # position of each row of each touched block
    last = seg["end"] // P
    ix = {"seq": seq, "pos": pos, "row_page": to(table.astype(np.int64))[seq, pos // P], "row_off": pos % P, "block": seg["block"], "page": seg["page"],
          "new": (p_of >= seg["pos0"][:, None]) & (p_of < seg["end"][:, None]), "token": (seg["first"][:, None] + p_of - seg["pos0"][:, None]).clamp(0, t - 1),
          "held": p_of < seg["end"][:, None], "half": 2 * seg["seq"] + seg["block"] % 2}
    full = (seg["block"] + 1) * P <= seg["end"]
    ix["full"] = torch.nonzero(full).flatten()
    ix["kept"] = torch.nonzero((seg["block"] >= last - 1)).flatten()
    # queries of every sequence side by side, padded to the longest, and the blocks a sequence has
    lens = to([p + n for p, n in _lengths(c)])
    most = max(n for _, n in _lengths(c))
    first = to(np.cumsum([0] + [n for _, n in _lengths(c)])[:-1].tolist())
    count = to([n for _, n in _lengths(c)])
    j = torch.arange(most, device="cuda")
    ix["pad_token"] = (first[:, None] + j).clamp(0, t - 1)
    ix["pad_pos"] = lens[:, None] - count[:, None] + j.clamp(max=most)  # positions of padded rows run past the end: their results are dropped
    ix["flat"] = seq * most + (pos - (lens - count)[seq])
    blocks = torch.arange(table.shape[1], device="cuda")
    ix["table"] = to(table.astype(np.int64))
    ix["open"] = (blocks[None] == (lens // P)[:, None])
    ix["open_half"] = 2 * torch.arange(c["seqs"], device="cuda") + (lens // P) % 2
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


def _prepare_own(s):
    """device tensors with the inputs, the plan of the step and the layer's cache"""
    from crabml_b200 import CudaTensor, CudaTensorDevice, capi, paged
    if not _device:
        _device.append(CudaTensorDevice(0))
    dev, c = _device[0], s["case"]
    types = {torch.float32: capi.F32, torch.float16: capi.F16, torch.int8: capi.I8}

    def give(t):
        ct = CudaTensor.alloc(list(t.shape), types[t.dtype], dev)
        dev.synchronize()
        torch.as_tensor(ct, device="cuda").copy_(t)
        return ct
    if c["kind"] == "product":
        s["h"] = {n: give(s[n]) for n in ("x", "w", "w_scale")}
        return
    s["h"] = {n: give(s[n]) for n in ("qkv", "freq", "q") if n in s}
    h = s["h"]
    h["plan"] = paged.PagePlan(dev, page_size=c["page"], n_pages=s["n_pages"], table=s["table"], pos0=[p for p, _ in _lengths(c)], counts=[n for _, n in _lengths(c)],
                               n_slots=c["seqs"])
    h["cache"] = paged.PagedCache(**{n: give(t) for n, t in s["cache"].items()})
    h["stream"] = torch.cuda.ExternalStream(dev.stream())
    # what the program sees of its cache: the same memory
    s["cache"] = {n: torch.as_tensor(getattr(h["cache"], n), device="cuda") for n in s["cache"]}


def _run_own(s):
    from crabml_b200 import paged, seqops
    c, h = s["case"], s["h"]
    if c["kind"] == "product":
        return torch.as_tensor(seqops.product_i8(h["w"], h["w_scale"], h["x"]), device="cuda")
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "attention":
        y = paged.attention(h["plan"], h["cache"], h["q"], H, d ** -0.5, window=c["window"], softcap=c["softcap"])
        return torch.as_tensor(y, device="cuda")
    qkv = h["qkv"]
    q = paged.append(h["plan"], h["cache"], qkv, 0, qkv, H * d, qkv, (H + G) * d, H, freq=h["freq"])
    with torch.cuda.stream(h["stream"]):
        return dict(_values(s["cache"]), q=torch.as_tensor(q, device="cuda"))


# ---- their plain form ---------------------------------------------------------------------------------------------------------------------
def _values(cache):
    """a cache as the numbers it stands for"""
    if "k_scale" not in cache:
        return {"k": cache["k"], "v": cache["v"]}
    return {"k": cache["k"] * cache["k_scale"][:, :, None, None], "v": cache["v"] * cache["v_scale"][:, :, None, None], "k_open": cache["k_open"], "v_open": cache["v_open"]}


def _turn(x, cos, sin):
    """x [T, heads, dim] in 64 bits, neighbouring columns turned"""
    x = x.to(F)
    u, v = x[..., 0::2], x[..., 1::2]
    return torch.stack([u * cos - v * sin, v * cos + u * sin], -1).reshape(x.shape).float()


def _plain_append(s):
    c, ix, cache = s["case"], s["ix"], s["cache"]
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = s["qkv"][:, :H * d], s["qkv"][:, H * d:(H + G) * d], s["qkv"][:, (H + G) * d:]
    angle = ix["pos"].to(F)[:, None, None] * s["freq"].to(F)
    cos, sin = angle.cos(), angle.sin()
    q = _turn(q.reshape(-1, H, d), cos, sin).reshape(-1, H * d)
    _plain_store(c, ix, cache, "k", _turn(k.reshape(-1, G, d), cos, sin).half())
    _plain_store(c, ix, cache, "v", v.reshape(-1, G, d).half())
    return dict(_values(cache), q=q)


def _plain_store(c, ix, cache, name, x):
    """rows x [T, heads, dim] into the pages"""
    if c["bits"] == 16:
        cache[name][ix["row_page"], :, ix["row_off"]] = x
        return
    opened = cache[name + "_open"]
    was = opened[ix["half"]]                                             # [touched blocks, heads, page, dim]
    block = torch.where(ix["new"][:, None, :, None], x[ix["token"]].transpose(1, 2), was)
    codes, factors = _blocks(block[ix["full"]])
    cache[name][ix["page"][ix["full"]]] = codes
    cache[name + "_scale"][ix["page"][ix["full"]]] = factors
    opened[ix["half"][ix["kept"]]] = torch.where(ix["held"][ix["kept"]][:, None, :, None], block[ix["kept"]], was[ix["kept"]])


def _plain_rows(c, ix, cache, name):
    """the keys or values of every sequence, [sequences, heads, positions, dim]"""
    x = cache[name][ix["table"]]                                         # [sequences, blocks, heads, page, dim]
    if c["bits"] == 8:
        x = x * cache[name + "_scale"][ix["table"]][..., None, None]
        x = torch.where(ix["open"][:, :, None, None, None], cache[name + "_open"][ix["open_half"]][:, None].float(), x)
    return x.float().transpose(1, 2).reshape(c["seqs"], c["kv_heads"], -1, c["dim"])


def _plain_attention(s):
    c, ix = s["case"], s["ix"]
    H, G, d, S = c["heads"], c["kv_heads"], c["dim"], c["seqs"]
    k, v = (_plain_rows(c, ix, s["cache"], n) for n in ("k", "v"))
    q = s["q"].reshape(-1, G, H // G, d)[ix["pad_token"]].permute(0, 2, 3, 1, 4).reshape(S, G, -1, d)      # [sequences, heads, group x tokens, dim]
    x = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    back = ix["pad_pos"][:, :, None] - torch.arange(k.shape[2], device="cuda")                          # [sequences, tokens, positions]
    seen = back >= 0
    if c["window"]:
        seen &= back < c["window"]
    x = x.reshape(S, G, H // G, -1, k.shape[2]).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    x = (x / x.sum(-1, keepdim=True)).reshape(S, G, -1, k.shape[2])
    y = torch.matmul(x, v).reshape(S, G, H // G, -1, d).permute(0, 3, 1, 2, 4).reshape(-1, H * d)
    return y[ix["flat"]]


def _plain_product(s):
    x = s["x"]
    a = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x.to(F) * 127.0 / a.to(F).clamp_min(1e-300)).float()      # numbers next to a border: in 64 bits
    return torch.matmul(codes, s["w"].float().T) * (a / 127.0) * s["w_scale"]


def run(s):
    if own:
        return _run_own(s)
    return {"product": _plain_product, "append": _plain_append, "attention": _plain_attention}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "product":
        n, m, k = c["rows"], c["m"], c["k"]
        return {"bytes": m * k + 4 * (m + n * (k + m)), "flops": 2 * n * m * k}
    H, G, d, P, wide = c["heads"], c["kv_heads"], c["dim"], c["page"], c["bits"] // 8
    T = sum(n for _, n in _lengths(c))
    if c["kind"] == "append":
        # rows in, queries out, rows into their pages; 8 bits: the rows of blocks that are not complete as 16-bit numbers, and the pages as the numbers they stand for
        pages = sum((p + n + P - 1) // P for p, n in _lengths(c))
        stay = sum(min(n, (p + n) % P) for p, n in _lengths(c))
        there = 2 * G * d * (2 * T if wide == 2 else T + 2 * stay + pages * P * 5)
        return {"bytes": 4 * T * (2 * H + 2 * G) * d + there, "flops": 6 * T * (H + G) * d}
    w = c["window"]
    pairs = sum(min(i + 1, w) if w else i + 1 for p, n in _lengths(c) for i in range(p, p + n))
    rows = sum(p + n - (max(0, p + 1 - w) if w else 0) for p, n in _lengths(c))
    return {"bytes": 2 * rows * G * d * wide + 4 * 2 * T * H * d, "flops": 4 * pairs * H * d}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------------------------
def _coded(x):
    """16-bit numbers of one block and head as (the numbers their codes stand for)"""
    a = x.to(F).abs().max()
    return torch.round(x.to(F) * 127.0 / a) * (a / 127.0) if a > 0 else torch.zeros_like(x, dtype=F)


def _exact_product(c, seed):
    t = _product_inputs(c, seed)
    x = t["x"].to(F)
    a = x.abs().amax(1, keepdim=True)
    return (torch.round(x * 127.0 / a) @ t["w"].to(F).T) * (a / 127.0) * t["w_scale"].to(F)


def _turned_exactly(x, pos, freq):
    out = torch.empty_like(x, dtype=F)
    a = pos.to(F)[:, None] * freq.to(F)
    for i in range(x.shape[1]):
        re, im = x[:, i, 0::2].to(F), x[:, i, 1::2].to(F)
        out[:, i, 0::2] = re * torch.cos(a) - im * torch.sin(a)
        out[:, i, 1::2] = im * torch.cos(a) + re * torch.sin(a)
    return out


def _exact_append(c, seed):
    t = _append_inputs(c, seed)
    H, G, d, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    cache = t["cache"]
    out = {}
    for name in ("k", "v"):
        out[name] = cache[name].to(F) if c["bits"] == 16 else cache[name].to(F) * cache[name + "_scale"].to(F)[:, :, None, None]
        if c["bits"] == 8:
            out[name + "_open"] = cache[name + "_open"].clone()
    x = t["qkv"].reshape(-1, H + 2 * G, d)
    q, at = [], 0
    for i, (p, n) in enumerate(_lengths(c)):
        rows = x[at:at + n]
        turned = _turned_exactly(rows[:, :H + G], torch.arange(p, p + n, device="cuda"), t["freq"])
        q.append(turned[:, :H].reshape(n, H * d))
        both = {"k": turned[:, H:].float().half(), "v": rows[:, H + G:].half()}
        for name, new in both.items():
            if c["bits"] == 16:
                for b in range(p // P, (p + n - 1) // P + 1):
                    lo, hi = max(p, b * P), min(p + n, (b + 1) * P)
                    out[name][int(t["table"][i, b]), :, lo - b * P:hi - b * P] = new[lo - p:hi - p].transpose(0, 1).to(F)
                continue
            started = cache[name + "_open"]                             # the call's rows may replace what its first block began with
            for b in range(p // P, (p + n - 1) // P + 1):
                lo, hi = max(p, b * P), min(p + n, (b + 1) * P)
                block = started[2 * i + b % 2].clone()
                block[:, lo - b * P:hi - b * P] = new[lo - p:hi - p].transpose(0, 1)
                if hi == (b + 1) * P:
                    out[name][int(t["table"][i, b])] = torch.stack([_coded(block[g]) for g in range(G)])
                if b >= (p + n) // P - 1:
                    out[name + "_open"][2 * i + b % 2, :, :hi - b * P] = block[:, :hi - b * P]
        at += n
    out["q"] = torch.cat(q)
    return out


def _exact_attention(c, seed):
    t = _attention_inputs(c, seed)
    H, G, d, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    cache, q = t["cache"], t["q"].to(F).reshape(-1, H, d)
    out, at = torch.empty_like(q), 0
    for i, (p, n) in enumerate(_lengths(c)):
        L = p + n
        rows = {}
        for name in ("k", "v"):
            pages = torch.tensor(t["table"][i, :(L + P - 1) // P].astype(np.int64), device="cuda")
            x = cache[name][pages].to(F)
            if c["bits"] == 8:
                x = x * cache[name + "_scale"][pages].to(F)[:, :, None, None]
                if L % P:
                    x[L // P] = cache[name + "_open"][2 * i + (L // P) % 2].to(F)
            rows[name] = x.transpose(0, 1).reshape(G, -1, d)[:, :L]
        mine, keys = torch.arange(p, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        hidden = keys > mine
        if c["window"]:
            hidden = hidden | (keys <= mine - c["window"])
        for h in range(H):
            z = q[at:at + n, h] @ rows["k"][h // (H // G)].T / math.sqrt(d)
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            z = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h] = z @ rows["v"][h // (H // G)]
        at += n
    return out.reshape(-1, H * d)


def exact(case, seed):
    return {"product": _exact_product, "append": _exact_append, "attention": _exact_attention}[case["kind"]](case, seed)
