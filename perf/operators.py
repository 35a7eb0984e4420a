"""Performance cases of the serving operators: one decoding step of many conversations over a paged cache.

Operators and ranges (`draw` spreads over them):
  append    rows of Q|K|V projections rotated, K and V written into a paged cache: 1 .. 4096 rows (one new token of
            many sequences, or the consecutive tokens of one prompt), heads of 64 and 128, pages of 16 .. 128 positions
  attend    attention of one new token per sequence over the paged cache: 1 .. 64 sequences, 1 .. 131072 cached
            positions, even and ragged, 1 .. 8 query heads per KV head
  linear    a projection of 1 .. 16 rows with 4-bit weights, one scale per 32, 64 or 128 of them
  logprobs  log probability of a given token, entropy and the most probable alternatives of each row of logits:
            1 .. 1024 rows of 1000 .. 200000 ids, 0 .. 32 alternatives

Heads, widths and vocabulary of the small cases are the TinyLlama-1.1B shape of bench.py (32 query / 4 KV heads of 64,
hidden 2048, FFN 5632, vocabulary 32000, up to 2048 positions); the others are generic.

Types: activations float32 (the framework's), bfloat16 or float16; the cache INT8 with one scale per KV head (the
framework's), bfloat16 or float16.  INT8 cache rows are defined by float32 steps, each rounded (rotation, division by
the scale, round to nearest even), as the framework's dense cache defines them, so they have no value in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}
THETA = 10000.0


def listed():
    return [
        # one conversation, one new token of the repository's shape into its INT8 cache
        {"name": "append_1_i8", "op": "append", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64, "page": 16,
         "seqs": 1, "rows": 1, "ctx": 500},
        # a decoding step of a ragged batch
        {"name": "append_61_bf16", "op": "append", "act": "bf16", "cache": "bf16", "heads": 32, "kv": 8, "hd": 128,
         "page": 16, "seqs": 61, "rows": 61, "ctx": 300},
        # a long prompt's rows
        {"name": "append_2048_f16", "op": "append", "act": "f16", "cache": "f16", "heads": 32, "kv": 8, "hd": 128,
         "page": 64, "seqs": 1, "rows": 2048, "ctx": 2048},
        # one conversation near the end of the repository's context: latency
        {"name": "attend_1x2047_i8", "op": "attend", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64,
         "page": 16, "seqs": 1, "ctx": 2047, "ragged": False},
        # the benchmark's batch, 32 sequences near the end of the context
        {"name": "attend_32x1984_i8", "op": "attend", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64,
         "page": 64, "seqs": 32, "ctx": 1984, "ragged": False},
        # a batch of conversations of very different lengths
        {"name": "attend_40x8192_bf16", "op": "attend", "act": "bf16", "cache": "bf16", "heads": 32, "kv": 8, "hd": 128,
         "page": 16, "seqs": 40, "ctx": 8192, "ragged": True},
        # one very long document
        {"name": "attend_1x131072_f16", "op": "attend", "act": "f16", "cache": "f16", "heads": 28, "kv": 4, "hd": 128,
         "page": 64, "seqs": 1, "ctx": 131071, "ragged": False},
        # gate projection of one token
        {"name": "linear_1_gate", "op": "linear", "act": "f32", "rows": 1, "n": 5632, "k": 2048, "group": 128,
         "scale": "f16", "residual": False},
        # down projection of a small batch onto the residual stream
        {"name": "linear_13_down", "op": "linear", "act": "bf16", "rows": 13, "n": 2048, "k": 5632, "group": 64,
         "scale": "bf16", "residual": True},
        # the head of one token
        {"name": "linear_1_head", "op": "linear", "act": "f32", "rows": 1, "n": 32000, "k": 2048, "group": 32,
         "scale": "f32", "residual": False},
        # one decoded token's log probability with alternatives
        {"name": "logprobs_1x32000", "op": "logprobs", "dtype": "f32", "rows": 1, "vocab": 32000, "top": 5,
         "masked": False},
        # a text scored at every position, over a larger odd vocabulary, some ids banned
        {"name": "logprobs_500x100003", "op": "logprobs", "dtype": "bf16", "rows": 500, "vocab": 100003, "top": 20,
         "masked": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, KV heads, head dimension)
HEADS = [(32, 4, 64), (8, 8, 64), (12, 12, 64), (16, 2, 128), (32, 8, 128), (28, 4, 128), (40, 8, 128), (5, 1, 64)]


def _draw_cache(rng):
    heads, kv, hd = rng.choice(HEADS)
    act = rng.choice(["f32", "f32", "bf16", "f16"])
    cache = "i8" if rng.random() < 0.5 else (act if act != "f32" else rng.choice(["bf16", "f16"]))
    return {"act": act, "cache": cache, "heads": heads, "kv": kv, "hd": hd, "page": rng.choice([16, 32, 64, 128])}


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "linear", "logprobs"])
    if op == "append":
        c = {"op": op, **_draw_cache(rng)}
        if rng.random() < 0.5:
            rows = _log_int(rng, 1, 256)
            return {**c, "seqs": rows, "rows": rows, "ctx": _log_int(rng, 1, 400)}
        rows = _log_int(rng, 1, 4096)
        return {**c, "seqs": 1, "rows": rows, "ctx": rows + rng.choice([0, rng.randint(0, 1000)])}
    if op == "attend":
        c = {"op": op, **_draw_cache(rng)}
        seqs = _log_int(rng, 1, 64)
        # no more cached bytes than the largest listed case has
        most = (40 * 8192 // 2) * 8 * 128 * 2 // (c["kv"] * c["hd"] * BYTES[c["cache"]] * seqs)
        # float32 results are held to float32's bound at the contexts a float32 engine serves
        most = min(most, 131072 if c["act"] != "f32" else 16384)
        return {**c, "seqs": seqs, "ctx": _log_int(rng, 1, most), "ragged": rng.random() < 0.6}
    if op == "linear":
        group = rng.choice([32, 64, 128])
        act = rng.choice(["f32", "f32", "bf16", "f16"])
        return {"op": op, "act": act, "rows": rng.choice([1, 1, 2, 3, _log_int(rng, 1, 16)]),
                "n": _log_int(rng, 64, 32000), "k": group * _log_int(rng, 512 // group, 8192 // group), "group": group,
                "scale": rng.choice(["f32", "bf16", "f16"]), "residual": rng.random() < 0.4}
    vocab = _log_int(rng, 1000, 200000)
    return {"op": op, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
            "rows": _log_int(rng, 1, min(1024, 25000000 // vocab)), "vocab": vocab, "top": rng.randint(0, 32),
            "masked": rng.random() < 0.3}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _lengths(c):
    """Cached positions of each sequence, the new token's among them: all ctx, or spread over 1 .. ctx."""
    if not c.get("ragged", True):
        return [c["ctx"]] * c["seqs"]
    return [c["ctx"] if i == 0 else max(1, math.ceil(c["ctx"] * math.fmod(i * 0.6180339887, 1.0)))
            for i in range(c["seqs"])]


def _rope_table(n, hd):
    """cos and sin [position][hd] float32, the two halves of a head alike."""
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().float(), ang.sin().float()


def _cache(c, g, lengths):
    """A pool of pages in a shuffled order, filled as a running server's is, and its page table."""
    pages = [-(-n // c["page"]) for n in lengths]
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda")[: sum(pages)].to(torch.int32)
    table = torch.zeros(c["seqs"], max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at: at + p]
        at += p
    shape = (n_pages, c["kv"], c["page"], c["hd"])
    s = {"table": table, "k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        x = torch.empty(shape, dtype=DTYPES[c["cache"]], device="cuda")
        for part in x.split(max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))):
            r = torch.randn(part.shape, generator=g, device="cuda")
            part.copy_((r * 36).round().clamp(-127, 127) if c["cache"] == "i8" else r * 1.2)
        s[name] = x
        if c["cache"] == "i8":
            s[name + "_scale"] = 0.02 + 0.04 * torch.rand(c["kv"], generator=g, device="cuda")
    return s


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] in ("append", "attend"):
        if c["op"] == "append" and c["seqs"] == 1:   # the last `rows` positions of one sequence
            lengths = [c["ctx"]]
            pos = torch.arange(c["ctx"] - c["rows"], c["ctx"], dtype=torch.int32, device="cuda")
            seq = torch.zeros(c["rows"], dtype=torch.int32, device="cuda")
        else:                                        # the newest position of every sequence
            lengths = _lengths(c)
            pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
            seq = torch.arange(c["seqs"], dtype=torch.int32, device="cuda")
        s = {"case": c, "pos": pos, "seq": seq, **_cache(c, g, lengths)}
        if c["op"] == "append":
            s["cos"], s["sin"] = _rope_table(max(lengths), c["hd"])
            s["qkv"] = torch.randn(c["rows"], (c["heads"] + 2 * c["kv"]) * c["hd"], generator=g,
                                   device="cuda").to(DTYPES[c["act"]])
        else:
            s["q"] = torch.randn(c["seqs"], c["heads"] * c["hd"], generator=g, device="cuda").to(DTYPES[c["act"]])
        if own:   # a server's handle on its cache, made once
            s["cache"] = _serving().PagedCache(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"],
                                               rope=(s["cos"], s["sin"]) if c["op"] == "append" else None)
        return s
    if c["op"] == "linear":
        n, k, group = c["n"], c["k"], c["group"]
        w = (torch.randn(n, k, generator=g, device="cuda") * 0.02).view(n, k // group, group)
        scales = (w.abs().amax(dim=2) / 7).to(DTYPES[c["scale"]])
        q = (w / scales.float()[:, :, None]).round().clamp(-8, 7).to(torch.int32).view(n, k) & 15
        x = torch.randn(c["rows"], k, generator=g, device="cuda")
        x[:, ::97] *= 12   # outlier channels
        s = {"case": c, "q": (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8), "scales": scales,
             "x": x.to(DTYPES[c["act"]]), "residual": None}
        if c["residual"]:
            s["residual"] = torch.randn(c["rows"], n, generator=g, device="cuda").to(DTYPES[c["act"]])
        if own:   # the layer of a loaded model
            s["linear"] = _serving().W4Linear(s["q"], s["scales"])
        return s
    x = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda") * 2.5
    x[:, ::1009] += 6
    if c["masked"]:
        x.masked_fill_(torch.rand(c["vocab"], generator=g, device="cuda") < 0.02, -math.inf)
        x[:, 0] = 1.0
    x = x.to(DTYPES[c["dtype"]])
    # the tokens that were sampled or given: one of the likely ones
    near = x.float() + 1.5 * torch.randn(x.shape, generator=g, device="cuda")
    return {"case": c, "logits": x, "targets": near.argmax(dim=1).to(torch.int32)}


# ---- one pass ---------------------------------------------------------------------------------------------------

def _serving():
    from __graft_entry__ import load_package
    load_package()
    from lpta import serving
    return serving


def _values(s, name):
    """The pages' values: the buffer itself, or what its INT8 stands for."""
    scale = s[name + "_scale"]
    return s[name] if scale is None else s[name] * scale[:, None, None]


def _append(s):
    c = s["case"]
    heads, kv, hd, page = c["heads"], c["kv"], c["hd"], c["page"]
    pos = s["pos"].long()
    x = s["qkv"].float().view(-1, heads + 2 * kv, hd)
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    turned = torch.cat([-qk[..., hd // 2:], qk[..., :hd // 2]], dim=-1)
    qk = qk * s["cos"][pos][:, None] + turned * s["sin"][pos][:, None]
    q, k = qk[:, :heads], qk[:, heads:]
    if c["cache"] == "i8":
        k = (k / s["k_scale"][:, None]).round().clamp(-127, 127)
        v = (v / s["v_scale"][:, None]).round().clamp(-127, 127)
    pages, at = s["table"][s["seq"].long(), pos // page].long(), pos % page
    s["k"][pages, :, at] = k.to(s["k"].dtype)
    s["v"][pages, :, at] = v.to(s["v"].dtype)
    return q.reshape(-1, heads * hd).to(s["qkv"].dtype)


def _attend(s):
    c = s["case"]
    heads, kv, hd, page = c["heads"], c["kv"], c["hd"], c["page"]
    b, rep = c["seqs"], heads // kv
    table = s["table"][s["seq"].long()].long()
    # [seq][page][KV head][position][hd]; the sum over positions is made page by page
    k, v = (s[name][table].float() for name in ("k", "v"))
    if c["cache"] == "i8":
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    q = s["q"].float().view(b, 1, kv, rep, hd) * (1.0 / math.sqrt(hd))
    x = torch.matmul(k, q.transpose(-1, -2).contiguous())            # [seq][page][KV head][position][rep]
    at = torch.arange(table.shape[1] * page, device="cuda").view(1, -1, 1, page, 1)
    x = x.masked_fill(at > s["pos"].view(b, 1, 1, 1, 1), -math.inf)
    e = torch.exp(x - x.amax(dim=(1, 3), keepdim=True))
    p = (e / e.sum(dim=(1, 3), keepdim=True)).transpose(-1, -2).contiguous()
    return torch.matmul(p, v).sum(dim=1).reshape(b, heads * hd).to(s["q"].dtype)


def _linear(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    q = s["q"].to(torch.int32)
    q = torch.stack([q & 15, q >> 4], dim=-1).view(n, k // group, group)
    w = (q - ((q & 8) << 1)).float() * s["scales"].float()[:, :, None]
    y = torch.matmul(s["x"].float(), w.view(n, k).t())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    x = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    lp = x.gather(1, s["targets"].long()[:, None])[:, 0] - log_total
    entropy = log_total - torch.where(e > 0, x * e, 0.0).sum(dim=1) / total
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)   # equal logits: the lowest id first
    return {"logprob": lp, "entropy": entropy, "top_ids": ids[:, :c["top"]].to(torch.int32),
            "top_logprobs": best[:, :c["top"]] - log_total[:, None]}


def run(state):
    s, op = state, state["case"]["op"]
    if op == "append":
        if own:
            q = s["cache"].append(s["qkv"], s["seq"], s["pos"])
        else:
            q = _append(s)
        return {"q": q, "k": _values(s, "k"), "v": _values(s, "v")}
    if op == "attend":
        if own:
            return s["cache"].attend(s["q"], s["seq"], s["pos"])
        return _attend(s)
    if op == "linear":
        if own:
            return s["linear"](s["x"], residual=s["residual"])
        return _linear(s)
    if own:
        got = _serving().token_logprobs(s["logits"], s["targets"], top=s["case"]["top"])
        return {"logprob": got.logprob, "entropy": got.entropy, "top_ids": got.top_ids,
                "top_logprobs": got.top_logprobs}
    return _logprobs(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "append":
        a, b, hd = BYTES[c["act"]], BYTES[c["cache"]], c["hd"]
        rows, width = c["rows"], (c["heads"] + c["kv"]) * hd
        moved = rows * ((c["heads"] + 2 * c["kv"]) * hd * a + c["heads"] * hd * a + 2 * c["kv"] * hd * b)
        tables = (rows if c["seqs"] == 1 else len(set(_lengths(c)))) * hd * 4
        return {"bytes": moved + tables + rows * 12, "flops": rows * width * 3}
    if c["op"] == "attend":
        n = sum(_lengths(c))
        pages = sum(-(-x // c["page"]) for x in _lengths(c))
        moved = n * 2 * c["kv"] * c["hd"] * BYTES[c["cache"]] + 2 * c["seqs"] * c["heads"] * c["hd"] * BYTES[c["act"]]
        return {"bytes": moved + pages * 4 + c["seqs"] * 8, "flops": 4 * n * c["heads"] * c["hd"]}
    if c["op"] == "linear":
        n, k, m = c["n"], c["k"], c["rows"]
        moved = n * k // 2 + n * (k // c["group"]) * BYTES[c["scale"]] + m * k * BYTES[c["act"]]
        return {"bytes": moved + m * n * BYTES[c["act"]] * (2 if c["residual"] else 1), "flops": 2 * m * n * k}
    moved = c["rows"] * (c["vocab"] * BYTES[c["dtype"]] + 12 + 8 * c["top"])
    return {"bytes": moved, "flops": 4 * c["rows"] * c["vocab"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        hd, heads, kv = c["hd"], c["heads"], c["kv"]
        x = s["qkv"].double().view(c["rows"], heads + 2 * kv, 2, hd // 2)
        pos = s["pos"].long()
        # a pair (x_d, x_{d + hd/2}) as a complex number, turned by its position's angle
        turn = torch.complex(s["cos"][pos, None, :hd // 2].double(), s["sin"][pos, None, :hd // 2].double())
        z = torch.complex(x[:, :heads + kv, 0], x[:, :heads + kv, 1]) * turn
        y = torch.cat([z.real, z.imag], dim=-1)
        q = y[:, :heads].reshape(c["rows"], heads * hd)
        if c["cache"] == "i8":
            return {"q": q, "k": None, "v": None}
        out = {"q": q}
        v = x[:, heads + kv:].reshape(c["rows"], kv, hd)
        slot = s["table"][s["seq"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]
        for name, new in (("k", y[:, heads:]), ("v", v)):
            rows = s[name].double().transpose(1, 2).contiguous()     # [page][position][KV head][hd]
            rows.view(-1, kv, hd)[slot] = new
            out[name] = rows.transpose(1, 2).contiguous()
        return out
    if c["op"] == "attend":
        kv, hd, rep = c["kv"], c["hd"], c["heads"] // c["kv"]
        out = torch.empty(c["seqs"], c["heads"], hd, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(c)):
            pages = s["table"][b, :-(-n // c["page"])].long()
            for h in range(kv):
                k, v = (s[name][pages, h].reshape(-1, hd)[:n].double() for name in ("k", "v"))
                if c["cache"] == "i8":
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                q = s["q"][b].view(c["heads"], hd)[h * rep:(h + 1) * rep].double()
                out[b, h * rep:(h + 1) * rep] = torch.softmax(q @ k.t() / math.sqrt(hd), dim=1) @ v
        return out.view(c["seqs"], c["heads"] * hd)
    if c["op"] == "linear":
        q = s["q"].long()
        low, high = q % 16, q // 16
        w = torch.empty(c["n"], c["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = torch.where(low > 7, low - 16, low), torch.where(high > 7, high - 16, high)
        w *= s["scales"].double().repeat_interleave(c["group"], dim=1)
        y = (w @ s["x"].double().t()).t()
        return y if s["residual"] is None else y + s["residual"].double()
    lp = torch.log_softmax(s["logits"].double(), dim=1)
    order = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :c["top"]]
    return {"logprob": lp.gather(1, s["targets"].long()[:, None])[:, 0], "entropy": torch.special.entr(lp.exp()).sum(dim=1),
            "top_ids": order.to(torch.int32), "top_logprobs": lp.gather(1, order)}
