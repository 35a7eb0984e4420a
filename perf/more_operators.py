"""Performance cases of further serving operators: one layer's step of many conversations that share a long prompt,
with 8-bit projections.

Operators and ranges (`draw` spreads over them):
  norm    rows of Q|K|V projections, q and k normed for each head and rotated, K and V written into a paged cache:
          1 .. 4096 rows (one new token of many sequences, or the consecutive tokens of one prompt), heads of 64 and 128
  shared  attention of one new token per sequence, whose first positions are one prompt's for all: 1 .. 256 sequences,
          a prompt of 1 .. 65536 positions, 1 .. 2000 positions of their own, 1 .. 8 query heads per KV head
  w8      a projection with 8-bit weights and activations, scales for each token and channel: 1 .. 8192 rows, odd
          sizes among them
  glu     gate and up projections of that kind and their product silu(gate) up: 1 .. 4096 rows

Heads and widths of the small cases are the TinyLlama-1.1B shape of bench.py (32 query / 4 KV heads of 64, hidden
2048, FFN 5632, up to 2048 positions); the others are generic.

Types: activations float32 (the framework's), bfloat16 or float16; the cache INT8 with one scale per KV head (the
framework's), bfloat16 or float16; weights INT8 with one float32 scale per channel.  What is rounded to INT8 on the
way (cache rows, rows of activations) is defined by float32 steps, each rounded: the norm's factor f = 1 / sqrt(mean
x^2 + eps) in 64 bits and rounded once, (x f) gain, the rotation, a division by the scale, round to nearest even; a
row's scale is max |x| / 127.  INT8 cache rows therefore have no value in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}
THETA = 10000.0
EPS = 1e-5


def listed():
    return [
        # one conversation, one new token of the repository's shape into its INT8 cache
        {"name": "norm_1_i8", "op": "norm", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64, "page": 16,
         "seqs": 1, "rows": 1, "ctx": 40},
        # a decoding step of a ragged batch
        {"name": "norm_75_bf16", "op": "norm", "act": "bf16", "cache": "bf16", "heads": 32, "kv": 8, "hd": 128,
         "page": 16, "seqs": 75, "rows": 75, "ctx": 300},
        # a long prompt's rows
        {"name": "norm_4000_f16", "op": "norm", "act": "f16", "cache": "f16", "heads": 32, "kv": 8, "hd": 128,
         "page": 64, "seqs": 1, "rows": 4000, "ctx": 4000},
        # a few conversations after a short instruction: latency
        {"name": "shared_4x500_i8", "op": "shared", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64,
         "page": 16, "seqs": 4, "prefix": 500, "own": 60, "ragged": True},
        # the benchmark's batch of 32 sequences near the end of the context, three quarters of it in common
        {"name": "shared_32x1536_i8", "op": "shared", "act": "f32", "cache": "i8", "heads": 32, "kv": 4, "hd": 64,
         "page": 64, "seqs": 32, "prefix": 1536, "own": 448, "ragged": False},
        # many questions about one long document
        {"name": "shared_64x32768_bf16", "op": "shared", "act": "bf16", "cache": "bf16", "heads": 32, "kv": 8,
         "hd": 128, "page": 16, "seqs": 64, "prefix": 32768, "own": 700, "ragged": True},
        # down projection of one token onto the residual stream
        {"name": "w8_1_down", "op": "w8", "act": "f32", "rows": 1, "n": 2048, "k": 5632, "residual": True},
        # Q|K|V of a decoding step of a batch
        {"name": "w8_45_qkv", "op": "w8", "act": "bf16", "rows": 45, "n": 6144, "k": 4096, "residual": False},
        # a prompt's rows through a wide projection
        {"name": "w8_4096_wide", "op": "w8", "act": "bf16", "rows": 4096, "n": 14336, "k": 4096, "residual": False},
        # gate and up of one token
        {"name": "glu_1", "op": "glu", "act": "f32", "rows": 1, "n": 5632, "k": 2048},
        # the benchmark's batch
        {"name": "glu_32", "op": "glu", "act": "f32", "rows": 32, "n": 5632, "k": 2048},
        # several prompts' rows together
        {"name": "glu_2001", "op": "glu", "act": "f16", "rows": 2001, "n": 14336, "k": 4096},
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
    op = rng.choice(["norm", "shared", "shared", "w8", "w8", "glu"])
    if op == "norm":
        c = {"op": op, **_draw_cache(rng)}
        if rng.random() < 0.5:
            rows = _log_int(rng, 1, 256)
            return {**c, "seqs": rows, "rows": rows, "ctx": _log_int(rng, 1, 400)}
        rows = _log_int(rng, 1, 4000)
        return {**c, "seqs": 1, "rows": rows, "ctx": rows + rng.choice([0, rng.randint(0, 1000)])}
    if op == "shared":
        c = {"op": op, **_draw_cache(rng)}
        seqs = _log_int(rng, 1, 256)
        # no more products and no more bytes of the sequences' own than the largest listed case has
        most = 64 * 32768 * 32 * 128 // (seqs * c["heads"] * c["hd"])
        # float32 results are held to float32's bound at the contexts a float32 engine serves
        most = min(most, 65536 if c["act"] != "f32" else 16384)
        kept = 64 * 350 * 8 * 128 * 2 // (seqs * c["kv"] * c["hd"] * BYTES[c["cache"]])
        return {**c, "seqs": seqs, "prefix": _log_int(rng, 1, most), "own": _log_int(rng, 1, min(2000, kept)),
                "ragged": rng.random() < 0.6}
    act = rng.choice(["f32", "bf16", "bf16", "f16"])
    k = rng.choice([_log_int(rng, 64, 16384), 64 * _log_int(rng, 4, 256), 64 * _log_int(rng, 4, 256)])
    most = 4096 * 14336 * 4096
    if op == "w8":
        n = _log_int(rng, 64, 32000)
        # no more bytes of results than the largest listed case has
        rows = _log_int(rng, 1, max(1, min(8192, most // (n * k), 4096 * 14336 * 2 // (n * BYTES[act]))))
        return {"op": op, "act": act, "rows": rows, "n": n, "k": k, "residual": rng.random() < 0.4}
    n = _log_int(rng, 64, 16384)
    return {"op": op, "act": act, "rows": _log_int(rng, 1, max(1, min(4096, most // (2 * n * k)))), "n": n, "k": k}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _spread(n, most, ragged):
    """n lengths: all `most`, or spread over 1 .. most."""
    if not ragged:
        return [most] * n
    return [most if i == 0 else max(1, math.ceil(most * math.fmod(i * 0.6180339887, 1.0))) for i in range(n)]


def _rope_table(n, hd):
    """cos and sin [position][hd] float32, the two halves of a head alike."""
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().float(), ang.sin().float()


def _pool(c, g, n_pages):
    """Pages filled as a running server's are."""
    shape = (n_pages, c["kv"], c["page"], c["hd"])
    s = {"k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        x = torch.empty(shape, dtype=DTYPES[c["cache"]], device="cuda")
        for part in x.split(max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))):
            r = torch.randn(part.shape, generator=g, device="cuda")
            part.copy_((r * 36).round().clamp(-127, 127) if c["cache"] == "i8" else r * 1.2)
        s[name] = x
        if c["cache"] == "i8":
            s[name + "_scale"] = 0.02 + 0.04 * torch.rand(c["kv"], generator=g, device="cuda")
    return s


def _table(g, counts, n_pages):
    """A page table that hands out pages in a shuffled order."""
    order = torch.randperm(n_pages, generator=g, device="cuda")[: sum(counts)].to(torch.int32)
    table = torch.zeros(len(counts), max(counts), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(counts):
        table[i, :p] = order[at: at + p]
        at += p
    return table


def _weights(g, n, k):
    """8-bit weights [n][k] and a scale for each channel."""
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    scale = w.abs().amax(dim=1) / 127
    return (w / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "norm":
        if c["seqs"] == 1:   # the last `rows` positions of one sequence
            lengths = [c["ctx"]]
            pos = torch.arange(c["ctx"] - c["rows"], c["ctx"], dtype=torch.int32, device="cuda")
            seq = torch.zeros(c["rows"], dtype=torch.int32, device="cuda")
        else:                # the newest position of every sequence
            lengths = _spread(c["seqs"], c["ctx"], True)
            pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
            seq = torch.arange(c["seqs"], dtype=torch.int32, device="cuda")
        counts = [-(-n // c["page"]) for n in lengths]
        s = {"case": c, "pos": pos, "seq": seq, **_pool(c, g, sum(counts) + 3)}
        s["table"] = _table(g, counts, sum(counts) + 3)
        s["cos"], s["sin"] = _rope_table(max(lengths), c["hd"])
        s["q_gain"], s["k_gain"] = (1 + 0.3 * torch.randn(c["hd"], generator=g, device="cuda") for _ in range(2))
        x = torch.randn(c["rows"], c["heads"] + 2 * c["kv"], c["hd"], generator=g, device="cuda")
        x *= torch.exp(torch.randn(c["rows"], c["heads"] + 2 * c["kv"], 1, generator=g, device="cuda"))
        s["qkv"] = x.view(c["rows"], -1).to(DTYPES[c["act"]])
        if own:   # a server's handle on its cache, made once
            s["cache"] = _serving().PagedCache(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"],
                                               rope=(s["cos"], s["sin"]))
        return s
    if c["op"] == "shared":
        # sequence 0 is the prompt; the conversations' first whole pages are its own, the rest theirs
        lens = _spread(c["seqs"], c["own"], c["ragged"])
        common = c["prefix"] // c["page"]
        first = -(-c["prefix"] // c["page"])
        counts = [first] + [-(-(c["prefix"] + n) // c["page"]) - common for n in lens]
        n_pages = sum(counts) + 3
        s = {"case": c, **_pool(c, g, n_pages)}
        t = _table(g, counts, n_pages)
        table = torch.zeros(1 + c["seqs"], max(first, common + max(counts[1:])), dtype=torch.int32, device="cuda")
        table[:, :common] = t[0, :common]
        table[0, :first] = t[0, :first]
        for i, p in enumerate(counts[1:], 1):
            table[i, common:common + p] = t[i, :p]
        s["table"] = table
        s["seq"] = torch.arange(1, 1 + c["seqs"], dtype=torch.int32, device="cuda")
        s["pos"] = torch.tensor(lens, dtype=torch.int32, device="cuda") + (c["prefix"] - 1)
        s["q"] = torch.randn(c["seqs"], c["heads"] * c["hd"], generator=g, device="cuda").to(DTYPES[c["act"]])
        if own:
            s["cache"] = _serving().PagedCache(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"])
        return s
    n, k = c["n"], c["k"]
    x = torch.randn(c["rows"], k, generator=g, device="cuda")
    x[:, ::97] *= 6   # outlier channels
    s = {"case": c, "x": x.to(DTYPES[c["act"]])}
    if c["op"] == "glu":
        s["w"], s["scale"] = _weights(g, n, k)
        s["w2"], s["scale2"] = _weights(g, n, k)
        if own:   # the layer of a loaded model
            s["linear"] = _serving().W8GatedLinear(s["w"], s["scale"], s["w2"], s["scale2"])
        return s
    s["w"], s["scale"] = _weights(g, n, k)
    s["residual"] = torch.randn(c["rows"], n, generator=g, device="cuda").to(DTYPES[c["act"]]) if c["residual"] else None
    if own:
        s["linear"] = _serving().W8Linear(s["w"], s["scale"])
    return s


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


def _norm(s):
    c = s["case"]
    heads, kv, hd, page = c["heads"], c["kv"], c["hd"], c["page"]
    pos = s["pos"].long()
    x = s["qkv"].float().view(-1, heads + 2 * kv, hd)
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    mean = (qk.double() * qk.double()).sum(dim=-1, keepdim=True) / hd
    qk = qk * (1.0 / torch.sqrt(mean + EPS)).float()
    gain = torch.cat([s["q_gain"].expand(heads, hd), s["k_gain"].expand(kv, hd)])
    qk = qk * gain
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


def _shared(s):
    """The prompt's keys in one product for all sequences, then each one's own; one softmax over both."""
    c = s["case"]
    heads, kv, hd, page, n = c["heads"], c["kv"], c["hd"], c["page"], c["prefix"]
    b, rep = c["seqs"], heads // kv

    def read(name, pages):     # [..., page][KV head][position][hd]
        x = s[name][pages].float()
        return x if s[name + "_scale"] is None else x * s[name + "_scale"][:, None, None]
    q = s["q"].float().view(b, kv, rep, hd) * (1.0 / math.sqrt(hd))
    qh = q.transpose(0, 1).reshape(kv, b * rep, hd)
    prompt = s["table"][0, :-(-n // page)].long()
    k, v = (read(name, prompt).transpose(0, 1).reshape(kv, -1, hd)[:, :n] for name in ("k", "v"))
    x = torch.matmul(qh, k.transpose(1, 2).contiguous())                        # [KV head][row, head][position]
    mine = s["table"][s["seq"].long(), n // page:].long()
    ko, vo = (read(name, mine) for name in ("k", "v"))                           # [row][page][KV head][position][hd]
    y = torch.matmul(ko, q[:, None].transpose(-1, -2).contiguous())              # [row][page][KV head][position][rep]
    at = (n // page * page + torch.arange(mine.shape[1] * page, device="cuda")).view(1, -1, 1, page, 1)
    y = y.masked_fill((at < n) | (at > s["pos"].view(b, 1, 1, 1, 1)), -math.inf)
    x = x.view(kv, b, rep, n)
    top = torch.maximum(x.amax(dim=3).permute(1, 0, 2), y.amax(dim=(1, 3)))      # [row][KV head][rep]
    x = torch.exp(x - top.permute(1, 0, 2)[..., None])
    y = torch.exp(y - top[:, None, :, None])
    total = x.sum(dim=3).permute(1, 0, 2) + y.sum(dim=(1, 3))
    o = torch.matmul(x.view(kv, b * rep, n), v).view(kv, b, rep, hd).transpose(0, 1)
    o = o + torch.matmul(y.transpose(-1, -2).contiguous(), vo).sum(dim=1)
    return (o / total[..., None]).reshape(b, heads * hd).to(s["q"].dtype)


def _product(x, w, scale):
    """Rows of x to INT8 with a scale each, their products with w's rows, in float32."""
    x = x.float()
    row = x.abs().amax(dim=1, keepdim=True) / 127
    row = torch.where(row == 0, 1.0, row)
    q = (x / row).round().clamp(-127, 127)
    return torch.matmul(q, w.float().t()) * (row * scale)


def run(state):
    s, op = state, state["case"]["op"]
    if op == "norm":
        if own:
            q = s["cache"].append(s["qkv"], s["seq"], s["pos"], norm=(s["q_gain"], s["k_gain"]), eps=EPS)
        else:
            q = _norm(s)
        return {"q": q, "k": _values(s, "k"), "v": _values(s, "v")}
    if op == "shared":
        if own:
            return s["cache"].attend_shared(s["q"], s["seq"], s["pos"], 0, s["case"]["prefix"])
        return _shared(s)
    if op == "w8":
        if own:
            return s["linear"](s["x"], residual=s["residual"])
        y = _product(s["x"], s["w"], s["scale"])
        return (y if s["residual"] is None else y + s["residual"].float()).to(s["x"].dtype)
    if own:
        return s["linear"](s["x"])
    gate, up = _product(s["x"], s["w"], s["scale"]), _product(s["x"], s["w2"], s["scale2"])
    return (gate / (1.0 + torch.exp(-gate)) * up).to(s["x"].dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "norm":
        a, b, hd = BYTES[c["act"]], BYTES[c["cache"]], c["hd"]
        rows, width = c["rows"], (c["heads"] + c["kv"]) * hd
        moved = rows * ((c["heads"] + 2 * c["kv"]) * hd * a + c["heads"] * hd * a + 2 * c["kv"] * hd * b)
        tables = (rows if c["seqs"] == 1 else len(set(_spread(c["seqs"], c["ctx"], True)))) * hd * 4
        return {"bytes": moved + tables + rows * 12 + 8 * hd, "flops": rows * width * 7}
    if c["op"] == "shared":
        lens = _spread(c["seqs"], c["own"], c["ragged"])
        keys = c["prefix"] + sum(lens)
        moved = keys * 2 * c["kv"] * c["hd"] * BYTES[c["cache"]] + 2 * c["seqs"] * c["heads"] * c["hd"] * BYTES[c["act"]]
        return {"bytes": moved + keys // c["page"] * 4 + c["seqs"] * 8,
                "flops": 4 * (c["seqs"] * c["prefix"] + sum(lens)) * c["heads"] * c["hd"]}
    n, k, m = c["n"], c["k"], c["rows"]
    two = 2 if c["op"] == "glu" else 1
    moved = two * n * (k + 4) + m * (k + n * (2 if c.get("residual") else 1)) * BYTES[c["act"]]
    return {"bytes": moved, "flops": 2 * two * m * n * k}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def _exact_product(x, w, scale):
    x = x.double()
    row = (x.abs().amax(dim=1) / 127).float().double()
    row[row == 0] = 1
    q = torch.round((x / row[:, None]).float()).clamp(-127, 127).double()
    return (w.double() @ q.t()).t() * row[:, None] * scale.double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        hd, heads, kv = c["hd"], c["heads"], c["kv"]
        x = s["qkv"].double().view(c["rows"], heads + 2 * kv, hd)
        pos = s["pos"].long()
        qk = x[:, :heads + kv]
        qk = qk / (qk.pow(2).mean(dim=-1, keepdim=True) + EPS).sqrt()
        qk = torch.cat([qk[:, :heads] * s["q_gain"].double(), qk[:, heads:] * s["k_gain"].double()], dim=1)
        qk = qk.view(c["rows"], heads + kv, 2, hd // 2)
        # a pair (x_d, x_{d + hd/2}) as a complex number, turned by its position's angle
        turn = torch.complex(s["cos"][pos, None, :hd // 2].double(), s["sin"][pos, None, :hd // 2].double())
        z = torch.complex(qk[:, :, 0], qk[:, :, 1]) * turn
        y = torch.cat([z.real, z.imag], dim=-1)
        q = y[:, :heads].reshape(c["rows"], heads * hd)
        if c["cache"] == "i8":
            return {"q": q, "k": None, "v": None}
        out = {"q": q}
        slot = s["table"][s["seq"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]
        for name, new in (("k", y[:, heads:]), ("v", x[:, heads + kv:])):
            rows = s[name].double().transpose(1, 2).contiguous()     # [page][position][KV head][hd]
            rows.view(-1, kv, hd)[slot] = new
            out[name] = rows.transpose(1, 2).contiguous()
        return out
    if c["op"] == "shared":
        kv, hd, rep, n, page = c["kv"], c["hd"], c["heads"] // c["kv"], c["prefix"], c["page"]
        out = torch.empty(c["seqs"], c["heads"], hd, dtype=torch.float64, device="cuda")
        for h in range(kv):
            def rows(row, end):
                pages = s["table"][row, :-(-end // page)].long()
                k, v = (s[name][pages, h].reshape(-1, hd)[:end].double() for name in ("k", "v"))
                if c["cache"] == "i8":
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                return k, v
            kp, vp = rows(0, n)
            for b, m in enumerate(_spread(c["seqs"], c["own"], c["ragged"])):
                # the prompt's last page may lie elsewhere in the conversation's table: from n on only its own count
                pages = s["table"][b + 1, n // page:-(-(n + m) // page)].long()
                ko, vo = (s[name][pages, h].reshape(-1, hd)[n % page:n % page + m].double() for name in ("k", "v"))
                if c["cache"] == "i8":
                    ko, vo = ko * s["k_scale"][h].double(), vo * s["v_scale"][h].double()
                q = s["q"][b].view(c["heads"], hd)[h * rep:(h + 1) * rep].double()
                p = torch.softmax(torch.cat([q @ kp.t(), q @ ko.t()], dim=1) / math.sqrt(hd), dim=1)
                out[b, h * rep:(h + 1) * rep] = p[:, :n] @ vp + p[:, n:] @ vo
        return out.view(c["seqs"], c["heads"] * hd)
    if c["op"] == "w8":
        y = _exact_product(s["x"], s["w"], s["scale"])
        return y if s["residual"] is None else y + s["residual"].double()
    gate, up = (_exact_product(s["x"], s[w], s[v]) for w, v in (("w", "scale"), ("w2", "scale2")))
    return torch.nn.functional.silu(gate) * up
