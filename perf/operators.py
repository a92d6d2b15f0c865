"""Timed cases of the serving operators: what a host runs between the
projections and the sampler when many sessions share one paged key-value
cache.

A case is a dict of plain values with a "kind":

* ``append`` -- the new tokens of every sequence: keys (RMS-normed per head and
  rotated) and values go into the cache's pages, the queries are normed and
  rotated for the attention that follows.
* ``decode`` -- attention of one new token per sequence over its pages.
* ``prompt`` -- causal attention of packed new tokens, sequences of different
  lengths, each behind the history that its pages hold.
* ``sample`` -- one draw per row of logits: temperature, top-k, top-p, min-p and
  a given random number for each row.

Sequence lengths follow from the case alone (its "mix"), values and page orders
from the seed. Sizes are those of the models in bench.py: 32 query heads on 8
key-value heads (4B shape) and 16 on 8 (1.7B shape), 128 values a head,
vocabulary 151936, sessions of 4096 positions, 8 of them together; the larger
ones stand for a server with more memory and more players.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 151936
EPS = 1e-6


def listed():
    return [
        # Eight players' sessions, a decode step's token each, in the engine's
        # own cache type. The smallest call.
        {"name": "append 8 tokens f32", "kind": "append", "type": "f32", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "seqs": 8, "len_lo": 1025, "len_hi": 1152, "new_lo": 1, "new_hi": 1, "mix": 1},
        # Prompts of a full server, some of them the next part of a longer
        # document.
        {"name": "append prompts bf16", "kind": "append", "type": "bf16", "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "seqs": 12, "len_lo": 300, "len_hi": 4096, "new_lo": 77, "new_hi": 1500, "mix": 2},
        # One player of the small model, early in a conversation: latency.
        {"name": "decode 1 short f16", "kind": "decode", "type": "f16", "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "seqs": 1, "len_lo": 95, "len_hi": 95, "mix": 3},
        # Eight sessions behind a prompt of 1024 tokens, in the engine's type.
        {"name": "decode 8 f32", "kind": "decode", "type": "f32", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "seqs": 8, "len_lo": 1025, "len_hi": 1152, "mix": 4},
        # A busy server: conversations of every length.
        {"name": "decode 64 ragged bf16", "kind": "decode", "type": "bf16", "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "seqs": 64, "len_lo": 200, "len_hi": 12000, "mix": 5},
        # One reader of a very long document.
        {"name": "decode 1 long f16", "kind": "decode", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "page": 256,
         "seqs": 1, "len_lo": 131000, "len_hi": 131000, "mix": 6},
        # The next messages of a few running conversations, together.
        {"name": "prompt turns f16", "kind": "prompt", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "seqs": 6, "len_lo": 400, "len_hi": 1703, "new_lo": 12, "new_hi": 203, "mix": 7},
        # The headline prompt in the engine's own type.
        {"name": "prompt 512 f32", "kind": "prompt", "type": "f32", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "seqs": 1, "len_lo": 512, "len_hi": 512, "new_lo": 512, "new_hi": 512, "mix": 8},
        # Documents that fill their contexts. The largest.
        {"name": "prompt documents bf16", "kind": "prompt", "type": "bf16", "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "seqs": 4, "len_lo": 2900, "len_hi": 4096, "new_lo": 2900, "new_hi": 4096, "mix": 9},
        # A single session's draw at the chat defaults: latency. The logits of
        # random weights are flat, so most of the vocabulary stays in.
        {"name": "sample 1 default f32", "kind": "sample", "type": "f32", "vocab": VOCAB, "rows": 1, "flat": True,
         "mixed": False, "temperature": 0.7, "top_k": 0, "top_p": 0.95, "min_p": 0.0},
        # Eight sessions with min-p, as role-playing hosts like it.
        {"name": "sample 8 min-p f32", "kind": "sample", "type": "f32", "vocab": VOCAB, "rows": 8, "flat": False,
         "mixed": False, "temperature": 1.1, "top_k": 0, "top_p": 1.0, "min_p": 0.05},
        # A full server: every row with parameters of its own.
        {"name": "sample 192 mixed bf16", "kind": "sample", "type": "bf16", "vocab": VOCAB, "rows": 192, "flat": False,
         "mixed": True, "temperature": 0.8, "top_k": 40, "top_p": 0.9, "min_p": 0.02},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "sample"])
    kind_type = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "sample":
        top_k, top_p, min_p = rng.choice([(0, 0.95, 0.0), (40, 0.95, 0.0), (0, 1.0, 0.1), (100, 1.0, 0.02), (0, 0.8, 0.01)])
        return {"kind": kind, "type": kind_type, "vocab": _log(rng, 1000, VOCAB), "rows": _log(rng, 1, 96),
                "flat": rng.random() < 0.3, "mixed": rng.random() < 0.5, "temperature": round(rng.uniform(0.2, 1.5), 2),
                "top_k": top_k, "top_p": top_p, "min_p": min_p}
    kv = rng.choice([1, 2, 4, 8, 8])
    case = {"kind": kind, "type": kind_type, "heads": kv * rng.choice([1, 2, 4, 4, 5, 8]), "kv": kv,
            "dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 256])}
    if kind == "decode":
        hi = _log(rng, 1, 16000)
        case |= {"seqs": _log(rng, 1, min(64, max(1, 400000 // hi))), "len_lo": max(1, int(hi * rng.uniform(0.05, 1))),
                 "len_hi": hi}
    else:
        new = _log(rng, 1, 3000 if kind == "append" else 2500)
        hi = min(4096, new + rng.choice([0, _log(rng, 1, 2500)]))
        case |= {"seqs": _log(rng, 1, min(24, max(1, 9000 // hi))), "len_lo": max(new, int(hi * rng.uniform(0.2, 1))),
                 "len_hi": hi, "new_lo": max(1, int(new * rng.uniform(0.1, 1))), "new_hi": new}
    return case | {"mix": rng.randrange(1 << 20)}


# ---- inputs


def _lengths(case):
    """(positions that each sequence's cache holds after the call, its new tokens among them)."""
    rng = random.Random(case["mix"])
    lens = [_log(rng, case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    if "new_lo" not in case:
        return lens, [1] * len(lens)
    return lens, [min(n, _log(rng, case["new_lo"], case["new_hi"])) for n in lens]


def _device(case):
    return torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")


def prepare(case, seed):
    dev = _device(case)
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = TYPES[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * by).to(dtype)

    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device=dev)
        if not case["flat"]:  # a trained model's: a broad floor, and some tens of tokens that stand out
            x = x * 2.2
            few = torch.randint(0, vocab, (rows, 48), generator=gen, device=dev)
            x.scatter_(1, few, torch.rand(rows, 48, generator=gen, device=dev) * 9.0 + 5.0)

        def column(value, choices, t):
            pick = torch.randint(0, len(choices), (rows,), generator=gen, device=dev)
            every = torch.tensor(choices, device=dev, dtype=t)[pick]
            return every if case["mixed"] else torch.full((rows,), value, device=dev, dtype=t)

        return {"case": case, "logits": x.to(dtype),
                "temperature": column(case["temperature"], [0.0, 0.3, 0.7, case["temperature"], 1.3], torch.float32),
                "top_k": column(case["top_k"], [0, 1, 20, case["top_k"], 400], torch.int32),
                "top_p": column(case["top_p"], [1.0, 0.5, 0.95, case["top_p"]], torch.float32),
                "min_p": column(case["min_p"], [0.0, 0.1, case["min_p"]], torch.float32),
                "u": torch.rand(rows, generator=gen, device=dev)}

    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, new = _lengths(case)
    pages = [-(-n // page) for n in lens]
    # A pool with some pages to spare, handed out in no order; the table's
    # entries behind a sequence's last page hold -1.
    pool = sum(pages) + 1 + sum(pages) // 16
    order = torch.randperm(pool, generator=gen, device=dev)[: sum(pages)].to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    tokens = sum(new)
    state = {"case": case, "table": table, "k_pool": normal(pool, kv, page, dim), "v_pool": normal(pool, kv, page, dim),
             "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "longest": max(new),
             "starts": torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)}
    if case["kind"] == "append":
        # One fused projection's output, as the QKV product writes it.
        qkv = normal(tokens, heads + 2 * kv, dim, by=2.0)
        state |= {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:],
                  "q_out": torch.empty(tokens, heads, dim, dtype=dtype, device=dev)}
        for name in ("q_norm", "k_norm"):
            state[name] = 1 + 0.1 * torch.randn(dim, generator=gen, device=dev)
        pos = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None]
        ang = pos * torch.pow(1e6, -2.0 * torch.arange(dim // 2, device=dev, dtype=torch.float64) / dim)
        state["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    else:
        state["q"] = normal(tokens, heads, dim, by=1.5)
        state["out"] = torch.empty(tokens, heads, dim, dtype=dtype, device=dev)
    if own:
        from rpgbarengine_amd import serving
        state["cache"] = serving.PagedCache(state["k_pool"], state["v_pool"])
    return state


# ---- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    return {"append": _append, "decode": _decode, "prompt": _prompt, "sample": _sample}[kind](state)


def _own(kind, s):
    from rpgbarengine_amd import serving
    if kind == "append":
        serving.append(s["cache"], s["table"], s["lens"], s["starts"], s["k"], s["v"], q=s["q"], q_out=s["q_out"],
                       q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rope=s["rope"])
        return s["q_out"], s["k_pool"], s["v_pool"]
    if kind == "decode":
        return serving.decode_attention(s["q"], s["cache"], s["table"], s["lens"], out=s["out"])
    if kind == "prompt":
        return serving.prompt_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], out=s["out"])
    return serving.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _places(s, tokens):
    """The sequence and the position of every new token."""
    t = torch.arange(tokens, device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:], t.to(torch.int32), right=True)
    return seq, s["lens"][seq] - s["starts"][seq + 1] + t


def _append(s):
    page, dtype = s["case"]["page"], s["k_pool"].dtype
    seq, pos = _places(s, s["k"].shape[0])
    half = s["case"]["dim"] // 2
    c, sn = s["rope"][pos, None, :half], s["rope"][pos, None, half:]

    def turned(x, gain):
        x = x.float()
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * gain
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * sn, b * c + a * sn], -1).to(dtype)

    at = s["table"][seq, torch.div(pos, page, rounding_mode="floor")].long()
    s["k_pool"][at, :, pos % page] = turned(s["k"], s["k_norm"])
    s["v_pool"][at, :, pos % page] = s["v"]
    return turned(s["q"], s["q_norm"]), s["k_pool"], s["v_pool"]


def _rows(pool, table):
    """The sequences' cache rows one behind the other, in 32 bits: [sequences, kv heads, positions, dim]."""
    x = pool[table.clamp(min=0).long()].float()
    return x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pool.shape[1], -1, pool.shape[3]).contiguous()


def _weights(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _decode(s):
    kv, dim = s["case"]["kv"], s["case"]["dim"]
    k, v = _rows(s["k_pool"], s["table"]), _rows(s["v_pool"], s["table"])
    q = s["q"].float().reshape(len(s["lens"]), kv, -1, dim) / math.sqrt(dim)
    seen = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None, None, None]
    p = _weights(torch.matmul(q, k.transpose(2, 3).contiguous()), seen)
    return torch.matmul(p, v).reshape(s["q"].shape).to(s["q"].dtype)


def _prompt(s):
    kv, dim, most = s["case"]["kv"], s["case"]["dim"], s["longest"]
    k, v = _rows(s["k_pool"], s["table"]), _rows(s["v_pool"], s["table"])
    n, heads = s["q"].shape[:2]
    g, seqs = heads // kv, len(s["lens"])
    at = (s["starts"][:-1, None] + torch.arange(most, device=k.device)).clamp(max=n - 1)
    q = s["q"][at].float().reshape(seqs, most, kv, g, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, g * most, dim)
    scores = torch.matmul(q / math.sqrt(dim), k.transpose(2, 3).contiguous()).reshape(seqs, kv, g, most, -1)
    first = s["lens"] - (s["starts"][1:] - s["starts"][:-1])
    pos = first[:, None] + torch.arange(most, device=k.device)
    p = _weights(scores, torch.arange(k.shape[2], device=k.device) <= pos[:, None, None, :, None])
    o = torch.matmul(p.reshape(seqs, kv, g * most, -1), v).reshape(seqs, kv, g, most, dim)
    seq, where = _places(s, n)
    return o[seq, :, :, where - first[seq]].reshape(s["q"].shape).to(s["q"].dtype)


def _sample(s):
    x = s["logits"].double()
    vocab = x.shape[1]
    top = x.max(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    w = torch.exp((x - top.values) / torch.where(t > 0, t, 1.0))
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    ordered = w.gather(1, order)
    k = s["top_k"].long()[:, None]
    k = torch.where((k > 0) & (k < vocab), k, vocab)
    ordered = ordered * (torch.arange(vocab, device=x.device) < k)
    cum = ordered.cumsum(1)
    p = s["top_p"].double()[:, None]
    stay = (ordered > 0) & (cum - ordered < torch.where((p > 0) & (p < 1), p, 2.0) * cum[:, -1:])
    stay &= ordered >= s["min_p"].double()[:, None].clamp(max=1.0)
    w = w * torch.zeros_like(stay).scatter(1, order, stay)
    cdf = w.cumsum(1)
    draw = (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(1, keepdim=True)
    last = vocab - 1 - (w > 0).flip(1).to(torch.uint8).argmax(1, keepdim=True)
    token = torch.where(t > 0, torch.minimum(draw, last), top.indices)
    logprob = torch.where(t > 0, torch.log(w.gather(1, token) / cdf[:, -1:]), 0.0)
    return token[:, 0].int(), logprob[:, 0].float()


# ---- what a pass cannot do without


def work(case):
    size = BYTES[case["type"]]
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}  # difference, scale, exponential, sum
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, new = _lengths(case)
    tokens, tables = sum(new), sum(4 * -(-n // case["page"]) + 8 for n in lens)
    if case["kind"] == "append":
        # keys, values and queries in and out; a rotation row for each position
        positions = len({p for n, m in zip(lens, new) for p in range(n - m, n)})
        return {"bytes": 2 * tokens * (heads + 2 * kv) * dim * size + positions * dim * 4 + 8 * dim + tables,
                "flops": tokens * (heads + kv) * dim * 7}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
    return {"bytes": 2 * sum(lens) * kv * dim * size + 2 * tokens * heads * dim * size + tables,
            "flops": 4 * pairs * heads * dim}


# ---- the operators' definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return [None, _exact_sample(s)]
    lens, new = _lengths(case)
    dim, page = case["dim"], case["page"]
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    q, at = s["q"].double(), 0
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if case["kind"] == "append":
        rope = s["rope"].double()
        for i, (n, m) in enumerate(zip(lens, new)):
            pos = torch.arange(n - m, n, device=q.device)
            turn = torch.complex(rope[pos, :dim // 2], rope[pos, dim // 2:])[:, None]

            def turned(x, gain):
                x = x[at:at + m].double()
                x = x / (x.square().sum(-1, keepdim=True) / dim + EPS).sqrt() * gain.double()
                z = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)

            out[at:at + m] = turned(s["q"], s["q_norm"])
            pages, rows = s["table"][i].long()[pos // page], pos % page
            k_pool[pages, :, rows] = turned(s["k"], s["k_norm"])
            v_pool[pages, :, rows] = s["v"][at:at + m].double()
            at += m
        return [out, k_pool, v_pool]
    group = case["heads"] // case["kv"]
    for i, (n, m) in enumerate(zip(lens, new)):
        pages = s["table"][i, : -(-n // page)].long()
        pos = torch.arange(n - m, n, device=q.device)[:, None]
        hidden = torch.arange(n, device=q.device)[None, :] > pos
        for h in range(case["heads"]):
            keys = k_pool[pages, h // group].reshape(-1, dim)[:n]
            values = v_pool[pages, h // group].reshape(-1, dim)[:n]
            scores = torch.mm(q[at:at + m, h].contiguous(), keys.t().contiguous()) * dim ** -0.5
            p = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1)
            out[at:at + m, h] = torch.mm(p, values)
        at += m
    return out


def _exact_sample(s):
    """The log-probabilities of the tokens drawn, row by row."""
    got = []
    for i in range(s["logits"].shape[0]):
        x = s["logits"][i].double()
        t, u = float(s["temperature"][i]), float(s["u"][i])
        if not t > 0:
            got.append(0.0)
            continue
        p = torch.softmax(x / t, 0)
        order = torch.argsort(x, descending=True, stable=True)
        k, top_p, min_p = int(s["top_k"][i]), float(s["top_p"][i]), float(s["min_p"][i])
        if 0 < k < len(order):
            order = order[:k]
        ranked = p[order] / p[order].sum()
        n = len(order)
        if 0 < top_p < 1:
            n = min(n, int((ranked.cumsum(0) < top_p).sum()) + 1)
        n = min(n, int((ranked >= min_p * ranked[0]).sum()))
        kept = order[:max(1, n)].sort().values
        cdf = p[kept].cumsum(0) / p[kept].sum()
        at = min(int((cdf <= u).sum()), len(kept) - 1)
        got.append(float(torch.log(p[kept[at]] / p[kept].sum())))
    return torch.tensor(got, dtype=torch.float64)
