"""Timed cases of what a server of many characters adds to a decode step: a
key-value cache held in 8 bits, attention of sessions that share a long prefix,
and the edits of logits before the sampler.

A case is a dict of plain values with a "kind":

* ``append`` -- the new tokens of every sequence: keys (RMS-normed per head and
  rotated) and values go into the pages of an 8-bit cache, each row as codes and a
  scale; the queries are normed and rotated.
* ``read`` -- the last positions of sequences out of an 8-bit cache, as rows.
* ``decode`` -- attention of one new token per sequence over an 8-bit cache.
* ``prompt`` -- causal attention of packed new tokens over an 8-bit cache.
* ``shared`` -- one new token per sequence, the sequences in groups whose first
  positions lie in the same pages; a cache of any kind.
* ``edit`` -- logits of many rows: penalties for the tokens so far, biases, the
  bits of a grammar's mask.

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
CODES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
LARGEST = {"e4m3": 448.0, "i8": 127.0}  # of a code
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 151936
EPS = 1e-6


def listed():
    return [
        # Eight players' sessions, a decode step's token each, rows in the
        # engine's own type. The smallest call.
        {"name": "append 8 tokens e4m3 f32", "kind": "append", "codes": "e4m3", "type": "f32", "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "seqs": 8, "len_lo": 1025, "len_hi": 1152, "new_lo": 1, "new_hi": 1, "mix": 1},
        # Prompts of a full server, some of them the next part of a longer
        # document.
        {"name": "append prompts e4m3 bf16", "kind": "append", "codes": "e4m3", "type": "bf16", "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "seqs": 12, "len_lo": 300, "len_hi": 4096, "new_lo": 77, "new_hi": 1500, "mix": 2},
        # One session on its way back into the engine's own cache.
        {"name": "read 1 session i8 f32", "kind": "read", "codes": "i8", "type": "f32", "heads": 16, "kv": 8,
         "dim": 128, "page": 16, "seqs": 1, "len_lo": 1100, "len_hi": 1100, "new_lo": 1100, "new_hi": 1100, "mix": 3},
        # Sessions of a server that moves to another one.
        {"name": "read 24 sessions e4m3 bf16", "kind": "read", "codes": "e4m3", "type": "bf16", "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "seqs": 24, "len_lo": 500, "len_hi": 4096, "new_lo": 500, "new_hi": 4096, "mix": 4},
        # Eight sessions of the small model behind a prompt of 1024 tokens.
        {"name": "decode 8 i8 f16", "kind": "decode", "codes": "i8", "type": "f16", "heads": 16, "kv": 8, "dim": 128,
         "page": 16, "seqs": 8, "len_lo": 1025, "len_hi": 1152, "mix": 5},
        # A busy server: conversations of every length.
        {"name": "decode 64 ragged e4m3 bf16", "kind": "decode", "codes": "e4m3", "type": "bf16", "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "seqs": 64, "len_lo": 200, "len_hi": 12000, "mix": 6},
        # The next messages of a few running conversations, together.
        {"name": "prompt turns i8 f16", "kind": "prompt", "codes": "i8", "type": "f16", "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "seqs": 6, "len_lo": 400, "len_hi": 1703, "new_lo": 12, "new_hi": 203, "mix": 7},
        # Documents that fill their contexts.
        {"name": "prompt documents e4m3 bf16", "kind": "prompt", "codes": "e4m3", "type": "bf16", "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "seqs": 4, "len_lo": 2900, "len_hi": 4096, "new_lo": 2900, "new_hi": 4096, "mix": 8},
        # Eight characters of one world, its description the prefix, in the
        # engine's own cache type.
        {"name": "shared 8 sessions f32", "kind": "shared", "codes": "", "type": "f32", "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "groups": 1, "seqs": 8, "shared_lo": 2000, "shared_hi": 2000, "len_lo": 60,
         "len_hi": 500, "mix": 9},
        # A server of three worlds.
        {"name": "shared 96 sessions bf16", "kind": "shared", "codes": "", "type": "bf16", "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "groups": 3, "seqs": 96, "shared_lo": 4000, "shared_hi": 12000, "len_lo": 100,
         "len_hi": 2500, "mix": 10},
        # Eight sessions at the chat defaults with a repetition penalty.
        {"name": "edit 8 rows f32", "kind": "edit", "type": "f32", "vocab": VOCAB, "rows": 8, "history": 1100,
         "biases": 0, "masked": 0.0, "mix": 11},
        # A full server: some rows bound to a grammar (tool calls), some biased.
        {"name": "edit 192 rows bf16", "kind": "edit", "type": "bf16", "vocab": VOCAB, "rows": 192, "history": 4096,
         "biases": 32, "masked": 0.3, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt", "shared", "shared", "shared", "edit"])
    rows = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "edit":
        return {"kind": kind, "type": rows, "vocab": _log(rng, 1000, VOCAB), "rows": _log(rng, 1, 128),
                "history": _log(rng, 1, 8000), "biases": rng.choice([0, 1, 40, 300]),
                "masked": rng.choice([0.0, 0.2, 1.0]), "mix": rng.randrange(1 << 20)}
    kv = rng.choice([1, 2, 4, 8, 8])
    codes = rng.choice(["e4m3", "i8"])
    if kind == "append":  # (whole numbers would have to be equal: e4m3 codes are returned as values)
        codes = "e4m3"
    if kind == "shared":
        codes = rng.choice(["", "", codes])
    case = {"kind": kind, "codes": codes, "type": rows, "heads": kv * rng.choice([1, 2, 4, 4, 5, 8]), "kv": kv,
            "dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 256])}
    if kind == "decode":
        hi = _log(rng, 1, 16000)
        case |= {"seqs": _log(rng, 1, min(64, max(1, 400000 // hi))), "len_lo": max(1, int(hi * rng.uniform(0.05, 1))),
                 "len_hi": hi}
    elif kind == "shared":
        shared, hi = _log(rng, 16, 12000), _log(rng, 1, 2500)
        groups = rng.choice([1, 1, 2, 5])
        most = min(96, max(2, 500000 // (shared + hi)))
        case |= {"groups": min(groups, most), "seqs": max(groups, _log(rng, 2, most)),
                 "shared_lo": max(1, int(shared * rng.uniform(0.2, 1))), "shared_hi": shared,
                 "len_lo": max(1, int(hi * rng.uniform(0.05, 1))), "len_hi": hi}
    else:
        new = _log(rng, 1, 2500 if kind == "prompt" else 3000)
        hi = min(4096, new + rng.choice([0, _log(rng, 1, 2500)]))
        case |= {"seqs": _log(rng, 1, min(24, max(1, 9000 // hi))), "len_lo": max(new, int(hi * rng.uniform(0.2, 1))),
                 "len_hi": hi, "new_lo": max(1, int(new * rng.uniform(0.1, 1))), "new_hi": new}
    return case | {"mix": rng.randrange(1 << 20)}


# ---- inputs


def _lengths(case):
    """(positions that each sequence's cache holds after the call, its new tokens
    among them and the pages that it shares; its new tokens)."""
    rng = random.Random(case["mix"])
    lens = [_log(rng, case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    if case["kind"] == "shared":
        _, shared, of = _groups(case)
        lens = [n + shared[g] for n, g in zip(lens, of)]
    if "new_lo" not in case:
        return lens, [1] * len(lens)
    return lens, [min(n, _log(rng, case["new_lo"], case["new_hi"])) for n in lens]


def _groups(case):
    """(the groups' first sequences and their end, the positions that each shares,
    each sequence's group)."""
    rng = random.Random(case["mix"] + 1)
    n, seqs, page = case["groups"], case["seqs"], case["page"]
    cuts = sorted(rng.sample(range(1, seqs), n - 1))
    starts = [0] + cuts + [seqs]
    # whole pages: the rest of a prefix is every sequence's own
    shared = [_log(rng, case["shared_lo"], case["shared_hi"]) // page * page for _ in range(n)]
    return starts, shared, [g for g in range(n) for _ in range(starts[g], starts[g + 1])]


def _edits(case):
    """The tokens so far of each row and how many of them are its prompt; the rows
    that a mask binds."""
    rng = random.Random(case["mix"])
    lens = [_log(rng, max(1, case["history"] // 20), case["history"]) for _ in range(case["rows"])]
    return lens, [int(n * rng.uniform(0, 0.9)) for n in lens], [rng.random() < case["masked"] for _ in lens]


def _device():
    return torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")


def _quantised(x, codes):
    """(codes, scales) of rows, as the cache holds them. The quotients in 64 bits:
    with 16-bit rows many of them lie midway between two codes."""
    most = x.abs().amax(-1)
    scaled = (x.double() * LARGEST[codes] / most.double()[..., None]).float()
    return (scaled.round() if codes == "i8" else scaled).to(CODES[codes]), most / LARGEST[codes]


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    if case["kind"] == "edit":
        return _prepare_edit(case, gen, dev)
    dtype = TYPES[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * by).to(dtype)

    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, new = _lengths(case)
    pages = [-(-n // page) for n in lens]
    head = [0] * len(lens)  # pages of a sequence that are its group's
    groups, shared, of = _groups(case) if case["kind"] == "shared" else ([], [], [])
    if groups:
        head = [shared[g] // page for g in of]
    used = sum(pages) - sum(head) + sum(n // page for n in shared)
    # A pool with some pages to spare, handed out in no order; the table's
    # entries behind a sequence's last page hold -1.
    pool = used + 1 + used // 16
    order = torch.randperm(pool, generator=gen, device=dev)[:used].to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=dev)
    at = 0
    for g, n in enumerate(shared):
        table[groups[g]:groups[g + 1], : n // page] = order[at:at + n // page]
        at += n // page
    for i, (h, n) in enumerate(zip(head, pages)):
        table[i, h:n] = order[at:at + n - h]
        at += n - h
    tokens = sum(new)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    ints = dict(dtype=torch.int32, device=dev)
    state = {"case": case, "table": table, "lens": torch.tensor(lens, **ints), "longest": max(new), "tokens": tokens,
             "starts": torch.tensor(starts, **ints)}
    if groups:
        state |= {"groups": torch.tensor(groups, **ints), "shared": torch.tensor(shared, **ints)}
    for name in ("k", "v"):
        if not case["codes"]:
            state[name + "_pool"] = normal(pool, kv, page, dim)
        elif case["kind"] == "append":
            state[name + "_pool"] = torch.zeros(pool, kv, page, dim, device=dev).to(CODES[case["codes"]])
            state[name + "_scale"] = torch.zeros(pool, kv, page, device=dev)
        else:
            rows = torch.randn(pool, kv, page, dim, generator=gen, device=dev)
            if name == "k":  # a model's keys have dimensions that stand out
                rows[..., :: dim // 4] *= 3.0
            state[name + "_pool"], state[name + "_scale"] = _quantised(rows, case["codes"])
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
    elif case["kind"] == "read":
        state |= {n: torch.empty(tokens, kv, dim, dtype=dtype, device=dev) for n in ("k_out", "v_out")}
    else:
        state["q"] = normal(tokens, heads, dim, by=1.5)
        state["out"] = torch.empty(tokens, heads, dim, dtype=dtype, device=dev)
    if own:
        from rpgbarengine_amd import serving
        if case["codes"]:
            state["cache"] = serving.QuantCache(state["k_pool"], state["v_pool"], state["k_scale"], state["v_scale"])
        else:
            state["cache"] = serving.PagedCache(state["k_pool"], state["v_pool"])
    return state


def _prepare_edit(case, gen, dev):
    rows, vocab, biases = case["rows"], case["vocab"], case["biases"]
    lens, prompts, bound = _edits(case)
    x = torch.randn(rows, vocab, generator=gen, device=dev) * 2.5
    # Text repeats itself: token numbers crowd at the low end, as a tokenizer's
    # frequent ones do.
    draw = torch.rand(rows, max(lens), generator=gen, device=dev)
    history = ((draw ** 4) * vocab).to(torch.int32).clamp_(max=vocab - 1)

    def each(choices):
        return torch.tensor(choices, device=dev)[torch.randint(0, len(choices), (rows,), generator=gen, device=dev)]

    ints = dict(dtype=torch.int32, device=dev)
    state = {"case": case, "logits": x.to(TYPES[case["type"]]), "history": history,
             "history_lens": torch.tensor(lens, **ints), "prompts": torch.tensor(prompts, **ints),
             "repetition": each([1.0, 1.1, 1.3]), "presence": each([0.0, 0.4]), "frequency": each([0.0, 0.2, 0.05]),
             "out": torch.empty(rows, vocab, dtype=TYPES[case["type"]], device=dev),
             "bias_ids": None, "bias": None, "mask": None, "mask_rows": None}
    if biases:
        # numbers of a row are distinct; shorter lists are filled up with -1
        ids = torch.rand(rows, vocab, generator=gen, device=dev).topk(biases, 1).indices.to(torch.int32)
        spare = torch.rand(rows, biases, generator=gen, device=dev) < 0.3
        state["bias_ids"] = ids.masked_fill(spare, -1)
        state["bias"] = torch.randn(rows, biases, generator=gen, device=dev) * 4
    if any(bound):
        # One mask for each row that a grammar binds: few tokens in most of
        # its states, most of them inside a string.
        n = sum(bound)
        words = -(-vocab // 32)
        bits = torch.randint(-(1 << 31), 1 << 31, (3, n, words), generator=gen, device=dev)
        loose = torch.rand(n, 1, generator=gen, device=dev) < 0.4
        state["mask"] = torch.where(loose, bits[0] | bits[1] | bits[2], bits[0] & bits[1] & bits[2]).to(torch.int32)
        of, at = [], 0
        for b in bound:
            of.append(at if b else -1)
            at += b
        state["mask_rows"] = torch.tensor(of, **ints)
    return state


# ---- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    return {"append": _append, "read": _read, "decode": _decode, "prompt": _prompt, "shared": _decode,
            "edit": _edit}[kind](state)


def _own(kind, s):
    from rpgbarengine_amd import serving
    if kind == "append":
        serving.append(s["cache"], s["table"], s["lens"], s["starts"], s["k"], s["v"], q=s["q"], q_out=s["q_out"],
                       q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rope=s["rope"])
        return s["q_out"], s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"]
    if kind == "read":
        return serving.read_rows(s["cache"], s["table"], s["lens"], s["starts"], k_out=s["k_out"], v_out=s["v_out"])
    if kind == "decode":
        return serving.decode_attention(s["q"], s["cache"], s["table"], s["lens"], out=s["out"])
    if kind == "prompt":
        return serving.prompt_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], out=s["out"])
    if kind == "shared":
        return serving.shared_attention(s["q"], s["cache"], s["table"], s["lens"], s["groups"], s["shared"], out=s["out"])
    return serving.edit_logits(s["logits"], s["history"], s["history_lens"], prompts=s["prompts"],
                               repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                               bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], mask_rows=s["mask_rows"],
                               out=s["out"])


def _places(s, tokens):
    """The sequence and the position of every new token."""
    t = torch.arange(tokens, device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:], t.to(torch.int32), right=True)
    return seq, s["lens"][seq] - s["starts"][seq + 1] + t


def _append(s):
    page, dtype = s["case"]["page"], TYPES[s["case"]["type"]]
    seq, pos = _places(s, s["tokens"])
    half = s["case"]["dim"] // 2
    c, sn = s["rope"][pos, None, :half], s["rope"][pos, None, half:]

    def turned(x, gain):
        x = x.float()
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * gain
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * sn, b * c + a * sn], -1)

    at = s["table"][seq, torch.div(pos, page, rounding_mode="floor")].long()
    k, ks = _quantised(turned(s["k"], s["k_norm"]), s["case"]["codes"])
    v, vs = _quantised(s["v"].float(), s["case"]["codes"])
    s["k_pool"][at, :, pos % page], s["k_scale"][at, :, pos % page] = k, ks
    s["v_pool"][at, :, pos % page], s["v_scale"][at, :, pos % page] = v, vs
    return turned(s["q"], s["q_norm"]).to(dtype), s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"]


def _read(s):
    page, dtype = s["case"]["page"], TYPES[s["case"]["type"]]
    seq, pos = _places(s, s["tokens"])
    at = s["table"][seq, torch.div(pos, page, rounding_mode="floor")].long()

    def rows(name):
        return (s[name + "_pool"][at, :, pos % page].float() * s[name + "_scale"][at, :, pos % page, None]).to(dtype)

    return rows("k"), rows("v")


def _rows(s, name):
    """The sequences' cache rows one behind the other, in 32 bits: [sequences, kv heads, positions, dim]."""
    pool, table = s[name + "_pool"], s["table"].clamp(min=0).long()
    x = pool[table].float()
    if s["case"]["codes"]:
        x = x * s[name + "_scale"][table][..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pool.shape[1], -1, pool.shape[3]).contiguous()


def _weights(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _decode(s):
    kv, dim = s["case"]["kv"], s["case"]["dim"]
    k, v = _rows(s, "k"), _rows(s, "v")
    q = s["q"].float().reshape(len(s["lens"]), kv, -1, dim) / math.sqrt(dim)
    seen = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None, None, None]
    p = _weights(torch.matmul(q, k.transpose(2, 3).contiguous()), seen)
    return torch.matmul(p, v).reshape(s["q"].shape).to(s["q"].dtype)


def _prompt(s):
    kv, dim, most = s["case"]["kv"], s["case"]["dim"], s["longest"]
    k, v = _rows(s, "k"), _rows(s, "v")
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


def _edit(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(s["history"].shape[1], device=x.device)
    here = at < s["history_lens"][:, None]
    made = here & (at >= s["prompts"][:, None])
    ids = s["history"].long()
    seen = torch.zeros_like(x).scatter_add_(1, ids, here.float())
    count = torch.zeros_like(x).scatter_add_(1, ids, made.float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long()
        x = x.scatter_add(1, ids.clamp(min=0), torch.where(ids >= 0, s["bias"], 0.0))
    if s["mask"] is not None:
        bit = torch.arange(vocab, device=x.device)
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        allowed = (words[:, bit // 32] >> (bit % 32)) & 1
        x = x.masked_fill((allowed == 0) & (s["mask_rows"][:, None] >= 0), -math.inf)
    return x.to(s["logits"].dtype)


# ---- what a pass cannot do without


def work(case):
    size = BYTES[case["type"]]
    if case["kind"] == "edit":
        lens, _, bound = _edits(case)
        n, rows = case["rows"] * case["vocab"], case["rows"]
        return {"bytes": 2 * n * size + 4 * sum(lens) + rows * (24 + 8 * case["biases"]) + sum(bound) * (case["vocab"] // 8),
                "flops": 6 * n}  # a quotient, two penalties and their product, a bias, the mask
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, new = _lengths(case)
    tokens, tables = sum(new), sum(4 * -(-n // case["page"]) + 8 for n in lens)
    row = dim + 4 if case["codes"] else dim * size  # of the cache
    if case["kind"] == "append":
        # keys, values and queries in, queries out, codes and scales; a rotation row for each position
        positions = len({p for n, m in zip(lens, new) for p in range(n - m, n)})
        return {"bytes": tokens * ((2 * heads + 2 * kv) * dim * size + 2 * kv * row) + positions * dim * 4 + 8 * dim + tables,
                "flops": tokens * (heads + kv) * dim * 7 + tokens * 2 * kv * dim * 2}
    if case["kind"] == "read":
        return {"bytes": 2 * tokens * kv * (row + dim * size) + tables, "flops": 2 * tokens * kv * dim}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
    held = sum(lens)
    if case["kind"] == "shared":  # a group's common positions once
        starts, shared, of = _groups(case)
        held += sum(shared) - sum(shared[g] for g in of)
    return {"bytes": 2 * held * kv * row + 2 * tokens * heads * dim * size + tables, "flops": 4 * pairs * heads * dim}


# ---- the operators' definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "edit":
        return _exact_edit(s)
    lens, new = _lengths(case)
    dim, page = case["dim"], case["page"]
    pools = {}
    for name in ("k", "v"):
        pools[name] = s[name + "_pool"].double()
        if case["codes"] and case["kind"] != "append":
            pools[name] *= s[name + "_scale"].double()[..., None]
    if case["kind"] == "append":
        return _exact_append(case, s, lens, new, pools)
    at = 0
    if case["kind"] == "read":
        got = [torch.zeros(s["tokens"], case["kv"], dim, dtype=torch.float64, device=s["table"].device) for _ in "kv"]
        for i, (n, m) in enumerate(zip(lens, new)):
            pos = torch.arange(n - m, n, device=s["table"].device)
            for out, name in zip(got, "kv"):
                out[at:at + m] = pools[name][s["table"][i].long()[pos // page], :, pos % page]
            at += m
        return got
    q = s["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = case["heads"] // case["kv"]
    for i, (n, m) in enumerate(zip(lens, new)):
        pages = s["table"][i, : -(-n // page)].long()
        pos = torch.arange(n - m, n, device=q.device)[:, None]
        hidden = torch.arange(n, device=q.device)[None, :] > pos
        for h in range(case["heads"]):
            keys = pools["k"][pages, h // group].reshape(-1, dim)[:n]
            values = pools["v"][pages, h // group].reshape(-1, dim)[:n]
            scores = torch.mm(q[at:at + m, h].contiguous(), keys.t().contiguous()) * dim ** -0.5
            p = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1)
            out[at:at + m, h] = torch.mm(p, values)
        at += m
    return out


def _exact_append(case, s, lens, new, pools):
    dim, page, codes = case["dim"], case["page"], case["codes"]
    q = s["q"].double()
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    rope = s["rope"].double()
    scales = {name: s[name + "_scale"].double() for name in "kv"}

    def code(x):
        """The nearest value that 8 bits hold, even where two are as near."""
        if codes == "i8":
            return torch.round(x)
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # three bits behind the first
        return torch.round(x / step) * step

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
        for name, x in (("k", turned(s["k"], s["k_norm"])), ("v", s["v"][at:at + m].double())):
            scale = x.abs().amax(-1) / LARGEST[codes]
            pools[name][pages, :, rows] = code(x * LARGEST[codes] / x.abs().amax(-1, keepdim=True))
            scales[name][pages, :, rows] = scale
        at += m
    return [out, pools["k"], scales["k"], pools["v"], scales["v"]]


def _exact_edit(s):
    """Row by row, from lists."""
    x = s["logits"].double()
    vocab = x.shape[1]
    for i in range(x.shape[0]):
        n, prompt = int(s["history_lens"][i]), int(s["prompts"][i])
        ids = s["history"][i, :n].long()
        seen = torch.unique(ids)
        r = float(s["repetition"][i])
        x[i, seen] = torch.where(x[i, seen] > 0, x[i, seen] / r, x[i, seen] * r)
        made, times = torch.unique(ids[prompt:], return_counts=True)
        x[i, made] -= float(s["frequency"][i]) * times + float(s["presence"][i])
        if s["bias_ids"] is not None:
            use = s["bias_ids"][i] >= 0
            x[i, s["bias_ids"][i][use].long()] += s["bias"][i][use].double()
        if s["mask"] is not None and int(s["mask_rows"][i]) >= 0:
            words = s["mask"][int(s["mask_rows"][i])].long()
            bits = (words[:, None] >> torch.arange(32, device=x.device)) & 1
            x[i, bits.reshape(-1)[:vocab] == 0] = -math.inf
    return x
