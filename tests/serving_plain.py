"""The serving operators' definitions in float64 on the CPU, and the error that
their kernels may make, derived from their arithmetic."""

import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}  # half the smallest step


def turned(x, gain, eps, rope_row):
    """(norm and rotation of x [heads, dim], sum of the two products' magnitudes)."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    if rope_row is None:
        return x, x.abs()
    half = x.shape[-1] // 2
    c, s = rope_row[:half].double(), rope_row[half:].double()
    a, b = x[..., :half], x[..., half:]
    return (torch.cat([a * c - b * s, b * c + a * s], -1),
            torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1))


def turned_bound(dtype, size, magnitude):
    """A sum of at most 32 squares a lane in fp32 and 5 adds across lanes, halved by
    the root; root, division, two products, the rotation's product and fma: under
    32 roundings of 2^-24; then the rounding to the type."""
    return 32 * 2.0 ** -24 * magnitude + EPS[dtype] * size.abs() + TINY[dtype]


def sequence_rows(pool, table_row, n):
    """[kv, n, dim] float64 rows of a sequence's positions and which of them exist."""
    pages, _, page, _ = pool.shape
    rows, there = [], []
    for p in range(n):
        at = int(table_row[p // page])
        ok = 0 <= at < pages
        rows.append(pool[at if ok else 0, :, p % page])
        there.append(ok)
    if not rows:
        return torch.zeros(pool.shape[1], 0, pool.shape[3], dtype=torch.float64), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows, 1).double(), torch.tensor(there)


def attention(q, k, v, seen, scale, dtype):
    """q [heads, dim] over k, v [kv, n, dim] where seen [n]: (out, bound), float64."""
    heads, dim = q.shape
    group = heads // k.shape[0]
    out, bound = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    if not bool(seen.any()):
        return out, bound
    for h in range(heads):
        kk, vv = k[h // group][seen], v[h // group][seen]
        qq = q[h].double()
        s = kk @ qq * scale
        p = torch.softmax(s, 0)
        out[h] = (p[:, None] * vv).sum(0)
        mass = (p[:, None] * vv.abs()).sum(0)
        # A score's dot product in fp32 (dim products, added in any order), its
        # scaling and the difference from the maximum; 2^x; sums over the keys and
        # the ranges' joins; then the weights' rounding to 16 bits.
        ds = float((kk.abs() @ qq.abs()).max()) * scale * (dim + 4) * 2.0 ** -24 + float(s.abs().max()) * 2.0 ** -21
        rel = math.expm1(2 * ds) + (len(s) + 16) * 2.0 ** -23
        if dtype != torch.float32:
            # An f16 weight is held times 2^7 at the least; below the type's normal
            # range it is off by at most 2^-25 absolutely; the largest weight is 1.
            rel += EPS[dtype]
            if dtype == torch.float16:
                bound[h] += 2.0 ** -32 * vv.abs().sum(0) * float(p.max())
        bound[h] += rel * mass
    return out, bound + EPS[dtype] * (out.abs() + bound) + TINY[dtype]


def sample(x, u, t, k, p, m):
    """(token, log of its probability) of one row, float64."""
    x = torch.where(x.isnan(), torch.tensor(-math.inf, dtype=torch.float64), x.double())
    top = float(x.max())
    if top == -math.inf:
        return -1, -math.inf
    best = int((x == top).nonzero()[0])
    if not t > 0:
        return best, 0.0
    d = torch.where(x == top, 0.0, top - x)
    w = torch.exp(-d / t)
    order = torch.sort(-x, stable=True).indices
    n = len(order) if not 0 < k < len(order) else k
    ranked = w[order][:n]
    if 0 < p < 1:
        before = ranked.cumsum(0) - ranked
        n = int((before < p * ranked.sum()).sum())
    if m > 0:
        n = min(n, int((ranked[:n] >= min(m, 1.0)).sum()))
    kept = torch.zeros_like(w)
    kept[order[:n]] = w[order[:n]]
    cdf = kept.cumsum(0)
    u = min(max(u, 0.0), 1.0)
    hits = (cdf > u * cdf[-1]).nonzero()
    token = int(hits[0]) if len(hits) else int(kept.nonzero()[-1])
    return token, float(torch.log(kept[token] / cdf[-1]))
