"""Serving operators in the batches of a busy server: as many sequences as fill the
card, whose ranges have a least length, tables far wider than their sequences, and
appends and reads of thousands of tokens."""

import ctypes

import pytest
import torch

from rpgbarengine_amd import serving
from serving_plain import attention as plain_attention
from test_gpu_serving import DTYPES, Batch, close
from test_gpu_serving_codes import CODES, attention, empty_cache, ident, on_cpu, random_cache, weight_bits

pytestmark = pytest.mark.gpu


def gathered(pool, table_row, n, page):
    """[kv, n, ...] of a sequence's positions, and which of them are there."""
    at = table_row[: -(-n // page)].long()
    there = ((at >= 0) & (at < pool.shape[0])).repeat_interleave(page)[:n]
    rows = pool[at.clamp(0, pool.shape[0] - 1)].transpose(0, 1)
    return rows.reshape(pool.shape[1], -1, *pool.shape[3:])[:, :n], there


def expected(b, cache, q, i):
    """(out, bound) of the token of sequence i, its positions all seen: a cache of codes
    (on_cpu) or of rows (k, v)."""
    n, scale = b.lens[i], b.dim ** -0.5
    if len(cache) == 2:
        (k, there), (v, _) = (gathered(x, b.table[i], n, b.page) for x in cache)
        return plain_attention(q[i], k.double(), v.double(), there, scale, b.dtype)
    (k, there), (v, _), (ks, _), (vs, _) = (gathered(x, b.table[i], n, b.page) for x in cache)
    return attention(q[i], k, v, ks, vs, there, scale, b.dtype, weight_bits(b.dtype, False))


def with_work(b, q, cache, table, lens, shared=None):
    """(out, work) of a call at the C entry whose work memory holds NaN before it: a range
    that is joined and was not written makes a NaN."""
    L, quant = serving._lib(), isinstance(cache, serving.QuantCache)
    seqs, n_seqs, pages = serving._seqs(cache, table, lens, None, 0)
    out = torch.full_like(q, 5.0)
    heads, kind = q.shape[1], serving._TYPES[b.dtype]
    groups, rows = (), (serving._rows(q, "q", cache, b.dtype), serving._rows(out, "out", cache, b.dtype), heads)
    if shared is not None:
        starts, common = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in shared)
        groups = (serving._GROUPS.pack(starts.data_ptr(), common.data_ptr(), len(common)),)
        n = (len(common),)
        need = (L.rpg_hip_quant_shared_work(cache._packed(), seqs, *n, kind, heads) if quant
                else L.rpg_hip_paged_shared_work(cache._packed(), seqs, *n, heads))
        f = L.rpg_hip_quant_shared if quant else L.rpg_hip_paged_shared
    else:
        need = (L.rpg_hip_quant_work(cache._packed(), seqs, kind, heads, 0) if quant
                else L.rpg_hip_paged_work(cache._packed(), seqs, heads, 0))
        f = L.rpg_hip_quant_decode if quant else L.rpg_hip_paged_decode
    assert need > 0
    work = torch.full((need // 4,), torch.nan, device="cuda")
    assert f(cache._packed(), seqs, *groups, *((kind,) if quant else ()), *rows, ctypes.c_float(b.dim ** -0.5), work.data_ptr(), need,
             torch.cuda.current_stream().cuda_stream) == 0
    return out, work


def ranges(b, work, heads):
    """The ranges that each row's positions were cut into, by what was written."""
    rows = len(b.lens) * heads
    splits = len(work) // (rows * (b.dim + 2))
    return (~work[:2 * rows * splits].isnan()).view(len(b.lens), heads, splits, 2).all(-1).sum(-1).cpu()


EDGES = [511, 512, 513, 0, 1023, 1024, 1025, 2049, 1, 2048, 2560, 4100, 0, 130]


def repeated(seqs, dtype, seed, extra_pages, common=0):
    """A batch of `seqs` sequences whose lengths lie at the borders of ranges, `common`
    positions behind; every fourteenth has the same pages, one position less each time."""
    b = Batch([n + common for n in EDGES], [1] * 14, dtype, 8, 64, 16, 8, seed=seed, extra_pages=extra_pages)
    b.table = b.table.repeat(-(-seqs // 14), 1)[:seqs].contiguous()
    b.lens = [max(0, EDGES[i % 14] - i // 14) for i in range(seqs)]
    return b


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("seqs,width", [(5, 17000), (18, 5000), (40, 5000), (70, 9000)])
def test_decode(codes, dtype, seqs, width):
    """40, 144, 320 and 560 workgroups of whole sequences on 8 key heads: less than one to
    two compute units, one to two, one to one and more; ranges of 384 and of 1024
    positions at the least, in tables for more than any sequence has."""
    b = repeated(seqs, dtype, 41, (width - 4100) // 16)
    q = b.normal(seqs, 8, 64, by=0.3)
    cache = random_cache(b, codes)
    table, lens = b.table.cuda(), torch.tensor(b.lens, dtype=torch.int32, device="cuda")
    out, _ = with_work(b, q.cuda(), cache, table, lens)
    held = on_cpu(cache)
    for i in (*range(min(14, seqs)), seqs - 1):
        close(out[i], *expected(b, held, q, i))
    assert torch.equal(serving.decode_attention(q.cuda(), cache, table, lens), out)


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("seqs,n", [(8, 1090), (1, 1000), (4, 2050)])
def test_a_wide_table_cuts_as_a_narrow_one(codes, dtype, seqs, n):
    """Sequences that do not fill the card, in a table of their own width, in one for 8192
    and in one for 131072 positions: a row is cut into as many ranges or more."""
    got = []
    for width in (n, 8192, 131072):
        b = Batch([n] * seqs, [1] * seqs, dtype, 8, 64, 16, 8, seed=42, extra_pages=(width - n) // 16)
        q = b.normal(seqs, 8, 64, by=0.3).cuda()
        _, table, lens, _ = b.gpu()
        out, work = with_work(b, q, random_cache(b, codes), table, lens)
        assert bool(out.isfinite().all())
        got.append(ranges(b, work, 8))
    assert int(got[0].min()) >= 3 and all(bool((x >= got[0]).all()) for x in got)


@pytest.mark.parametrize("kind", ["rows", *CODES], ids=lambda x: x if x == "rows" else ident(x))
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("seqs", [40, 70])
def test_shared(kind, dtype, seqs):
    """Own ranges of 512 positions at the least, behind 640, 1104 and no common ones."""
    common = [640, 1104]
    starts = [0, seqs // 2, seqs - 3]
    b = repeated(seqs, dtype, 43, 200, common[1])
    for g in range(2):
        for i in range(starts[g], starts[g + 1]):
            b.lens[i] += common[g] if b.lens[i] else 0
            b.table[i, :common[g] // 16] = b.table[starts[g], :common[g] // 16]
    q = b.normal(seqs, 8, 64, by=0.3)
    table, lens = b.table.cuda(), torch.tensor(b.lens, dtype=torch.int32, device="cuda")
    cache = serving.PagedCache(b.k.cuda(), b.v.cuda()) if kind == "rows" else random_cache(b, kind)
    held = (b.k, b.v) if kind == "rows" else on_cpu(cache)
    out, _ = with_work(b, q.cuda(), cache, table, lens, (starts, common))
    for i in (*range(14), starts[1] - 1, *range(starts[1], starts[1] + 8), *range(starts[2] - 1, seqs)):
        close(out[i], *expected(b, held, q, i))
    groups, shared = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, common))
    assert torch.equal(serving.shared_attention(q.cuda(), cache, table, lens, groups, shared), out)


# ---- thousands of tokens: the same bits as a few at a time


def pieces(b, before):
    """(sequence, its first packed row, its new tokens, how many of them are behind) of
    calls of at most 97 tokens."""
    for i, m in enumerate(b.new):
        for a in range(0, m, 97):
            yield i, before + int(b.starts[i]) + a, min(97, m - a), max(0, m - a - 97)


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 6, 3, 16), (64, 15, 5, 64), (128, 32, 8, 32)])
def test_append(codes, dtype, dim, heads, kv, page):
    """Heads that fill their units and that do not; rows in front of the first sequence
    and behind the last, sequences of no new token and of one, more new tokens than
    positions, an unnamed page, positions past the rotation's."""
    b = Batch([900, 40, 333, 1, 64, 3], [700, 0, 333, 1, 64, 7], dtype, kv, dim, page, heads, seed=44)
    b.table[2, 1] = -1
    before, behind = 3, 2
    n = before + b.tokens + behind
    assert b.tokens >= 1024
    qkv = b.normal(n, heads + 2 * kv, dim, by=3.0).cuda()
    gains = [(1 + 0.2 * torch.randn(dim, generator=b.gen)).cuda() for _ in "qk"]
    ang = torch.rand(890, dim // 2, generator=b.gen) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    _, table, lens, starts = b.gpu()
    kw = dict(q_norm=gains[0], k_norm=gains[1], eps=1e-5, rope=rope)
    whole, parts = empty_cache(b, codes), empty_cache(b, codes)
    outs = [torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    serving.append(whole, table, lens, starts + before, k, v, q=q, q_out=outs[0], **kw)
    for i, t, m, left in pieces(b, before):
        rows = slice(t, t + m)
        serving.append(parts, table[i:i + 1], lens[i:i + 1] - left, torch.tensor([0, m], dtype=torch.int32, device="cuda"),
                       k[rows], v[rows], q=q[rows], q_out=outs[1][rows], **kw)
    assert torch.equal(outs[0], outs[1])
    for x, y in ((whole.k, parts.k), (whole.v, parts.v)):
        assert torch.equal(x.view(torch.int8), y.view(torch.int8))
    assert torch.equal(whole.k_scale, parts.k_scale) and torch.equal(whole.v_scale, parts.v_scale)
    written = whole.k_scale != 7.0
    assert int(written[:, 0].sum()) == b.tokens - page - 10 - 4  # the unnamed page, 890 .. 899, four without a place
    assert bool((outs[0][:before] == 7).all()) and bool((outs[0][n - behind:] == 7).all())


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,kv,page", [(128, 3, 16), (64, 5, 64), (128, 8, 32)])
def test_read(codes, dtype, dim, kv, page):
    """Borders of sequences at any place of a workgroup's four tokens, and the same edges."""
    new = [1401, 0, 2, 333, 0, 1, 3, 1, 1, 2, 300, 4, 7]
    lens = [1500, 20, 2, 333, 0, 1, 50, 1, 9, 2, 310, 4, 3]
    b = Batch(lens, new, dtype, kv, dim, page, kv, seed=45)
    b.table[3, 1] = -1
    b.table[10, 2] = b.n_pages
    before, behind = 2, 5
    n = before + b.tokens + behind
    assert n >= 2048 and n % 4
    _, table, lens_d, starts = b.gpu()
    cache = random_cache(b, codes)
    got = [torch.full((n, kv, dim), 7.0, dtype=dtype, device="cuda") for _ in range(4)]
    serving.read_rows(cache, table, lens_d, starts + before, *got[:2])
    for i, t, m, left in pieces(b, before):
        serving.read_rows(cache, table[i:i + 1], lens_d[i:i + 1] - left,
                          torch.tensor([0, m], dtype=torch.int32, device="cuda"), got[2][t:t + m], got[3][t:t + m])
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    for x in got[:2]:
        left = (x == 7).all(-1).all(-1)
        last = before + int(b.starts[12])  # four tokens of the last sequence have no place
        assert left.nonzero().flatten().tolist() == [0, 1, *range(last, last + 4), *range(n - behind, n)]
