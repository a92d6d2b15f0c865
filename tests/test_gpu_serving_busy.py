"""Serving operators in the batches of a busy server: as many sequences as fill the
card, whose ranges have a least length, and tables far wider than their sequences."""

import ctypes

import pytest
import torch

from rpgbarengine_amd import serving
from serving_plain import attention as plain_attention
from test_gpu_serving import DTYPES, Batch, close
from test_gpu_serving_codes import CODES, attention, ident, on_cpu, random_cache, weight_bits

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
