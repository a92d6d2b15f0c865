"""A cache held in 8 bits (rpgbarengine_amd.serving.QuantCache): rows in and out,
against their definitions in float64."""

import math

import pytest
import torch

import rpgbarengine_amd as eng
import serving_more_plain as more
import serving_plain as plain
from rpgbarengine_amd import serving
from test_gpu_serving import DTYPES, IDS, Batch, close

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
NAMES = {**IDS, torch.int8: "i8", torch.float8_e4m3fn: "e4m3"}


def ident(x):
    return NAMES.get(x, None) if isinstance(x, torch.dtype) else None


def empty_cache(b, codes, fill=0x33):
    """A QuantCache over the batch's pages whose every byte is `fill`, scales 7."""
    shape = (b.n_pages, b.kv, b.page, b.dim)
    k, v = (torch.full(shape, fill, dtype=torch.int8, device="cuda").view(codes) for _ in "kv")
    return serving.QuantCache(k, v, *(torch.full(shape[:3], 7.0, device="cuda") for _ in "kv"))


def held(cache):
    return [x.cpu() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 32, 8, 16), (128, 5, 1, 64), (64, 6, 3, 32)])
def test_append(codes, dtype, dim, heads, kv, page):
    b = Batch([37, 16, 1, 200, 33], [5, 16, 1, 0, 33], dtype, kv, dim, page, heads, seed=1)
    behind = 4  # rows behind the last sequence
    n = b.tokens + behind
    qkv = b.normal(n, heads + 2 * kv, dim, by=3.0)
    qn, kn = 1 + 0.2 * torch.randn(dim, generator=b.gen), 1 + 0.2 * torch.randn(dim, generator=b.gen)
    ang = torch.rand(256, dim // 2, generator=b.gen) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1)
    _, table, lens, starts = b.gpu()
    cache = empty_cache(b, codes)
    before = held(cache)
    x = qkv.cuda()
    out = torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda")
    got = serving.append(cache, table, lens, starts, x[:, heads:heads + kv], x[:, heads + kv:], q=x[:, :heads], q_out=out,
                         q_norm=qn.cuda(), k_norm=kn.cuda(), eps=1e-5, rope=rope.cuda())
    assert got is out
    after = held(cache)
    k, v = cache.k.cpu().double(), cache.v.cpu().double()
    ks, vs = after[2].double(), after[3].double()
    touched = torch.zeros(b.n_pages, page, dtype=torch.bool)
    for i, (ln, m) in enumerate(zip(b.lens, b.new)):
        for j in range(m):
            t, pos = int(b.starts[i]) + j, ln - m + j
            at, r = int(b.table[i, pos // page]), pos % page
            touched[at, r] = True
            want, mag = plain.turned(qkv[t, heads:heads + kv], kn, 1e-5, rope[pos])
            more.check_row(k[at, :, r], ks[at, :, r], want, plain.turned_bound(torch.float32, 0 * want, mag), codes)
            y = qkv[t, heads + kv:].double()
            more.check_row(v[at, :, r], vs[at, :, r], y, 0 * y, codes)
            if dtype != torch.float32:  # y M is exact, the quotient rounded once: the codes are the nearest
                assert torch.equal(v[at, :, r], more.nearest(y * more.LARGEST[codes] / y.abs().amax(-1, keepdim=True), codes))
            want, mag = plain.turned(qkv[t, :heads], qn, 1e-5, rope[pos])
            close(out[t], want, plain.turned_bound(dtype, want, mag))
    for was, now in zip(before, after):  # every other row as it was
        assert torch.equal(now.transpose(1, 2)[~touched], was.transpose(1, 2)[~touched])
    assert bool((out[b.tokens:] == 7).all())


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_append_odd_rows(codes, dtype):
    """Zeros, a single value, the type's largest and smallest magnitudes, rows that are
    not finite; signs of zero and of the largest."""
    b = Batch([40], [12], dtype, 2, 128, 16, 4, seed=2)
    rows = b.normal(12, 2, 128)
    big = torch.finfo(dtype).max
    rows[0] = 0.0
    rows[1], rows[1, 0, 5], rows[1, 1, 7] = 0.0, -3.0, 1e-3
    rows[2] *= big / 8
    rows[2, :, 3] = -big
    rows[3] = (rows[3].double() * 1e-3 * float(torch.finfo(dtype).smallest_normal)).to(dtype)
    rows[4, 0, 9], rows[4, 1, 9] = math.inf, -math.inf
    rows[5, 0, 0], rows[5, 1, 127] = math.nan, -math.nan
    rows[6] = (rows[6].double() * 2.0 ** -70).to(dtype)  # f16: zeros
    rows[7] = torch.where(rows[7] < 0, -2.5, 2.5).to(dtype)
    rows[8] = (rows[8].double() * (2.0 ** 90 if dtype != torch.float16 else 1000)).to(dtype)
    _, table, lens, starts = b.gpu()
    cache = empty_cache(b, codes)
    x = rows.cuda()
    assert serving.append(cache, table, lens, starts, x, x) is None
    k, v, ks, vs = cache.k.cpu().double(), cache.v.cpu().double(), cache.k_scale.cpu().double(), cache.v_scale.cpu().double()
    assert torch.equal(k, v) or codes == torch.float8_e4m3fn
    assert torch.equal(cache.k.view(torch.int8), cache.v.view(torch.int8))
    assert torch.equal(ks.nan_to_num(-1.0), vs.nan_to_num(-1.0))
    for j in range(12):
        pos = 28 + j
        at, r = int(b.table[0, pos // 16]), pos % 16
        for h in range(2):
            y = rows[j, h].double()
            if not bool(y.isfinite().all()):
                assert math.isnan(float(ks[at, h, r])) and bool((k[at, h, r] == 0).all())
            elif float(y.abs().max()) < 2.0 ** -112:
                assert float(ks[at, h, r]) == 0.0 and bool((k[at, h, r] == 0).all())
            else:
                more.check_row(k[at, h, r], ks[at, h, r], y, 0 * y, codes)
    kr, vr = torch.empty_like(x), torch.empty_like(x)
    serving.read_rows(cache, table, lens, starts, kr, vr)
    for j in (4, 5):
        assert bool(kr[j].isnan().all()) and bool(vr[j].isnan().all())
    assert bool((kr[0] == 0).all()) and bool(kr[[1, 2, 6, 7, 8, 9, 10, 11]].isfinite().all())


@pytest.mark.parametrize("codes", CODES, ids=ident)
def test_append_leaves_out_tokens_without_a_place(codes):
    """More new tokens than positions, positions past the rotation table, pages
    that the table does not name; queries in place."""
    b = Batch([3, 40, 20], [5, 2, 20], torch.bfloat16, seed=3)
    b.table[2, 0] = b.n_pages  # no such page
    b.table[2, 1] = -7
    _, table, lens, starts = b.gpu()
    cache = empty_cache(b, codes)
    before = held(cache)
    k, v, q = (b.normal(b.tokens, h, 128).cuda() for h in (2, 2, 4))
    rope = torch.ones(39, 128).cuda()
    apart = torch.full_like(q, 9.0)
    serving.append(cache, table, lens, starts, k, v, q=q, q_out=apart, rope=rope)
    same = [int(b.starts[0]), int(b.starts[0]) + 1, int(b.starts[1]) + 1]  # positions -2, -1; 39
    for t in range(b.tokens):
        assert bool((apart[t] == 9).all()) == (t in same), t
    want = torch.zeros(b.n_pages, 16, dtype=torch.bool)
    for pos in range(3):
        want[int(b.table[0, 0]), pos] = True
    want[int(b.table[1, 2]), 38 - 32] = True
    for was, now in zip(before, held(cache)):
        changed = now != was
        changed = (changed if changed.dim() == 3 else changed.any(-1)).any(1)
        assert torch.equal(changed, want)
    mine = q.clone()
    assert serving.append(cache, table, lens, starts, k, v, q=mine, q_out=mine, rope=rope) is mine
    there = [t for t in range(b.tokens) if t not in same]
    assert torch.equal(mine[there], apart[there]) and torch.equal(mine[same], q[same])


def random_cache(b, codes, by=1.0):
    """Codes of any value (NaN apart) and scales over some orders of magnitude."""
    shape = (b.n_pages, b.kv, b.page, b.dim)

    def pool():
        if codes == torch.int8:
            return torch.randint(-127, 128, shape, generator=b.gen, dtype=torch.int8)
        x = torch.randint(0, 254, shape, generator=b.gen)
        return torch.where(x >= 127, x + 1, x).to(torch.uint8).view(codes)

    def scales():
        return torch.exp(torch.randn(shape[:3], generator=b.gen)) * by / more.LARGEST[codes]

    return serving.QuantCache(pool().cuda(), pool().cuda(), scales().cuda(), scales().cuda())


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,kv,page", [(128, 8, 16), (128, 1, 64), (64, 3, 32)])
def test_read(codes, dtype, dim, kv, page):
    b = Batch([37, 16, 1, 200, 33, 3], [5, 16, 1, 0, 33, 5], dtype, kv, dim, page, kv, seed=4)
    b.table[4, 0] = -1
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    ko, vo = (torch.full((b.tokens + 3, kv, dim), 7.0, dtype=dtype, device="cuda") for _ in "kv")
    got = serving.read_rows(cache, table, lens, starts, ko, vo)
    assert got[0] is ko and got[1] is vo
    for out, pool, scale in ((ko, cache.k, cache.k_scale), (vo, cache.v, cache.v_scale)):
        want = torch.full((b.tokens + 3, kv, dim), 7.0, dtype=torch.float64)
        rows = more.values(pool.cpu(), scale.cpu())
        for i, (ln, m) in enumerate(zip(b.lens, b.new)):
            for j in range(m):
                pos = ln - m + j
                if pos < 0:
                    continue
                at = int(b.table[i, pos // page])
                want[int(b.starts[i]) + j] = rows[at, :, pos % page] if at >= 0 else 0.0
        # The product of a code (8 bits) and a scale (24) is exact in float64. The kernel
        # rounds it to f32, by 2^-24 at most, and then to the type, or to the type at
        # once (the compiler may join the two); to f32 once.
        twice = 0.0 if dtype == torch.float32 else 2.0 ** -24
        bound = (plain.EPS[dtype] * (1 + twice) + twice) * want.abs() + plain.TINY[dtype]
        close(out, want, bound)


def test_every_code_reads_as_its_value():
    for codes in CODES:
        b = Batch([16], [16], torch.float32, 1, 128, 16, 1, seed=5)
        _, table, lens, starts = b.gpu()
        every = torch.arange(256, dtype=torch.uint8).repeat(b.n_pages * 8).view(b.n_pages, 1, 16, 128)
        k = every.view(codes).cuda()
        one = torch.ones(b.n_pages, 1, 16, device="cuda")
        cache = serving.QuantCache(k, k.clone(), one, one.clone())
        for dtype in DTYPES:
            ko, vo = (torch.empty(16, 1, 128, dtype=dtype, device="cuda") for _ in "kv")
            serving.read_rows(cache, table, lens, starts, ko, vo)
            want = every[int(b.table[0, 0]), 0].view(codes).float().view(16, 1, 128)
            assert torch.equal(ko.cpu().float().nan_to_num(1e9), want.nan_to_num(1e9))


def test_views_of_larger_pools():
    """Pages, heads and positions at any strides of 16 bytes, rows behind one another."""
    b = Batch([50, 20], [50, 20], torch.bfloat16, 3, 64, 16, 3, seed=6)
    _, table, lens, starts = b.gpu()
    pool = torch.zeros(b.n_pages, 16, 2, 3, 80, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, b.n_pages, 5, 16, device="cuda")
    k, v = (pool[:, :, i, :, :64].transpose(1, 2) for i in range(2))
    ks, vs = (scales[i, :, 1:4] for i in range(2))
    cache = serving.QuantCache(k, v, ks, vs)
    rows = b.normal(70, 3, 64).cuda()
    serving.append(cache, table, lens, starts, rows, -rows)
    flat = serving.QuantCache.zeros(b.n_pages, 16, 3, 64, torch.int8)
    serving.append(flat, table, lens, starts, rows, -rows)
    for x, y in ((cache.k, flat.k), (cache.v, flat.v), (cache.k_scale, flat.k_scale), (cache.v_scale, flat.v_scale)):
        assert torch.equal(x, y)
    assert bool((pool[..., 64:] == 0).all()) and bool((scales[:, :, [0, 4]] == 0).all())
    ko, vo = torch.empty_like(rows), torch.empty_like(rows)
    serving.read_rows(cache, table, lens, starts, ko, vo)
    assert torch.equal(ko, -vo)


@pytest.mark.parametrize("codes", CODES, ids=ident)
def test_pages_past_32_bits(codes):
    """Pages two GiB apart, scales as far: what each operator gives is that of the same
    pages side by side, to the bit."""
    b = Batch([33, 16], [33, 16], torch.bfloat16, 2, 64, 16, 4, seed=17, spare=1)
    assert b.n_pages == 5
    apart = (1 << 31) - (1 << 20)
    pool = torch.empty(5 * apart, dtype=torch.int8, device="cuda")

    def view(at, dtype, shape, stride):
        return torch.as_strided(pool.view(dtype), shape, stride, at // dtype.itemsize)

    k, v = (view(at << 16, codes, (5, 2, 16, 64), (apart, 1024, 64, 1)) for at in (0, 1))
    ks, vs = (view(at << 16, torch.float32, (5, 2, 16), (apart // 4, 16, 1)) for at in (2, 3))
    far, near = serving.QuantCache(k, v, ks, vs), serving.QuantCache.zeros(5, 16, 2, 64, codes)
    for x in (k, v):
        x.view(torch.int8).zero_()
    ks.zero_(), vs.zero_()
    _, table, lens, starts = b.gpu()
    rows, q = b.normal(49, 2, 64).cuda(), b.normal(49, 4, 64, by=0.5).cuda()
    groups, shared = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([16], dtype=torch.int32).cuda()
    table[1, 0] = table[0, 0]
    got = []
    for cache in (far, near):
        serving.append(cache, table[:1], lens[:1], starts[:2], rows, -rows)
        ko, vo = torch.zeros_like(rows), torch.zeros_like(rows)
        serving.read_rows(cache, table, lens, starts, ko, vo)
        got.append((ko, vo, serving.prompt_attention(q, cache, table, lens, starts),
                    serving.decode_attention(q[:2], cache, table, lens),
                    serving.shared_attention(q[:2], cache, table, lens, groups, shared)))
    for x, y in zip(*got):
        assert torch.equal(x, y) and bool(x.isfinite().all()) and bool((x != 0).any())


def test_a_cache_whose_tensors_moved_is_refused():
    cache = serving.QuantCache.zeros(4, 16, 2, 64)
    b = Batch([5], [5], torch.float32, 2, 64, 16, 2)
    _, table, lens, starts = b.gpu()
    rows = b.normal(5, 2, 64).cuda()
    cache.k_scale.set_(torch.zeros(4, 2, 16, device="cuda"))
    with pytest.raises(eng.EngineError, match="lie elsewhere"):
        serving.append(cache, table, lens, starts, rows, rows)


# ---- attention


def attention(q, k, v, ks, vs, seen, scale, dtype, weight_bits, prompt=False):
    """q [heads, dim] over codes k, v [kv, n, dim] with scales ks, vs [kv, n], where
    seen [n]: (out, bound), float64. weight_bits: of a weight times its scale in the
    second product."""
    heads, dim = q.shape
    group = heads // k.shape[0]
    out, bound = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    if not bool(seen.any()):
        return out, bound
    for h in range(heads):
        kv = h // group
        kk, vv = k[kv][seen].double(), v[kv][seen].double()
        ss, tt = ks[kv][seen].double(), vs[kv][seen].double()
        qq = q[h].double()
        s = (kk @ qq) * ss * scale
        p = torch.softmax(s, 0)
        out[h] = ((p * tt)[:, None] * vv).sum(0)
        mass = ((p * tt)[:, None] * vv.abs()).sum(0)
        # A score: dim products in fp32, added in any order (three parts of an f32
        # query are exact), two products with scales, the difference from the maximum;
        # 2^x; the weight's product with its scale; sums over the keys and the ranges'
        # joins; the weight's rounding.
        ds = float(((kk.abs() @ qq.abs()) * ss).max()) * scale * (3 * dim + 6) * 2.0 ** -24 + float(s.abs().max()) * 2.0 ** -21
        rel = math.expm1(2 * ds) + (3 * len(s) + 18) * 2.0 ** -23 + 2.0 ** -weight_bits
        # (the scales of all of the sequence's keys count: later tokens' too)
        bound[h] = rel * mass + 2.0 ** -140 * len(s) * 448 + least_weight(dtype, prompt, vs[kv].double(), tt, vv) * float(p.max())
    return out, bound + plain.EPS[dtype] * (out.abs() + bound) + plain.TINY[dtype]


def rows_of(pool, b, i, n):
    return plain.sequence_rows(pool, b.table[i], n)


def scales_of(pool, b, i, n):
    rows, there = plain.sequence_rows(pool[..., None], b.table[i], n)
    return rows[..., 0], there


def on_cpu(cache):
    return cache.k.cpu().float(), cache.v.cpu().float(), cache.k_scale.cpu(), cache.v_scale.cpu()


def expect(b, cache, q, scale, i, pos, row, prompt=False):
    """(out, bound) of the token at position pos of sequence i, row `row` of q. Weights
    go to the second product in three parts of 8 bits (f32), two (16-bit rows), in
    prompts of 16-bit rows rounded once to their type."""
    k, v, ks, vs = cache
    n = b.lens[i]
    kk, there = rows_of(k, b, i, n)
    seen = there & (torch.arange(n) <= pos)
    return attention(q[row], kk, rows_of(v, b, i, n)[0], scales_of(ks, b, i, n)[0], scales_of(vs, b, i, n)[0], seen, scale,
                     b.dtype, weight_bits(b.dtype, prompt), prompt)


def weight_bits(dtype, prompt):
    return {torch.float32: 24, torch.float16: 11 if prompt else 16, torch.bfloat16: 8 if prompt else 16}[dtype]


def least_weight(dtype, prompt, every, ss, vv):
    """What f16 weights of prompts lose below the type's range. A code is multiplied times
    the power of two in its scale, within 2^-24 .. 2^5 (e4m3 2^-15 .. 2^7), and its weight
    takes the rest of the scale: held times 2^7, over a power of two that the rests (of
    `every` scale) reach half of at least, each off by 2^-25. (The larger of the two
    types' bounds.) ss, vv: of the keys that are seen."""
    if not prompt or dtype != torch.float16 or not len(ss):
        return 0.0

    def power(x):
        return 2.0 ** x.clamp(min=2.0 ** -149).log2().floor().clamp(lo, hi)

    least = []
    for lo, hi in ((-24, 5), (-15, 7)):
        least.append(2.0 ** -32 * 2 * float((every / power(every)).max()) * (power(ss)[..., None] * vv.abs()).sum(-2))
    return torch.maximum(*least)


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300, 0]


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (128, 3, 3, 64), (64, 40, 2, 32), (64, 8, 1, 16),
                                               (128, 17, 1, 256)])
def test_decode(codes, dtype, dim, heads, kv, page):
    b = Batch(LENS, [1] * len(LENS), dtype, kv, dim, page, heads, seed=7)
    q = b.normal(len(LENS), heads, dim, by=0.3)
    _, table, lens, _ = b.gpu()
    cache = random_cache(b, codes)
    out = torch.full((len(LENS), heads, dim), 5.0, dtype=dtype, device="cuda")
    assert serving.decode_attention(q.cuda(), cache, table, lens, scale=0.11, out=out) is out
    held_ = on_cpu(cache)
    for i, n in enumerate(LENS):
        close(out[i], *expect(b, held_, q, 0.11, i, n - 1, i))
    assert torch.equal(serving.decode_attention(q.cuda(), cache, table, lens, scale=0.11), out)  # the same bits


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_decode_long_and_split(codes, dtype):
    """Many ranges joined; lengths next to a range's border in a table that has room
    for more; peaked scores (the maximum moves from range to range)."""
    b = Batch([3001, 1, 640, 513, 2049], [1] * 5, dtype, 1, 64, 16, 2, seed=8, extra_pages=70)
    q = b.normal(5, 2, 64, by=0.4)
    _, table, lens, _ = b.gpu()
    cache = random_cache(b, codes)
    cache.k_scale[int(b.table[0, 100]), 0, 3] *= 6
    got = serving.decode_attention(q.cuda(), cache, table, lens)
    held_ = on_cpu(cache)
    for i, n in enumerate(b.lens):
        close(got[i], *expect(b, held_, q, 64 ** -0.5, i, n - 1, i))


def spoil(b, cache, used, odd_scale):
    """Every place that no position uses: NaN codes, scales of odd_scale."""
    hold = (~used)[:, None, :].expand(-1, b.kv, -1).cuda()
    for x in (cache.k, cache.v):
        bits = x.view(torch.uint8)
        bits[hold] = 0x7F if x.dtype == torch.float8_e4m3fn else 0x80
    for x in (cache.k_scale, cache.v_scale):
        x[hold] = odd_scale


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("prompt", [0, 1], ids=["decode", "prompt"])
def test_masked_places_hold_anything(codes, dtype, value, prompt):
    """Rows past the length, spare pages and pages that the table names no more."""
    new = [3, 40, 1, 2] if prompt else [1] * 4
    b = Batch([37, 130, 16, 700], new, dtype, 2, 128, 16, 8, seed=9)
    used = torch.zeros(b.n_pages, 16, dtype=torch.bool)
    b.table[1, 3] = -1
    b.table[3, 20] = b.n_pages + 5
    b.table[2, 0] = 1 << 30  # the whole of a sequence
    for i, n in enumerate(b.lens):
        for p in range(n):
            at = int(b.table[i, p // 16])
            if 0 <= at < b.n_pages:
                used[at, p % 16] = True
    q = b.normal(b.tokens, 8, 128, by=0.3)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    held_ = on_cpu(cache)
    spoil(b, cache, used, value)
    if prompt:
        got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    else:
        got = serving.decode_attention(q.cuda(), cache, table, lens)
    for i, n in enumerate(b.lens):
        for j in range(b.new[i]):
            row = int(b.starts[i]) + j
            close(got[row], *expect(b, held_, q, 128 ** -0.5, i, n - b.new[i] + j, row, prompt=bool(prompt)))


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_a_row_that_was_not_finite(codes, dtype):
    """NaN for the tokens that see it, nothing for those before it and for other
    sequences; keys' and values' rows."""
    for name in ("k_scale", "v_scale"):
        b = Batch([90, 50], [60, 50], dtype, 2, 64, 16, 4, seed=10)
        q = b.normal(b.tokens, 4, 64, by=0.3)
        _, table, lens, starts = b.gpu()
        cache = random_cache(b, codes)
        held_ = on_cpu(cache)
        getattr(cache, name)[int(b.table[0, 70 // 16]), 1, 70 % 16] = math.nan
        got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
        one = serving.decode_attention(q[[59, 109]].cuda(), cache, table, lens)
        for i in range(2):
            for j in range(b.new[i]):
                row, pos = int(b.starts[i]) + j, b.lens[i] - b.new[i] + j
                hit = i == 0 and pos >= 70
                want, bound = expect(b, held_, q, 64 ** -0.5, i, pos, row, prompt=True)
                heads = slice(0, 2) if hit else slice(0, 4)
                close(got[row, heads], want[heads], bound[heads])
                assert not hit or bool(got[row, 2:].isnan().all())
        assert bool(one[0, 2:].isnan().all()) and bool(one[0, :2].isfinite().all()) and bool(one[1].isfinite().all())


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("power", [-100, -60, 60, 90])
def test_scales_of_any_size(codes, dtype, power):
    """Values' scales far from 1, where an f16 product's operands would not hold them."""
    if dtype == torch.float16:
        power //= 10
    b = Batch([33, 200], [1, 1], dtype, 2, 128, 16, 4, seed=11)
    q = b.normal(2, 4, 128, by=0.3)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    cache.v_scale.mul_(2.0 ** power)
    held_ = on_cpu(cache)
    for got, prompt in ((serving.decode_attention(q.cuda(), cache, table, lens), False),
                        (serving.prompt_attention(q.cuda(), cache, table, lens, starts), True)):
        for i, n in enumerate(b.lens):
            close(got[i], *expect(b, held_, q, 128 ** -0.5, i, n - 1, i, prompt))


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,new", [(128, 4, 2, 9), (64, 192, 32, 300)], ids=["few", "many"])
def test_a_large_row_that_weighs_nothing(codes, dtype, dim, heads, kv, new):
    """One row of values 2^22 times as large as the others, with next to no weight: the
    output is the others'."""
    b = Batch([330], [new], dtype, kv, dim, 16, heads, seed=16)
    q = b.normal(b.tokens, heads, dim, by=0.3).abs().add(0.5).to(dtype)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    cache.v_scale.copy_(torch.exp(torch.randn(cache.v_scale.shape, generator=b.gen)).mul(2.0 ** -15))
    page, at = int(b.table[0, 1]), 5
    cache.v_scale[page, :, at] = 100.0
    cache.k[page, :, at] = torch.full((kv, dim), -96.0, device="cuda").to(codes)
    cache.k_scale[page, :, at] = 0.1
    held_ = on_cpu(cache)
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    for h in (0, heads // 2, heads - 1):
        close(got[:, h], *expect_head(b, held_, q, dim ** -0.5, 0, h, heads))


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (64, 5, 1, 32), (128, 3, 3, 64), (64, 34, 2, 16)])
def test_prompt(codes, dtype, dim, heads, kv, page):
    lens, new = [70, 33, 1, 5, 130, 64, 0, 100], [70, 3, 1, 0, 40, 64, 0, 1]
    b = Batch(lens, new, dtype, kv, dim, page, heads, seed=12)
    q = b.normal(b.tokens + 3, heads, dim, by=0.3)
    _, table, lens_d, starts = b.gpu()
    cache = random_cache(b, codes)
    out = torch.full((b.tokens + 3, heads, dim), 5.0, dtype=dtype, device="cuda")
    assert serving.prompt_attention(q.cuda(), cache, table, lens_d, starts, scale=0.1, out=out) is out
    held_ = on_cpu(cache)
    for i, n in enumerate(b.lens):
        for j in range(b.new[i]):
            row = int(b.starts[i]) + j
            close(out[row], *expect(b, held_, q, 0.1, i, n - b.new[i] + j, row, prompt=True))
    assert bool((out[b.tokens:] == 5).all())  # rows behind the last sequence
    again = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts, scale=0.1)
    assert torch.equal(again[:b.tokens], out[:b.tokens])


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_prompt_behind_a_long_history(codes, dtype):
    b = Batch([900, 1500, 333], [7, 1, 20], dtype, 1, 128, 64, 2, seed=13)
    q = b.normal(b.tokens, 2, 128, by=0.3)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    cache.k_scale[int(b.table[0, 5]), 0, 3] *= 5  # the maximum moves
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    held_ = on_cpu(cache)
    for i, n in enumerate(b.lens):
        for j in range(b.new[i]):
            row = int(b.starts[i]) + j
            close(got[row], *expect(b, held_, q, 128 ** -0.5, i, n - b.new[i] + j, row, prompt=True))


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_more_new_tokens_than_positions(codes, dtype):
    """Tokens at positions below 0 see nothing: zeros."""
    b = Batch([3, 20], [8, 20], dtype, 2, 64, 16, 4, seed=14)
    q = b.normal(b.tokens, 4, 64)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    assert bool((got[:5] == 0).all()) and bool((got[5:] != 0).any(-1).all())


def expect_head(b, cache, q, scale, i, h, heads):
    """(out, bound) of all new tokens of sequence i for query head h, as `attention`
    has them for one token."""
    k, v, ks, vs = cache
    n, m = b.lens[i], b.new[i]
    kv = h // (heads // b.kv)
    kk, there = rows_of(k, b, i, n)
    kk, vv = kk[kv], rows_of(v, b, i, n)[0][kv]
    ss, tt = scales_of(ks, b, i, n)[0][kv], scales_of(vs, b, i, n)[0][kv]
    qq = q[int(b.starts[i]):int(b.starts[i]) + m, h].double()
    seen = there[None, :] & (torch.arange(n)[None, :] <= torch.arange(n - m, n)[:, None])
    s = (qq @ kk.t()) * ss * scale
    p = torch.softmax(s.masked_fill(~seen, -math.inf), 1) * tt
    out, mass = p @ vv, p @ vv.abs()
    size = (qq.abs() @ kk.abs().t()) * ss
    ds = (size * seen).amax(1) * scale * (3 * q.shape[2] + 6) * 2.0 ** -24 + (s.abs() * seen).amax(1) * 2.0 ** -21
    rel = torch.expm1(2 * ds) + (3 * seen.sum(1) + 18) * 2.0 ** -23 + 2.0 ** -weight_bits(b.dtype, True)
    bound = rel[:, None] * mass + 2.0 ** -140 * n * 448 + least_weight(b.dtype, True, tt, tt, vv)
    return out, bound + plain.EPS[b.dtype] * (out.abs() + bound) + plain.TINY[b.dtype]


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 128, 32, 16), (64, 96, 32, 64)])
def test_prompts_of_many_rows(codes, dtype, dim, heads, kv, page):
    """Enough rows for tiles of 128, in sequences that begin and end inside them, one
    with a history, one with an unnamed page and one with a row that was not finite."""
    lens, new = [150, 300, 64, 97], [150, 70, 64, 33]
    b = Batch(lens, new, dtype, kv, dim, page, heads, seed=15)
    b.table[1, 1] = -1
    q = b.normal(b.tokens + 2, heads, dim, by=0.3)
    _, table, lens_d, starts = b.gpu()
    cache = random_cache(b, codes)
    held_ = on_cpu(cache)
    cache.v_scale[int(b.table[2, 40 // page]), 5, 40 % page] = math.nan
    out = torch.full((b.tokens + 2, heads, dim), 5.0, dtype=dtype, device="cuda")
    serving.prompt_attention(q.cuda(), cache, table, lens_d, starts, out=out)
    group = heads // kv
    for i in range(4):
        at = slice(int(b.starts[i]), int(b.starts[i]) + new[i])
        for h in (0, 5 * group, 5 * group + group - 1, heads - 1):
            want, bound = expect_head(b, held_, q, dim ** -0.5, i, h, heads)
            got = out[at, h]
            if i == 2 and h // group == 5:
                assert bool(got[40:].isnan().all())
                got, want, bound = got[:40], want[:40], bound[:40]
            close(got, want, bound)
    assert bool((out[b.tokens:] == 5).all())
    again = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts)[:b.tokens]
    assert torch.equal(again.nan_to_num(7.0), out[:b.tokens].nan_to_num(7.0))


# ---- refusals of the binding


def test_refusals_on_tensors():
    b = Batch([20, 5], [4, 1], torch.float32, 2, 64, 16, 4, seed=16)
    rows, table, lens, starts = b.gpu()
    cache = random_cache(b, torch.int8)
    k, q, one = b.normal(5, 2, 64).cuda(), b.normal(5, 4, 64).cuda(), b.normal(2, 4, 64).cuda()
    groups, shared = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([16], dtype=torch.int32).cuda()
    E = eng.EngineError
    for call in (lambda: serving.append(cache, table, lens, starts, k, k.half()),
                 lambda: serving.append(cache, table, lens, starts, k.double(), k.double()),
                 lambda: serving.append(cache, table, lens, starts, k[:, :1], k[:, :1]),
                 lambda: serving.append(cache, table, lens, starts, k, k, q=q.half()),
                 lambda: serving.append(cache, table, lens, starts, k.requires_grad_(), k.detach()),
                 lambda: serving.read_rows(rows, table, lens, starts, k.detach(), k.detach()),
                 lambda: serving.read_rows(cache, table, lens, None, k.detach(), k.detach()),
                 lambda: serving.read_rows(cache, table, lens, starts, k.detach(), k.detach()[:4]),
                 lambda: serving.read_rows(cache, table, lens, starts, q, q),
                 lambda: serving.decode_attention(q, cache, table, lens),
                 lambda: serving.decode_attention(one.double(), cache, table, lens),
                 lambda: serving.decode_attention(one.cpu(), cache, table, lens),
                 lambda: serving.decode_attention(one, cache, table.long(), lens),
                 lambda: serving.decode_attention(one, cache, table, lens, out=one.half()),
                 lambda: serving.prompt_attention(q, cache, table, lens, None),
                 lambda: serving.prompt_attention(q, cache, table, lens, starts[:2]),
                 lambda: serving.shared_attention(one, cache, table, lens, groups[:1], shared),
                 lambda: serving.shared_attention(one, cache, table, lens, groups.long(), shared),
                 lambda: serving.shared_attention(one, cache, table, lens, groups, shared.cpu()),
                 lambda: serving.shared_attention(q, rows, table, lens, groups, shared),
                 lambda: serving.shared_attention(one.half(), rows, table, lens, groups, shared),
                 lambda: serving.shared_attention(one.clone().requires_grad_(), rows, table, lens, groups, shared)):
        with pytest.raises(E):
            call()
    with torch.no_grad():  # nothing is recorded: parameters are fine
        serving.decode_attention(one.clone().requires_grad_(), cache, table, lens)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(one, torch.ones_like(one))
        for call in (lambda: serving.decode_attention(dual, cache, table, lens),
                     lambda: serving.shared_attention(dual, cache, table, lens, groups, shared)):
            with pytest.raises(E, match="tangent"):
                call()


def test_what_is_written_is_a_new_version():
    b = Batch([20], [4], torch.float32, 2, 64, 16, 2, seed=17)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, torch.float8_e4m3fn)
    k = b.normal(4, 2, 64).cuda()
    held_ = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    was = [x._version for x in held_]
    serving.append(cache, table, lens, starts, k, k)
    assert all(x._version > v for x, v in zip(held_, was))
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    was = ko._version, vo._version
    serving.read_rows(cache, table, lens, starts, ko, vo)
    assert ko._version > was[0] and vo._version > was[1]


@pytest.mark.parametrize("prompt", [0, 1], ids=["decode", "prompt"])
def test_on_another_stream_and_replayed(prompt):
    """A stream of the caller's; a captured call takes lengths and pages of its moment."""
    b = Batch([700, 33], [2, 1] if prompt else [1, 1], torch.float16, 2, 128, 16, 8, seed=18)
    q = b.normal(b.tokens, 8, 128, by=0.3)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, torch.int8)
    held_, qd, out = on_cpu(cache), q.cuda(), torch.empty(b.tokens, 8, 128, dtype=torch.float16, device="cuda")

    def call():
        if prompt:
            serving.prompt_attention(qd, cache, table, lens, starts, out=out)
        else:
            serving.decode_attention(qd, cache, table, lens, out=out)

    def check():
        for i, n in enumerate(b.lens):
            for j in range(b.new[i]):
                row = int(b.starts[i]) + j
                close(out[row], *expect(b, held_, q, 128 ** -0.5, i, n - b.new[i] + j, row, prompt=bool(prompt)))

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(3):
        b.lens = [700 - 200 * step, 33 - 16 * step]
        b.table[0, 1] = b.table[0, 2 + step]
        lens.copy_(torch.tensor(b.lens, dtype=torch.int32)), table.copy_(b.table)
        out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        check()
