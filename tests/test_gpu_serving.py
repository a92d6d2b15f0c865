"""The serving operators (rpgbarengine_amd.serving) against their definitions in
float64: cache pages, decode and prompt attention, the row sampler, at the
sizes, masks and layouts where they can go wrong."""

import itertools
import math

import pytest
import torch

import rpgbarengine_amd as eng
import serving_plain as plain
from rpgbarengine_amd import serving

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}


def ident(x):
    return IDS.get(x, None) if isinstance(x, torch.dtype) else None


class Batch:
    """Sequences of given lengths and new tokens over a shuffled pool of pages,
    some of them spare; on the CPU, with device copies by gpu()."""

    def __init__(self, lens, new, dtype, kv=2, dim=128, page=16, heads=4, seed=0, spare=3, extra_pages=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.dtype, self.page, self.dim, self.kv, self.heads = lens, new, dtype, page, dim, kv, heads
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((len(lens), max(need, default=0) + extra_pages), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, kv, page, dim)
        self.k = torch.randn(shape, generator=g).to(dtype)
        self.v = torch.randn(shape, generator=g).to(dtype)
        self.tokens = sum(new)
        self.starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
        self.len_t = torch.tensor(lens, dtype=torch.int32)
        self.gen = g

    def normal(self, *shape, by=1.0):
        return (torch.randn(shape, generator=self.gen) * by).to(self.dtype)

    def gpu(self):
        self.cache = serving.PagedCache(self.k.cuda(), self.v.cuda())
        return self.cache, self.table.cuda(), self.len_t.cuda(), self.starts.cuda()


def expect_prompt(b, q, scale, k=None, v=None):
    """(out, bound) of every packed token."""
    k, v = (b.k if k is None else k), (b.v if v is None else v)
    outs, bounds = [], []
    for i, (n, m) in enumerate(zip(b.lens, b.new)):
        kk, there = plain.sequence_rows(k, b.table[i], n)
        vv, _ = plain.sequence_rows(v, b.table[i], n)
        for j in range(m):
            pos = n - m + j
            seen = there & (torch.arange(n) <= pos)
            o, e = plain.attention(q[int(b.starts[i]) + j], kk, vv, seen, scale, b.dtype)
            outs.append(o)
            bounds.append(e)
    return torch.stack(outs), torch.stack(bounds)


def close(got, want, bound):
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float((d / bound).nan_to_num(math.inf).max())} of the bound"


# ---- append


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 32, 8, 16), (128, 5, 1, 64), (64, 6, 3, 32)])
def test_append(dtype, dim, heads, kv, page):
    b = Batch([37, 16, 1, 200, 33], [5, 16, 1, 0, 33], dtype, kv, dim, page, heads, seed=1)
    behind = 4  # rows behind the last sequence
    n = b.tokens + behind
    qkv = b.normal(n, heads + 2 * kv, dim, by=3.0)
    qn, kn = 1 + 0.2 * torch.randn(dim, generator=b.gen), 1 + 0.2 * torch.randn(dim, generator=b.gen)
    ang = torch.rand(256, dim // 2, generator=b.gen) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1)
    cache, table, lens, starts = b.gpu()
    x = qkv.cuda()
    out = torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda")
    got = serving.append(cache, table, lens, starts, x[:, heads:heads + kv], x[:, heads + kv:], q=x[:, :heads], q_out=out,
                         q_norm=qn.cuda(), k_norm=kn.cuda(), eps=1e-5, rope=rope.cuda())
    assert got is out
    k, v = cache.k.cpu(), cache.v.cpu()
    touched = torch.zeros(b.n_pages, page, dtype=torch.bool)
    for i, (ln, m) in enumerate(zip(b.lens, b.new)):
        for j in range(m):
            t, pos = int(b.starts[i]) + j, ln - m + j
            at, r = int(b.table[i, pos // page]), pos % page
            touched[at, r] = True
            want, mag = plain.turned(qkv[t, heads:heads + kv], kn, 1e-5, rope[pos])
            close(k[at, :, r], want, plain.turned_bound(dtype, want, mag))
            assert torch.equal(v[at, :, r], qkv[t, heads + kv:])
            want, mag = plain.turned(qkv[t, :heads], qn, 1e-5, rope[pos])
            close(out[t], want, plain.turned_bound(dtype, want, mag))
    for pool, was in ((k, b.k), (v, b.v)):  # every other row as it was
        assert torch.equal(pool.transpose(1, 2)[~touched], was.transpose(1, 2)[~touched])
    assert bool((out[b.tokens:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_append_plain_copies_and_in_place(dtype):
    """Without gains and rotation rows are stored as they are; q_out may be q."""
    b = Batch([20, 40], [3, 2], dtype, seed=2)
    cache, table, lens, starts = b.gpu()
    k, v = b.normal(5, 2, 128).cuda(), b.normal(5, 2, 128).cuda()
    assert serving.append(cache, table, lens, starts, k, v) is None
    for i in range(2):
        for j in range(b.new[i]):
            pos = b.lens[i] - b.new[i] + j
            at = int(b.table[i, pos // 16])
            assert torch.equal(cache.k[at, :, pos % 16], k[int(b.starts[i]) + j])
            assert torch.equal(cache.v[at, :, pos % 16], v[int(b.starts[i]) + j])
    ang = torch.rand(64, 64, generator=b.gen)
    rope = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    q = b.normal(5, 4, 128).cuda()
    apart = serving.append(cache, table, lens, starts, k, v, q=q, rope=rope)
    assert serving.append(cache, table, lens, starts, k, v, q=q, q_out=q, rope=rope) is q
    assert torch.equal(apart, q)


def test_append_leaves_out_tokens_without_a_place():
    """More new tokens than positions, positions past the rotation table, pages
    that the table does not name, lengths past the table."""
    b = Batch([3, 40, 20], [5, 2, 20], torch.bfloat16, seed=3)
    b.table[2, 0] = b.n_pages  # no such page
    b.table[2, 1] = -7
    cache, table, lens, starts = b.gpu()
    before_k = cache.k.clone()
    k, v, q = (b.normal(b.tokens, h, 128).cuda() for h in (2, 2, 4))
    out = torch.full_like(q, 9.0)
    rope = torch.ones(39, 128).cuda()
    serving.append(cache, table, lens, starts, k, v, q=q, q_out=out, rope=rope)
    same = [int(b.starts[0]), int(b.starts[0]) + 1, int(b.starts[1]) + 1]  # positions -2, -1; 39
    for t in range(b.tokens):
        assert bool((out[t] == 9).all()) == (t in same), t
    changed = (cache.k != before_k).any(-1).any(1).cpu()
    want = torch.zeros_like(changed)
    for pos in range(3):
        want[int(b.table[0, 0]), pos] = True
    want[int(b.table[1, 2]), 38 - 32] = True
    assert torch.equal(changed, want)
    # a length past the table's pages is cut to them
    lens2 = torch.tensor([10 ** 6, 0, -5], dtype=torch.int32).cuda()
    starts2 = torch.tensor([0, 1, 1, 1], dtype=torch.int32).cuda()
    full = torch.arange(b.table.shape[1], dtype=torch.int32)[None].repeat(3, 1).cuda()
    serving.append(cache, full, lens2, starts2, k[:1], v[:1])
    last = b.table.shape[1] - 1
    assert torch.equal(cache.v[last, :, 15], v[0])


# ---- decode attention

LENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300, 0]


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (128, 3, 3, 64), (64, 40, 2, 32), (64, 8, 1, 16),
                                               (128, 17, 1, 256)])
def test_decode(dtype, dim, heads, kv, page):
    b = Batch(LENS, [1] * len(LENS), dtype, kv, dim, page, heads, seed=4)
    q = b.normal(len(LENS), heads, dim, by=1.5)
    cache, table, lens, _ = b.gpu()
    out = torch.full((len(LENS), heads, dim), 5.0, dtype=dtype, device="cuda")
    assert serving.decode_attention(q.cuda(), cache, table, lens, scale=0.11, out=out) is out
    for i, n in enumerate(LENS):
        kk, there = plain.sequence_rows(b.k, b.table[i], n)
        vv, _ = plain.sequence_rows(b.v, b.table[i], n)
        want, bound = plain.attention(q[i], kk, vv, there, 0.11, dtype)
        close(out[i], want, bound)
    again = serving.decode_attention(q.cuda(), cache, table, lens, scale=0.11)
    assert torch.equal(again, out)  # the same bits


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_decode_long_and_split(dtype):
    """Many ranges joined; lengths next to a range's border in a table that has
    room for more; peaked scores (the maximum moves from range to range)."""
    b = Batch([3001, 1, 640, 513, 2049], [1] * 5, dtype, 1, 64, 16, 2, seed=5, extra_pages=70)
    b.k[int(b.table[0, 100]), 0, 3] *= 6
    q = b.normal(5, 2, 64, by=2.0)
    cache, table, lens, _ = b.gpu()
    got = serving.decode_attention(q.cuda(), cache, table, lens)
    for i, n in enumerate(b.lens):
        kk, there = plain.sequence_rows(b.k, b.table[i], n)
        vv, _ = plain.sequence_rows(b.v, b.table[i], n)
        want, bound = plain.attention(q[i], kk, vv, there, 64 ** -0.5, dtype)
        close(got[i], want, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ident)
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_weights_keep_more_bits_than_the_type(dtype, dim):
    """Values +-1, whose weighted sums cancel down to near nothing: what a weight's
    rounding to 16 bits takes off would stand out. Two parts leave its square."""
    b = Batch([40, 300, 3000], [1] * 3, dtype, 2, dim, 16, 8, seed=33)
    b.v = torch.where(b.v < 0, -1.0, 1.0).to(dtype)
    q = b.normal(3, 8, dim, by=1.5)
    cache, table, lens, _ = b.gpu()
    got = serving.decode_attention(q.cuda(), cache, table, lens)
    half = plain.EPS[dtype]
    for i, n in enumerate(b.lens):
        kk, there = plain.sequence_rows(b.k, b.table[i], n)
        vv, _ = plain.sequence_rows(b.v, b.table[i], n)
        want, bound = plain.attention(q[i], kk, vv, there, dim ** -0.5, torch.float32)
        # The weights sum to 1 and the values are 1: a first part is within half of
        # a step, relative, and the second part within half a step of what is left;
        # an f16 second part, held times 2^15, not closer than 2^-25.
        bound += half * half + (n * 2.0 ** -40 if dtype == torch.float16 else 0.0)
        close(got[i], want, bound + half * (want.abs() + bound) + plain.TINY[dtype])


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("n", [37, 3000])
def test_decode_infinities(dtype, n):
    """Infinite values that a token sees, of either sign, beside weights that are
    whole numbers of steps and others; NaN where both signs meet."""
    b = Batch([n, 20], [1, 1], dtype, 2, 128, 16, 8, seed=34)
    at = int(b.table[0, 1])
    b.v[at, 0, 2, 5], b.v[at, 0, 9, 6] = math.inf, -math.inf
    b.v[at, 1, 3, 7], b.v[at, 1, 4, 7] = math.inf, -math.inf
    q = b.normal(2, 8, 128)
    q[0, 0] = 0.0  # every weight is the largest
    cache, table, lens, _ = b.gpu()
    got = serving.decode_attention(q.cuda(), cache, table, lens).double().cpu()
    assert bool((got[0, :4, 5] == math.inf).all()) and bool((got[0, :4, 6] == -math.inf).all())
    assert bool(got[0, 4:, 7].isnan().all())
    ok = torch.ones_like(got, dtype=torch.bool)
    ok[0, :4, 5:7] = False
    ok[0, 4:, 7] = False
    assert bool(got[ok].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prompt", [0, 1], ids=["decode", "prompt"])
def test_an_odd_number_of_partials(dtype, dim, prompt):
    """Five rows in an odd number of ranges, in work memory of exactly the size asked
    for, the bytes behind it as they were."""
    n = 1300 if dtype == torch.float32 else 2300
    b = Batch([n], [1], dtype, 1, dim, 16, 5, seed=28)
    q = b.normal(1, 5, dim, by=1.5).cuda()
    cache, table, lens, starts = b.gpu()
    L = serving._lib()
    size = serving._work_bytes(1, 16, dim, serving._TYPES[dtype], table.shape[1], 1, prompt, 5, prompt)
    assert size // (4 * (dim + 2)) % 2 == 1
    work = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    args = (cache._c, serving._seqs(cache, table, lens, starts, prompt)[0], serving._rows(q, "q", cache),
            serving._rows(out, "out", cache), 5, 0.1, work.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert (L.rpg_hip_paged_prompt if prompt else L.rpg_hip_paged_decode)(*args) == 0
    kk, there = plain.sequence_rows(b.k, b.table[0], n)
    vv, _ = plain.sequence_rows(b.v, b.table[0], n)
    close(out[0], *plain.attention(q[0].cpu(), kk, vv, there, float(torch.tensor(0.1)), dtype))
    assert bool((work[size:] == 0xA5).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_decode_masked_places_hold_anything(dtype, value):
    """Rows past the length, spare pages and pages that the table names no more."""
    b = Batch([37, 130, 16, 700], [1] * 4, dtype, 2, 128, 16, 8, seed=6)
    used = torch.zeros(b.n_pages, 16, dtype=torch.bool)
    b.table[1, 3] = -1
    b.table[3, 20] = b.n_pages + 5
    b.table[2, 0] = 1 << 30  # the whole of a sequence
    for i, n in enumerate(b.lens):
        for p in range(n):
            at = int(b.table[i, p // 16])
            if 0 <= at < b.n_pages:
                used[at, p % 16] = True
    hold = (~used)[:, None, :, None]
    kb, vb = b.k.clone(), b.v.clone()
    b.k, b.v = b.k.masked_fill(hold, value), b.v.masked_fill(hold, value)
    q = b.normal(4, 8, 128)
    cache, table, lens, _ = b.gpu()
    got = serving.decode_attention(q.cuda(), cache, table, lens)
    for i, n in enumerate(b.lens):
        kk, there = plain.sequence_rows(kb, b.table[i], n)
        vv, _ = plain.sequence_rows(vb, b.table[i], n)
        want, bound = plain.attention(q[i], kk, vv, there, 128 ** -0.5, dtype)
        close(got[i], want, bound)


# ---- prompt attention


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (64, 5, 1, 32), (128, 3, 3, 64), (64, 34, 2, 16)])
def test_prompt(dtype, dim, heads, kv, page):
    lens, new = [70, 33, 1, 5, 130, 64, 0, 100], [70, 3, 1, 0, 40, 64, 0, 1]
    b = Batch(lens, new, dtype, kv, dim, page, heads, seed=7)
    q = b.normal(b.tokens + 3, heads, dim, by=1.5)
    cache, table, lens_d, starts = b.gpu()
    out = torch.full((b.tokens + 3, heads, dim), 5.0, dtype=dtype, device="cuda")
    assert serving.prompt_attention(q.cuda(), cache, table, lens_d, starts, scale=0.1, out=out) is out
    want, bound = expect_prompt(b, q, 0.1)
    close(out[:b.tokens], want, bound)
    assert bool((out[b.tokens:] == 5).all())  # rows behind the last sequence
    assert torch.equal(serving.prompt_attention(q.cuda(), cache, table, lens_d, starts, scale=0.1)[:b.tokens],
                       out[:b.tokens])


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_prompt_behind_a_long_history(dtype):
    b = Batch([900, 1500, 333], [7, 1, 20], dtype, 1, 128, 64, 2, seed=8)
    b.k[int(b.table[0, 5]), 0, 3] *= 5  # the maximum moves
    q = b.normal(b.tokens, 2, 128, by=1.5)
    cache, table, lens, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    close(got, *expect_prompt(b, q, 128 ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_prompt_masked_places_hold_anything(dtype, value):
    """Nothing of a later token, a row past the length or an unnamed page reaches a
    query that does not see it; the queries that see it have it."""
    b = Batch([70, 30, 97], [70, 12, 50], dtype, 2, 128, 16, 8, seed=9)
    b.table[2, 1] = -1
    used = torch.zeros(b.n_pages, 16, dtype=torch.bool)
    for i, n in enumerate(b.lens):
        for p in range(n):
            at = int(b.table[i, p // 16])
            if at >= 0:
                used[at, p % 16] = True
    hold = (~used)[:, None, :, None]
    b.k, b.v = b.k.masked_fill(hold, value), b.v.masked_fill(hold, value)
    clean = b.v.clone()
    pos, head, d = 41, 1, 77  # a value of the first sequence's own
    b.v[int(b.table[0, pos // 16]), head, pos % 16, d] = value
    q = b.normal(b.tokens, 8, 128)
    cache, table, lens, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts).double().cpu()
    hit = got[pos:70, 4 * head:4 * head + 4, d]
    assert bool(hit.isnan().all()) if math.isnan(value) else bool((hit == value).all())
    v2 = clean.masked_fill(hold, 0.0)
    k2 = b.k.masked_fill(hold, 0.0)
    want, bound = expect_prompt(b, q, 128 ** -0.5, k2, v2)
    got[pos:70, 4 * head:4 * head + 4, d] = want[pos:70, 4 * head:4 * head + 4, d]
    close(got, want, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("lens,new", [([300], [150]), ([900], [3]), ([700] * 8, [300] * 8)], ids=["mid", "few", "many"])
def test_prompt_infinities_that_every_query_sees(dtype, lens, new):
    """Infinite values early in a sequence: every query has them, of either sign,
    and NaN where both meet."""
    b = Batch(lens, new, dtype, 2, 128, 16, 8, seed=23)
    at = int(b.table[0, 0])
    b.v[at, 0, 2, 5], b.v[at, 0, 9, 6] = math.inf, -math.inf
    b.v[at, 1, 3, 7], b.v[at, 1, 4, 7] = math.inf, -math.inf
    q = b.normal(b.tokens, 8, 128)
    cache, table, lens_d, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts).double().cpu()
    n = new[0]
    assert bool((got[:n, :4, 5] == math.inf).all()) and bool((got[:n, :4, 6] == -math.inf).all())
    assert bool(got[:n, 4:, 7].isnan().all())
    ok = torch.ones_like(got, dtype=torch.bool)
    ok[:n, :4, 5:7] = False
    ok[:n, 4:, 7] = False
    assert bool(got[ok].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("lens,new", [([300], [150]), ([900], [3]), ([700] * 8, [300] * 8)], ids=["mid", "few", "many"])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_an_infinite_key(dtype, lens, new, value):
    """A score of -inf gives its key no weight; one of +inf makes the row NaN
    (inf - inf). The same for one new token."""
    b = Batch(lens, new, dtype, 2, 128, 16, 8, seed=24)
    d, pos = 37, 5
    b.k[int(b.table[0, 0]), :, pos, d] = value
    q = b.normal(b.tokens, 8, 128)
    q[:, :, d] = torch.where(q[:, :, d] < 0, -1.0, 1.0).to(dtype)
    cache, table, lens_d, starts = b.gpu()
    last = starts[1:].long() - 1
    many = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts)
    one = serving.decode_attention(q.cuda()[last], cache, table, lens_d)
    kk, there = plain.sequence_rows(b.k, b.table[0], lens[0])
    vv, _ = plain.sequence_rows(b.v, b.table[0], lens[0])
    kk[:, pos] = 0.0
    for j in (0, new[0] // 2, new[0] - 1):
        seen = there & (torch.arange(lens[0]) <= lens[0] - new[0] + j)
        seen[pos] = False
        want, bound = plain.attention(q[j], kk, vv, seen, 128 ** -0.5, dtype)
        up = q[j, :, d].double() * value > 0
        for got in [many[j]] + ([one[0]] if j == new[0] - 1 else []):
            assert bool(got.cpu()[up].isnan().all())
            close(got.cpu()[~up], want[~up], bound[~up])
    assert bool(many[new[0]:].isfinite().all()) and bool(one[1:].isfinite().all())


@pytest.mark.parametrize("tokens", [1, 2])
def test_f16_many_light_keys_beside_a_heavy_one(tokens):
    """One key takes nearly all the weight, 20000 others have 2^-25.4 of it each:
    less than half of f16's smallest step, and together all of the output."""
    n, page = 20000, 16
    k, v = torch.zeros(2, 1, page, 64, dtype=torch.float16), torch.ones(2, 1, page, 64, dtype=torch.float16)
    k[0, 0, 0, :16] = 1.1
    v[0, 0, 0] = 0.0
    table = torch.ones(1, n // page, dtype=torch.int32)
    table[0, 0] = 0
    q = torch.zeros(tokens, 1, 64, dtype=torch.float16)
    q[:, :, :16] = 8.0
    cache = serving.PagedCache(k.cuda(), v.cuda())
    lens = torch.tensor([n], dtype=torch.int32)
    if tokens == 1:
        got = serving.decode_attention(q.cuda(), cache, table.cuda(), lens.cuda()).double().cpu()
    else:
        starts = torch.tensor([0, tokens], dtype=torch.int32)
        got = serving.prompt_attention(q.cuda(), cache, table.cuda(), lens.cuda(), starts.cuda()).double().cpu()
    heavy = float(k[0, 0, 0, 0].double()) * 8.0 * 16 * 0.125
    assert 2.0 ** -26 < math.exp(-heavy) < 2.0 ** -25
    for t in range(tokens):
        rest = (n - tokens + t) * math.exp(-heavy)
        want = rest / (1.0 + rest)
        # A weight's rounding: half a step of 2^-24 / 2^7 (the least lift) of the
        # heaviest; sums of 20000 in fp32; the score (18 roundings of at most 2^-24
        # of it, twice); the output's rounding.
        rel = 2.0 ** -32 / math.exp(-heavy) + n * 2.0 ** -23 + 36 * heavy * 2.0 ** -24 + 2.0 ** -11
        assert float((got[t] - want).abs().max()) <= rel * want


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("lens,new", [([70, 30], [70, 12]), ([900, 40], [3, 1]), ([500] * 9, [140] * 9)])
def test_attention_in_place(dtype, lens, new):
    """out = q: the same bits as out of its own."""
    b = Batch(lens, new, dtype, 2, 64, 16, 8, seed=25)
    q = b.normal(b.tokens, 8, 64).cuda()
    cache, table, lens_d, starts = b.gpu()
    want = serving.prompt_attention(q, cache, table, lens_d, starts)
    one = q[: len(lens)].clone()
    want_one = serving.decode_attention(one, cache, table, lens_d)
    assert serving.prompt_attention(q, cache, table, lens_d, starts, out=q) is q
    serving.decode_attention(one, cache, table, lens_d, out=one)
    assert torch.equal(q, want) and torch.equal(one, want_one)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_one_token_in_place_with_another_token_stride(dtype):
    """The distance of tokens says nothing where there is one."""
    b = Batch([70], [1], dtype, 2, 64, 16, 8, seed=29)
    q = b.normal(1, 8, 64).cuda()
    cache, table, lens, starts = b.gpu()
    L = serving._lib()
    wants = [(L.rpg_hip_paged_decode, serving.decode_attention(q, cache, table, lens)),
             (L.rpg_hip_paged_prompt, serving.prompt_attention(q, cache, table, lens, starts))]
    seqs = serving._seqs(cache, table, lens, starts, 1)[0]
    stream = torch.cuda.current_stream().cuda_stream
    for call, want in wants:
        x = q.clone()
        r, o = (serving._ROWS.pack(x.data_ptr(), n, 64) for n in (512, 4096))
        assert serving._work_bytes(2, 16, 64, serving._TYPES[dtype], table.shape[1], 1, 1, 8, 1) == 0
        assert call(cache._c, seqs, r, o, 8, 0.125, None, 0, stream) == 0
        assert torch.equal(x, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_prompt_many_short_turns(dtype):
    """More row tiles than compute units, most of them partly filled: ragged ends,
    pages that are not named, NaN in every place that no query sees."""
    lens = [5 + 7 * i % 101 for i in range(44)]
    new = [min(n, 1 + 5 * i % 13) for i, n in enumerate(lens)]
    b = Batch(lens, new, dtype, 8, 128, 16, 8, seed=26)
    used = torch.zeros(b.n_pages, 16, dtype=torch.bool)
    for i, n in enumerate(lens):
        if i % 9 == 4 and n > 16:
            b.table[i, 0] = b.n_pages + i
        for p in range(n):
            at = int(b.table[i, p // 16])
            if at < b.n_pages:
                used[at, p % 16] = True
    hold = (~used)[:, None, :, None]
    k2, v2 = b.k.masked_fill(hold, 0.0), b.v.masked_fill(hold, 0.0)
    b.k, b.v = b.k.masked_fill(hold, math.nan), b.v.masked_fill(hold, math.nan)
    q = b.normal(b.tokens, 8, 128)
    cache, table, lens_d, starts = b.gpu()
    want, bound = expect_prompt(b, q, 128 ** -0.5, k2, v2)
    close(serving.prompt_attention(q.cuda(), cache, table, lens_d, starts), want, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("lens", [[530, 690, 41], [2300, 1700, 3]], ids=["groups", "ranges"])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_few_rows_of_many_keys(dtype, lens, dim):
    """Turns behind long histories, a page of each not named, NaN in the places that
    no query sees, and a value of the history infinite."""
    new = [9, 4, 2]
    b = Batch(lens, new, dtype, 2, dim, 32, 6, seed=27)
    used = torch.zeros(b.n_pages, 32, dtype=torch.bool)
    for i, n in enumerate(lens):
        if n > 100:
            b.table[i, 3] = -5
        for p in range(n):
            at = int(b.table[i, p // 32])
            if at >= 0:
                used[at, p % 32] = True
    hold = (~used)[:, None, :, None]
    k2, v2 = b.k.masked_fill(hold, 0.0), b.v.masked_fill(hold, 0.0)
    b.k, b.v = b.k.masked_fill(hold, math.nan), b.v.masked_fill(hold, math.nan)
    at, d = int(b.table[0, 8]), 33
    b.v[at, 1, 7, d] = -math.inf
    q = b.normal(b.tokens, 6, dim)
    cache, table, lens_d, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts).double().cpu()
    want, bound = expect_prompt(b, q, dim ** -0.5, k2, v2)
    assert bool((got[:9, 3:, d] == -math.inf).all())
    got[:9, 3:, d] = want[:9, 3:, d]
    close(got, want, bound)


def test_prompt_more_tokens_than_positions():
    """Tokens before the cache's first position see no key: zeros."""
    b = Batch([3, 0], [5, 2], torch.float16, seed=10)
    q = b.normal(7, 4, 128)
    cache, table, lens, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    assert bool((got[:2] == 0).all()) and bool((got[5:] == 0).all())
    want, bound = expect_prompt(b, q, 128 ** -0.5)
    close(got, want, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_prompt_agrees_with_decode(dtype):
    """A sequence's last token alone, and as the end of its prompt."""
    b = Batch([200, 77], [9, 3], dtype, 2, 128, 32, 8, seed=11)
    q = b.normal(b.tokens, 8, 128)
    cache, table, lens, starts = b.gpu()
    many = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    one = serving.decode_attention(q.cuda()[[8, 11]], cache, table, lens)
    want, bound = expect_prompt(b, q, 128 ** -0.5)
    close(many, want, bound)
    close(one, want[[8, 11]], bound[[8, 11]])


def test_prompt_agrees_with_the_engine():
    """The engine's own prefill attention on a contiguous f32 cache."""
    b = Batch([150], [60], torch.float32, 2, 128, 16, 8, seed=12)
    q = b.normal(60, 8, 128)
    cache, table, lens, starts = b.gpu()
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    k, _ = plain.sequence_rows(b.k, b.table[0], 150)
    v, _ = plain.sequence_rows(b.v, b.table[0], 150)
    theirs = eng.attention(q.numpy(), k.float().numpy(), v.float().numpy(), 90)
    want, bound = expect_prompt(b, q, 128 ** -0.5)
    close(got, want, bound)
    # theirs: 22-bit operands and one more product's rounding of 2^-22 each
    assert float((got.cpu() - torch.from_numpy(theirs)).abs().max()) <= float(2 * bound.max()) + 1e-5


# ---- layouts, streams, graphs


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_strided_pools_queries_and_outputs(dtype):
    """One pool holding k and v side by side, rows with gaps, heads in front of
    positions, queries and outputs inside larger tensors."""
    b = Batch([45, 18], [6, 2], dtype, 2, 64, 16, 4, seed=13)
    kv = torch.zeros(b.n_pages, 16, 2, 2, 64 + 16, dtype=dtype, device="cuda")  # [page, position, k or v, head, dim + gap]
    k, v = kv[:, :, 0, :, :64].permute(0, 2, 1, 3), kv[:, :, 1, :, :64].permute(0, 2, 1, 3)
    k.copy_(b.k)
    v.copy_(b.v)
    cache = serving.PagedCache(k, v)
    wide_table = torch.full((2, 40), 12345, dtype=torch.int32, device="cuda")
    wide_table[:, :b.table.shape[1]] = b.table.cuda()
    table = wide_table[:, :b.table.shape[1]]
    lens, starts = b.len_t.cuda(), b.starts.cuda()
    big_q = b.normal(8, 9, 64 * 2).cuda()
    q = big_q[:, 2:6, 64:]
    big_o = torch.full((4, 8, 64), 3.0, dtype=dtype, device="cuda")
    out = big_o.transpose(0, 1)  # heads in front of tokens
    serving.prompt_attention(q, cache, table, lens, starts, out=out)
    close(out, *expect_prompt(b, q.cpu(), 64 ** -0.5))
    one = serving.decode_attention(q[[5, 7]], cache, table, lens, out=out[:2])
    want, bound = expect_prompt(b, q.cpu(), 64 ** -0.5)
    close(one, want[[5, 7]], bound[[5, 7]])
    new = b.normal(8, 2, 64).cuda()
    serving.append(cache, table, lens, starts, new, new)
    at = int(b.table[0, 2])
    assert torch.equal(k[at, :, 44 % 16], new[5]) and torch.equal(v[at, :, 44 % 16], new[5])
    assert float(kv[..., 64:].abs().max()) == 0  # the gaps


def test_pages_past_32_bit_offsets():
    """A pool of more than 2^32 bytes and elements: its far pages."""
    dtype, kv, dim, page = torch.float16, 8, 128, 256
    n = (1 << 32) // (kv * dim * page) + 40
    k = torch.empty(n, kv, page, dim, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(14)
    pages = [n - 1, 3, n - 2]
    for p in pages:
        k[p] = torch.randn(kv, page, dim, generator=g).to(dtype).cuda()
        v[p] = torch.randn(kv, page, dim, generator=g).to(dtype).cuda()
    cache = serving.PagedCache(k, v)
    table = torch.tensor([pages], dtype=torch.int32, device="cuda")
    lens = torch.tensor([700], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    new = torch.randn(2, kv, dim, generator=g).to(dtype).cuda()
    serving.append(cache, table, lens, starts, new, new)
    q = torch.randn(2, kv, dim, generator=g).to(dtype)
    kk = torch.cat([k[p].cpu() for p in pages], 1).double()[:, :700]
    vv = torch.cat([v[p].cpu() for p in pages], 1).double()[:, :700]
    assert torch.equal(kk[:, 699], new[1].cpu().double())
    want, bound = plain.attention(q[1], kk, vv, torch.ones(700, dtype=torch.bool), dim ** -0.5, dtype)
    close(serving.decode_attention(q[1:].cuda(), cache, table, lens)[0], want, bound)
    close(serving.prompt_attention(q.cuda(), cache, table, lens, starts)[1], want, bound)


def test_other_streams():
    b = Batch([500, 33], [1, 1], torch.bfloat16, 2, 128, 16, 8, seed=15)
    q = b.normal(2, 8, 128).cuda()
    cache, table, lens, _ = b.gpu()
    want = serving.decode_attention(q, cache, table, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(serving.decode_attention(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_graphs_replay_with_the_lengths_of_the_moment():
    """A serving step captured twice (two graphs, replayed in turn) with eager work
    between the replays: each replay takes the lengths, tables, random numbers
    and tokens that are there then."""
    b = Batch([40, 9], [1, 1], torch.float32, 2, 64, 16, 4, seed=16, spare=20, extra_pages=20)
    cache, table, lens, starts = b.gpu()
    free = [p for p in range(b.n_pages) if p not in b.table.tolist()[0] + b.table.tolist()[1]]
    for i in range(2):
        for j in range(3, 12):
            table[i, j] = free[i * 9 + j - 3]
    k, v, q = (b.normal(2, h, 64).cuda() for h in (2, 2, 4))
    logits = torch.randn(2, 501, generator=b.gen).cuda()
    u = torch.tensor([0.3, 0.8]).cuda()
    temp = torch.tensor([0.7, 0.0]).cuda()
    top_p = torch.tensor([0.9, 0.9]).cuda()

    def step():
        serving.append(cache, table, lens, starts, k, v)
        out = serving.decode_attention(q, cache, table, lens)
        tokens, lp = serving.sample(logits, u, temp, None, top_p)
        return out, serving.prompt_attention(q, cache, table, lens, starts), tokens, lp

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for r in range(6):
        g, outs = graphs[r % 2]
        lens += 11
        u.copy_(torch.rand(2, generator=b.gen))
        logits.copy_(torch.randn(2, 501, generator=b.gen))
        q.copy_(torch.randn(2, 4, 64, generator=b.gen))
        k.copy_(torch.randn(2, 2, 64, generator=b.gen))
        for o in outs:
            o.fill_(0)
        g.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w), r


def test_a_conversation():
    """Prompts of three sequences, then decode steps, as a host runs them: append,
    attention, sample; every step against float64 over the whole history."""
    kv, heads, dim, page, vocab = 2, 8, 128, 16, 300
    g = torch.Generator().manual_seed(17)
    cache = serving.PagedCache.zeros(40, page, kv, dim, torch.float32)
    table = torch.full((3, 10), -1, dtype=torch.int32)
    order = torch.randperm(40, generator=g)
    table[:, :] = order[:30].reshape(3, 10)
    ang = torch.arange(160)[:, None] * torch.pow(1e4, -torch.arange(64) / 64.0)
    rope = torch.cat([ang.cos(), ang.sin()], 1).float()
    head = torch.randn(heads * dim, vocab, generator=g) / 30
    hist = [[torch.zeros(kv, 0, dim), torch.zeros(kv, 0, dim)] for _ in range(3)]
    lens = [0, 0, 0]
    gain = torch.ones(dim)
    for new in [[50, 17, 1], [1, 1, 1], [1, 1, 1], [4, 1, 20], [1, 1, 1]]:
        n = sum(new)
        q, k, v = (torch.randn(n, h, dim, generator=g) for h in (heads, kv, kv))
        starts = [sum(new[:i]) for i in range(4)]
        lens = [a + b for a, b in zip(lens, new)]
        ld, sd = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda()
        qr = serving.append(cache, table.cuda(), ld, sd, k.cuda(), v.cuda(), q=q.cuda(), q_norm=gain.cuda(),
                            k_norm=gain.cuda(), rope=rope.cuda())
        one = max(new) == 1
        out = (serving.decode_attention(qr, cache, table.cuda(), ld) if one else
               serving.prompt_attention(qr, cache, table.cuda(), ld, sd))
        for i in range(3):
            for j in range(new[i]):
                t, pos = starts[i] + j, lens[i] - new[i] + j
                kk, _ = plain.turned(k[t], gain, 1e-6, rope[pos])
                hist[i][0] = torch.cat([hist[i][0], kk[:, None].float()], 1)
                hist[i][1] = torch.cat([hist[i][1], v[t][:, None]], 1)
                qq, _ = plain.turned(q[t], gain, 1e-6, rope[pos])
                want, bound = plain.attention(qq, hist[i][0].double(), hist[i][1].double(),
                                              torch.ones(pos + 1, dtype=torch.bool), dim ** -0.5, torch.float32)
                # the cache's keys and the queries are each 32 roundings off (turned_bound):
                # scores by 2 x 2 x 32 x 2^-24 of sum |q k| <= dim, weights by twice that
                close(out[t], want, bound + 4 * 64 * 2.0 ** -24 * dim ** 0.5 * hist[i][1].abs().max())
        last = out[[s - 1 for s in starts[1:]]].reshape(3, -1)
        logits = last.cpu() @ head
        u = torch.rand(3, generator=g)
        tokens, lp = serving.sample(logits.cuda(), u.cuda(), torch.tensor([0.8, 1.0, 0.0]).cuda(), None, None,
                                    torch.tensor([0.05, 0.0, 0.5]).cuda())
        for i, t in enumerate([0.8, 1.0, 0.0]):
            tok, want = plain.sample(logits[i], float(u[i]), float(torch.tensor(t)), 0, 1.0, [float(torch.tensor(0.05)), 0.0, 0.5][i])
            assert int(tokens[i]) == tok
            assert abs(float(lp[i]) - want) <= 2.0 ** -24 * abs(want) + 1e-7


# ---- sampling

GRID = list(itertools.product([0.0, 0.4, 1.0, 3.0], [0, 1, 7, 50], [1.0, 0.3, 0.95], [0.0, 0.1, 1.0]))


def check_samples(x, u, t, k, p, m):
    tokens, lp = serving.sample(x.cuda(), u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    tokens, lp = tokens.cpu(), lp.cpu()
    for i in range(x.shape[0]):
        want, logp = plain.sample(x[i], float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        assert int(tokens[i]) == want, (i, float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        # the sum of V weights is within V 2^-45 of exact; then one rounding
        if logp == -math.inf:
            assert float(lp[i]) == logp
        else:
            assert abs(float(lp[i]) - logp) <= 2.0 ** -24 * abs(logp) + x.shape[1] * 2.0 ** -44 + 1e-10, i


def params(rows, dtype=torch.float32):
    g = [GRID[i % len(GRID)] for i in range(rows)]
    return (torch.tensor([r[0] for r in g]), torch.tensor([r[1] for r in g], dtype=torch.int32),
            torch.tensor([r[2] for r in g]), torch.tensor([r[3] for r in g]))


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 4097, 20011])
def test_sample_grid(dtype, vocab):
    """Every combination of the limits, at odd sizes (rows that start at no
    multiple of 16 bytes)."""
    g = torch.Generator().manual_seed(vocab)
    rows = len(GRID)
    x = (torch.randn(rows, vocab, generator=g) * 2.5).to(dtype)
    check_samples(x, torch.rand(rows, generator=g), *params(rows))


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_sample_full_vocabulary(dtype):
    g = torch.Generator().manual_seed(18)
    rows, vocab = 24, 151936
    x = torch.randn(rows, vocab, generator=g)
    x[::2] *= 2.5
    x[::3, 77:120] += 8
    t = torch.tensor([0.7, 1.0, 0.3, 5.0]).repeat(6)
    k = torch.tensor([0, 40, 0, 30000, 5000, 0], dtype=torch.int32).repeat(4)
    p = torch.tensor([0.95, 1.0, 0.9]).repeat(8)
    m = torch.tensor([0.0, 0.0, 0.0, 0.02, 0.0]).repeat(5)[:rows]
    check_samples(x.to(dtype), torch.rand(rows, generator=g), t, k, p, m)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("vocab", [4099, 20011, 65541])
def test_sample_small_top_k(dtype, vocab):
    """Few tokens of many: the best ones side by side at the row's end, in
    order, spread, alike, among NaN of every kind."""
    g = torch.Generator().manual_seed(vocab + 1)
    x = torch.randn(7, vocab, generator=g)
    x[0, -3:] += 20
    x[1] = torch.arange(vocab) * (40.0 / vocab)
    x[2] = torch.arange(vocab, 0, -1) * (40.0 / vocab)
    x[3] = torch.arange(vocab) % 2
    x[4, ::2] = -math.inf
    x[5, 7:] = -math.inf
    x = x.to(dtype)
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    one = {torch.float32: 0x7F800001, torch.float16: 0x7C01, torch.bfloat16: 0x7F81}[dtype]  # a signalling NaN
    bits[6, ::3], x[6, 1::3] = one, math.nan
    for k in (1, 2, 3, 5, 16, 40, 64, 100, 128):
        rows = x.shape[0]
        check_samples(x, torch.rand(rows, generator=g), torch.full((rows,), 0.8), torch.full((rows,), k, dtype=torch.int32),
                      torch.tensor([1.0, 0.9, 1.0, 0.5, 1.0, 0.9, 0.7]), torch.tensor([0.0, 0.0, 0.1, 0.0, 0.2, 0.0, 0.0]))


def test_sample_ties_and_flat_rows():
    """Equal values: the lowest indices stay; lists longer than the kernel ranks in
    shared memory; temperatures that flatten or sharpen everything."""
    vocab = 9000
    rows = []
    g = torch.Generator().manual_seed(19)
    rows.append(torch.zeros(vocab))                                   # all equal
    rows.append(torch.randint(0, 3, (vocab,), generator=g).float())   # three values
    rows.append(torch.randint(-40, 40, (vocab,), generator=g) / 16)   # some tens
    rows.append(torch.randn(vocab, generator=g))
    rows.append(torch.full((vocab,), -3.0))
    rows[4][8999] = 20.0
    x, u, t, k, p, m = [], [], [], [], [], []
    for r, tt, (kk, pp, mm) in itertools.product(rows, [1.0, 1e-3, 1e6, math.inf], [
            (0, 1.0, 0.0), (1500, 1.0, 0.0), (0, 0.37, 0.0), (4000, 0.5, 0.0), (100, 0.9, 0.0), (0, 1.0, 0.9),
            (8999, 0.99, 1e-3)]):
        x.append(r)
        u.append(float(torch.rand(1, generator=g)))
        t.append(tt)
        k.append(kk)
        p.append(pp)
        m.append(mm)
    check_samples(torch.stack(x), torch.tensor(u), torch.tensor(t), torch.tensor(k, dtype=torch.int32), torch.tensor(p),
                  torch.tensor(m))


def sample_into(x, u, t, k, p, m, fill):
    """serving.sample's call with work memory and outputs that hold `fill` in every byte."""
    rows, vocab = x.shape
    L = serving._lib()
    size = L.rpg_hip_sample_rows_work(rows, vocab)
    work = torch.full((size,), fill, dtype=torch.uint8, device="cuda")
    tokens, lp = (torch.full((4 * rows,), fill, dtype=torch.uint8, device="cuda").view(d) for d in (torch.int32, torch.float32))
    dev = [v.cuda() for v in (x, t, k, p, m, u)]
    rc = L.rpg_hip_sample_rows(serving._TYPES[x.dtype], dev[0].data_ptr(), rows, vocab, vocab, *[v.data_ptr() for v in dev[1:]],
                               tokens.data_ptr(), lp.data_ptr(), work.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return tokens.cpu(), lp.cpu()


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("vocab", [700, 20011, 151936])
def test_sample_temperatures_next_to_zero(dtype, vocab):
    """Down to the smallest number above 0 they are temperatures: the best token,
    or a draw among those that are equal, or nearly so, to it. Nothing is taken
    from what work memory and outputs held."""
    g = torch.Generator().manual_seed(vocab + 3)
    base = torch.randn(4, vocab, generator=g) * 2.5
    base[1, [5, vocab // 2, vocab - 1]] = 30.0  # equal ones
    base[2, ::3] = 25.0                         # more of them than a list holds
    base[3] = torch.where(torch.rand(vocab, generator=g) < 0.01, torch.randn(vocab, generator=g) * 1e-37, -1.0)
    x, u, t, k, p, m = [], [], [], [], [], []
    for row, tt, (kk, pp, mm) in itertools.product(base, [1e-30, 1e-36, 2e-37, 1e-37, torch.finfo(torch.float32).tiny, 1e-39, 1e-45], [
            (0, 1.0, 0.0), (1, 1.0, 0.0), (40, 1.0, 0.0), (5000, 1.0, 0.0), (0, 0.9, 0.0), (1, 0.9, 0.0), (40, 0.9, 0.0),
            (5000, 0.9, 0.0), (0, 1.0, 0.5), (40, 0.5, 0.5)]):
        x.append(row)
        for v, w in zip((u, t, k, p, m), (float(torch.rand(1, generator=g)), tt, kk, pp, mm)):
            v.append(w)
    x = torch.stack(x).to(dtype)
    u, t, p, m = (torch.tensor(v) for v in (u, t, p, m))
    k = torch.tensor(k, dtype=torch.int32)
    assert bool((t > 0).all())
    want = [plain.sample(x[i], float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i])) for i in range(len(u))]
    for fill in (0x7F, 0xFF):
        tokens, lp = sample_into(x, u, t, k, p, m, fill)
        for i, (token, logp) in enumerate(want):
            assert int(tokens[i]) == token, (i, float(t[i]), int(k[i]), float(p[i]), float(m[i]))
            # as in check_samples
            assert abs(float(lp[i]) - logp) <= 2.0 ** -24 * abs(logp) + vocab * 2.0 ** -44 + 1e-10, i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ident)
def test_sample_temperatures_next_to_infinity(dtype):
    """Rows whose values lie further apart than a float reaches, at temperatures at
    which all of them, or many, have weight."""
    vocab = 3000
    g = torch.Generator().manual_seed(32)
    # (in float64: the step of one in float32 is infinite, and an infinite value
    # over an infinite temperature is nothing)
    rows = [torch.linspace(-3e38, 3e38, vocab, dtype=torch.float64).float(), torch.where(torch.rand(vocab, generator=g) < 0.5, -3.3e38, 3.3e38),
            torch.randn(vocab, generator=g)]
    x, u, t, k, p, m = [], [], [], [], [], []
    for row, tt, (kk, pp, mm) in itertools.product(rows, [5e36, 1.2e37, 3e37, 1e38, 3e38, math.inf], [
            (0, 1.0, 0.0), (5, 1.0, 0.0), (450, 0.9, 0.0), (2900, 1.0, 0.0), (0, 0.9, 0.0), (2500, 0.7, 0.0), (0, 1.0, 0.1),
            (0, 0.99, 0.5)]):
        x.append(row)
        for v, w in zip((u, t, k, p, m), (float(torch.rand(1, generator=g)), tt, kk, pp, mm)):
            v.append(w)
    check_samples(torch.stack(x).to(dtype), torch.tensor(u), torch.tensor(t), torch.tensor(k, dtype=torch.int32),
                  torch.tensor(p), torch.tensor(m))


def test_sample_rows_that_hold_little():
    """Infinities, NaN, rows with one value, with none."""
    inf, nan = math.inf, math.nan
    vocab = 300
    x = torch.full((8, vocab), -inf)
    x[1, 299] = -4.0
    x[2, :] = nan
    x[3, 5:9] = torch.tensor([1.0, nan, 1.5, 0.2])
    x[4] = torch.linspace(-2, 2, vocab)
    x[4, [20, 250]] = inf
    x[5] = torch.finfo(torch.float32).min
    x[6] = torch.linspace(-3e38, 3e38, vocab)
    x[7, 3], x[7, 9] = -0.0, 0.0
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.5, 2, 0.9, 0.1), (0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.0), (2.0, 0, 0.6, 0.0)]:
        for uu in (0.0, 0.4, 0.99):
            full = [torch.full((8,), float(v)) for v in (uu, t, p, m)]
            check_samples(x, full[0], full[1], torch.full((8,), k, dtype=torch.int32), full[2], full[3])


def test_sample_numbers_outside_and_absent_parameters():
    g = torch.Generator().manual_seed(20)
    x = torch.randn(5, 1000, generator=g).cuda()
    u = torch.tensor([-1.0, 0.0, 1.0, 2.0, math.nan]).cuda()
    tokens, _ = serving.sample(x, u)
    assert tokens.tolist() == [0, 0, 999, 999, 999]
    params = [torch.tensor([math.nan] * 5).cuda() for _ in range(3)]
    tokens, lp = serving.sample(x, u.clamp(0, 0.5).nan_to_num(0.5), params[0], None, params[1], params[2])
    assert tokens.tolist() == x.argmax(1).tolist() and lp.tolist() == [0.0] * 5  # no temperature: the best
    a = serving.sample(x, u, torch.ones(5).cuda(), None, params[1], params[2])[0]
    assert a.tolist() == [0, 0, 999, 999, 999]  # no limits


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
def test_sample_limits_that_are_absent(dtype):
    """No top_k and top_p: as arrays that set none; other calls in between."""
    g = torch.Generator().manual_seed(22)
    x = (torch.randn(9, 20011, generator=g) * 3).to(dtype).cuda()
    u, t = torch.rand(9, generator=g).cuda(), torch.full((9,), 0.9).cuda()
    k, p, m = torch.zeros(9, dtype=torch.int32).cuda(), torch.ones(9).cuda(), torch.full((9,), 0.05).cuda()
    for min_p in (None, m):
        want = serving.sample(x, u, t, k, p, min_p)
        serving.sample(x, u, t, k + 5, p * 0.5, min_p)
        for top_k, top_p in ((None, None), (k, None), (None, p)):
            got = serving.sample(x, u, t, top_k, top_p, min_p)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sample_strided_rows_and_repeats():
    g = torch.Generator().manual_seed(21)
    big = (torch.randn(6, 5000, generator=g) * 2).to(torch.bfloat16)
    x = big[:, 3:4000]
    u = torch.rand(6, generator=g)
    check_samples(x.contiguous(), u, *[v[:6] for v in params(40)])
    t, k, p, m = [v[20:26].cuda() for v in params(40)]
    a = serving.sample(x.cuda(), u.cuda(), t, k, p, m)
    b = serving.sample(big.cuda()[:, 3:4000], u.cuda(), t, k, p, m)
    same = serving.sample(big.cuda()[:1, 3:4000].expand(6, -1), u.cuda())
    first = serving.sample(big.cuda()[:1, 3:4000].repeat(6, 1), u.cuda())
    for v, w in zip(a + same, b + first):
        assert torch.equal(v, w)


# ---- refusals that need tensors on a GPU


def test_refusals():
    b = Batch([20], [1], torch.float16, seed=22)
    cache, table, lens, starts = b.gpu()
    q = b.normal(1, 4, 128).cuda()
    bad = [
        lambda: serving.decode_attention(q.float(), cache, table, lens),
        lambda: serving.decode_attention(q[:, :3], cache, table, lens),
        lambda: serving.decode_attention(q, cache, table.long(), lens),
        lambda: serving.decode_attention(q, cache, table, lens.cpu()),
        lambda: serving.decode_attention(q, cache, table, lens, scale=0.0),
        lambda: serving.decode_attention(q, cache, table, lens, scale=math.nan),
        lambda: serving.decode_attention(q, cache, table, lens, out=q[:, :2]),
        lambda: serving.decode_attention(q, cache, table, lens, out=q[:, :1].expand(1, 4, 128)),
        lambda: serving.decode_attention(q.expand(2, 4, 128), cache, table, lens),
        lambda: serving.decode_attention(q.detach().requires_grad_(), cache, table, lens),
        lambda: serving.prompt_attention(q, cache, table, lens, starts[:1]),
        lambda: serving.prompt_attention(torch.zeros(1, 4, 136, dtype=torch.float16).cuda()[..., 4:132], cache, table, lens,
                                         starts),
        lambda: serving.append(cache, table, lens, starts, q[:, :2], q[:, :1]),
        lambda: serving.append(cache, table, lens, starts, q[:, :2], q[:, :2], q=q, q_out=q[:, :2]),
        lambda: serving.append(cache, table, lens, starts, q[:, :2], q[:, :2], rope=torch.zeros(9, 64).cuda()),
        lambda: serving.append(cache, table, lens, starts, q[:, :2], q[:, :2], k_norm=torch.zeros(64).cuda()),
        lambda: serving.PagedCache(cache.k.cpu(), cache.v.cpu()),
        lambda: serving.PagedCache(cache.k, cache.v[:1]),
        lambda: serving.PagedCache(cache.k.double(), cache.v.double()),
        lambda: serving.sample(q[0], torch.zeros(3).cuda()),
        lambda: serving.sample(q[0].double(), torch.zeros(4).cuda()),
        lambda: serving.sample(q[0], torch.zeros(4)),
        lambda: serving.sample(q[0], torch.zeros(4).cuda(), top_k=torch.zeros(4).cuda()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(eng.EngineError):
            f()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        serving.decode_attention(q.detach().requires_grad_(), cache, table, lens)


def test_parameters_that_require_gradients_are_refused():
    b = Batch([4], [1], torch.float32, 1, 64, 16, 2)
    cache, table, lens, starts = b.gpu()
    k, q = b.normal(1, 1, 64).cuda(), b.normal(1, 2, 64).cuda()
    gain = torch.nn.Parameter(torch.ones(64, device="cuda"))
    rope = torch.nn.Parameter(torch.ones(64, 64, device="cuda"))
    one = torch.nn.Parameter(torch.ones(1, device="cuda"))
    x = torch.zeros(1, 5, device="cuda")
    for call in (lambda: serving.append(cache, table, lens, starts, k, k, q=q, q_norm=gain),
                 lambda: serving.append(cache, table, lens, starts, k, k, k_norm=gain),
                 lambda: serving.append(cache, table, lens, starts, k, k, rope=rope),
                 lambda: serving.sample(x, one.detach(), temperature=one),
                 lambda: serving.PagedCache(torch.nn.Parameter(cache.k), cache.v)):
        with pytest.raises(eng.EngineError, match="gradients"):
            call()
    with torch.no_grad():
        serving.append(cache, table, lens, starts, k, k, q=q, q_norm=gain, k_norm=gain, rope=rope)
    for call in (lambda: serving.append(cache, table, lens, starts, k[0], k[0]),
                 lambda: serving.append(cache, table, lens, starts, k, k, q=q[0, 0]),
                 lambda: serving.decode_attention(q[0, 0], cache, table, lens),
                 lambda: serving.prompt_attention(q, cache, table, lens, None)):
        with pytest.raises(eng.EngineError):
            call()


def test_a_cache_whose_tensors_moved_is_refused():
    """Its k and v are those that it was made of, and where they were."""
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, starts = torch.zeros(1, 1, **i32), torch.ones(1, **i32), torch.tensor([0, 1], **i32)
    k, q = torch.ones(1, 1, 64, device="cuda"), torch.ones(1, 2, 64, device="cuda")
    for move in (lambda t: setattr(t, "data", torch.zeros(4, 1, 16, 64, device="cuda")),
                 lambda t: t.untyped_storage().resize_(0)):
        for which in ("k", "v"):
            cache = serving.PagedCache.zeros(2, 16, 1, 64)
            with pytest.raises(AttributeError):
                setattr(cache, which, torch.zeros(4, 1, 16, 64, device="cuda"))
            calls = (lambda: serving.append(cache, table, lens, starts, k, k),
                     lambda: serving.decode_attention(q, cache, table, lens),
                     lambda: serving.prompt_attention(q, cache, table, lens, starts))
            for call in calls:
                call()
            move(getattr(cache, which))
            for call in calls:
                with pytest.raises(eng.EngineError, match="lie elsewhere"):
                    call()


def test_tensors_with_tangents_are_refused():
    """Forward-mode gradients, which the outputs would lose without a word."""
    from torch.autograd import forward_ad
    b = Batch([4], [1], torch.float32, 1, 64, 16, 2, seed=31)
    cache, table, lens, starts = b.gpu()
    k, q, gain, rope, x, one = (torch.ones(*s, device="cuda") for s in ((1, 1, 64), (1, 2, 64), (64,), (64, 64), (1, 5), (1,)))
    calls = [
        (k, lambda t: serving.append(cache, table, lens, starts, t, k)),
        (k, lambda t: serving.append(cache, table, lens, starts, k, t)),
        (q, lambda t: serving.append(cache, table, lens, starts, k, k, q=t)),
        (q, lambda t: serving.append(cache, table, lens, starts, k, k, q=q, q_out=t)),
        (gain, lambda t: serving.append(cache, table, lens, starts, k, k, q=q, q_norm=t)),
        (gain, lambda t: serving.append(cache, table, lens, starts, k, k, k_norm=t)),
        (rope, lambda t: serving.append(cache, table, lens, starts, k, k, rope=t)),
        (q, lambda t: serving.decode_attention(t, cache, table, lens)),
        (q, lambda t: serving.decode_attention(q, cache, table, lens, out=t)),
        (q, lambda t: serving.prompt_attention(t, cache, table, lens, starts)),
        (cache.k, lambda t: serving.PagedCache(t, cache.v)),
        (cache.v, lambda t: serving.PagedCache(cache.k, t)),
        (x, lambda t: serving.sample(t, one)),
        (one, lambda t: serving.sample(x, t)),
        (one, lambda t: serving.sample(x, one, temperature=t)),
    ]
    with forward_ad.dual_level():
        for i, (value, call) in enumerate(calls):
            call(value.clone())  # without one, in the same place
            with pytest.raises(eng.EngineError, match="tangent"):
                call(forward_ad.make_dual(value.clone(), torch.ones_like(value)))
                pytest.fail(f"call {i} was not refused")
    for value, call in calls:
        call(value.clone())


def test_tensors_written_in_place_are_new_versions():
    """The pool, out and q_out: a backward pass that saved one of them refuses,
    instead of taking what was written over it."""
    b = Batch([20], [2], torch.float32, 2, 64, 16, 4, seed=30)
    cache, table, lens, starts = b.gpu()
    k, q = b.normal(2, 2, 64).cuda(), b.normal(2, 4, 64).cuda()
    calls = [(lambda: serving.append(cache, table, lens, starts, k, k), [cache.k, cache.v]),
             (lambda: serving.append(cache, table, lens, starts, k, k, q=q, q_out=q), [cache.k, cache.v, q]),
             (lambda: serving.decode_attention(q[:1], cache, table, lens, out=q[:1]), [q]),
             (lambda: serving.prompt_attention(q, cache, table, lens, starts, out=q), [q])]
    for i, (call, written) in enumerate(calls):
        for x in written:
            leaf = torch.ones_like(x, requires_grad=True)
            loss = (leaf * x).sum()  # saves x
            was = x._version
            call()
            assert x._version > was, i
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():  # tensors without versions
        out = torch.empty_like(q)
        serving.append(cache, table, lens, starts, k, k, q=q, q_out=out)
        serving.prompt_attention(q, cache, table, lens, starts, out=out)
        pool = serving.PagedCache.zeros(2, 16, 2, 64)
        serving.append(pool, table, lens, starts, k, k)


def test_nothing_to_do():
    """No sequence, no token, no row."""
    cache = serving.PagedCache.zeros(2, 16, 1, 64, torch.float32)
    i32 = dict(dtype=torch.int32, device="cuda")
    empty = torch.zeros(0, 2, 64, device="cuda")
    assert serving.decode_attention(empty, cache, torch.zeros(0, 3, **i32), torch.zeros(0, **i32)).shape == (0, 2, 64)
    out = serving.prompt_attention(empty, cache, torch.zeros(1, 3, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32))
    assert out.shape == (0, 2, 64)
    serving.append(cache, torch.zeros(1, 3, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32), empty[:, :1],
                   empty[:, :1])
    none = serving.decode_attention(torch.ones(1, 2, 64, device="cuda"), cache, torch.zeros(1, 0, **i32),
                                    torch.ones(1, **i32))
    assert bool((none == 0).all())  # a table without pages
    assert serving.sample(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda"))[0].shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("tokens", [0, 3])
def test_no_sequences(dtype, tokens):
    """Tables of any width and no sequence: rows of none are left as they were."""
    cache = serving.PagedCache.zeros(2, 16, 2, 128, dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, starts = torch.zeros(0, **i32), torch.zeros(1, **i32)
    for pages in (1, 64, 256):
        table = torch.zeros(0, pages, **i32)
        q = torch.ones(tokens, 8, 128, dtype=dtype, device="cuda")
        out = torch.full_like(q, 7.0)
        serving.prompt_attention(q, cache, table, lens, starts, out=out)
        assert serving.decode_attention(q[:0], cache, table, lens).shape == (0, 8, 128)
        serving.append(cache, table, lens, starts, q[:, :2], q[:, :2], q=q, q_out=out)
        assert bool((out == 7).all()) and bool((cache.k == 0).all()) and bool((cache.v == 0).all())
