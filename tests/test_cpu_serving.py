"""Refusals of the serving operators (include/rpg_hip.h), which come before
anything touches a GPU, and the plain definitions that the GPU tests hold the
kernels to."""

import ctypes
import math

import pytest
import torch

import rpgbarengine_amd as eng
import serving_plain as plain
from rpgbarengine_amd import serving

A = 0x10000  # an address: refused calls follow none
P, I32, I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("page_stride", I64), ("head_stride", I64), ("row_stride", I64), ("n_pages", I32),
                ("page_size", I32), ("n_kv", I32), ("head_dim", I32), ("type", I32)]


class Seqs(ctypes.Structure):
    _fields_ = [("table", P), ("table_stride", I64), ("lens", P), ("starts", P), ("pages", I32), ("n_seqs", I32),
                ("n_tokens", I32)]


class Rows(ctypes.Structure):
    _fields_ = [("data", P), ("token_stride", I64), ("head_stride", I64)]


def cache(**over):
    f = dict(k=A, v=A, page_stride=4 * 16 * 128, head_stride=16 * 128, row_stride=128, n_pages=9, page_size=16, n_kv=4,
             head_dim=128, type=1)
    f.update(over)
    return Cache(**f)


def seqs(**over):
    f = dict(table=A, table_stride=8, lens=A, starts=A, pages=8, n_seqs=3, n_tokens=7)
    f.update(over)
    return Seqs(**f)


def rows(**over):
    f = dict(data=A, token_stride=1024, head_stride=128)
    f.update(over)
    return Rows(**f)


def refused(rc, word):
    assert rc == -1
    said = eng.lib().rpg_hip_last_error().decode()
    assert word in said, said


def ref(x):
    return None if x is None else ctypes.byref(x)


BAD_CACHES = [
    (dict(type=8), "element type"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
    (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=131072), "page_size"),
    (dict(page_size=-16), "page_size"), (dict(n_pages=0), "pages"), (dict(n_kv=0), "key heads"),
    (dict(row_stride=64), "row_stride"), (dict(row_stride=132), "row_stride"), (dict(row_stride=1 << 27), "row_stride"),
    (dict(row_stride=-128), "row_stride"), (dict(head_stride=8), "head_stride"), (dict(page_stride=0), "page_stride"),
    (dict(page_stride=1 << 33), "page_stride"),
]


@pytest.mark.parametrize("over,word", BAD_CACHES, ids=[str(i) for i in range(len(BAD_CACHES))])
def test_bad_caches(over, word):
    L = serving._lib()
    c, s, r = cache(**over), seqs(), rows()
    refused(L.rpg_hip_paged_decode(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, 1 << 40, None), word)
    refused(L.rpg_hip_paged_prompt(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, 1 << 40, None), word)
    refused(L.rpg_hip_paged_append(ref(c), ref(s), ref(r), ref(r), None, None, 0, None, None, 0.0, None, 0, None), word)
    refused(L.rpg_hip_paged_work(ref(c), ref(s), 8, 0), word)


BAD_CALLS = [
    (dict(cache=None), "cache is null"), (dict(seqs=None), "sequences are null"), (dict(cache=cache(k=None)), "k is null"),
    (dict(cache=cache(v=A + 8)), "v does not lie"), (dict(seqs=seqs(n_seqs=-1)), "sequences"),
    (dict(seqs=seqs(n_tokens=-1)), "tokens"), (dict(seqs=seqs(pages=-1)), "pages"),
    (dict(seqs=seqs(pages=1 << 28, table_stride=1 << 28)), "pages"), (dict(seqs=seqs(table=None)), "table is null"),
    (dict(seqs=seqs(table_stride=7)), "table_stride"), (dict(seqs=seqs(lens=None)), "lens is null"),
    (dict(seqs=seqs(lens=A + 2)), "lens does not lie"), (dict(q=None), "q is null"), (dict(q=rows(data=None)), "q is null"),
    (dict(q=rows(data=A + 8)), "q does not lie"), (dict(q=rows(token_stride=1028)), "16 bytes"),
    (dict(out=rows(head_stride=0)), "overlap"), (dict(out=rows(token_stride=64)), "overlap"), (dict(heads=6), "query heads"),
    (dict(heads=0), "query heads"), (dict(heads=-4), "query heads"), (dict(heads=1 << 29), "query rows"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
]


@pytest.mark.parametrize("over,word", BAD_CALLS, ids=[str(i) for i in range(len(BAD_CALLS))])
def test_bad_attention_calls(over, word):
    f = dict(cache=cache(), seqs=seqs(), q=rows(), out=rows(), heads=8, scale=0.1)
    f.update(over)
    L = serving._lib()
    for call in (L.rpg_hip_paged_decode, L.rpg_hip_paged_prompt):
        refused(call(ref(f["cache"]), ref(f["seqs"]), ref(f["q"]), ref(f["out"]), f["heads"], f["scale"], A, 1 << 50,
                     None), word)


@pytest.mark.parametrize("over", [dict(head_stride=256, token_stride=2048), dict(head_stride=512), dict(token_stride=4096)],
                         ids=["both", "heads", "tokens"])
def test_outputs_at_the_queries_with_other_strides(over):
    """They would overwrite queries that are not read yet."""
    L = serving._lib()
    c, s, r = cache(), seqs(), rows()
    for call in (L.rpg_hip_paged_decode, L.rpg_hip_paged_prompt):
        refused(call(ref(c), ref(s), ref(r), ref(rows(**over)), 8, 0.1, A, 1 << 50, None), "out is q with other strides")
    refused(L.rpg_hip_paged_append(ref(c), ref(s), ref(r), ref(r), ref(r), ref(rows(**over)), 8, None, None, 0.0, None, 0,
                                   None), "q_out is q with other strides")


def test_starts_and_work_memory():
    L = serving._lib()
    c, r = cache(), rows()
    s = seqs(starts=None)
    refused(L.rpg_hip_paged_prompt(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, 1 << 40, None), "starts is null")
    s = seqs(pages=1000, table_stride=1000)
    need = L.rpg_hip_paged_work(ref(c), ref(s), 8, 0)
    assert need > 0 and need % 4 == 0
    refused(L.rpg_hip_paged_decode(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, need - 1, None), "work memory")
    refused(L.rpg_hip_paged_decode(ref(c), ref(s), ref(r), ref(r), 8, 0.1, None, need, None), "work is null")
    refused(L.rpg_hip_paged_decode(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A + 4, need, None), "work does not lie")
    assert L.rpg_hip_paged_work(ref(c), ref(seqs(pages=1, n_seqs=1)), 8, 0) == 0  # one range: none


@pytest.mark.parametrize("kind", [0, 1, 30])
@pytest.mark.parametrize("pages", [1, 64, 256, 8192])
@pytest.mark.parametrize("n_seqs,n_tokens,prompt", [(0, 0, 0), (0, 0, 1), (0, 3, 0), (0, 3, 1), (5, 0, 1)])
def test_nothing_to_do_takes_no_work_memory(kind, pages, n_seqs, n_tokens, prompt):
    """No sequences, with tokens or without, or no tokens: no bytes and no refusal,
    and a call that returns at once with no work memory."""
    L = serving._lib()
    r = rows()
    s = seqs(pages=pages, table_stride=pages, n_seqs=n_seqs, n_tokens=n_tokens)
    for c in (cache(type=kind), cache(type=kind, n_kv=1)):
        assert L.rpg_hip_paged_work(ref(c), ref(s), 8, prompt) == 0
        call = L.rpg_hip_paged_prompt if prompt else L.rpg_hip_paged_decode
        assert call(ref(c), ref(s), ref(r), ref(r), 8, 0.1, None, 0, None) == 0
    assert serving._work_bytes(8, 16, 128, kind, pages, n_seqs, n_tokens, 32, prompt) == 0


@pytest.mark.parametrize("kind,pages,prompt", [(30, 72, 0), (1, 200, 0), (0, 72, 0), (0, 90, 1), (1, 160, 1), (30, 288, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_partial_outputs_lie_at_multiples_of_16_bytes(kind, pages, prompt, dim):
    """An odd number of (maximum, sum) pairs in front of them: rows of five heads in
    an odd number of ranges. Work memory is in whole 16 bytes then, as the outputs are."""
    L = serving._lib()
    c = cache(type=kind, n_kv=1, head_dim=dim, row_stride=dim)
    odd = 0
    for tokens in (1, 3):
        s = seqs(pages=pages, table_stride=pages, n_seqs=tokens if prompt == 0 else 1, n_tokens=tokens)
        size = L.rpg_hip_paged_work(ref(c), ref(s), 5, prompt)
        pairs = size // (4 * (dim + 2))
        odd += pairs % 2
        assert size > 0 and pairs % (5 * tokens) == 0
        assert size == 4 * (pairs * dim + (2 * pairs + 3) // 4 * 4)
        assert size % 16 == 0
    assert odd > 0


def test_more_than_one_launch_holds():
    """2^24 workgroups and more, and positions that a step would count past 2^31."""
    L = serving._lib()
    c, r = cache(), rows(token_stride=1024)
    s = seqs(n_seqs=1 << 22, n_tokens=1 << 22)
    refused(L.rpg_hip_paged_decode(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, 1 << 60, None), "query rows in one launch")
    refused(L.rpg_hip_paged_prompt(ref(c), ref(s), ref(r), ref(r), 8, 0.1, A, 1 << 60, None), "query rows in one launch")
    s = seqs(n_tokens=1 << 24)
    refused(L.rpg_hip_paged_append(ref(c), ref(s), ref(r), ref(r), None, None, 0, None, None, 0.0, None, 0, None),
            "new tokens in one launch")
    most = (1 << 30) // 16
    assert L.rpg_hip_paged_work(ref(c), ref(seqs(pages=most, table_stride=most)), 8, 0) > 0
    refused(L.rpg_hip_paged_work(ref(c), ref(seqs(pages=most + 1, table_stride=most + 1)), 8, 0), "pages")


BAD_APPENDS = [
    (dict(k=None), "k is null"), (dict(v=rows(data=None)), "v is null"), (dict(q_out=None), "q_out is null"),
    (dict(q_out=rows(head_stride=256, token_stride=4096)), "other strides"), (dict(heads=5), "query heads"),
    (dict(q_norm=A + 4), "q_norm"), (dict(k_norm=A + 8), "k_norm"), (dict(rope=A + 8), "rope"),
    (dict(rope=A, rope_rows=-1), "rotation rows"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(seqs=seqs(starts=None)), "starts is null"), (dict(q_out=rows(data=A + 4096, head_stride=64)), "overlap"),
]


@pytest.mark.parametrize("over,word", BAD_APPENDS, ids=[str(i) for i in range(len(BAD_APPENDS))])
def test_bad_appends(over, word):
    f = dict(cache=cache(), seqs=seqs(), k=rows(), v=rows(), q=rows(), q_out=rows(), heads=8, q_norm=A, k_norm=A, eps=1e-6,
             rope=A, rope_rows=10)
    f.update(over)
    refused(serving._lib().rpg_hip_paged_append(
        ref(f["cache"]), ref(f["seqs"]), ref(f["k"]), ref(f["v"]), ref(f["q"]), ref(f["q_out"]), f["heads"], f["q_norm"],
        f["k_norm"], f["eps"], f["rope"], f["rope_rows"], None), word)


BAD_SAMPLES = [
    (dict(type=8), "element type"), (dict(rows=-1), "rows"), (dict(rows=65536), "rows"), (dict(vocab=0), "logits"),
    (dict(vocab=262145), "logits"), (dict(logits=None), "logits is null"), (dict(logits=A + 2), "logits does not lie"),
    (dict(stride=-1), "row_stride"), (dict(u=None), "u is null"), (dict(tokens=None), "tokens is null"),
    (dict(k=A + 1), "row parameter"), (dict(work=None), "work is null"), (dict(size=100), "work memory"),
]


@pytest.mark.parametrize("over,word", BAD_SAMPLES, ids=[str(i) for i in range(len(BAD_SAMPLES))])
def test_bad_samples(over, word):
    f = dict(type=0, logits=A, rows=4, vocab=1000, stride=1000, t=A, k=A, p=A, m=A, u=A, tokens=A, lp=A, work=A, size=1 << 40)
    f.update(over)
    refused(serving._lib().rpg_hip_sample_rows(f["type"], f["logits"], f["rows"], f["vocab"], f["stride"], f["t"], f["k"],
                                               f["p"], f["m"], f["u"], f["tokens"], f["lp"], f["work"], f["size"], None),
            word)


def test_work_sizes():
    L = serving._lib()
    assert L.rpg_hip_sample_rows_work(0, 10) >= 0
    assert L.rpg_hip_sample_rows_work(1, 1) > 0
    refused(L.rpg_hip_sample_rows_work(1, 262145), "logits")
    refused(L.rpg_hip_sample_rows_work(70000, 10), "rows")
    assert L.rpg_hip_sample_rows_work(300, 151936) > L.rpg_hip_sample_rows_work(1, 151936)


def test_packed_structs_are_laid_out_as_c_does():
    c = Cache(1, 2, 3, 4, 5, 6, 7, 8, 9, 10)
    assert bytes(c)[:serving._CACHE.size] == serving._CACHE.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10)
    s = Seqs(1, 2, 3, 4, 5, 6, 7)
    assert bytes(s)[:serving._SEQS.size] == serving._SEQS.pack(1, 2, 3, 4, 5, 6, 7)
    assert bytes(Rows(1, -2, 3)) == serving._ROWS.pack(1, -2, 3)


def test_tensors_without_a_gpu_are_refused():
    z = torch.zeros(2, 1, 16, 64)
    with pytest.raises(eng.EngineError, match="one GPU"):
        serving.PagedCache(z, z)
    with pytest.raises(eng.EngineError, match="on a GPU"):
        serving.sample(torch.zeros(2, 5), torch.zeros(2))


# ---- the definitions themselves


def test_plain_sample_by_hand():
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.2, 0.1]))
    lp = lambda p: pytest.approx(math.log(p), abs=1e-6)  # noqa: E731
    assert plain.sample(x, 0.05, 1.0, 0, 1.0, 0.0) == (0, lp(0.1))
    assert plain.sample(x, 0.45, 1.0, 0, 1.0, 0.0) == (1, lp(0.4))
    assert plain.sample(x, 0.95, 1.0, 0, 1.0, 0.0) == (4, lp(0.1))
    assert plain.sample(x, 0.95, 1.0, 2, 1.0, 0.0) == (2, lp(0.2 / 0.6))  # the first of the equal ones stays
    assert plain.sample(x, 0.95, 1.0, 0, 0.5, 0.0) == (2, lp(0.2 / 0.6))
    assert plain.sample(x, 0.95, 1.0, 0, 1.0, 0.45) == (3, lp(0.25))
    assert plain.sample(x, 0.95, 0.0, 0, 1.0, 0.0) == (1, 0.0)
    assert plain.sample(x * math.nan, 0.5, 1.0, 0, 1.0, 0.0) == (-1, -math.inf)


def test_plain_attention_by_hand():
    k = torch.tensor([[[0.0] * 64, [1.0] + [0.0] * 63]])
    v = torch.stack([torch.full((64,), 1.0), torch.full((64,), 3.0)])[None]
    q = torch.zeros(1, 64)
    q[0, 0] = math.log(3.0)
    out, bound = plain.attention(q, k.double(), v.double(), torch.tensor([True, True]), 1.0, torch.float32)
    assert torch.allclose(out, torch.full((1, 64), 2.5, dtype=torch.float64))
    assert float(bound.max()) < 1e-3
    out, _ = plain.attention(q, k.double(), v.double(), torch.tensor([True, False]), 1.0, torch.float32)
    assert bool((out == 1).all())
