"""Refusals of the operators on 8-bit caches, of shared positions and of the edits of
logits (include/rpg_hip.h), which come before anything touches a GPU; sizes of work
memory; and the plain definitions that the GPU tests hold the kernels to."""

import ctypes
import math

import pytest
import torch

import rpgbarengine_amd as eng
import serving_more_plain as more
from rpgbarengine_amd import serving
from test_cpu_serving import A, I32, I64, P, cache, ref, refused, rows, seqs


class Quant(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("page_stride", I64), ("head_stride", I64),
                ("row_stride", I64), ("scale_page_stride", I64), ("scale_head_stride", I64), ("n_pages", I32),
                ("page_size", I32), ("n_kv", I32), ("head_dim", I32), ("code", I32)]


class Groups(ctypes.Structure):
    _fields_ = [("starts", P), ("shared", P), ("n_groups", I32)]


class Edits(ctypes.Structure):
    _fields_ = [("history", P), ("history_stride", I64), ("history_lens", P), ("prompts", P), ("repetition", P),
                ("presence", P), ("frequency", P), ("bias_ids", P), ("bias_ids_stride", I64), ("bias", P),
                ("bias_stride", I64), ("mask", P), ("mask_stride", I64), ("mask_rows", P), ("history_size", I32),
                ("n_biases", I32), ("n_masks", I32)]


def test_structures_are_packed_as_c_lays_them_out():
    assert serving._QUANT.size == ctypes.sizeof(Quant) - 4 and Quant.code.offset == serving._QUANT.size - 4
    assert serving._GROUPS.size == Groups.n_groups.offset + 4
    assert serving._EDITS.size == Edits.n_masks.offset + 4


def quant(**over):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, page_stride=4 * 16 * 128, head_stride=16 * 128, row_stride=128,
             scale_page_stride=64, scale_head_stride=16, n_pages=9, page_size=16, n_kv=4, head_dim=128, code=1)
    f.update(over)
    return Quant(**f)


def groups(**over):
    f = dict(starts=A, shared=A, n_groups=2)
    f.update(over)
    return Groups(**f)


BIG = 1 << 50  # bytes of work memory


def quant_calls(c, s=None, q=None, out=None, heads=8, scale=0.1, kind=1, work=A, size=BIG, g=None):
    """The return values of every operator on a cache of codes."""
    L = serving._lib()
    s, q = s or seqs(), q or rows()
    out = out or q
    yield L.rpg_hip_quant_decode(ref(c), ref(s), kind, ref(q), ref(out), heads, scale, work, size, None)
    yield L.rpg_hip_quant_prompt(ref(c), ref(s), kind, ref(q), ref(out), heads, scale, work, size, None)
    yield L.rpg_hip_quant_shared(ref(c), ref(s), ref(g or groups()), kind, ref(q), ref(out), heads, scale, work, size, None)


BAD_CACHES = [
    (dict(code=2), "code"), (dict(code=-1), "code"), (dict(head_dim=96), "head_dim"), (dict(page_size=24), "page_size"),
    (dict(page_size=8), "page_size"), (dict(n_pages=0), "pages"), (dict(n_kv=0), "key heads"),
    (dict(row_stride=64), "row_stride"), (dict(row_stride=136), "row_stride"), (dict(row_stride=1 << 28), "row_stride"),
    (dict(head_stride=64), "head_stride"), (dict(page_stride=0), "page_stride"), (dict(page_stride=8), "page_stride"),
    (dict(scale_head_stride=8), "scale_head_stride"), (dict(scale_page_stride=0), "scale_head_stride"),
    (dict(scale_page_stride=66), "scale_page_stride"), (dict(scale_head_stride=1 << 40), "scale_head_stride"),
]


@pytest.mark.parametrize("over,word", BAD_CACHES, ids=[str(i) for i in range(len(BAD_CACHES))])
def test_bad_caches(over, word):
    L = serving._lib()
    c, s, r = quant(**over), seqs(), rows()
    for rc in quant_calls(c):
        refused(rc, word)
    refused(L.rpg_hip_quant_append(ref(c), ref(s), 1, ref(r), ref(r), None, None, 0, None, None, 0.0, None, 0, None), word)
    refused(L.rpg_hip_quant_read(ref(c), ref(s), 1, ref(r), ref(r), None), word)
    refused(L.rpg_hip_quant_work(ref(c), ref(s), 1, 8, 0), word)
    refused(L.rpg_hip_quant_shared_work(ref(c), ref(s), 2, 1, 8), word)


BAD_POINTERS = [(dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(k=A + 8), "k does not lie"),
                (dict(k_scale=None), "k_scale is null"), (dict(v_scale=None), "v_scale is null"),
                (dict(v_scale=A + 4), "v_scale does not lie")]


@pytest.mark.parametrize("over,word", BAD_POINTERS, ids=[str(i) for i in range(len(BAD_POINTERS))])
def test_bad_pools(over, word):
    L = serving._lib()
    c, s, r = quant(**over), seqs(), rows()
    for rc in quant_calls(c):
        refused(rc, word)
    refused(L.rpg_hip_quant_append(ref(c), ref(s), 1, ref(r), ref(r), None, None, 0, None, None, 0.0, None, 0, None), word)
    refused(L.rpg_hip_quant_read(ref(c), ref(s), 1, ref(r), ref(r), None), word)


BAD_CALLS = [
    (dict(kind=8), "element type"), (dict(s=seqs(n_seqs=-1)), "sequences"), (dict(s=seqs(pages=-1)), "pages"),
    (dict(s=seqs(table=None)), "table is null"), (dict(s=seqs(table_stride=7)), "table_stride"),
    (dict(s=seqs(lens=None)), "lens is null"), (dict(q=rows(data=None)), "q is null"), (dict(q=rows(data=A + 8)), "q does not lie"),
    (dict(q=rows(token_stride=1028)), "16 bytes"), (dict(out=rows(data=A + 4096, head_stride=0)), "overlap"),
    (dict(out=rows(token_stride=2048)), "out is q with other strides"), (dict(heads=6), "query heads"),
    (dict(heads=0), "query heads"), (dict(heads=1 << 29), "query rows"), (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
]


@pytest.mark.parametrize("over,word", BAD_CALLS, ids=[str(i) for i in range(len(BAD_CALLS))])
def test_bad_attention_calls(over, word):
    for rc in quant_calls(quant(), **over):
        refused(rc, word)


def test_append_and_read_refusals():
    L = serving._lib()
    c, s, r = quant(), seqs(), rows()

    def append(k=r, v=r, q=None, q_out=None, heads=8, qn=None, kn=None, eps=0.0, rope=None, n=0, kind=1, s=s):
        return L.rpg_hip_quant_append(ref(c), ref(s), kind, ref(k), ref(v), ref(q), ref(q_out), heads, qn, kn, eps, rope, n, None)

    refused(append(k=None), "k is null")
    refused(append(v=rows(data=A + 2)), "v does not lie")
    refused(append(kind=24), "element type")
    refused(append(q=r, q_out=None), "q_out is null")
    refused(append(q=r, q_out=rows(head_stride=256, token_stride=2048)), "q_out is q with other strides")
    refused(append(q=r, q_out=r, heads=6), "query heads")
    refused(append(kn=A + 4), "k_norm does not lie")
    refused(append(rope=A, n=-1), "rotation rows")
    refused(append(eps=-1.0), "eps")
    refused(append(eps=math.nan), "eps")
    refused(append(s=seqs(starts=None)), "starts is null")
    refused(L.rpg_hip_quant_read(ref(c), ref(s), 1, None, ref(r), None), "k is null")
    refused(L.rpg_hip_quant_read(ref(c), ref(s), 1, ref(r), ref(rows(head_stride=64)), None), "overlap")
    refused(L.rpg_hip_quant_read(ref(c), ref(seqs(starts=None)), 1, ref(r), ref(r), None), "starts is null")
    assert append(s=seqs(n_seqs=0)) == 0 and append(s=seqs(n_tokens=0)) == 0
    assert L.rpg_hip_quant_read(ref(c), ref(seqs(n_seqs=0)), 1, None, None, None) == 0


@pytest.mark.parametrize("kind", [0, 1, 30])
def test_work_memory(kind):
    L = serving._lib()
    c, r = quant(), rows()
    s = seqs(pages=1000, table_stride=1000)
    need = [L.rpg_hip_quant_work(ref(c), ref(s), kind, 8, 0), L.rpg_hip_quant_work(ref(c), ref(s), kind, 8, 1),
            L.rpg_hip_quant_shared_work(ref(c), ref(s), 2, kind, 8)]
    assert all(n > 0 and n % 4 == 0 for n in need)
    for size_less, word, at in ((1, "work memory", A), (0, "work is null", None), (0, "work does not lie", A + 4)):
        f = [L.rpg_hip_quant_decode, L.rpg_hip_quant_prompt]
        for call, n in zip(f, need):
            refused(call(ref(c), ref(s), kind, ref(r), ref(r), 8, 0.1, at, n - size_less, None), word)
        refused(L.rpg_hip_quant_shared(ref(c), ref(s), ref(groups()), kind, ref(r), ref(r), 8, 0.1, at, need[2] - size_less,
                                       None), word)
    assert L.rpg_hip_quant_work(ref(c), ref(seqs(pages=1, n_seqs=1)), kind, 8, 0) == 0  # one range: none
    for n_seqs, n_tokens, prompt in ((0, 0, 0), (0, 3, 1), (5, 0, 1)):
        s = seqs(pages=500, table_stride=500, n_seqs=n_seqs, n_tokens=n_tokens)
        assert L.rpg_hip_quant_work(ref(c), ref(s), kind, 8, prompt) == 0
        call = L.rpg_hip_quant_prompt if prompt else L.rpg_hip_quant_decode
        assert call(ref(c), ref(s), kind, ref(r), ref(r), 8, 0.1, None, 0, None) == 0
    s = seqs(n_seqs=0)
    assert L.rpg_hip_quant_shared(ref(c), ref(s), ref(groups()), kind, ref(r), ref(r), 8, 0.1, None, 0, None) == 0
    assert L.rpg_hip_quant_shared_work(ref(c), ref(s), 2, kind, 8) == 0


def test_shared_refusals():
    L = serving._lib()
    for c, call, sizes in ((cache(), lambda c, s, g, r, o, h, sc, w, n: L.rpg_hip_paged_shared(c, s, g, r, o, h, sc, w, n, None),
                            lambda c, s, g, h: L.rpg_hip_paged_shared_work(c, s, g, h)),
                           (quant(), lambda c, s, g, r, o, h, sc, w, n: L.rpg_hip_quant_shared(c, s, g, 1, r, o, h, sc, w, n, None),
                            lambda c, s, g, h: L.rpg_hip_quant_shared_work(c, s, g, 1, h))):
        s, r = seqs(), rows()

        def run(g=groups(), s=s, r=r, o=None, heads=8, scale=0.1, work=A, size=BIG):
            return call(ref(c), ref(s), ref(g), ref(r), ref(o or r), heads, scale, work, size)

        refused(run(g=None), "groups are null")
        refused(run(g=groups(n_groups=-1)), "groups")
        refused(run(g=groups(starts=None)), "starts is null")
        refused(run(g=groups(shared=None)), "shared is null")
        refused(run(g=groups(shared=A + 2)), "shared does not lie")
        refused(run(s=seqs(lens=None)), "lens is null")
        refused(run(heads=7), "query heads")
        refused(run(scale=-1.0), "scale")
        refused(run(o=rows(head_stride=256, token_stride=2048)), "out is q with other strides")
        need = sizes(ref(c), ref(s), 2, 8)
        assert need > 0 and need % 4 == 0
        refused(run(size=need - 1), "work memory")
        refused(run(work=None, size=need), "work is null")
        refused(sizes(ref(c), ref(s), -1, 8), "groups")
        refused(sizes(ref(c), ref(s), 2, 7), "query heads")
        assert run(s=seqs(n_seqs=0)) == 0


@pytest.mark.parametrize("kind", [0, 1, 30])
@pytest.mark.parametrize("n_seqs", [1, 3, 64, 5000])
@pytest.mark.parametrize("n_groups", [0, 1, 2, 7, 5000])
@pytest.mark.parametrize("pages", [0, 1, 40, 100000])
def test_shared_sizes_hold_at_any_shape(kind, n_seqs, n_groups, pages):
    """Sizes are asked for without pointers; every range has its place."""
    for heads, n_kv in ((8, 4), (4, 4), (64, 4)):
        got = serving._shared_bytes(False, n_kv, 16, 128, kind, pages, n_seqs, n_groups, heads)
        codes = serving._shared_bytes(True, n_kv, 16, 128, kind, pages, n_seqs, n_groups, heads)
        rows_ = n_seqs * heads
        for n in (got, codes):
            slots = n // (4 * rows_ * 130)
            assert 2 <= slots <= 512 and n == 4 * ((2 * rows_ * slots + 3) // 4 * 4 + rows_ * slots * 128)


def edits(**over):
    f = dict(history=A, history_stride=50, history_size=50, bias_ids=A, bias=A, bias_ids_stride=4, bias_stride=4, n_biases=4,
             mask=A, mask_stride=10, n_masks=3)
    f.update(over)
    return Edits(**f)


BAD_EDITS = [
    (dict(kind=8), "element type"), (dict(e=None), "edits are null"), (dict(n=-1), "rows"), (dict(n=65536), "rows"),
    (dict(vocab=0), "logits outside"), (dict(vocab=(1 << 24) + 1), "logits outside"), (dict(x=None), "logits is null"),
    (dict(x=A + 1), "logits does not lie"), (dict(out=None), "out is null"), (dict(out=A + 1), "out does not lie"),
    (dict(stride=-1), "row_stride"), (dict(out_stride=299), "out_stride"), (dict(stride=1 << 40), "row_stride"),
    (dict(out=A, x=A, stride=400), "out is logits with another stride"), (dict(e=edits(history_stride=-1)), "history"),
    (dict(e=edits(history=A + 2)), "history does not lie"), (dict(e=edits(history_size=-1)), "history"),
    (dict(e=edits(history_size=(1 << 20) + 1)), "history"), (dict(e=edits(history=None, repetition=A)), "without a history"),
    (dict(e=edits(history=None, history_lens=A)), "without a history"), (dict(e=edits(repetition=A + 1)), "row parameter"),
    (dict(e=edits(bias=None)), "bias"), (dict(e=edits(bias_ids=None)), "bias"), (dict(e=edits(n_biases=-1)), "biases"),
    (dict(e=edits(n_biases=1024)), "biases"), (dict(e=edits(bias_stride=-4)), "bias"), (dict(e=edits(n_masks=-1)), "masks"),
    (dict(e=edits(mask=None, mask_rows=A)), "without a mask"), (dict(e=edits(mask_rows=A + 2)), "row parameter"),
    (dict(e=edits(mask_stride=-1)), "mask"),
]


@pytest.mark.parametrize("over,word", BAD_EDITS, ids=[str(i) for i in range(len(BAD_EDITS))])
def test_bad_edits(over, word):
    f = dict(kind=1, x=A, n=3, vocab=300, stride=300, e=edits(), out=A + 4096, out_stride=300)
    f.update(over)
    refused(serving._lib().rpg_hip_edit_logits(f["kind"], f["x"], f["n"], f["vocab"], f["stride"], ref(f["e"]), f["out"],
                                               f["out_stride"], None), word)


def test_no_rows_no_edits():
    assert serving._lib().rpg_hip_edit_logits(0, None, 0, 300, 300, ref(edits()), None, 300, None) == 0


# ---- the binding's own refusals (tensors on the CPU)


def test_quant_caches_of_bad_tensors():
    k, s = torch.zeros(3, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2, 16)
    for args, word in (((k[0], k, s, s), "are \\[pages"), ((k, k.view(torch.float8_e4m3fn), s, s), "both int8"),
                       ((k.short(), k.short(), s, s), "both int8"), ((k, k, s[:, :1], s), "k_scale and v_scale"),
                       ((k, k, s, s.double()), "k_scale and v_scale"), ((k, k, s, s), "one GPU")):
        with pytest.raises(eng.EngineError, match=word):
            serving.QuantCache(*args)


def test_edits_of_tensors_on_the_cpu():
    with pytest.raises(eng.EngineError, match="on a GPU"):
        serving.edit_logits(torch.zeros(2, 8))


# ---- the definitions


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_nearest_code(codes):
    """Against the conversion of torch, ties among them."""
    u = torch.cat([torch.linspace(-127, 127, 4001, dtype=torch.float64), torch.arange(-127, 127) + 0.5])
    if codes == torch.float8_e4m3fn:
        u = torch.cat([u * 3.5, u * 2.0 ** -7, u * 2.0 ** -12]).clamp(-448, 448)
        assert torch.equal(more.nearest(u, codes), u.float().to(codes).double())
    else:
        assert torch.equal(more.nearest(u, codes), torch.round(u))
    assert bool(((more.nearest(u, codes) - u).abs() <= more.half_step(u, codes)).all())


def test_check_row_sees_a_code_that_is_off():
    y = torch.randn(4, 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    top = y.abs().amax(-1, keepdim=True)
    for codes in more.LARGEST:
        code = more.nearest(y * more.LARGEST[codes] / top, codes)
        scale = top[..., 0] / more.LARGEST[codes]
        more.check_row(code, scale, y, 0 * y, codes)
        bad = code.clone()
        bad[2, 7] += 1 if codes == torch.int8 else 32
        with pytest.raises(AssertionError):
            more.check_row(bad, scale, y, 0 * y, codes)
        with pytest.raises(AssertionError):
            more.check_row(code, scale * 1.001, y, 0 * y, codes)


def test_edit_by_hand():
    x, mag = more.edit(torch.tensor([1.0, -1.0, 2.0, 3.0, 4.0], dtype=torch.float64), [0, 1, 1, 2, 9, -1], 2, 2.0, 0.5, 0.25,
                       [(3, 1.0), (3, 2.0), (7, 1.0)], torch.tensor([True, True, True, True, False]))
    assert x.tolist() == [0.5, -2.75, 0.25, 5.0, -math.inf]
