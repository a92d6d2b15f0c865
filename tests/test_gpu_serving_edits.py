"""The edits of logits (rpgbarengine_amd.serving.edit_logits) against their
definition in float64."""

import math

import pytest
import torch

import serving_more_plain as more
import serving_plain as plain
from rpgbarengine_amd import serving
from test_gpu_serving import DTYPES, ident

pytestmark = pytest.mark.gpu


class Edits:
    """Random edits of `rows` rows; everything on the CPU."""

    def __init__(self, rows, vocab, dtype, size, biases=5, masks=None, seed=0, stride=None):
        g = self.gen = torch.Generator().manual_seed(seed)
        self.rows, self.vocab, self.dtype = rows, vocab, dtype
        wide = torch.randn(rows, stride or vocab, generator=g) * 3
        self.logits = wide.to(dtype)
        # numbers of the vocabulary, some twice and more, some outside it
        self.history = (torch.rand(rows, size, generator=g) ** 2 * (vocab + 2)).int() - 1
        self.lens = torch.randint(0, size + 3, (rows,), generator=g, dtype=torch.int32) - 1
        self.prompts = torch.randint(-1, size + 2, (rows,), generator=g, dtype=torch.int32)
        self.repetition = 1 + torch.rand(rows, generator=g)
        self.presence = torch.randn(rows, generator=g)
        self.frequency = torch.randn(rows, generator=g)
        self.bias_ids = torch.randint(-2, vocab + 2, (rows, biases), generator=g, dtype=torch.int32)
        self.bias = torch.randn(rows, biases, generator=g) * 4
        n = rows if masks is None else masks
        self.mask = torch.randint(-(1 << 31), 1 << 31, (n, (vocab + 31) // 32), generator=g).int()
        self.mask_rows = torch.randint(-2, n + 2, (rows,), generator=g, dtype=torch.int32)

    def want(self, use):
        """(rows, bounds) float64 with the edits named in `use`."""
        outs, bounds = [], []
        for r in range(self.rows):
            n = max(0, min(int(self.lens[r]), self.history.shape[1])) if "lens" in use else self.history.shape[1]
            history = self.history[r, :n].tolist() if "history" in use else []
            allowed = None
            if "mask" in use:
                at = int(self.mask_rows[r]) if "mask_rows" in use else r
                if 0 <= at < len(self.mask):
                    bits = (self.mask[at].long()[:, None] >> torch.arange(32)) & 1
                    allowed = bits.reshape(-1)[: self.vocab] == 1
            x, mag = more.edit(self.logits[r, : self.vocab].double(), history,
                               int(self.prompts[r]) if "prompts" in use else 0,
                               float(self.repetition[r]) if "repetition" in use else 1.0,
                               float(self.presence[r]) if "presence" in use else 0.0,
                               float(self.frequency[r]) if "frequency" in use else 0.0,
                               list(zip(self.bias_ids[r].tolist(), self.bias[r].double().tolist())) if "bias" in use else [],
                               allowed)
            outs.append(x)
            # a quotient or product, a product, two differences, a sum: five roundings of fp32, then one to the type
            size = torch.where(x.isfinite(), x.abs(), 0.0)
            bounds.append(5 * 2.0 ** -24 * mag + plain.EPS[self.dtype] * (size + 5 * 2.0 ** -24 * mag) + plain.TINY[self.dtype])
        return torch.stack(outs), torch.stack(bounds)

    def call(self, use, out=None, logits=None):
        d = {"history": self.history, "history_lens": self.lens if "lens" in use else None,
             "prompts": self.prompts, "repetition": self.repetition, "presence": self.presence,
             "frequency": self.frequency, "mask": self.mask, "mask_rows": self.mask_rows}
        kw = {k: (v.cuda() if v is not None and (k in use or k == "history_lens") else None) for k, v in d.items()}
        if "bias" in use:
            kw |= {"bias_ids": self.bias_ids.cuda(), "bias": self.bias.cuda()}
        x = self.logits.cuda()[:, : self.vocab] if logits is None else logits
        return serving.edit_logits(x, out=out, **kw)


ALL = ("history", "lens", "prompts", "repetition", "presence", "frequency", "bias", "mask", "mask_rows")


def same(got, want, bound):
    got = got.double().cpu()
    low = want == -math.inf
    assert torch.equal(got == -math.inf, low)
    bad = ~((got - want).abs() <= bound) & ~low
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / bound)[~low].max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("rows,vocab,size", [(3, 1, 1), (2, 31, 40), (5, 4096, 300), (3, 4097, 1), (4, 9001, 1500), (1, 12288, 5000)])
def test_all_edits(dtype, rows, vocab, size):
    e = Edits(rows, vocab, dtype, size, seed=rows + vocab)
    got = e.call(ALL)
    assert got.dtype is dtype and got.shape == (rows, vocab)
    same(got, *e.want(ALL))


USES = [(), ("history", "repetition"), ("history", "lens", "presence"), ("history", "prompts", "frequency", "presence"),
        ("bias",), ("mask",), ("mask", "mask_rows"), ("history", "repetition", "prompts", "lens", "bias"),
        ("bias", "mask", "mask_rows")]


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("use", USES, ids=["+".join(u) or "none" for u in USES])
def test_some_edits_apart_and_in_place(dtype, use):
    e = Edits(4, 5003, dtype, 200, seed=7)
    want = e.want(use)
    got = e.call(use)
    same(got, *want)
    x = e.logits.cuda()
    assert e.call(use, out=x, logits=x) is x
    assert torch.equal(x, got)


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_rows_at_any_place(dtype, shift):
    """Rows that do not lie at multiples of 16 bytes, apart, alike or in place, with
    what lies between rows left as it was; broadcast lists and logits."""
    rows, vocab = 5, 4999
    e = Edits(rows, vocab, dtype, 64, seed=9)
    want = e.want(ALL)
    wide = torch.full((rows, vocab + 11), 3.0, dtype=dtype, device="cuda")
    wide[:, shift:shift + vocab] = e.logits.cuda()
    out = torch.full((rows, vocab + 2 * shift + 8), 5.0, dtype=dtype, device="cuda")
    got = e.call(ALL, out=out[:, shift + 1:shift + 1 + vocab], logits=wide[:, shift:shift + vocab])
    same(got, *want)
    assert bool((out[:, :shift + 1] == 5).all()) and bool((out[:, shift + 1 + vocab:] == 5).all())
    place = wide[:, shift:shift + vocab]
    assert torch.equal(e.call(ALL, out=place, logits=place), got)
    assert bool((wide[:, :shift] == 3).all()) and bool((wide[:, shift + vocab:] == 3).all())
    e.logits[:] = e.logits[:1].clone()
    e.history[:], e.bias_ids[:], e.bias[:] = e.history[:1].clone(), e.bias_ids[:1].clone(), e.bias[:1].clone()
    want = e.want(ALL)
    one = e.logits[:1].cuda().expand(rows, vocab)
    got = serving.edit_logits(one, e.history[:1].cuda().expand(rows, -1), e.lens.cuda(), e.prompts.cuda(),
                              e.repetition.cuda(), e.presence.cuda(), e.frequency.cuda(),
                              e.bias_ids[:1].cuda().expand(rows, -1), e.bias[:1].cuda().expand(rows, -1), e.mask.cuda(),
                              e.mask_rows.cuda())
    same(got, *want)


def test_many_times_the_same_token():
    """Counts past what 16 bits hold, from more lanes than there are at once."""
    n = 70000
    history = torch.zeros(2, n, dtype=torch.int32)
    history[1, :] = 4099
    x = torch.ones(2, 4100)
    got = serving.edit_logits(x.cuda(), history.cuda(), frequency=torch.tensor([0.5, 2.0]).cuda()).cpu()
    assert float(got[0, 0]) == 1 - 0.5 * n and float(got[1, 4099]) == 1 - 2.0 * n
    got[0, 0] = got[1, 4099] = 1.0
    assert bool((got == 1).all())


def test_values_that_are_not_finite_and_a_mask_that_leaves_nothing():
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0, -2.0, 0.0]]).repeat(3, 1)
    history = torch.tensor([[0, 1, 2, 3, 4, 5]], dtype=torch.int32).repeat(3, 1)
    mask = torch.tensor([[0x3F], [0], [0x3B]], dtype=torch.int32)
    got = serving.edit_logits(x.cuda(), history.cuda(), repetition=torch.tensor([2.0, 2.0, -1.0]).cuda(), mask=mask.cuda()).cpu()
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and bool(got[0, 2].isnan())
    assert got[0, 3:].tolist() == [0.5, -4.0, 0.0]
    assert bool((got[1] == -math.inf).all())
    assert got[2, 0] == math.inf and got[2, 2] == -math.inf and got[2, 3:].tolist() == [1.0, -2.0, 0.0]  # not above 0: none
    tokens, _ = serving.sample(got.cuda(), torch.full((3,), 0.5).cuda(), temperature=torch.zeros(3).cuda())
    assert tokens.tolist() == [0, -1, 0]


def test_the_last_of_several_biases_counts():
    ids = torch.tensor([[7, 3, 7, -1, 7, 99]], dtype=torch.int32)
    bias = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]])
    got = serving.edit_logits(torch.zeros(1, 10).cuda(), bias_ids=ids.cuda(), bias=bias.cuda()).cpu()
    assert got.tolist() == [[0, 0, 0, 2.0, 0, 0, 0, 5.0, 0, 0]]


def test_empty_lists_and_rows():
    x = torch.randn(2, 50).cuda()
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    got = serving.edit_logits(x, none, repetition=torch.full((2,), 3.0).cuda(), bias_ids=none, bias=none.float())
    assert torch.equal(got, x)
    assert serving.edit_logits(x[:0]).shape == (0, 50)


def test_no_masks_for_rows_that_go_by_none():
    x = torch.randn(3, 70, device="cuda")
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    rows = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(serving.edit_logits(x, mask=none, mask_rows=rows), x)


def test_captured_and_replayed():
    """A replay takes the history, its length and the masks of its moment."""
    e = Edits(3, 5000, torch.bfloat16, 100, seed=11)
    x, history, lens = e.logits.cuda(), e.history.cuda(), e.lens.cuda()
    mask, of, r = e.mask.cuda(), e.mask_rows.cuda(), e.repetition.cuda()
    out = torch.empty_like(x)
    serving.edit_logits(x, history, lens, repetition=r, mask=mask, mask_rows=of, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.edit_logits(x, history, lens, repetition=r, mask=mask, mask_rows=of, out=out)
    use = ("history", "lens", "repetition", "mask", "mask_rows")
    for step in range(4):
        e.lens[:] = torch.tensor([step * 20, 100 - step, 3])
        e.mask_rows[:] = torch.tensor([step % 3, -1, 2])
        e.history[0, :50] += 1
        lens.copy_(e.lens), of.copy_(e.mask_rows), history.copy_(e.history)
        out.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        same(out, *e.want(use))


def test_refusals_on_tensors():
    from rpgbarengine_amd import EngineError
    x, ids = torch.randn(2, 64).cuda(), torch.zeros(2, 3, dtype=torch.int32).cuda()
    two, bits = torch.ones(2).cuda(), torch.zeros(2, 2, dtype=torch.int32).cuda()
    for kw in (dict(repetition=two), dict(history_lens=ids[:, 0]), dict(history=ids.long()), dict(history=ids[:1]),
               dict(history=ids.t().contiguous().t()), dict(history=ids.cpu()), dict(history=ids, repetition=two.double()),
               dict(history=ids, repetition=two[:1]), dict(history=ids, history_lens=two), dict(bias_ids=ids),
               dict(bias=two[:, None]), dict(bias_ids=ids, bias=two[:, None]), dict(mask=bits[:, :1]), dict(mask=bits[:1]),
               dict(mask_rows=ids[:, 0].contiguous()), dict(out=x.half()), dict(out=x[:1]), dict(out=x.t().contiguous().t()),
               dict(bias_ids=ids, bias=torch.zeros(2, 3, device="cuda", requires_grad=True)),
               dict(bias_ids=torch.zeros(2, 1024, dtype=torch.int32, device="cuda"), bias=torch.zeros(2, 1024, device="cuda"))):
        with pytest.raises(EngineError):
            serving.edit_logits(x, **kw)
    for bad in (x[0], x.double(), x.cpu(), x.t().contiguous().t(), x.clone().requires_grad_()):
        with pytest.raises(EngineError):
            serving.edit_logits(bad)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(EngineError, match="tangent"):
            serving.edit_logits(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    version = x._version
    serving.edit_logits(x, out=x)
    assert x._version > version


def test_as_many_biases_as_may_be():
    g = torch.Generator().manual_seed(5)
    ids = torch.randperm(6000, generator=g)[:1023].int()[None]
    bias = torch.randn(1, 1023, generator=g)
    x = torch.randn(1, 6000, generator=g)
    got = serving.edit_logits(x.cuda(), ids.cuda(), bias_ids=ids.cuda(), bias=bias.cuda(), presence=torch.ones(1).cuda()).cpu()
    want = x.double()
    want[0, ids[0].long()] += bias[0].double() - 1.0
    assert float((got.double() - want).abs().max()) <= 2 * 2.0 ** -24 * 12  # two roundings of values below 12
