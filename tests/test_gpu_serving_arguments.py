"""Arguments of the serving operators that lie in each other's memory, and caches of a
class of the caller's."""

import pytest
import torch

import rpgbarengine_amd as eng
from rpgbarengine_amd import serving
from test_gpu_serving import DTYPES, Batch, ident

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=ident)
@pytest.mark.parametrize("vocab", [1000, 9001])
def test_logits_edited_within_one_matrix(dtype, vocab):
    """Into the other part of the same rows; over themselves, some tokens on, is refused."""
    gen = torch.Generator().manual_seed(51)
    both = torch.randn(5, 2 * vocab + 8, generator=gen).to(dtype).cuda()
    history = torch.randint(0, vocab, (5, 30), generator=gen, dtype=torch.int32).cuda()
    r = torch.full((5,), 1.3, device="cuda")
    x = both[:, :vocab]
    want = serving.edit_logits(x.clone(), history, repetition=r)
    before = both.clone()
    for off in (1, vocab - 1):
        with pytest.raises(eng.EngineError, match="out overlaps logits"):
            serving.edit_logits(both[:, off:off + vocab][:4], history[:4], repetition=r[:4], out=both[1:, :vocab])
        with pytest.raises(eng.EngineError, match="out overlaps logits"):
            serving.edit_logits(both.view(-1)[:vocab][None], history[:1], repetition=r[:1],
                                out=both.view(-1)[off:][:vocab][None])
    assert torch.equal(both, before)
    out = both[:, vocab + 8:]
    assert serving.edit_logits(x, history, repetition=r, out=out) is out
    assert torch.equal(out, want) and torch.equal(both[:, :vocab + 8], before[:, :vocab + 8])
    assert torch.equal(serving.edit_logits(x, history, repetition=r, out=x), want)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_a_cache_of_a_class_of_the_callers(codes):
    """Is what its base is."""
    class Mine(serving.QuantCache):
        pass

    b = Batch([37, 20], [37, 20], torch.bfloat16, 2, 64, 16, 4, seed=52)
    _, table, lens, starts = b.gpu()
    groups, shared = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 2], [0]))
    k, q = b.normal(57, 2, 64).cuda(), b.normal(57, 4, 64).cuda()
    got = []
    for kind in (serving.QuantCache, Mine):
        cache = kind.zeros(b.n_pages, 16, 2, 64, codes)
        assert type(cache) is kind
        serving.append(cache, table, lens, starts, k, -k)
        got.append((serving.prompt_attention(q, cache, table, lens, starts), serving.decode_attention(q[:2], cache, table, lens),
                    serving.shared_attention(q[:2], cache, table, lens, groups, shared),
                    *serving.read_rows(cache, table, lens, starts, torch.empty_like(k), torch.empty_like(k))))
    assert all(torch.equal(x, y) for x, y in zip(*got))
