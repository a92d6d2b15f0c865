"""How exact the serving operators over an 8-bit cache are: their outputs against
float64 definitions, measured by what the outputs' own rounding leaves."""

import pytest
import torch

from rpgbarengine_amd import serving
from test_gpu_serving import Batch, close
from test_gpu_serving_codes import CODES, expect, ident, on_cpu, random_cache, rows_of, scales_of

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
# tiles of 32 rows by eight waves, by four, in several ranges, and tiles of 128 rows
SIZES = {"few": ([70, 290, 33], [9, 20, 33], 128, 8, 2), "short": ([64, 30], [64, 30], 64, 6, 3),
         "long": ([1500], [12], 128, 4, 1), "many": ([150, 330], [150, 200], 64, 192, 32)}


def exact(b, cache, q, scale):
    """The packed tokens' outputs in float64, without any rounding."""
    k, v, ks, vs = cache
    out = torch.zeros(b.tokens, b.heads, b.dim, dtype=torch.float64)
    for i, (n, m) in enumerate(zip(b.lens, b.new)):
        kk, vv = rows_of(k, b, i, n)[0], rows_of(v, b, i, n)[0]
        ss, tt = scales_of(ks, b, i, n)[0].double(), scales_of(vs, b, i, n)[0].double()
        at = slice(int(b.starts[i]), int(b.starts[i]) + m)
        hidden = torch.arange(n)[None, :] > torch.arange(n - m, n)[:, None]
        for h in range(b.heads):
            g = h // (b.heads // b.kv)
            s = (q[at, h].double() @ kk[g].t()) * ss[g] * scale
            out[at, h] = (torch.softmax(s.masked_fill(hidden, -torch.inf), 1) * tt[g]) @ vv[g]
    return out


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", HALVES, ids=ident)
@pytest.mark.parametrize("size", SIZES)
def test_prompts_are_as_exact_as_their_rounding(codes, dtype, size):
    """Root mean squares of the error and of what rounding the exact output leaves, a
    half step of 2^-12 (f16) or 2^-9 over the square root of 3 of the output. A weight
    times its scale is held in 16 bits: 2^-17 over that root, each apart from the
    others, so of the output of values of either sign as much; that is 1/32 of an f16
    rounding. Scores of up to a few units in f32 add some 2^-19 of the output, 1/60 of
    it. Together less than a thousandth of the whole; 5 hundredths are allowed. (Weights
    rounded to the rows' type once would make it 1.41.)"""
    lens, new, dim, heads, kv = SIZES[size]
    b = Batch(lens, new, dtype, kv, dim, 16, heads, seed=31)
    q = b.normal(b.tokens, heads, dim, by=0.2)
    _, table, lens_d, starts = b.gpu()
    cache = random_cache(b, codes)
    got = serving.prompt_attention(q.cuda(), cache, table, lens_d, starts).double().cpu()
    want = exact(b, on_cpu(cache), q, dim ** -0.5)
    # the first tokens see one key: their weight is 1 in any form
    least = (want.to(dtype).double() - want).square().mean().sqrt()
    assert float((got - want).square().mean().sqrt()) <= 1.05 * float(least)


@pytest.mark.parametrize("codes", CODES, ids=ident)
@pytest.mark.parametrize("dtype", [torch.float32, *HALVES], ids=ident)
@pytest.mark.parametrize("dim,heads,kv,new", [(128, 4, 2, 20), (64, 192, 32, 300)], ids=["few", "many"])
@pytest.mark.parametrize("power", [30, 110])
def test_a_large_value_of_a_later_token(codes, dtype, dim, heads, kv, new, power):
    """The last token's value row has a scale far above the others': the tokens before
    it do not see it and come out as they are without it."""
    b = Batch([330], [new], dtype, kv, dim, 16, heads, seed=32)
    q = b.normal(b.tokens, heads, dim, by=0.3)
    _, table, lens, starts = b.gpu()
    cache = random_cache(b, codes)
    held = on_cpu(cache)
    cache.v_scale[int(b.table[0, 329 // 16]), :, 329 % 16] = 2.0 ** power
    got = serving.prompt_attention(q.cuda(), cache, table, lens, starts)
    for j in (0, new // 2, new - 9, new - 2):
        # (weights in 16 bits, f32 in 24: what decode attention is held to)
        close(got[j], *expect(b, held, q, dim ** -0.5, 0, 330 - new + j, j))
