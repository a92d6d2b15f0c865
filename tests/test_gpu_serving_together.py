"""A decode step of characters of one world, as a host runs it: new tokens into an
8-bit cache, attention behind the pages that the sessions share, edits of the logits
and a draw, captured once and replayed."""

import math

import pytest
import torch

import serving_more_plain as more
import serving_plain as plain
from rpgbarengine_amd import serving
from test_gpu_serving import close
from test_gpu_serving_codes import attention, weight_bits

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, VOCAB = 8, 2, 64, 16, 500
SHARED, SESSIONS, ROOM, STEPS = 48, 5, 8, 5


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn, None], ids=["i8", "e4m3", "rows"])
def test_steps_of_a_shared_world(codes):
    g = torch.Generator().manual_seed(3)
    dtype = torch.bfloat16

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g) * by).to(dtype)

    # The world's description once, in pages that every session's table names; then each
    # session's own turn, of another length each.
    world_pages, own_pages = SHARED // PAGE, ROOM
    n_pages = world_pages + SESSIONS * own_pages + 2
    order = torch.randperm(n_pages, generator=g).int()
    table = torch.empty(SESSIONS, world_pages + own_pages, dtype=torch.int32)
    table[:, :world_pages] = order[:world_pages]
    table[:, world_pages:] = order[world_pages:world_pages + SESSIONS * own_pages].view(SESSIONS, own_pages)
    if codes is None:
        cache = serving.PagedCache.zeros(n_pages, PAGE, KV, DIM, dtype)
    else:
        cache = serving.QuantCache.zeros(n_pages, PAGE, KV, DIM, codes)
    ang = torch.rand(200, DIM // 2, generator=g) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    gain = (1 + 0.1 * torch.randn(DIM, generator=g)).cuda()
    table_d = table.cuda()

    def prompt(row, lens, k, v, q):
        """The last k.shape[0] positions of a session: cached and attended."""
        starts = torch.tensor([0, k.shape[0]], dtype=torch.int32).cuda()
        n = torch.tensor([lens], dtype=torch.int32).cuda()
        t = table_d[row:row + 1]
        q = serving.append(cache, t, n, starts, k.cuda(), v.cuda(), q=q.cuda(), q_norm=gain, k_norm=gain, rope=rope)
        return serving.prompt_attention(q, cache, t, n, starts)

    prompt(0, SHARED, normal(SHARED, KV, DIM), normal(SHARED, KV, DIM), normal(SHARED, HEADS, DIM))
    lens = [SHARED]
    for s in range(SESSIONS):
        turn = 3 + 7 * s
        if s:
            lens.append(SHARED)
        lens[s] += turn
        prompt(s, lens[s], normal(turn, KV, DIM), normal(turn, KV, DIM), normal(turn, HEADS, DIM))

    # One step's buffers: the projections write into qkv and logits.
    qkv = torch.zeros(SESSIONS, HEADS + 2 * KV, DIM, dtype=dtype, device="cuda")
    logits = torch.zeros(SESSIONS, VOCAB, dtype=dtype, device="cuda")
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    starts = torch.arange(SESSIONS + 1, dtype=torch.int32).cuda()
    groups, shared = torch.tensor([0, SESSIONS], dtype=torch.int32).cuda(), torch.tensor([SHARED], dtype=torch.int32).cuda()
    history = torch.randint(0, VOCAB, (SESSIONS, 64), generator=g, dtype=torch.int32).cuda()
    history_lens = torch.tensor([7, 0, 20, 1, 5], dtype=torch.int32).cuda()
    repetition = torch.tensor([1.3, 1.0, 1.1, 2.0, 1.2]).cuda()
    frequency = torch.tensor([0.0, 0.5, 0.1, 0.0, 0.3]).cuda()
    mask = torch.randint(-(1 << 31), 1 << 31, (2, (VOCAB + 31) // 32), generator=g).int().cuda()
    mask_rows = torch.tensor([-1, 0, 1, -1, 0], dtype=torch.int32).cuda()
    u, greedy = torch.zeros(SESSIONS).cuda(), torch.zeros(SESSIONS).cuda()

    def step():
        q = serving.append(cache, table_d, lens_d, starts, qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:], q=qkv[:, :HEADS],
                           q_norm=gain, k_norm=gain, rope=rope)
        out = serving.shared_attention(q, cache, table_d, lens_d, groups, shared)
        x = serving.edit_logits(logits, history, history_lens, repetition=repetition, frequency=frequency, mask=mask,
                                mask_rows=mask_rows)
        return q, out, x, serving.sample(x, u, greedy)[0]

    def pools():
        return [x.cpu().float() for x in ((cache.k, cache.v) if codes is None else
                                          (cache.k, cache.v, cache.k_scale, cache.v_scale))]

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        lens_d.add_(1)
        step()  # (what it caches is cached again by the first replay)
        lens_d.sub_(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for at in range(STEPS):
        qkv.copy_(normal(SESSIONS, HEADS + 2 * KV, DIM))
        x = normal(SESSIONS, VOCAB, by=3.0)
        logits.copy_(x)
        lens_d.add_(1)
        before = [p.clone() for p in pools()]
        graph.replay()
        torch.cuda.synchronize()
        q, out, edited, tokens = (t.cpu() for t in got)
        held = pools()
        n_now = lens_d.tolist()
        assert n_now == [n + at + 1 for n in lens]
        for s, n in enumerate(n_now):
            # one row of each head changed, and only there
            page, r = int(table[s, (n - 1) // PAGE]), (n - 1) % PAGE
            for p in before:
                p[page, :, r] = 0
            rows = [plain.sequence_rows(p, table[s], n)[0] for p in held[:2]]
            there = torch.ones(n, dtype=torch.bool)
            if codes is None:
                close(out[s], *plain.attention(q[s], *rows, there, DIM ** -0.5, dtype))
            else:
                scales = [plain.sequence_rows(p[..., None], table[s], n)[0][..., 0] for p in held[2:]]
                close(out[s], *attention(q[s], *rows, *scales, there, DIM ** -0.5, dtype, weight_bits(dtype, False)))
        for p, now in zip(before, held):
            now = now.clone()
            for s, n in enumerate(n_now):
                now[int(table[s, (n - 1) // PAGE]), :, (n - 1) % PAGE] = 0
            assert torch.equal(p, now)
        for s in range(SESSIONS):
            m = int(mask_rows[s])
            allowed = None if m < 0 else (((mask[m].cpu().long()[:, None] >> torch.arange(32)) & 1).reshape(-1)[:VOCAB] == 1)
            want, mag = more.edit(x[s].double(), history[s, :int(history_lens[s])].tolist(), 0, float(repetition[s]), 0.0,
                                  float(frequency[s]), [], allowed)
            low = want == -math.inf
            assert torch.equal(edited[s].double() == -math.inf, low)
            bound = 5 * 2.0 ** -24 * mag + plain.EPS[dtype] * (1 + 2.0 ** -20) * mag
            assert bool(((edited[s].double() - want).abs() <= bound)[~low].all())
            assert int(tokens[s]) == int(edited[s].float().argmax())
            # the token goes into the history, as a host does it
            history[s, int(history_lens[s])] = int(tokens[s])
        history_lens.add_(1)
