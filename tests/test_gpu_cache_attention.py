"""mesh_transformer.cache.cache_attention against 64-bit attention over the same bf16 cache.

Tolerance of an output row, from the arithmetic: its storage rounds by half a step of its type relative to the value; scores in 32 bits
(sums of up to 256 products) and exponentials are off by under 2^-18 of the largest score (below 16 here) and the weights are multiplied
as bf16 numbers on the prompt path, half a step each, which the sum over values bounds by 2^-8 of the sum of |a v| at worst; the few-token
path keeps the weights to 2^-16."""
import numpy as np
import pytest
import torch

from cache_util import PAGE, Cache, host, rounding
from oracle import cache_oracle

pytestmark = pytest.mark.gpu


def _reference(c, q, lengths, fresh, window, sinks, scale):
    kp, vp = host(c.kpool), host(c.vpool)
    outs, received, spread = [], [], []
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        keys, values = cache_oracle.slots_of(kp, c.table[b], n), cache_oracle.slots_of(vp, c.table[b], n)
        o, r = cache_oracle.attention(host(q[b, :f]), keys, values, n, f, window, sinks, scale)
        m, _ = cache_oracle.attention(host(q[b, :f]), keys, np.abs(values), n, f, window, sinks, scale)
        outs.append(o)
        received.append(r)
        spread.append(m)
    return outs, received, spread


def _check(out, outs, spread, dtype, weight_rounding):
    for b, o in enumerate(outs):
        got = host(out[b, :len(o)])
        assert np.isfinite(got).all(), b
        room = rounding(dtype) * np.abs(o) + (weight_rounding + 2.0 ** -14) * spread[b]
        assert (np.abs(got - o) <= room + 1e-30).all(), (b, np.abs(got - o).max(), (np.abs(got - o) / room).max())
        assert float(out[b, len(o):].float().abs().sum()) == 0.0, b


def _run(seed, batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks, dtype, append=True, weights=False, scale=None,
         padded=0):
    from mesh_transformer.cache import cache_attention
    pages = max(1, (max(max(lengths), tokens) + PAGE - 1) // PAGE) + 1
    c = Cache(seed, batch, pages, kv_heads, d_head, lengths)
    q = c.rows(batch, tokens, heads, d_head, dtype, 1.5)
    k, v = c.rows(batch, tokens, kv_heads, d_head, dtype), c.rows(batch, tokens, kv_heads, d_head, dtype)
    if padded:                                            # slices of one fused row
        fused = torch.full((batch, tokens, (heads + 2 * kv_heads) * d_head + padded), float("nan"), dtype=dtype, device="cuda")
        fused[..., :heads * d_head] = q.flatten(2)
        fused[..., heads * d_head:(heads + kv_heads) * d_head] = k.flatten(2)
        fused[..., (heads + kv_heads) * d_head:(heads + 2 * kv_heads) * d_head] = v.flatten(2)
        q = fused[..., :heads * d_head].unflatten(2, (heads, d_head))
        k = fused[..., heads * d_head:(heads + kv_heads) * d_head].unflatten(2, (kv_heads, d_head))
        v = fused[..., (heads + kv_heads) * d_head:(heads + 2 * kv_heads) * d_head].unflatten(2, (kv_heads, d_head))
    before = [c.kpool.clone(), c.vpool.clone()]
    want = [c.kpool.clone(), c.vpool.clone()]
    if append:
        for b, (n, f) in enumerate(zip(lengths, fresh)):
            for t in range(f):
                slot = n - f + t
                for pool, rows in zip(want, (k, v)):
                    pool[int(c.table[b, slot // PAGE]), :, slot % PAGE] = rows[b, t].to(torch.bfloat16)
    new = torch.tensor(fresh, dtype=torch.int32, device="cuda")
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    w_in = w_out = None
    if weights:
        w_in = torch.rand((batch, kv_heads, pages * PAGE), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
        w_out = torch.full_like(w_in, -7.0)
    out = cache_attention(q, k if append else None, v if append else None, c.kpool, c.vpool, c.page_table, c.lengths_dev, new=new,
                          window=window, sinks=sinks, scale=scale, weights=w_in, weights_out=w_out, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for got, exp in zip((c.kpool, c.vpool), want if append else before):
        assert torch.equal(got.view(torch.int16), exp.view(torch.int16)), "slots other than the new ones changed, or the new ones did not"
    outs, received, spread = _reference(c, q, lengths, fresh, window or pages * PAGE, sinks, d_head ** -0.5 if scale is None else scale)
    return c, out, outs, received, spread, (w_in, w_out)


FEW = [
    # batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks
    (1, 4, 4, 64, 1, [1], [1], 1, 0),                                      # a token that sees itself
    (1, 4, 4, 64, 1, [127], [1], None, 0),
    (2, 16, 16, 256, 1, [300, 1], [1, 1], 128, 4),
    (3, 8, 2, 128, 1, [65, 64, 63], [1, 1, 1], 64, 1),                     # page borders
    (4, 8, 1, 128, 5, [700, 5, 130, 64], [5, 1, 3, 0], 100, 70),           # drafts, first tokens beyond a page, nothing new
    (2, 40, 8, 64, 3, [200, 77], [3, 2], 7, 16),                           # odd group
    (2, 6, 2, 256, 8, [513, 90], [8, 8], 33, 0),
    (1, 64, 1, 64, 2, [1000], [2], 999, 2),                                # the largest group
    (5, 3, 3, 128, 1, [0, 1, 2, 1500, 129], [0, 1, 1, 1, 1], None, 5),     # an empty sequence beside a long one
    (1, 2, 2, 128, 1, [6000], [1], None, 0),                               # one long sequence, cut into many pieces
    (1, 8, 8, 64, 1, [4100], [1], 70, 130),                                # first tokens and window far apart
    (2, 4, 2, 64, 16, [40, 16], [16, 16], 3, 2),                           # more new tokens than the window holds
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", FEW)
def test_few_tokens(cuda_device, case, dtype):
    batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks = case
    _, out, outs, _, spread, _ = _run(3, batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks, dtype)
    _check(out, outs, spread, dtype, 2.0 ** -16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", FEW)
def test_received_weights(cuda_device, case, dtype):
    """Every slot's weight to 2^-13 of itself (scores as above, so exponentials to 2^-14, and the same for the sum below them);
    slots that nobody sees keep what they had, slots behind the sequence are not written."""
    batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks = case
    _, out, outs, received, spread, (w_in, w_out) = _run(5, batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks, dtype,
                                                         weights=True)
    _check(out, outs, spread, dtype, 2.0 ** -16)
    w_in, w_out = w_in.double().cpu().numpy(), w_out.double().cpu().numpy()
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        before = w_in[b, :, :n].copy()
        before[:, n - f:] = 0
        want = before + received[b]
        assert (np.abs(w_out[b, :, :n] - want) <= 2.0 ** -13 * received[b] + 2.0 ** -22 * want).all()
        assert (w_out[b, :, n:] == -7.0).all()


def test_weights_in_place_and_from_nothing(cuda_device):
    from mesh_transformer.cache import cache_attention
    c = Cache(1, 2, 3, 2, 64, [150, 20])
    q = c.rows(2, 1, 4, 64, torch.bfloat16)
    a = torch.zeros((2, 2, 192), device="cuda")
    cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, weights_out=a)
    total = a.sum(-1).cpu().numpy()
    assert np.abs(total - 2.0).max() <= 1e-4                     # two heads a group, shares of one each
    b = torch.ones_like(a)
    cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, weights=b)
    for i, n in enumerate((150, 20)):
        want = a[i, :, :n] + 1.0
        want[:, n - 1] -= 1.0                                    # the new token's slot begins at zero
        assert torch.allclose(b[i, :, :n], want, atol=1e-6)
        assert (b[i, :, n:] == 1.0).all()


PROMPT = [
    (1, 2, 2, 256, 200, [200], [200], None, 0),
    (2, 4, 2, 128, 333, [500, 333], [333, 100], 64, 4),                    # history, ragged
    (1, 4, 4, 64, 129, [129], [129], 1, 0),                                # every token sees itself alone
    (1, 5, 1, 64, 257, [900], [257], 130, 70),                             # first tokens beyond a page
    (3, 2, 2, 128, 64, [64, 0, 1], [64, 0, 1], 10, 3),                     # an empty sequence
    (1, 2, 1, 256, 300, [1000], [300], 300, 16),
    (2, 3, 3, 64, 100, [640, 639], [100, 99], 65, 64),                     # last token at a page's end and before it
    (1, 8, 8, 128, 700, [700], [700], 2000, 4),                            # a window that hides nothing
]


@pytest.mark.parametrize("padded", [0, 24])
@pytest.mark.parametrize("case", PROMPT)
def test_prompts(cuda_device, case, padded):
    batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks = case
    _, out, outs, _, spread, _ = _run(7, batch, heads, kv_heads, d_head, tokens, lengths, fresh, window, sinks, torch.bfloat16, padded=padded)
    _check(out, outs, spread, torch.bfloat16, 2.0 ** -8)


@pytest.mark.parametrize("tokens,weights", [(90, False), (40, True)])
def test_prompts_in_32_bits_and_with_weights(cuda_device, tokens, weights):
    _, out, outs, received, spread, (w_in, w_out) = _run(9, 2, 4, 2, 128, tokens, [200, tokens], [tokens, tokens - 3], 50, 4, torch.float32,
                                                         weights=weights)
    _check(out, outs, spread, torch.float32, 2.0 ** -16)
    if weights:
        got = w_out[0, :, :200].double().cpu().numpy()
        before = w_in[0, :, :200].double().cpu().numpy()
        before[:, 200 - tokens:] = 0
        assert (np.abs(got - before - received[0]) <= 2.0 ** -13 * received[0] + 2.0 ** -22 * (before + received[0])).all()


@pytest.mark.parametrize("tokens", [1, 4, 150])
def test_rows_that_are_in_the_cache_already(cuda_device, tokens):
    _, out, outs, _, spread, _ = _run(11, 2, 4, 2, 64, tokens, [tokens + 60, tokens], [tokens, tokens], 40, 4, torch.bfloat16, append=False)
    _check(out, outs, spread, torch.bfloat16, 2.0 ** -8)


@pytest.mark.parametrize("tokens", [1, 100])
def test_scale_and_one_key_that_outweighs_all(cuda_device, tokens):
    """A score 60 above the others anywhere in the cache, the first and last slots of pages among its places."""
    from mesh_transformer.cache import cache_attention
    length = 400
    for place in (0, 3, 63, 64, 200, 319, length - tokens):
        c = Cache(13, 1, 7, 2, 128, [length])
        q = c.rows(1, tokens, 2, 128, torch.bfloat16)
        q[:] = q[:, :1]
        row = q[0, 0].float()
        c.kpool[int(c.table[0, place // PAGE]), :, place % PAGE] = (row * 60.0 / row.square().sum(-1, keepdim=True) / 0.5).to(torch.bfloat16)
        out = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=250, sinks=4, scale=0.5)
        for t in {0, tokens // 2, tokens - 1}:
            p = length - tokens + t
            keys, values = (cache_oracle.slots_of(host(x), c.table[0], p + 1) for x in (c.kpool, c.vpool))
            o, _ = cache_oracle.attention(host(q[0, t:t + 1]), keys, values, p + 1, 1, 250, 4, 0.5)
            m, _ = cache_oracle.attention(host(q[0, t:t + 1]), keys, np.abs(values), p + 1, 1, 250, 4, 0.5)
            # a score of 60 in 32 bits: 60 * 2^-18
            assert (np.abs(host(out[0, t]) - o[0]) <= 2.0 ** -9 * np.abs(o[0]) + (2.0 ** -8 + 60 * 2.0 ** -18) * m[0]).all(), (place, t)


def test_a_page_shared_by_two_sequences(cuda_device):
    """A common beginning is stored once."""
    from mesh_transformer.cache import cache_attention
    c = Cache(17, 2, 3, 2, 64, [130, 130])
    c.table[1, 0] = c.table[0, 0]
    c.page_table = torch.from_numpy(c.table).to("cuda")
    q = c.rows(2, 1, 4, 64, torch.bfloat16)
    out = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=100, sinks=4)
    outs, _, spread = _reference(c, q, [130, 130], [1, 1], 100, 4, 0.125)
    _check(out, outs, spread, torch.bfloat16, 2.0 ** -16)


@pytest.mark.parametrize("tokens", [1, 90])
def test_bad_lengths_and_pages_are_reported_and_left_alone(cuda_device, tokens):
    """A length beyond the pages, one below the new tokens, a negative one, and page numbers outside the pool: status bit 1, zeros or the
    other pages' result, and nothing written."""
    from mesh_transformer.cache import cache_attention
    c = Cache(19, 4, 3, 2, 64, [150, 150, 150, 150])
    q, k, v = (c.rows(4, tokens, h, 64, torch.bfloat16) for h in (4, 2, 2))
    lengths = torch.tensor([193, tokens - 1, -5, 150], dtype=torch.int32, device="cuda")
    before = c.kpool.clone()
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    out = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, lengths, window=100, sinks=4, status=status)
    assert int(status) == 2
    assert float(out[:3].float().abs().sum()) == 0.0
    outs, _, spread = _reference(c, q, [150] * 4, [tokens] * 4, 100, 4, 0.125)
    _check(out[3:], outs[3:], spread[3:], torch.bfloat16, 2.0 ** -8)
    # the new tokens' pages do not exist: nothing is stored
    table = c.page_table.clone()
    table[:, 1:] = torch.tensor([[-1], [8 * 12], [2 ** 31 - 1], [-2 ** 31]], dtype=torch.int32, device="cuda")
    status.zero_()
    short = torch.full((4,), 64 + tokens, dtype=torch.int32, device="cuda")
    cache_attention(q, k, v, c.kpool, c.vpool, table, short, window=100, sinks=4, status=status)
    torch.cuda.synchronize()
    assert int(status) == 2
    assert torch.equal(c.kpool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("tokens", [1, 6, 200])
def test_captured_and_replayed_on_another_stream(cuda_device, tokens):
    """The call is captured once and replayed with other lengths, queries and page tables in the same tensors."""
    from mesh_transformer.cache import cache_attention
    c = Cache(23, 2, 6, 2, 128, [300, 210])
    q, k, v = (c.rows(2, tokens, h, 128, torch.bfloat16) for h in (4, 2, 2))
    weights = torch.zeros((2, 2, 384), device="cuda") if tokens < 10 else None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=90, sinks=4, weights_out=weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=90, sinks=4, weights_out=weights)
    for lengths in ([300, 210], [280, 201]):
        q.copy_(c.rows(2, tokens, 4, 128, torch.bfloat16))
        c.lengths_dev.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got, got_w = out.clone(), None if weights is None else weights.clone()
        again = cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=90, sinks=4, weights_out=weights)
        torch.cuda.synchronize()
        assert torch.equal(got, again)
        if weights is not None:
            assert torch.equal(got_w, weights)
        outs, _, spread = _reference(c, q, lengths, [tokens] * 2, 90, 4, 128 ** -0.5)
        _check(got, outs, spread, torch.bfloat16, 2.0 ** -8)


def test_two_calls_at_once(cuda_device):
    """Two streams at work on caches of their own give what each gives alone."""
    from mesh_transformer.cache import cache_attention
    sets = []
    for seed in (29, 31):
        c = Cache(seed, 8, 20, 4, 128, [1200 - 9 * i for i in range(8)])
        sets.append((c, c.rows(8, 1, 16, 128, torch.bfloat16), torch.zeros((8, 4, 1280), device="cuda")))
    call = lambda c, q, w: cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, weights_out=w)
    alone = [(call(*s), s[2].clone()) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        outs = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                outs.append(call(*s))
        torch.cuda.synchronize()
        for (want, w), got, s in zip(alone, outs, sets):
            assert torch.equal(want, got) and torch.equal(w, s[2])


def test_same_bits_every_time(cuda_device):
    from mesh_transformer.cache import cache_attention
    for tokens in (1, 5, 300):
        c = Cache(37, 3, 30, 2, 128, [1900, 900, 350])
        q = c.rows(3, tokens, 16, 128, torch.bfloat16)
        first = None
        for _ in range(10):
            w = torch.zeros((3, 2, 1920), device="cuda") if tokens < 10 else None
            out = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=800, sinks=4, weights_out=w)
            if first is None:
                first = out, w
            assert torch.equal(first[0], out) and (w is None or torch.equal(first[1], w))


def test_output_of_the_callers_own_with_wide_rows(cuda_device):
    from mesh_transformer.cache import cache_attention
    for tokens in (1, 80):
        c = Cache(41, 2, 4, 2, 64, [200, 100])
        q = c.rows(2, tokens, 4, 64, torch.bfloat16)
        wide = torch.full((2, tokens, 4 * 64 + 40), 5.0, dtype=torch.bfloat16, device="cuda")
        out = wide[..., :256].unflatten(2, (4, 64))
        assert cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=50, out=out) is not None
        want = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=50)
        assert torch.equal(wide[..., :256].reshape(want.shape), want) and (wide[..., 256:] == 5.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,d_head,tokens", [(8, 8, 64, 1), (16, 4, 64, 5), (16, 4, 128, 1), (24, 4, 128, 4), (6, 6, 256, 1), (16, 2, 256, 2)])
def test_many_long_sequences(cuda_device, heads, kv_heads, d_head, tokens, dtype):
    """More tiles than blocks: a block works on parts of several sequences, and rings go round many times."""
    from mesh_transformer.cache import cache_attention
    lengths = [6000 - 331 * i for i in range(17)]
    window, sinks, group = 4000, 4, heads // kv_heads
    c = Cache(43, 17, 94, kv_heads, d_head, lengths)
    q, k, v = (c.rows(17, tokens, h, d_head, dtype) for h in (heads, kv_heads, kv_heads))
    w = torch.zeros((17, kv_heads, 94 * 64), device="cuda")
    for _ in range(3):
        out = cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=window, sinks=sinks, weights_out=w)
    for b, n in enumerate(lengths):
        table = c.page_table[b].long()
        keys, values = (x[table].transpose(0, 1).reshape(kv_heads, -1, d_head)[:, :n].double() for x in (c.kpool, c.vpool))
        p = torch.arange(n - tokens, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = (j > p) | ((j >= sinks) & (p - j >= window))
        qb = q[b].double().reshape(tokens, kv_heads, group, d_head).permute(1, 2, 0, 3)
        share = torch.softmax((torch.einsum("hgtd,hjd->hgtj", qb, keys) * d_head ** -0.5).masked_fill(hidden, float("-inf")), -1)
        want = torch.einsum("hgtj,hjd->thgd", share, values).reshape(tokens, heads, d_head)
        spread = torch.einsum("hgtj,hjd->thgd", share, values.abs()).reshape(tokens, heads, d_head)
        assert ((out[b].double() - want).abs() <= rounding(dtype) * want.abs() + 2.0 ** -13 * spread).all(), b
        received = share.sum((1, 2))
        assert ((w[b, :, :n].double() - received).abs() <= 2.0 ** -13 * received).all(), b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,d_head,heads,weights", [(1, 64, 4, True), (1, 128, 2, False), (6, 256, 4, True), (150, 64, 2, False), (150, 128, 2, False),
                                                         (300, 128, 4, False), (150, 256, 2, False), (40, 256, 4, False)])
def test_slots_that_no_token_sees_may_hold_anything(cuda_device, tokens, d_head, heads, weights, dtype):
    """Between the first tokens and the window: NaN and infinities in pages that are seen in part, no page at all elsewhere."""
    from mesh_transformer.cache import cache_attention
    for length, window, sinks in ((tokens + 900, 200, 4), (tokens + 900, 129, 70), (tokens + 400, 320, 64), (tokens + 130, 100, 1)):
        pages = (length + PAGE - 1) // PAGE
        c = Cache(47, 1, pages, 2, d_head, [length])
        q = c.rows(1, tokens, heads, d_head, dtype, 1.5)
        outs, _, spread = _reference(c, q, [length], [tokens], window, sinks, d_head ** -0.5)
        low = length - tokens - window + 1
        for j in range(sinks, low):
            c.kpool[int(c.table[0, j // PAGE]), :, j % PAGE] = (float("nan"), float("inf"), float("-inf"))[j % 3]
            c.vpool[int(c.table[0, j // PAGE]), :, j % PAGE] = (float("inf"), float("nan"), float("-inf"))[j % 3]
        hidden = [i for i in range(pages) if i * PAGE >= sinks and (i + 1) * PAGE <= low]
        c.page_table[0, hidden] = -1
        status = torch.zeros((1,), dtype=torch.int32, device="cuda")
        w = torch.zeros((1, 2, pages * PAGE), device="cuda") if weights else None
        out = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=window, sinks=sinks, weights_out=w, status=status)
        assert int(status) == 0
        _check(out, outs, spread, dtype, 2.0 ** -8)
        if weights:
            assert torch.isfinite(w).all() and float(w[:, :, sinks:low].abs().sum()) == 0.0


@pytest.mark.parametrize("tokens,d_head", [(1, 128), (4, 64), (200, 64), (200, 128), (200, 256)])
def test_a_key_that_is_not_a_number(cuda_device, tokens, d_head):
    """Rows that see it are NaN throughout, the others as without it, wherever in a block the key lies."""
    from mesh_transformer.cache import cache_attention
    length = tokens + 300
    for place in list(range(120, 136)) + [length - tokens // 2 - 1]:
        c = Cache(53, 1, 9, 2, d_head, [length])
        q = c.rows(1, tokens, 4, d_head, torch.bfloat16)
        call = lambda: cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=250, sinks=4)
        want = call()
        c.kpool[int(c.table[0, place // PAGE]), 1, place % PAGE] = float("nan")
        got = call()
        p = torch.arange(length - tokens, length, device="cuda")
        sees = (place <= p) & (p - place < 250)
        assert got[0, sees][:, 2:].isnan().all()
        assert torch.equal(got[0, :, :2], want[0, :, :2]) and torch.equal(got[0, ~sees], want[0, ~sees])


def _dense(q, keys, values, p, j, window, sinks):
    """64-bit attention [batch, tokens, heads, d] over slots of their own; ``p`` [batch, tokens] slots of the tokens, -1: none."""
    batch, tokens, heads, d = q.shape
    kv_heads, group = keys.shape[1], heads // keys.shape[1]
    hidden = (j > p[..., None]) | ((j >= sinks) & (p[..., None] - j >= window))
    s = torch.einsum("btghd,bgjd->bghtj", q.double().unflatten(2, (kv_heads, group)), keys.double()) * d ** -0.5
    share = torch.nan_to_num(torch.softmax(s.masked_fill(hidden[:, None, None], float("-inf")), -1))
    out = lambda v: torch.einsum("bghtj,bgjd->btghd", share, v).flatten(2, 3)
    return out(values.double()), out(values.double().abs()), share.sum((2, 3))


@pytest.mark.parametrize("batch,tokens,heads,kv_heads,weights", [(300, 1, 4, 2, True), (300, 5, 2, 2, False), (513, 2, 2, 1, True),
                                                                 (8300, 65, 2, 2, False), (1100, 129, 1, 1, False)])
def test_more_sequences_than_a_launch_plans(cuda_device, batch, tokens, heads, kv_heads, weights):
    from mesh_transformer.cache import cache_attention
    d_head, pages, window, sinks = 64, 3, 70, 3
    g = torch.Generator("cuda").manual_seed(59)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    kpool, vpool = rand(batch * pages, kv_heads, PAGE, d_head), rand(batch * pages, kv_heads, PAGE, d_head)
    table = torch.randperm(batch * pages, generator=g, device="cuda").to(torch.int32).reshape(batch, pages)
    new = torch.randint(0, tokens + 1, (batch,), generator=g, device="cuda").to(torch.int32)
    lengths = (new + torch.randint(0, pages * PAGE - tokens + 1, (batch,), generator=g, device="cuda")).to(torch.int32)
    q = rand(batch, tokens, heads, d_head)
    w = torch.zeros((batch, kv_heads, pages * PAGE), device="cuda") if weights else None
    out = cache_attention(q, None, None, kpool, vpool, table, lengths, new=new, window=window, sinks=sinks, weights_out=w)
    for b in range(0, batch, 512):
        part = slice(b, b + 512)
        keys, values = (x[table[part].long()].transpose(1, 2).flatten(2, 3) for x in (kpool, vpool))
        t = torch.arange(tokens, device="cuda")
        p = torch.where(t < new[part, None], lengths[part, None] - new[part, None] + t, -1)
        want, spread, received = _dense(q[part], keys, values, p, torch.arange(pages * PAGE, device="cuda"), window, sinks)
        assert ((out[part].double() - want).abs() <= rounding(torch.bfloat16) * want.abs() + 2.0 ** -8 * spread).all(), b
        if weights:
            assert ((w[part].double() - received).abs() <= 2.0 ** -13 * received).all(), b


@pytest.mark.parametrize("tokens", [1, 130])
def test_a_pool_of_more_than_32_bits(cuda_device, tokens):
    """Pages behind the pool's first 2^32 bytes and 2^31 elements: attention, storing and eviction."""
    from mesh_transformer.cache import cache_attention, cache_evict
    d_head, kv_heads, heads, pages = 256, 4, 4, 5
    n_pages = 2 ** 31 // (kv_heads * PAGE * d_head) + 40
    if torch.cuda.mem_get_info()[0] < 5 * n_pages * kv_heads * PAGE * d_head:
        pytest.skip("not enough memory")
    g = torch.Generator("cuda").manual_seed(61)
    kpool = torch.empty((n_pages, kv_heads, PAGE, d_head), dtype=torch.bfloat16, device="cuda")
    vpool = torch.empty_like(kpool)
    for pool in (kpool, vpool):
        pool[-40:].normal_(generator=g)
    table = (n_pages - 40 + torch.randperm(40, generator=g, device="cuda")[:2 * pages]).to(torch.int32).reshape(2, pages)
    lengths = torch.tensor([300, 257], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn((2, tokens, heads, d_head), generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    out = cache_attention(q, k, v, kpool, vpool, table, lengths, window=200, sinks=4)
    keys, values = (x[table.long()].transpose(1, 2).flatten(2, 3) for x in (kpool, vpool))
    p = lengths[:, None] - tokens + torch.arange(tokens, device="cuda")
    for b in range(2):
        assert torch.equal(keys[b, :, p[b].long()].transpose(0, 1), k[b]) and torch.equal(values[b, :, p[b].long()].transpose(0, 1), v[b])
    want, spread, _ = _dense(q, keys, values, p, torch.arange(pages * PAGE, device="cuda"), 200, 4)
    assert ((out.double() - want).abs() <= rounding(torch.bfloat16) * want.abs() + 2.0 ** -8 * spread).all()
    used = set(table.flatten().tolist())
    spare = torch.tensor([x for x in range(n_pages - 40, n_pages) if x not in used][:2], dtype=torch.int32, device="cuda").reshape(2, 1)
    weights = torch.rand((2, kv_heads, pages * PAGE), generator=g, device="cuda")
    kept, _, _, cut = cache_evict(kpool, vpool, table, lengths, weights, spare, 64, first=4, last=16)
    assert torch.equal(cut[:, :1], spare)
    for b in range(2):
        for h in range(kv_heads):
            for pool, rows in ((kpool, keys), (vpool, values)):
                assert torch.equal(pool[int(spare[b, 0]), h], rows[b, h, kept[b, h].long()])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,d_head,tokens", [(10, 2, 64, 4), (24, 4, 128, 3), (40, 8, 64, 5), (8, 1, 128, 5), (12, 2, 64, 9), (5, 1, 256, 4)])
def test_rows_that_fill_three_eighths_and_five(cuda_device, heads, kv_heads, d_head, tokens, dtype):
    """17 to 24 rows a key head, and 25 to 54 in tiles of which the last has rows left over; weights and ragged lengths with them."""
    lengths, fresh = [700, tokens, 65, 1300], [tokens, tokens, tokens - 1, tokens]
    _, out, outs, received, spread, (w_in, w_out) = _run(67, 4, heads, kv_heads, d_head, tokens, lengths, fresh, 500, 9, dtype, weights=True)
    _check(out, outs, spread, dtype, 2.0 ** -16)
    _, out, outs, _, spread, _ = _run(67, 4, heads, kv_heads, d_head, tokens, lengths, fresh, 500, 9, dtype)
    _check(out, outs, spread, dtype, 2.0 ** -16)
    w_in, w_out = w_in.double().cpu().numpy(), w_out.double().cpu().numpy()
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        before = w_in[b, :, :n].copy()
        before[:, n - f:] = 0
        assert (np.abs(w_out[b, :, :n] - before - received[b]) <= 2.0 ** -13 * received[b] + 2.0 ** -22 * (before + received[b])).all()


@pytest.mark.parametrize("d_heads", [(256, 256), (128, 64), (256, 128)])
def test_two_prompts_at_once(cuda_device, d_heads):
    """Two streams with prompts of their own, each storing its keys and values, replayed from graphs: what each gives alone."""
    from mesh_transformer.cache import cache_attention
    sets = []
    for seed, d_head in zip((71, 73), d_heads):
        c = Cache(seed, 3, 12, 2, d_head, [700, 333, 512])
        sets.append((c, *(c.rows(3, 320, h, d_head, torch.bfloat16) for h in (4, 2, 2))))
    call = lambda c, q, k, v: cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=300, sinks=4)
    alone = [call(*s) for s in sets]
    pools = [s[0].kpool.clone() for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(*s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for want, got, s, pool in zip(alone, outs, sets, pools):
            assert torch.equal(want, got) and torch.equal(s[0].kpool.view(torch.int16), pool.view(torch.int16))


def test_python_refusals_with_tensors_on_a_gpu(cuda_device):
    from mesh_transformer.cache import cache_attention, cache_evict
    from mesh_transformer.sampling import verify_drafts
    c = Cache(79, 2, 3, 2, 64, [100, 90])
    q, k = c.rows(2, 3, 4, 64, torch.bfloat16), c.rows(2, 3, 2, 64, torch.bfloat16)
    good = dict(q=q, k=k, v=k, kpool=c.kpool, vpool=c.vpool, page_table=c.page_table, lengths=c.lengths_dev)
    before = c.kpool.clone()
    w = torch.zeros((2, 2, 192), device="cuda")
    for bad in (dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[:, :, 0]), dict(q=None), dict(k=None), dict(v=None),
                dict(k=k.float()), dict(k=k.cpu()), dict(v=k[:, :2]), dict(v=q), dict(kpool=c.kpool.float()), dict(kpool=c.kpool.cpu()),
                dict(kpool=c.kpool.transpose(0, 1)), dict(kpool=c.kpool[:, :, :32]), dict(vpool=c.vpool[1:]), dict(vpool=c.vpool.cpu()),
                dict(vpool=None), dict(page_table=c.page_table.long()), dict(page_table=c.page_table[0]), dict(page_table=c.page_table.cpu()),
                dict(page_table=c.page_table.t().contiguous().t()), dict(lengths=c.lengths_dev[:1]), dict(lengths=c.lengths_dev.float()),
                dict(lengths=[100, 90]), dict(new=c.lengths_dev[:1]), dict(new=c.lengths_dev.cpu()), dict(status=c.lengths_dev), dict(weights=w.double()),
                dict(weights=w[:, :1]), dict(weights_out=w.cpu()), dict(out=q.float()), dict(out=torch.empty_like(q)[:1]),
                dict(out=torch.empty((2, 3, 4, 128), dtype=torch.bfloat16, device="cuda")[..., ::2]), dict(window=0), dict(window=1.5), dict(sinks=-1),
                dict(scale=0.0), dict(scale="1")):
        with pytest.raises(ValueError):
            cache_attention(**{**good, **bad})
    spare = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    for bad in (dict(weights=w.half()), dict(weights=w[:, :, :64]), dict(spare_pages=spare.long()), dict(spare_pages=spare[:1]), dict(keep=0), dict(keep=65),
                dict(first=60, last=5), dict(first=-1), dict(status=spare), dict(lengths=c.lengths_dev.cpu())):
        with pytest.raises(ValueError):
            cache_evict(**{**dict(kpool=c.kpool, vpool=c.vpool, page_table=c.page_table, lengths=c.lengths_dev, weights=w, spare_pages=spare, keep=64), **bad})
    logits, u = torch.zeros((2, 3, 50), device="cuda"), torch.full((2, 50), 0.5, device="cuda")
    drafts = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    good = dict(target_logits=logits, draft_logits=logits[:, :2], draft_tokens=drafts, accept=u[:, :2], noise=u)
    for bad in (dict(target_logits=logits.half()), dict(target_logits=logits.cpu()), dict(target_logits=logits[0]), dict(target_logits=None),
                dict(draft_logits=logits), dict(draft_logits=logits[:, :2].bfloat16()), dict(draft_tokens=drafts.long()), dict(draft_tokens=drafts[:1]),
                dict(accept=u), dict(noise=u.double()), dict(noise=u.cpu()), dict(count=drafts), dict(temp=None), dict(temp="1"), dict(temp=float("inf")),
                dict(temp=u), dict(temp=torch.ones(2, dtype=torch.float64, device="cuda"))):
        with pytest.raises(ValueError):
            verify_drafts(**{**good, **bad})
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.int16), c.kpool.view(torch.int16))


@pytest.mark.parametrize("tokens,d_head", [(1, 64), (5, 128), (200, 64), (200, 128), (200, 256)])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 40, 2 ** 40), (1, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_windows_and_first_tokens_at_the_ends_of_their_range(cuda_device, tokens, d_head, window, sinks):
    _, out, outs, _, spread, _ = _run(83, 2, 4, 2, d_head, tokens, [tokens + 310, tokens], [tokens, tokens], window, sinks, torch.bfloat16)
    _check(out, outs, spread, torch.bfloat16, 2.0 ** -8)
