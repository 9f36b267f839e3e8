"""mesh_transformer.cache.cache_evict against the plain form: whole numbers and copied rows, so everything is equal."""
import numpy as np
import pytest
import torch

from cache_util import PAGE, Cache
from oracle import cache_oracle

pytestmark = pytest.mark.gpu


def _weights(c, batch, kv_heads, slots, kind):
    if kind == "spread":
        w = c.rng.random((batch, kv_heads, slots), dtype=np.float32) ** -0.7
    elif kind == "equal":
        w = np.full((batch, kv_heads, slots), 0.25, np.float32)
    elif kind == "few":                                              # many ties, zeros of both signs
        w = c.rng.choice(np.array([0.0, -0.0, 1.0, 2.0, 2.0000002], np.float32), (batch, kv_heads, slots))
    else:                                                            # signs, infinities, denormals
        w = c.rng.choice(np.array([-np.inf, -3.0, -1e-40, 0.0, 1e-40, 1e-38, 5.0, np.inf], np.float32), (batch, kv_heads, slots))
    return w


@pytest.mark.parametrize("kind", ["spread", "equal", "few", "wild"])
@pytest.mark.parametrize("batch,kv_heads,d_head,lengths,keep,first,last", [
    (1, 4, 64, [511], 256, 4, 32),
    (3, 2, 128, [700, 100, 300], 200, 0, 0),                          # one sequence stays as it is
    (2, 1, 256, [65, 64], 64, 1, 63),                                 # one slot goes; nothing goes
    (2, 3, 64, [5000, 1], 1, 0, 1),                                   # one slot stays
    (1, 2, 128, [1025], 1024, 1000, 24),                              # nothing between first and last stays
    (4, 1, 64, [0, 2, 130, 129], 129, 3, 7),                          # an empty sequence
    (1, 2, 64, [9000], 4097, 16, 512),
    (1, 1, 128, [100], 5000, 4, 4),                                   # more than the cache holds
])
def test_eviction(cuda_device, batch, kv_heads, d_head, lengths, keep, first, last, kind):
    from mesh_transformer.cache import cache_evict
    pages = max(1, (max(lengths) + PAGE - 1) // PAGE)
    n_spare = (keep + PAGE - 1) // PAGE
    c = Cache(len(lengths) * 100 + keep, batch, pages, kv_heads, d_head, lengths, spare=batch * n_spare)
    slots = pages * PAGE
    w = _weights(c, batch, kv_heads, slots, kind)
    wd = torch.from_numpy(w).to("cuda")
    spare = torch.from_numpy(c.spare.reshape(batch, n_spare)).to("cuda")
    pools = [c.kpool.clone(), c.vpool.clone()]
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    kept, lengths_out, weights_out, table = cache_evict(c.kpool, c.vpool, c.page_table, c.lengths_dev, wd, spare, keep, first=first, last=last,
                                                        status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    assert lengths_out.tolist() == [min(n, keep) for n in lengths]
    assert c.lengths_dev.tolist() == lengths and torch.equal(wd.cpu(), torch.from_numpy(w))
    kept, weights_out, table = kept.cpu().numpy(), weights_out.cpu().numpy(), table.cpu().numpy()
    for b, n in enumerate(lengths):
        for h in range(kv_heads):
            want = cache_oracle.evict(w[b, h], n, keep, first, last)
            assert kept[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert np.array_equal(weights_out[b, h], np.concatenate([w[b, h, want], np.zeros(slots - len(want), np.float32)]))
            if n > keep:
                for pool in pools:
                    rows = torch.stack([pool[int(c.table[b, j // PAGE]), h, j % PAGE] for j in want])
                    for i in range(n_spare):
                        part = rows[i * PAGE:(i + 1) * PAGE]
                        pool[int(spare[b, i]), h, :len(part)] = part
        if n > keep:
            assert table[b].tolist() == (spare[b].tolist() + [-1] * pages)[:pages]
        else:
            assert table[b].tolist() == c.table[b].tolist()
    for got, want in zip((c.kpool, c.vpool), pools):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_bad_lengths_and_pages(cuda_device):
    """A length beyond the pages counts as none, rows of pages that do not exist are not copied; the status says so."""
    from mesh_transformer.cache import cache_evict
    c = Cache(5, 3, 4, 2, 64, [256, 256, 256], spare=3)
    lengths = torch.tensor([257, -1, 256], dtype=torch.int32, device="cuda")
    table = c.page_table.clone()
    table[2, 1] = 999
    w = torch.rand((3, 2, 256), device="cuda")
    before = c.kpool.clone()
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    spare = torch.from_numpy(c.spare.reshape(3, 1)).to("cuda")
    spare[1] = -7                                                        # not used: its sequence gives nothing up
    kept, lengths_out, _, _ = cache_evict(c.kpool, c.vpool, table, lengths, w, spare, 64, status=status)
    torch.cuda.synchronize()
    assert int(status) == 2 and lengths_out.tolist() == [0, 0, 64]
    assert (kept[:2] == -1).all()
    changed = (c.kpool.view(torch.int16) != before.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(c.spare[2])]
    status.zero_()
    spare[2] = 10 ** 6
    before = c.kpool.clone()
    cache_evict(c.kpool, c.vpool, c.page_table, c.lengths_dev, w, spare, 64, status=status)
    assert int(status) == 2


def test_captured(cuda_device):
    from mesh_transformer.cache import cache_evict
    c = Cache(7, 2, 8, 2, 128, [500, 400], spare=8)
    spare = torch.from_numpy(c.spare.reshape(2, 4)).to("cuda")
    w = torch.rand((2, 2, 512), device="cuda")
    call = lambda: cache_evict(c.kpool, c.vpool, c.page_table, c.lengths_dev, w, spare, 200, first=4, last=30)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for _ in range(3):
        w.copy_(torch.rand_like(w))
        graph.replay()
        torch.cuda.synchronize()
        pool = c.kpool.clone()
        for a, b in zip(captured, call()):
            assert torch.equal(a, b)
        assert torch.equal(pool.view(torch.int16), c.kpool.view(torch.int16))


def test_a_conversation_on_a_bounded_cache(cuda_device):
    """Prompt, tokens that count weights, eviction, more tokens, as a program uses them: against the same steps with the kept slots
    followed on the host."""
    from mesh_transformer.cache import cache_attention, cache_evict
    kv_heads, heads, d_head, pages, keep = 2, 4, 64, 4, 100
    c = Cache(11, 1, pages, kv_heads, d_head, [0], spare=2 * pages)
    dev = c.kpool.device
    weights = torch.zeros((1, kv_heads, pages * PAGE), device=dev)
    table, lengths = c.page_table, c.lengths_dev
    free = [int(p) for p in c.spare]
    held = [np.zeros((2, 0, d_head)) for _ in range(kv_heads)]            # per key head: keys and values of its slots
    total = np.zeros((kv_heads, 0))
    for tokens in [150] + [1] * 30 + [4] * 5 + [1] * 40:
        length = int(lengths) + tokens
        if length > pages * PAGE:
            break
        lengths = lengths + tokens
        q, k, v = (c.rows(1, tokens, h, d_head, torch.bfloat16) for h in (heads, kv_heads, kv_heads))
        out = cache_attention(q, k, v, c.kpool, c.vpool, table, lengths, weights=weights)
        qf, kf, vf = (x.double().cpu().numpy()[0] for x in (q, k, v))
        got = out.double().cpu().numpy()[0]
        received = np.zeros((kv_heads, length))
        for h in range(kv_heads):
            held[h] = np.concatenate([held[h], np.stack([kf[:, h], vf[:, h]])], 1)
            mine = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            want, r = cache_oracle.attention(qf[:, mine], held[h][0][:, None], held[h][1][:, None], length, tokens, 10 ** 6, 0, d_head ** -0.5)
            m, _ = cache_oracle.attention(qf[:, mine], held[h][0][:, None], np.abs(held[h][1])[:, None], length, tokens, 10 ** 6, 0, d_head ** -0.5)
            assert (np.abs(got[:, mine] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * m).all()
            received[h] = r[0]
        total = np.concatenate([total, np.zeros((kv_heads, tokens))], 1) + received
        assert np.abs(weights[0, :, :length].double().cpu().numpy() - total).max() <= 2.0 ** -12 * max(1.0, total.max())
        if length > 200:
            spare = torch.tensor([free[:2]], dtype=torch.int32, device=dev)
            old = table[0].tolist()
            kept, lengths, weights, table = cache_evict(c.kpool, c.vpool, table, lengths, weights, spare, keep, first=4, last=16)
            free = free[2:] + old[:2]
            table[0, 2:] = torch.tensor(old[2:], dtype=torch.int32, device=dev)
            kept = kept[0].cpu().numpy()
            for h in range(kv_heads):
                assert len(set(kept[h].tolist())) == keep and (np.diff(kept[h]) > 0).all()
                held[h] = held[h][:, kept[h]]
            total = np.take_along_axis(total, kept, 1)
