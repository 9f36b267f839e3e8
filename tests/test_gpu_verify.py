"""mesh_transformer.sampling.verify_drafts against the plain form in 64 bits: the same tokens, logarithms to 2^-20."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle

pytestmark = pytest.mark.gpu
TINY = float(np.finfo(np.float32).tiny)


def _inputs(seed, batch, drafts, vocab, dtype, spread=2.5, apart=0.7, agree=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    target = torch.randn((batch, drafts + 1, vocab), generator=g, device="cuda") * spread
    draft = target[:, :drafts] + apart * torch.randn((batch, drafts, vocab), generator=g, device="cuda")
    tokens = (draft - torch.log(-torch.log(torch.rand((batch, drafts, vocab), generator=g, device="cuda").clamp_(min=1e-30)))).argmax(-1)
    accept = torch.rand((batch, drafts), generator=g, device="cuda").clamp_(min=TINY) * (1.0 - agree) + TINY
    noise = torch.rand((batch, vocab), generator=g, device="cuda").clamp_(min=TINY)
    return target.to(dtype), draft.to(dtype), tokens.to(torch.int32), accept, noise


def _check(got, target, draft, tokens, accept, noise, counts, temps):
    out, taken, logs = (x.cpu().numpy() for x in got)
    target, accept, noise, tokens = (x.float().cpu().numpy() if x.is_floating_point() else x.cpu().numpy() for x in (target, accept, noise, tokens))
    draft = None if draft is None else draft.float().cpu().numpy()
    for b, n in enumerate(counts):
        want, k, lp = cache_oracle.verify(target[b, :n + 1], None if draft is None else draft[b, :n], tokens[b, :n], accept[b, :n], noise[b],
                                          float(np.float32(temps[b])))
        assert int(taken[b]) == k, b
        assert out[b].tolist() == want + [-1] * (out.shape[1] - len(want)), b
        assert np.abs(logs[b, :len(lp)] - lp).max() <= 2.0 ** -20 * max(1.0, np.abs(lp).max()), b
        assert (logs[b, len(lp):] == 0.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("batch,drafts,vocab,temp,agree", [
    (1, 4, 50400, 0.8, 0.0),
    (3, 1, 512, 1.0, 0.5),
    (5, 8, 997, 1.3, 0.9),            # odd rows: no two begin alike within 16 bytes
    (2, 3, 4096 + 3, 0.25, 0.99),
    (4, 2, 1, 1.0, 0.0),              # a vocabulary of one
    (2, 5, 33, 5.0, 0.0),
    (2, 40, 300, 1.0, 1.0),           # more drafts than a warp has lanes
    (6, 4, 20001, 0.0, 0.0),          # greedy
    (3, 6, 50400, 0.0, 0.0),
])
def test_verification(cuda_device, batch, drafts, vocab, temp, agree, known, dtype):
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(batch * 7 + drafts, batch, drafts, vocab, dtype, agree=agree, apart=0.2 if agree else 0.7)
    if temp == 0.0:                   # some drafts are the target's choice
        best = target[:, :drafts].float().argmax(-1).to(torch.int32)
        tokens = torch.where(torch.rand(tokens.shape, device="cuda") < 0.7, best, tokens)
    counts = [(3 * i + drafts) % (drafts + 1) for i in range(batch)]
    count = torch.tensor(counts, dtype=torch.int32, device="cuda")
    d = draft if known else None
    got = verify_drafts(target, d, tokens, accept, noise, count=count, temp=temp)
    _check(got, target, d, tokens, accept, noise, counts, [temp] * batch)
    got = verify_drafts(target, d, tokens, accept, noise, temp=torch.full((batch,), temp, device="cuda"))
    _check(got, target, d, tokens, accept, noise, [drafts] * batch, [temp] * batch)


def test_temperatures_of_their_own_and_filtered_logits(cuda_device):
    from mesh_transformer.sampling import nucleaus_filter, verify_drafts
    target, draft, tokens, accept, noise = _inputs(5, 4, 3, 2000, torch.float32)
    target = nucleaus_filter(target.reshape(-1, 2000), top_p=0.8).reshape(target.shape)
    draft = nucleaus_filter(draft.reshape(-1, 2000), top_p=0.7).reshape(draft.shape)
    temps = [0.0, 0.5, 1.0, 2.0]
    got = verify_drafts(target, draft, tokens, accept, noise, temp=torch.tensor(temps, device="cuda"))
    _check(got, target, draft, tokens, accept, noise, [3] * 4, temps)


@pytest.mark.parametrize("low", [float("-inf"), float(np.finfo(np.float32).min)])
def test_masked_entries(cuda_device, low):
    """Entries at -inf or the lowest value have no share: a masked draft is refused, a masked entry never comes out."""
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(9, 3, 4, 700, torch.float32)
    tokens = tokens.clone()
    target[:, :, ::2] = low
    draft[:, :, 1::3] = low
    tokens[0, 1] = 10                                     # masked in the target
    tokens[1, 0] = -1                                     # no token at all
    tokens[2, 2] = 700
    target[2, 3] = low
    target[2, 3, 5] = 1.0                                 # a row with one entry left
    for temp in (1.0, 0.6):
        got = verify_drafts(target, draft, tokens, accept, noise, temp=temp)
        _check(got, target, draft, tokens, accept, noise, [4] * 3, [temp] * 3)
        assert all(x < 0 or x % 2 == 1 for x in got[0].flatten().tolist())


def test_equal_distributions_take_everything_and_equal_logits_the_lowest(cuda_device):
    from mesh_transformer.sampling import verify_drafts
    target, _, tokens, accept, noise = _inputs(11, 4, 6, 1000, torch.float32)
    got = verify_drafts(target, target[:, :6].clone(), tokens, accept, noise)
    assert got[1].tolist() == [6] * 4
    _check(got, target, target[:, :6], tokens, accept, noise, [6] * 4, [1.0] * 4)
    flat = torch.zeros((2, 3, 5000), device="cuda")
    got = verify_drafts(flat, None, torch.zeros((2, 2), dtype=torch.int32, device="cuda"), accept[:2, :2].contiguous(),
                        torch.full((2, 5000), 0.5, device="cuda"), temp=0.0)
    assert got[0].tolist() == [[0, 0, 0]] * 2 and got[1].tolist() == [2, 2]
    got = verify_drafts(flat, None, torch.full((2, 2), 4999, dtype=torch.int32, device="cuda"), accept[:2, :2].contiguous(),
                        torch.full((2, 5000), 0.5, device="cuda"), temp=0.0)
    assert got[0].tolist() == [[0, -1, -1]] * 2
    # equal shares and equal noise: the lowest index, and not the refused one
    got = verify_drafts(flat, None, torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.full((2, 2), 0.9, device="cuda"),
                        torch.full((2, 5000), 0.5, device="cuda"), temp=1.0)
    assert got[0].tolist() == [[1, -1, -1]] * 2


def test_no_drafts_sample_the_target(cuda_device):
    from mesh_transformer.sampling import verify_drafts
    target, _, _, _, noise = _inputs(13, 3, 0, 3001, torch.float32)
    empty = torch.empty((3, 0), device="cuda")
    got = verify_drafts(target, None, empty.to(torch.int32), empty, noise, temp=0.9)
    _check(got, target, None, empty.to(torch.int32), empty, noise, [0] * 3, [0.9] * 3)


def test_strided_rows(cuda_device):
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(17, 3, 2, 501, torch.bfloat16)
    wide_t = torch.full((3, 5, 777), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_t[:, 1:4, 3:504] = target
    wide_d = torch.full((3, 2, 600), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_d[..., 7:508] = draft
    got = verify_drafts(wide_t[:, 1:4, 3:504], wide_d[..., 7:508], tokens, accept, noise)
    _check(got, target, draft, tokens, accept, noise, [2] * 3, [1.0] * 3)


def test_shares_of_the_samples(cuda_device):
    """Over many sequences the token behind refused and taken drafts is distributed as the target's samples: every share of the first
    token within six standard deviations of a binomial count."""
    from mesh_transformer.sampling import verify_drafts
    n, vocab = 40000, 6
    g = torch.Generator("cuda").manual_seed(3)
    target = torch.randn((1, 2, vocab), generator=g, device="cuda").expand(n, 2, vocab).contiguous()
    draft = torch.randn((1, 1, vocab), generator=g, device="cuda").expand(n, 1, vocab).contiguous()
    tokens = torch.multinomial(torch.softmax(draft[0, 0], -1), n, replacement=True, generator=g).to(torch.int32)[:, None].contiguous()
    accept = torch.rand((n, 1), generator=g, device="cuda").clamp_(min=TINY)
    noise = torch.rand((n, vocab), generator=g, device="cuda").clamp_(min=TINY)
    out, _, _ = verify_drafts(target, draft, tokens, accept, noise)
    p = torch.softmax(target[0, 0].double(), -1).cpu().numpy()
    seen = np.bincount(out[:, 0].cpu().numpy(), minlength=vocab) / n
    assert (np.abs(seen - p) <= 6 * np.sqrt(p * (1 - p) / n)).all()


def test_captured(cuda_device):
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(19, 2, 3, 9000, torch.float32)
    verify_drafts(target, draft, tokens, accept, noise)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_drafts(target, draft, tokens, accept, noise)
    for seed in (20, 21):
        for mine, new in zip((target, draft, tokens, accept, noise), _inputs(seed, 2, 3, 9000, torch.float32)):
            mine.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        _check(got, target, draft, tokens, accept, noise, [3] * 2, [1.0] * 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("batch,drafts,vocab,temp", [
    (1, 2, 200003, 1.0),              # a block goes over its part of a row in several steps, a lane over a row's chunks
    (1, 3, 140001, 0.0),
    (160, 1, 2500, 0.7),              # two blocks a sequence, and one
    (400, 2, 300, 1.1),
])
def test_long_rows_and_many_sequences(cuda_device, batch, drafts, vocab, temp, known, dtype):
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(31 + batch, batch, drafts, vocab, dtype, apart=0.3, agree=0.5)
    if temp == 0.0:
        tokens = target[:, :drafts].float().argmax(-1).to(torch.int32)
    d = draft if known else None
    got = verify_drafts(target, d, tokens, accept, noise, temp=temp)
    _check(got, target, d, tokens, accept, noise, [drafts] * batch, [temp] * batch)


def test_more_sequences_than_a_launch_takes(cuda_device):
    """The parts of the batch that are launched one after another give what each gives alone."""
    from mesh_transformer.sampling import verify_drafts
    target, draft, tokens, accept, noise = _inputs(37, 4500, 2, 70, torch.float32, agree=0.5)
    count = torch.randint(0, 3, (4500,), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.int32)
    temp = torch.rand((4500,), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) + 0.5
    got = verify_drafts(target, draft, tokens, accept, noise, count=count, temp=temp)
    for part in (slice(0, 1000), slice(3600, 4500)):
        alone = verify_drafts(target[part], draft[part], tokens[part], accept[part], noise[part], count=count[part], temp=temp[part])
        assert all(torch.equal(x[part], y) for x, y in zip(got, alone))
    tail = slice(4400, 4500)
    _check(tuple(x[tail] for x in got), target[tail], draft[tail], tokens[tail], accept[tail], noise[tail], count[tail].tolist(), temp[tail].tolist())


def test_drafts_over_a_cache(cuda_device):
    """Drafted tokens through an attention layer over a paged cache, checked, the refused ones taken back by the length alone; the
    cache is cut when it is full.  Every step's attention against 64 bits over the tokens that were kept so far, every check against
    the plain form on the step's logits."""
    from cache_util import PAGE, host, rounding
    from mesh_transformer.cache import cache_attention, cache_evict
    from mesh_transformer.sampling import verify_drafts
    g = torch.Generator("cuda").manual_seed(41)
    vocab, heads, kv_heads, d_head, pages, drafts, keep = 500, 4, 2, 64, 3, 3, 64
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    embed_q, embed_k, embed_v, head = (rand(vocab, heads, d_head), rand(vocab, kv_heads, d_head), rand(vocab, kv_heads, d_head),
                                       rand(heads * d_head, vocab).float() * 0.3)
    kpool, vpool = (torch.full((pages + 2, kv_heads, PAGE, d_head), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[4, 1, 3]], dtype=torch.int32, device="cuda")
    free = [0, 2]
    weights = torch.zeros((1, kv_heads, pages * PAGE), device="cuda")
    lengths = torch.zeros((1,), dtype=torch.int32, device="cuda")
    held = [np.zeros((0, 2, d_head)) for _ in range(kv_heads)]
    last, cuts, accepted = 7, 0, 0
    for step in range(200):
        guess = torch.randint(0, vocab, (1, drafts), generator=g, device="cuda").to(torch.int32)
        if step % 3 < 2:                                  # what the layer itself would say: the row is stored again by the step
            t = torch.tensor([[last]], device="cuda")
            y = cache_attention(embed_q[t], embed_k[t], embed_v[t], kpool, vpool, table, lengths + 1)
            guess[0, 0] = (y.float().flatten(2) @ head)[0, 0].argmax()
        tokens = torch.cat([torch.tensor([[last]], dtype=torch.int32, device="cuda"), guess], 1).long()
        n = int(lengths)
        lengths = lengths + (drafts + 1)
        out = cache_attention(embed_q[tokens], embed_k[tokens], embed_v[tokens], kpool, vpool, table, lengths, weights=weights)
        for h in range(kv_heads):
            rows = np.concatenate([held[h], np.stack([host(embed_k[tokens[0], h]), host(embed_v[tokens[0], h])], 1)])
            mine = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            qh = host(embed_q[tokens[0]])[:, mine]
            want, _ = cache_oracle.attention(qh, rows[:, :1], rows[:, 1:], len(rows), drafts + 1, 10 ** 6, 0, d_head ** -0.5)
            room, _ = cache_oracle.attention(qh, rows[:, :1], np.abs(rows[:, 1:]), len(rows), drafts + 1, 10 ** 6, 0, d_head ** -0.5)
            # a bf16 number has 8 significant bits: its step is 2^-7 of a power of two, half of it at most 2^-8 of the value
            assert (np.abs(host(out[0])[:, mine] - want) <= rounding(torch.bfloat16) * np.abs(want) + 2.0 ** -13 * room).all(), step
            held[h] = rows
        logits = out.float().flatten(2) @ head
        accept = torch.rand((1, drafts), generator=g, device="cuda").clamp_(min=TINY)
        noise = torch.rand((1, vocab), generator=g, device="cuda").clamp_(min=TINY)
        got = verify_drafts(logits, None, guess, accept, noise, temp=0.0 if step % 2 else 0.5)
        _check(got, logits, None, guess, accept, noise, [drafts], [0.0 if step % 2 else 0.5])
        taken = int(got[1])
        accepted += taken
        last = int(got[0][0, taken])
        lengths = lengths - (drafts - taken)
        held = [x[:n + 1 + taken] for x in held]
        if int(lengths) + drafts + 1 > pages * PAGE:
            spare = torch.tensor([[free[0]]], dtype=torch.int32, device="cuda")
            old = table[0].tolist()
            kept, lengths, weights, table = cache_evict(kpool, vpool, table, lengths, weights, spare, keep, first=2, last=20)
            assert int(lengths) == keep
            free = free[1:] + old
            table[0, 1:] = torch.tensor(free[:pages - 1], dtype=torch.int32, device="cuda")
            free = free[pages - 1:]
            kept = kept[0].cpu().numpy()
            held = [x[kept[h]] for h, x in enumerate(held)]
            cuts += 1
    assert int(lengths) == len(held[0]) and accepted >= 20 and cuts >= 1


def test_two_checks_at_once(cuda_device):
    from mesh_transformer.sampling import verify_drafts
    sets = [_inputs(seed, 30, 4, 20000, torch.float32, agree=0.5) for seed in (43, 47)]
    alone = [verify_drafts(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(verify_drafts(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for want, have in zip(alone, got) for x, y in zip(want, have))
