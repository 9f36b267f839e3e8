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
