"""mesh_transformer.sampling.verify_drafts at the ends of its ranges, against the plain form in 64 bits: tokens and counts are equal.

Logarithms: a row's sum is of 32-bit exponentials, off by at most 2^-22 each and by their arguments' roundings (the difference, the
scale twice, the product: 2^-24 each of an argument a, which counts with the share of its entry; the mean of a under the shares is at
most log(entries) < 11, so 2^-18.5 at most), and by the roundings of at most 16 sums (2^-20): below 2^-18 together.  The
result is rounded to 32 bits: 2^-24 of it."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle

pytestmark = pytest.mark.gpu
TINY = float(np.finfo(np.float32).tiny)


def _same(got, target, draft, tokens, accept, noise, temp):
    out, taken, logs = (x.cpu().numpy() for x in got)
    host = lambda x: None if x is None else x.float().cpu().numpy() if x.is_floating_point() else x.cpu().numpy()
    target, draft, tokens, accept, noise = (host(x) for x in (target, draft, tokens, accept, noise))
    for b in range(len(out)):
        want, k, lp = cache_oracle.verify(target[b], None if draft is None else draft[b], tokens[b], accept[b], noise[b], float(np.float32(temp)))
        assert int(taken[b]) == k, b
        assert out[b].tolist() == want + [-1] * (out.shape[1] - len(want)), b
        assert (np.abs(logs[b, :len(lp)] - lp) <= 2.0 ** -18 + 2.0 ** -24 * np.abs(lp)).all(), (b, logs[b], lp)


def _uniforms(g, *shape):
    return torch.rand(shape, generator=g, device="cuda").clamp_(min=TINY)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("offset", [0.0, 100.0, -100.0, 1e4, -1e4])
@pytest.mark.parametrize("temp", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-15, 1e-18])
def test_low_temperatures(cuda_device, temp, offset, known, dtype):
    """Drafts sampled at the temperature itself, logits far from zero beside their differences."""
    from mesh_transformer.sampling import verify_drafts
    batch, drafts, vocab = 4, 4, 1501
    g = torch.Generator("cuda").manual_seed(int(offset) % 97 + 5)
    target = (torch.randn((batch, drafts + 1, vocab), generator=g, device="cuda") * 2.5 + offset).to(dtype)
    draft = (target[:, :drafts].float() + 0.7 * torch.randn((batch, drafts, vocab), generator=g, device="cuda")).to(dtype)
    gumbel = -torch.log(-torch.log(_uniforms(g, batch, drafts, vocab).double().clamp_(max=1 - 2.0 ** -53)))
    tokens = (draft.double() + temp * gumbel).argmax(-1).to(torch.int32)
    accept, noise = _uniforms(g, batch, drafts), _uniforms(g, batch, vocab)
    d = draft if known else None
    _same(verify_drafts(target, d, tokens, accept, noise, temp=temp), target, d, tokens, accept, noise, temp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("drafts,known", [(1014, True), (1015, True), (1024, True), (1024, False)])
def test_the_most_drafts(cuda_device, drafts, known, dtype):
    """All of them taken, all but the last few, and a few: the shares of every row are in shared memory at once."""
    from mesh_transformer.sampling import verify_drafts
    vocab = 40
    g = torch.Generator("cuda").manual_seed(drafts)
    target = (torch.randn((3, drafts + 1, vocab), generator=g, device="cuda") * 2.5).to(dtype)
    draft = target[:, :drafts].clone()
    tokens = torch.randint(0, vocab, (3, drafts), generator=g, device="cuda").to(torch.int32)
    accept = _uniforms(g, 3, drafts) * 1e-6 if not known else _uniforms(g, 3, drafts) * 0.9 + 0.05
    tokens[1, drafts - 3] = -1
    tokens[2, 5] = vocab
    noise = _uniforms(g, 3, vocab)
    d = draft if known else None
    got = verify_drafts(target, d, tokens, accept.contiguous(), noise)
    if known:                         # equal rows: whatever there is is taken (a looked-up one hangs on its own share)
        assert got[1].tolist() == [drafts, drafts - 3, 5]
    _same(got, target, d, tokens, accept, noise, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("temp", [1e10, 1e28, 1e30, 1e38, 3e38])
def test_high_temperatures(cuda_device, temp, known, dtype):
    """All shares nearly alike, masked entries still without one: the refused token and masked entries would win the race."""
    from mesh_transformer.sampling import verify_drafts
    vocab = 600
    g = torch.Generator("cuda").manual_seed(7)
    target = (torch.randn((3, 3, vocab), generator=g, device="cuda") * 2.5).to(dtype)
    target[..., 1::2] = float("-inf")
    draft = target[:, :2].clone()
    draft[..., 2::4] = float("-inf")                       # the draft has half of the target's entries
    tokens = torch.tensor([[0, 4], [4, 8], [12, 0]], dtype=torch.int32, device="cuda")
    accept = torch.full((3, 2), 0.75, device="cuda")
    noise = _uniforms(g, 3, vocab)
    noise[:, 1::2] = 1 - 2.0 ** -24
    noise[torch.arange(3), tokens[:, 0].long()] = 1 - 2.0 ** -23
    d = draft if known else None
    got = verify_drafts(target, d, tokens, accept, noise, temp=temp)
    assert got[1].tolist() == [0, 0, 0]
    _same(got, target, d, tokens, accept, noise, temp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [50, 9001])
@pytest.mark.parametrize("temp", [1.0, 0.5])
def test_differences_below_the_32_bit_range(cuda_device, temp, vocab, dtype):
    """Target and draft agree on one token to the last bit of 64; what is left of the difference are shares of e^-100 to e^-300."""
    from mesh_transformer.sampling import verify_drafts
    g = torch.Generator("cuda").manual_seed(vocab)
    target = torch.full((3, 2, vocab), -2000.0, device="cuda")
    draft = torch.full((3, 1, vocab), -2000.0, device="cuda")
    target[..., 7], draft[..., 7] = 0.0, 0.0
    target[..., 3], draft[..., 3] = -1000.0, -280.0 * temp         # the drafted token: no share in the target
    noise = _uniforms(g, 3, vocab) * 0.5
    target[0, 0, 11], draft[0, 0, 11] = -100.0 * temp, -130.0 * temp                       # the one that is left
    target[1, 0, 11:20], draft[1, 0, 11:20] = -100.0 * temp, -130.0 * temp                 # several: the race decides
    noise[1, 14] = 0.999
    target[2, 0, vocab - 1], draft[2, 0, vocab - 1] = -300.0 * temp, -1000.0               # a late entry, and a smaller one that waits less
    target[2, 0, 20], draft[2, 0, 20] = -304.0 * temp, -1000.0
    noise[2, 20], noise[2, vocab - 1] = 1 - 2.0 ** -24, 0.25
    tokens = torch.full((3, 1), 3, dtype=torch.int32, device="cuda")
    accept = torch.full((3, 1), 0.5, device="cuda")
    target, draft = target.to(dtype), draft.to(dtype)
    got = verify_drafts(target, draft, tokens, accept, noise, temp=temp)
    assert got[0].tolist() == [[11, -1], [14, -1], [20, -1]]
    _same(got, target, draft, tokens, accept, noise, temp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("vocab", [300, 5000])
@pytest.mark.parametrize("what", ["-inf", "nan", "inf", "all nan", "a part nan"])
def test_rows_without_shares(cuda_device, what, vocab, known, dtype):
    """In the target's first row, in a later one, in the row behind all drafts, and in the draft's: refused, token 0 with a logarithm that is
    NaN where there is no distribution, the target's own where only the draft has none."""
    from mesh_transformer.sampling import verify_drafts
    g = torch.Generator("cuda").manual_seed(vocab)
    target = torch.randn((4, 3, vocab), generator=g, device="cuda") * 2.5
    draft = target[:, :2].clone()
    tokens = torch.randint(1, 60, (4, 2), generator=g, device="cuda").to(torch.int32)
    accept, noise = _uniforms(g, 4, 2) * (0.9 if known else 1e-9), _uniforms(g, 4, vocab)
    bad = [target[0, 0], target[1, 1], target[2, 2], draft[3, 0]]
    for row in bad:
        if what == "-inf":
            row.fill_(float("-inf"))
        elif what == "nan":
            row[70] = float("nan")
        elif what == "inf":
            row[70] = float("inf")
        elif what == "all nan":
            row.fill_(float("nan"))
        else:                                               # whole chunks of it
            row[100:].fill_(float("-inf"))
            row[vocab - 3:].fill_(float("nan"))
    target, draft = target.to(dtype), draft.to(dtype)
    d = draft if known else None
    out, taken, logs = verify_drafts(target, d, tokens, accept, noise)
    assert taken.tolist() == [0, 1, 2, 0 if known else 2]
    assert [int(out[b, b]) for b in range(3)] == [0, 0, 0]
    assert [bool(torch.isnan(logs[b, b])) for b in range(3)] == [True] * 3 and not torch.isnan(logs[3]).any()
    host = lambda x: x.float().cpu().numpy()
    with np.errstate(all="ignore"):
        for b in range(4):
            want, k, lp = cache_oracle.verify(host(target[b]), host(draft[b]) if known else None, tokens[b].tolist(), host(accept[b]), host(noise[b]), 1.0)
            assert out[b].tolist() == want + [-1] * (3 - len(want))
            near = np.abs(host(logs[b])[:len(lp)] - lp) <= 2.0 ** -18 + 2.0 ** -24 * np.abs(lp)
            assert (near | np.isnan(lp)).all()
