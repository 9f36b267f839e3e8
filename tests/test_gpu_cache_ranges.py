"""mesh_transformer.cache at the ends of its ranges, against 64 bits."""
import pytest
import torch

from cache_util import PAGE, rounding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 3, 70])
@pytest.mark.parametrize("d_head,pages", [(256, 2 ** 21), (64, 2 ** 23)])
def test_a_sequence_of_very_many_slots(cuda_device, d_head, pages, tokens):
    """2^27 and 2^29 slots of which a few pages exist: places of tiles times pieces of a sequence are beyond 32 bits.

    Tolerance: the weights enter the products as bf16 numbers (two terms, prompts one: 2^-8 of each at most), the result is rounded."""
    from mesh_transformer.cache import cache_attention
    heads, held = 2, 24
    g = torch.Generator("cuda").manual_seed(d_head)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    kpool, vpool = rand(held, 1, PAGE, d_head), rand(held, 1, PAGE, d_head)
    length = pages * PAGE - 5
    places = torch.randperm(pages - 3, generator=g, device="cuda")[:held - 3].sort().values
    places = torch.cat([places, torch.arange(pages - 3, pages, device="cuda")])           # the new tokens' pages among them
    table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    table[0, places] = torch.arange(held, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    q, k, v = rand(1, tokens, heads, d_head), rand(1, tokens, 1, d_head), rand(1, tokens, 1, d_head)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    out = cache_attention(q, k, v, kpool, vpool, table, lengths, status=status)
    assert int(status) == 2                                                               # pages that do not exist, no wait
    slots = (places[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
    new = slots - (length - tokens)
    keys, values = (x[:, 0].flatten(0, 1).double() for x in (kpool, vpool))
    for rows, fresh in ((keys, k), (values, v)):
        stored = (new >= 0) & (new < tokens)
        assert torch.equal(rows[stored], fresh[0, :, 0].double()[new[stored]])
    p = length - tokens + torch.arange(tokens, device="cuda")
    scores = torch.einsum("thd,sd->ths", q[0].double(), keys) * d_head ** -0.5
    a = torch.softmax(scores.masked_fill((slots[None, :] > p[:, None])[:, None], float("-inf")), -1)
    want, spread = a @ values, a @ values.abs()
    assert ((out[0].double() - want).abs() <= rounding(torch.bfloat16) * want.abs() + 2.0 ** -8 * spread).all()


@pytest.mark.parametrize("length", [200, 20000])
def test_eviction_by_weights_that_are_not_numbers(cuda_device, length):
    """NaN is heavier than any number, infinities included, and equals itself: the lower slot first.  Exact: nothing is computed."""
    from mesh_transformer.cache import cache_evict
    keep, first, last, nan, inf = 60, 2, 8, float("nan"), float("inf")
    pages = (length + PAGE - 1) // PAGE
    g = torch.Generator("cuda").manual_seed(length)
    pools = [torch.randn((pages + 1, 1, PAGE, 64), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    for nans in (5, 70):                                          # fewer than are kept, and more
        weights = torch.rand((1, 1, pages * PAGE), generator=g, device="cuda")
        at = first + torch.randperm(length - first - last, generator=g, device="cuda")[:nans + 3]
        weights[0, 0, at] = torch.tensor([nan] * nans + [inf, inf, -inf], device="cuda")
        ranks = torch.where(torch.isnan(weights[0, 0]), torch.full((), inf, device="cuda"), torch.where(weights[0, 0] == inf, 1e30, weights[0, 0].double()))
        middle = ranks[first:length - last]
        heaviest = first + torch.sort(middle, descending=True, stable=True).indices[:keep - first - last]
        want = torch.cat([torch.arange(first, device="cuda"), heaviest, torch.arange(length - last, length, device="cuda")]).sort().values
        kept, _, _, _ = cache_evict(*pools, table, torch.tensor([length], dtype=torch.int32, device="cuda"), weights,
                                    torch.tensor([[pages]], dtype=torch.int32, device="cuda"), keep, first=first, last=last)
        assert torch.equal(kept[0, 0].long(), want)
        assert all(torch.equal(p[pages, 0, :keep], p[:pages, 0].flatten(0, 1)[want]) for p in pools)
