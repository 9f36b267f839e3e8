"""Received weights and drafted tokens: only tokens that stay in the text count in what is evicted later."""
import numpy as np
import pytest
import torch

from cache_util import Cache, host
from oracle import cache_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d_head,heads,kv_heads", [(64, 4, 2), (128, 8, 2), (256, 2, 2)])
def test_weights_of_taken_tokens_alone(cuda_device, d_head, heads, kv_heads, dtype):
    """The sequence that the documentation gives: attend without weights, check, call again with the tokens that were taken.  Weights to the
    tolerance of test_received_weights: 2^-13 of what is received, and the sum's rounding."""
    from mesh_transformer.cache import cache_attention
    from mesh_transformer.sampling import verify_drafts
    drafts, vocab, window, sinks = 4, 50, 60, 3
    lengths = [7, 64, 200, 131]                                   # with the last token and the drafts
    c = Cache(d_head, 4, 5, kv_heads, d_head, lengths)
    q = c.rows(4, drafts + 1, heads, d_head, dtype, 1.5)
    k, v = c.rows(4, drafts + 1, kv_heads, d_head, dtype), c.rows(4, drafts + 1, kv_heads, d_head, dtype)
    g = torch.Generator("cuda").manual_seed(d_head)
    weights = torch.rand((4, kv_heads, 5 * 64), generator=g, device="cuda")
    before = weights.double().cpu().numpy()
    out = cache_attention(q, k, v, c.kpool, c.vpool, c.page_table, c.lengths_dev, window=window, sinks=sinks)
    logits = torch.zeros((4, drafts + 1, vocab), device="cuda")
    guess = torch.arange(1, drafts + 1, dtype=torch.int32, device="cuda").expand(4, drafts).contiguous()
    for b in range(4):                                            # greedy: sequence b takes b drafts, the last one of them all
        for t in range(drafts if b == 3 else b):
            logits[b, t, int(guess[b, t])] = 1.0
    ones = torch.full((4, drafts), 0.5, device="cuda")
    taken = verify_drafts(logits, None, guess, ones, torch.full((4, vocab), 0.5, device="cuda"), temp=0.0)[1]
    assert taken.tolist() == [0, 1, 2, 4]
    now = c.lengths_dev - (drafts - taken)
    again = cache_attention(q, None, None, c.kpool, c.vpool, c.page_table, now, new=taken + 1, window=window, sinks=sinks, weights=weights)
    for b in range(4):
        n, fresh = lengths[b] - drafts + int(taken[b]), int(taken[b]) + 1
        assert torch.allclose(again[b, :fresh].float(), out[b, :fresh].float(), rtol=2.0 ** -7, atol=2.0 ** -7)
        keys, values = (cache_oracle.slots_of(host(x), c.table[b], n) for x in (c.kpool, c.vpool))
        _, received = cache_oracle.attention(host(q[b, :fresh]), keys, values, n, fresh, window, sinks, d_head ** -0.5)
        want = before[b, :, :n].copy()
        want[:, n - fresh:] = 0
        want += received
        got = weights[b].double().cpu().numpy()
        assert (np.abs(got[:, :n] - want) <= 2.0 ** -13 * received + 2.0 ** -22 * want).all()
        assert np.array_equal(got[:, n:], before[b, :, n:])       # slots of refused drafts and behind
