"""Paged caches with marked slots for the tests of mesh_transformer.cache."""
import numpy as np
import torch

PAGE = 64


class Cache:
    """Pools whose slots in use hold random numbers and whose other slots hold NaN, through a shuffled page table."""

    def __init__(self, seed, batch, pages, kv_heads, d_head, lengths, spare=0, device="cuda", key_scale=1.0):
        rng = np.random.Generator(np.random.PCG64(seed))
        self.rng, self.lengths = rng, list(lengths)
        n = batch * pages + spare
        order = rng.permutation(n).astype(np.int32)
        self.table = order[:batch * pages].reshape(batch, pages).copy()
        self.spare = order[batch * pages:].copy()
        pools = []
        for scale in (key_scale, 1.0):
            pool = np.full((n, kv_heads, PAGE, d_head), np.nan, np.float32)
            for b, length in enumerate(lengths):
                for i in range((length + PAGE - 1) // PAGE):
                    rows = min(PAGE, length - i * PAGE)
                    pool[self.table[b, i], :, :rows] = scale * rng.standard_normal((kv_heads, rows, d_head), dtype=np.float32)
            pools.append(torch.from_numpy(pool).to(torch.bfloat16).to(device))
        self.kpool, self.vpool = pools
        self.page_table = torch.from_numpy(self.table).to(device)
        self.lengths_dev = torch.tensor(self.lengths, dtype=torch.int32, device=device)

    def rows(self, batch, tokens, heads, d_head, dtype, scale=1.0):
        x = scale * self.rng.standard_normal((batch, tokens, heads, d_head), dtype=np.float32)
        return torch.from_numpy(x).to(dtype).to(self.kpool.device)


def host(t):
    return t.detach().float().cpu().numpy()


def rounding(dtype):
    """Half a step of a stored number, relative."""
    return torch.finfo(dtype).eps / 2
