"""What the entry points over caller-owned caches and drafts refuse, before anything is launched: no GPU is needed."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    import __graft_entry__ as ge
    ge.build()
    from mesh_transformer import _lib
    return _lib


BUF = ctypes.create_string_buffer(1 << 16)
BASE = (ctypes.addressof(BUF) + 255) // 256 * 256


def _attn(L, **kw):
    a = dict(kpool=BASE, vpool=BASE, page_table=BASE, lengths=BASE, new_tokens=BASE, status=None, q=BASE, k_new=BASE, v_new=BASE, out=BASE,
             weights_in=None, weights_out=None, ld_q=512, ld_k=256, ld_v=256, ld_out=512, n_pages=8, batch=2, pages=4, heads=4, kv_heads=2,
             d_head=128, tokens=3, dtype=L.MTJ_BF16, window=100, sinks=4, scale=0.1)
    a.update(kw)
    return L.MtjCacheAttnArgs(**a)


ATTN_BAD = [
    dict(kpool=None), dict(vpool=None), dict(page_table=None), dict(lengths=None), dict(q=None), dict(out=None), dict(k_new=None), dict(v_new=None),
    dict(n_pages=0), dict(batch=0), dict(batch=-1), dict(pages=0), dict(heads=0), dict(kv_heads=0), dict(tokens=0), dict(tokens=257),
    dict(heads=3), dict(heads=130, kv_heads=2, ld_q=130 * 128, ld_out=130 * 128), dict(window=0), dict(window=-3), dict(sinks=-1),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(weights_in=BASE),
    dict(ld_q=504), dict(ld_q=516), dict(ld_out=511), dict(ld_k=248), dict(ld_v=260), dict(q=BASE + 8), dict(kpool=BASE + 2), dict(out=BASE + 4),
    dict(k_new=BASE + 8), dict(pages=2 ** 30), dict(batch=2 ** 30), dict(batch=2 ** 20, heads=64, kv_heads=64, ld_q=64 * 128, ld_out=64 * 128,
                                                                         ld_k=64 * 128, ld_v=64 * 128, tokens=200),
]


@pytest.mark.parametrize("bad", ATTN_BAD)
def test_attention_refuses(L, bad):
    a = _attn(L, **bad)
    assert L.lib.mtj_k_cache_attn_scratch_bytes(ctypes.byref(a)) == -1
    assert L.lib.mtj_k_cache_attn(ctypes.byref(a), BASE, 1 << 40, None) == 1
    assert L.lib.mtj_last_error()


def test_attention_refuses_types_and_scratch(L):
    for bad in (dict(d_head=32), dict(d_head=96), dict(d_head=512), dict(dtype=7)):
        a = _attn(L, **bad)
        assert L.lib.mtj_k_cache_attn(ctypes.byref(a), BASE, 1 << 40, None) == 4
    a = _attn(L)
    n = L.lib.mtj_k_cache_attn_scratch_bytes(ctypes.byref(a))
    assert n > 0
    for scratch, size in ((None, n), (BASE, n - 1), (BASE + 16, n)):
        assert L.lib.mtj_k_cache_attn(ctypes.byref(a), scratch, size, None) == 1
    assert L.lib.mtj_k_cache_attn(None, BASE, n, None) == 1
    assert L.lib.mtj_k_cache_attn_scratch_bytes(None) == -1


def _evict(L, **kw):
    a = dict(kpool=BASE, vpool=BASE, page_table=BASE, lengths=BASE, weights=BASE, spare_pages=BASE, kept_out=BASE, lengths_out=BASE + 256,
             weights_out=BASE, page_table_out=BASE + 256, status=None, n_pages=8, batch=2, pages=4, kv_heads=2, d_head=64, keep=100, first=4, last=10)
    a.update(kw)
    return L.MtjCacheEvictArgs(**a)


@pytest.mark.parametrize("bad", [
    *({n: None} for n in ("kpool", "vpool", "page_table", "lengths", "weights", "spare_pages", "kept_out", "lengths_out", "weights_out",
                          "page_table_out")),
    dict(n_pages=0), dict(batch=0), dict(pages=-1), dict(kv_heads=0), dict(keep=0), dict(keep=-5), dict(first=-1), dict(last=-1),
    dict(first=60, last=41), dict(first=2 ** 31 - 1, last=2 ** 31 - 1), dict(lengths_out=BASE), dict(page_table_out=BASE), dict(kpool=BASE + 8),
    dict(pages=2 ** 26), dict(batch=2 ** 28), dict(keep=2 ** 31 - 1)])
def test_eviction_refuses(L, bad):
    assert L.lib.mtj_k_cache_evict(ctypes.byref(_evict(L, **bad)), None) == 1
    assert L.lib.mtj_last_error()


def test_eviction_refuses_head_sizes(L):
    assert L.lib.mtj_k_cache_evict(ctypes.byref(_evict(L, d_head=80)), None) == 4
    assert L.lib.mtj_k_cache_evict(None, None) == 1


def _verify(L, **kw):
    a = dict(target=BASE, draft=BASE, draft_tokens=BASE, accept=BASE, noise=BASE, counts=None, temp_per_row=None, tokens_out=BASE,
             accepted_out=BASE, logprobs_out=None, ld_target=100, batch_target=400, ld_draft=100, batch_draft=300, batch=2, drafts=3, vocab=100,
             dtype=L.MTJ_F32, temp=1.0)
    a.update(kw)
    return L.MtjVerifyArgs(**a)


@pytest.mark.parametrize("bad", [
    *({n: None} for n in ("target", "draft_tokens", "accept", "noise", "tokens_out", "accepted_out")),
    dict(batch=0), dict(vocab=0), dict(vocab=-1), dict(drafts=-1), dict(drafts=1025), dict(ld_target=99), dict(ld_draft=99), dict(target=BASE + 2),
    dict(draft=BASE + 1), dict(batch_target=-1), dict(batch_draft=-4), dict(batch=2 ** 30), dict(vocab=2 ** 31 - 5, ld_target=2 ** 31, ld_draft=2 ** 31)])
def test_verification_refuses(L, bad):
    a = _verify(L, **bad)
    assert L.lib.mtj_verify_scratch_bytes(ctypes.byref(a)) == -1
    assert L.lib.mtj_verify_drafts(ctypes.byref(a), BASE, 1 << 40, None) == 1
    assert L.lib.mtj_last_error()


def test_verification_refuses_types_and_scratch(L):
    assert L.lib.mtj_verify_drafts(ctypes.byref(_verify(L, dtype=3)), BASE, 1 << 40, None) == 4
    a = _verify(L)
    n = L.lib.mtj_verify_scratch_bytes(ctypes.byref(a))
    assert n > 0
    for scratch, size in ((None, n), (BASE, n - 1), (BASE + 8, n)):
        assert L.lib.mtj_verify_drafts(ctypes.byref(a), scratch, size, None) == 1


def test_host_layer_wants_tensors_of_one_gpu(L):
    from mesh_transformer.cache import cache_attention, cache_evict
    from mesh_transformer.sampling import verify_drafts
    pool = torch.zeros((4, 2, 64, 64), dtype=torch.bfloat16)
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.ones((1,), dtype=torch.int32)
    q = torch.zeros((1, 1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        cache_attention(q, None, None, pool, pool, table, lengths)
    with pytest.raises(ValueError):
        cache_evict(pool, pool, table, lengths, torch.zeros((1, 2, 128)), table[:, :1], 64)
    with pytest.raises(ValueError):
        verify_drafts(torch.zeros((1, 2, 10)), None, torch.zeros((1, 1), dtype=torch.int32), torch.zeros((1, 1)), torch.zeros((1, 10)))


def test_packed_arguments_are_laid_out_as_the_structures(L):
    """The host layer packs the arguments itself: same size, and every field at its place."""
    import struct
    for cls, fmt in ((L.MtjCacheAttnArgs, "@12P4q10if4x"), (L.MtjCacheEvictArgs, "@11P8i"), (L.MtjVerifyArgs, "@10P4q4if4x")):
        assert struct.calcsize(fmt) == ctypes.sizeof(cls)
        values = [i + 1 for i in range(len(cls._fields_))]
        back = cls.from_buffer_copy(struct.pack(fmt, *values))
        assert [getattr(back, n) for n, _ in cls._fields_] == values
    src = open(__import__("mesh_transformer.cache", fromlist=["x"]).__file__).read() + open(__import__("mesh_transformer.sampling", fromlist=["x"]).__file__).read()
    assert all(f'"{fmt}"' in src for fmt in ("@12P4q10if4x", "@11P8i", "@10P4q4if4x"))


def test_numbers_beyond_the_kernels_own(L):
    """Slots of a sequence, entries of a row and temperatures up to which places and scaled logits stay in 32 bits."""
    err = lambda: L.lib.mtj_last_error().decode()
    assert L.lib.mtj_k_cache_attn(ctypes.byref(_attn(L, pages=2 ** 24 + 1, batch=1, kv_heads=1)), BASE, 1 << 40, None) == 1 and "2^30 slots" in err()
    assert L.lib.mtj_k_cache_evict(ctypes.byref(_evict(L, pages=2 ** 24 + 1, batch=1, kv_heads=1)), None) == 1 and "slots" in err()
    long = dict(vocab=2 ** 30 + 1, ld_target=2 ** 31, ld_draft=2 ** 31, batch=1, drafts=0)
    assert L.lib.mtj_verify_drafts(ctypes.byref(_verify(L, **long)), BASE, 1 << 40, None) == 1 and "vocabulary" in err()
    assert L.lib.mtj_verify_drafts(ctypes.byref(_verify(L, temp=float("inf"))), BASE, 1 << 40, None) == 1 and "temp" in err()


def test_prompts_beyond_the_plan(L):
    """New tokens of a sequence, and the key blocks that all of them see, are counted in 32 bits."""
    size = lambda **kw: L.lib.mtj_k_cache_attn_scratch_bytes(ctypes.byref(_attn(L, batch=1, heads=1, kv_heads=1, **kw)))
    assert size(tokens=2 ** 20, pages=2 ** 15, window=2 ** 30) > 0
    assert size(tokens=2 ** 21 + 1, pages=2 ** 16) == -1
    assert size(tokens=2 ** 20, pages=2 ** 20, window=2 ** 30) == -1 and "new tokens" in L.lib.mtj_last_error().decode()
    assert size(tokens=2 ** 20, pages=2 ** 20, window=2 ** 12) > 0
