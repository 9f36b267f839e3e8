"""Attention over caller-owned caches whose waits run out: a build of its kernels with the shortest limit, a wait that looks once.  The call
reports it, nothing is read or written outside the call's own rows and slots, copies in flight land before their blocks leave, and the next
call is as ever.

What a block does behind a wait that ran out stays in bounds: the few-row kernel leaves its loop as one and its second kernel checks what it
takes for an index; in the prompt kernel the warps that load and multiply stop, and the others go on over their own rows with whatever
tensor memory holds, their waits and the block's barriers as many as ever."""
import ctypes
import os
import subprocess

import pytest
import torch

from cache_util import PAGE

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mesh-transformer-jax_b200", "csrc")
UNITS = ("mtj_cache_attn", "mtj_cache_few", "mtj_cache_prompt")


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    import __graft_entry__ as ge
    from mesh_transformer import _lib
    build = ge._load_build_module()
    d = tmp_path_factory.mktemp("impatient")
    procs = [subprocess.Popen([build.NVCC, *build.FLAGS, "-DMTJ_WAIT_POLLS=0", "-c", os.path.join(CSRC, u + ".cu"), "-o", str(d / (u + ".o"))]) for u in UNITS]
    assert [p.wait() for p in procs] == [0] * len(procs)
    out = str(d / "impatient.so")
    subprocess.run([build.NVCC, "-shared", "-o", out, *(str(d / (u + ".o")) for u in UNITS), build.library(), "-lcudart", "-Xlinker", "-Bsymbolic",
                    "-Xlinker", "-rpath=" + os.path.dirname(build.library())], check=True)
    lib = ctypes.CDLL(out)
    for name in ("mtj_k_cache_attn_scratch_bytes", "mtj_k_cache_attn"):
        getattr(lib, name).restype, getattr(lib, name).argtypes = getattr(_lib.lib, name).restype, getattr(_lib.lib, name).argtypes
    lib.mtj_last_error = _lib.lib.mtj_last_error
    return lib


def _run(monkeypatch, impatient, batch, heads, kv_heads, d_head, tokens, length, dtype, weighed):
    from mesh_transformer import cache as module
    pages, spare = (length + PAGE - 1) // PAGE, 3
    g = torch.Generator("cuda").manual_seed(length + d_head)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    n = batch * pages + spare
    pools = [rand(n, kv_heads, PAGE, d_head).to(torch.bfloat16) for _ in range(2)]
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    table = order[:batch * pages].reshape(batch, pages).contiguous()
    lengths = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    q, k, v = rand(batch, tokens, heads, d_head), rand(batch, tokens, kv_heads, d_head), rand(batch, tokens, kv_heads, d_head)
    weights = torch.rand((batch, kv_heads, pages * PAGE), generator=g, device="cuda") if weighed else None

    def call(status):
        mine = [p.clone() for p in pools]
        out = torch.full((batch + 2, tokens, heads, d_head), 7.0, dtype=dtype, device="cuda")
        w = torch.full((batch + 2, kv_heads, pages * PAGE), 7.0, device="cuda") if weighed else None
        module.cache_attention(q, k, v, *mine, table, lengths, window=length - 100, sinks=4, weights=weights, weights_out=w[1:-1] if weighed else None,
                               out=out[1:-1], status=status)
        torch.cuda.synchronize()
        assert all((x[::len(x) - 1] == 7.0).all() for x in ([out, w] if weighed else [out]))
        for now, before in zip(mine, pools):
            assert torch.equal(now[order[batch * pages:].long()], before[order[batch * pages:].long()])
            rows = lambda p: p[table.long()].transpose(2, 3).flatten(1, 2)[:, :length - tokens]
            assert torch.equal(rows(now), rows(before))
        return [x[1:-1].clone() for x in ([out, w] if weighed else [out])]

    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    want = call(status)
    assert int(status) == 0
    for _ in range(4):
        with monkeypatch.context() as m:
            m.setattr(module, "lib", impatient)
            call(status)
        assert int(status) == 1
        status.zero_()
        got = call(status)
        assert int(status) == 0 and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("weighed", [False, True])
@pytest.mark.parametrize("batch,heads,kv_heads,d_head,tokens,length", [
    (2, 32, 8, 128, 1, 16000),        # few units: pieces end where units do
    (32, 16, 8, 64, 1, 9000),         # many: a block has parts of several
    (20, 8, 8, 256, 1, 4000),
    (12, 32, 8, 128, 5, 8000),        # drafts
])
def test_few_tokens(cuda_device, monkeypatch, impatient, batch, heads, kv_heads, d_head, tokens, length, weighed, dtype):
    _run(monkeypatch, impatient, batch, heads, kv_heads, d_head, tokens, length, dtype, weighed)


@pytest.mark.parametrize("batch,heads,kv_heads,d_head,tokens,length", [
    (1, 32, 8, 128, 2000, 2000),      # whole jobs
    (2, 8, 2, 64, 333, 5003),         # pieces that are joined
    (1, 16, 16, 256, 2047, 2047),     # pairs of blocks
    (3, 6, 2, 256, 200, 3000),
])
def test_prompts(cuda_device, monkeypatch, impatient, batch, heads, kv_heads, d_head, tokens, length):
    _run(monkeypatch, impatient, batch, heads, kv_heads, d_head, tokens, length, torch.bfloat16, False)
