"""Samplers of the reference's sampling.py on the B200 path.

``nucleaus_sample`` / ``softmax_sample`` keep the reference signature
``(key, logits, sampler_input, **options) -> (token, info)``
(sampling.py:6-7,41-44).  ``key`` is what the randomness comes from: a float32
tensor of pre-drawn uniforms in [tiny, 1) with the shape of ``logits`` (the
form the parity tests use), a ``torch.Generator``, or an int seed.  The
arithmetic runs in libmtj_b200's sampling kernel (``nucleaus_filter`` returns
the kernel's own selection); the top-k branch of the reference filter
(sampling.py:15-26) is not implemented.
"""
from __future__ import annotations

import struct

import numpy as np
import torch

from ._lib import MTJ_BF16, MTJ_F32, check, lib

TINY = float(np.finfo(np.float32).tiny)


def draw_uniforms(key, shape, device) -> torch.Tensor:
    """Uniforms in [tiny, 1) like jax.random.gumbel's input (minval=tiny)."""
    if isinstance(key, torch.Tensor):
        return key.to(device=device, dtype=torch.float32).contiguous()
    if isinstance(key, torch.Generator):
        gen = key
    else:
        gen = torch.Generator(device=device)
        gen.manual_seed(int(key) & ((1 << 63) - 1))
    u = torch.rand(shape, generator=gen, device=device, dtype=torch.float32)
    return u.clamp_(min=TINY)


def _per_row(value, rows, device):
    t = torch.as_tensor(np.asarray(value, dtype=np.float32)).reshape(-1)
    if t.numel() == 1:
        t = t.expand(rows)
    return t.to(device).contiguous()


def _per_row_int(value, rows, device):
    """None stays None (the reference's top_k = None); a scalar or [rows] becomes an int32 device tensor."""
    if value is None:
        return None
    t = torch.as_tensor(np.asarray(value, dtype=np.int64).clip(-2**31, 2**31 - 1).astype(np.int32)).reshape(-1)
    if t.numel() == 1:
        t = t.expand(rows)
    return t.to(device).contiguous()


def nucleaus_sample(key, logits, _=None, top_p=0.9, temp=1, top_k=None):
    """logits [rows, vocab] (CUDA tensor or array) -> (uint32 token ids [rows], None)."""
    if not isinstance(logits, torch.Tensor):
        logits = torch.as_tensor(np.asarray(logits, dtype=np.float32))
    if not logits.is_cuda:
        logits = logits.cuda()
    logits = logits.to(torch.float32).contiguous()
    rows, vocab = logits.shape
    dev = logits.device
    with torch.cuda.device(dev):
        u = draw_uniforms(key, (rows, vocab), dev)
        tp, tt, tk = _per_row(top_p, rows, dev), _per_row(temp, rows, dev), _per_row_int(top_k, rows, dev)
        nbytes = lib.mtj_sample_scratch_bytes(rows, vocab)
        scratch = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        out = torch.empty((rows,), dtype=torch.int32, device=dev)
        check(lib.mtj_sample_top_p(logits.data_ptr(), u.data_ptr(), tp.data_ptr(),
                                   tk.data_ptr() if tk is not None else None, tt.data_ptr(), rows, vocab,
                                   scratch.data_ptr(), nbytes, out.data_ptr(),
                                   torch.cuda.current_stream(dev).cuda_stream))
        return out.cpu().numpy().view(np.uint32), None


def softmax_sample(key, logits, _=None, temp=1):
    """sampling.py:6-7: categorical(logits / temp), i.e. no nucleus filter."""
    return nucleaus_sample(key, logits, None, top_p=float("inf"), temp=temp)


def nucleaus_filter(logits, top_p=0.9, top_k=None):
    """sampling.py:10-38: ``logits - 1e10 * removed`` as a CUDA tensor [rows, vocab]; with ``top_k`` also
    ``- 1e10 * index`` for the entries of sorted rank >= top_k (:15-26)."""
    if not isinstance(logits, torch.Tensor):
        logits = torch.as_tensor(np.asarray(logits, dtype=np.float32))
    if not logits.is_cuda:
        logits = logits.cuda()
    logits = logits.to(torch.float32).contiguous()
    rows, vocab = logits.shape
    dev = logits.device
    with torch.cuda.device(dev):
        out = torch.empty_like(logits)
        tp, tk = _per_row(top_p, rows, dev), _per_row_int(top_k, rows, dev)
        check(lib.mtj_nucleus_filter(logits.data_ptr(), tp.data_ptr(), tk.data_ptr() if tk is not None else None,
                                     rows, vocab, out.data_ptr(),
                                     torch.cuda.current_stream(dev).cuda_stream))
        return out


_LOGIT_TYPES = {torch.float32: MTJ_F32, torch.bfloat16: MTJ_BF16}
_VERIFY_ARGS = struct.Struct("@10P4q4if4x").pack           # mtj_verify_args, the fields of MtjVerifyArgs


def _logit_rows(t, shape):
    """``t`` [batch, rows, vocab] with unit stride inside a row; anything else is copied."""
    vocab, s = shape[2], t.stride()
    if s[2] != 1 and vocab > 1 or s[1] < vocab:
        t = t.contiguous()
        s = t.stride()
    return t, max(s[1], vocab), s[0]


def _plain_rows(t, name, dtype, shape, index):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != index or t.shape != shape:
        raise ValueError(f"{name} must be a {dtype} tensor {list(shape)} on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def verify_drafts(target_logits, draft_logits, draft_tokens, accept, noise, count=None, temp=1.0):
    """Speculative decoding: which drafted tokens the target model takes, and the token behind them.

    The reference samples one token a step (transformer_shard.py:198-210); with drafts a step yields up to ``drafts + 1``, whose
    distribution is that of the target's own samples.  ``target_logits`` [batch, drafts + 1, vocab] float32 or bf16, row k behind k
    drafted tokens; ``draft_logits`` [batch, drafts, vocab] the logits that the drafts were sampled from at the same temperature, or
    None for tokens that were looked up rather than sampled; ``draft_tokens`` int32 [batch, drafts]; ``accept`` [batch, drafts] and
    ``noise`` [batch, vocab] float32 uniforms in [tiny, 1) (``draw_uniforms``); ``count`` int32 [batch] drafted tokens of each sequence
    (default: all); ``temp`` a number or float32 [batch], 0: greedy, where a draft is taken if it is the first largest logit.
    Logits filtered by ``nucleaus_filter`` make it nucleus sampling.

    Draft k is taken while ``accept * q_k(x_k) < p_k(x_k)``.  The next token is sampled from ``max(p_k - q_k, 0)`` at the first that
    is not, from ``p`` behind the last.  A row with NaN or +inf in it, or with nothing above -inf, has no shares: its draft is refused, and
    where the next token hangs on a target row of that kind it is 0 with a logarithm that is NaN.  Returns device tensors, nothing is read back: tokens int32 [batch, drafts + 1] (the
    taken ones, the next one, -1 behind it), the number taken int32 [batch], and log p_k of every token that comes out float32
    [batch, drafts + 1] (0 behind the last)."""
    shape = target_logits.shape if isinstance(target_logits, torch.Tensor) else ()
    kind = target_logits.dtype if len(shape) == 3 and target_logits.is_cuda and min(shape) >= 1 else None
    dtype = _LOGIT_TYPES.get(kind)
    if dtype is None:
        raise ValueError("target_logits must be a float32 or bfloat16 CUDA tensor [batch, drafts + 1, vocab]")
    batch, rows, vocab = shape
    drafts, index, dev = rows - 1, target_logits.get_device(), target_logits.device
    target, ld_target, batch_target = _logit_rows(target_logits, shape)
    draft, ld_draft, batch_draft = None, 0, 0
    if draft_logits is not None:
        if not isinstance(draft_logits, torch.Tensor) or draft_logits.dtype != kind or draft_logits.get_device() != index or \
                draft_logits.shape != (batch, drafts, vocab):
            raise ValueError(f"draft_logits must be a {kind} tensor {[batch, drafts, vocab]} on cuda:{index}")
        draft, ld_draft, batch_draft = _logit_rows(draft_logits, (batch, drafts, vocab))
    tokens = _plain_rows(draft_tokens, "draft_tokens", torch.int32, (batch, drafts), index)
    accept = _plain_rows(accept, "accept", torch.float32, (batch, drafts), index)
    noise = _plain_rows(noise, "noise", torch.float32, (batch, vocab), index)
    if count is not None:
        count = _plain_rows(count, "count", torch.int32, (batch,), index)
    temps = None
    if isinstance(temp, torch.Tensor):
        temps, temp = _plain_rows(temp, "temp", torch.float32, (batch,), index), 1.0
    out = torch.empty(batch, rows, dtype=torch.int32, device=dev)
    taken = torch.empty(batch, dtype=torch.int32, device=dev)
    logprobs = torch.empty(batch, rows, dtype=torch.float32, device=dev)
    try:
        a = _VERIFY_ARGS(target.data_ptr(), draft.data_ptr() if draft is not None and drafts else 0, tokens.data_ptr(),
                         accept.data_ptr(), noise.data_ptr(), count.data_ptr() if count is not None else 0,
                         temps.data_ptr() if temps is not None else 0, out.data_ptr(), taken.data_ptr(), logprobs.data_ptr(),
                         ld_target, batch_target, ld_draft, batch_draft, batch, drafts, vocab, dtype, temp)
    except (struct.error, OverflowError, TypeError) as e:
        raise ValueError(f"temp must be a number or a tensor: {e}") from None
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            _run_verify(a, dev, index)
    else:
        _run_verify(a, dev, index)
    return out, taken, logprobs


def _run_verify(a, dev, index):
    nbytes = lib.mtj_verify_scratch_bytes(a)
    if nbytes < 0:
        raise ValueError(lib.mtj_last_error().decode("utf-8", "replace"))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    check(lib.mtj_verify_drafts(a, scratch.data_ptr(), nbytes, torch._C._cuda_getCurrentRawStream(index)))
