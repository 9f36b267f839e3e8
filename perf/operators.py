"""Operators over the paged cache and its sampler, as they are measured: attention of new tokens with a sliding window and first
tokens that stay visible, eviction by accumulated attention weight, and verification of drafted tokens.

A case has an ``op``:
    "attend"  ``tokens`` new tokens per sequence are appended and attend (``ragged``: sequences have between one and that many);
              ``cached`` slots are in use at the longest sequence with the new ones, ``shortest`` at the shortest; heads query heads
              over kv_heads key heads of ``dim`` numbers; ``weighed``: the weight that every slot received is added up
    "evict"   every key head of every sequence keeps ``keep`` slots: the first ``first``, the last ``last``, and the heaviest others
    "verify"  ``drafts`` drafted tokens per sequence (``ragged``: between none and that many) against the target's logits, and the
              logarithm of the target's share of every token that comes out;
              ``known``: drafts with logits of their own (otherwise looked up, i.e. drawn with certainty); ``temp`` 0: greedy
"""
import os
import sys

import torch

own = False

PAGE = 64
MOST_BYTES = 2.2e9                                   # of the largest listed case
MOST_FLOPS = 5.0e11
GPTJ_VOCAB = 50400


def listed():
    return [
        # one token of two short conversations on the smallest model: what a call costs besides its arithmetic
        dict(name="tiny_token", op="attend", batch=2, heads=4, kv_heads=4, dim=64, tokens=1, ragged=False, cached=127, shortest=90,
             window=96, sinks=4, dtype="bfloat16", weighed=False),
        # one token behind a full window of the 6B model, queries in 32 bits as its decode step has them
        dict(name="gptj_token", op="attend", batch=1, heads=16, kv_heads=16, dim=256, tokens=1, ragged=False, cached=3001, shortest=3001,
             window=2048, sinks=4, dtype="float32", weighed=False),
        # a serving batch checks up to five drafted tokens a sequence, conversations of very different length
        dict(name="grouped_drafts", op="attend", batch=8, heads=32, kv_heads=8, dim=128, tokens=5, ragged=True, cached=8191, shortest=700,
             window=4096, sinks=4, dtype="bfloat16", weighed=False),
        # a full batch on long caches that counts what every cached token is worth
        dict(name="grouped_weighed", op="attend", batch=32, heads=32, kv_heads=8, dim=128, tokens=1, ragged=False, cached=16383,
             shortest=2000, window=16384, sinks=0, dtype="bfloat16", weighed=True),
        # a whole prompt of the 6B model
        dict(name="gptj_prompt", op="attend", batch=1, heads=16, kv_heads=16, dim=256, tokens=2047, ragged=False, cached=2047,
             shortest=2047, window=1024, sinks=4, dtype="bfloat16", weighed=False),
        # a long document
        dict(name="grouped_document", op="attend", batch=1, heads=32, kv_heads=8, dim=128, tokens=8191, ragged=False, cached=8191,
             shortest=8191, window=4096, sinks=4, dtype="bfloat16", weighed=False),
        # portions of several prompts of odd length behind what is cached already
        dict(name="grouped_portions", op="attend", batch=4, heads=8, kv_heads=2, dim=64, tokens=333, ragged=True, cached=5003,
             shortest=1200, window=2000, sinks=16, dtype="bfloat16", weighed=False),
        # one short conversation gives back half of its cache
        dict(name="evict_one", op="evict", batch=1, kv_heads=4, dim=64, cached=511, shortest=511, keep=256, first=4, last=32),
        # a batch of long ones keeps a quarter
        dict(name="evict_batch", op="evict", batch=8, kv_heads=8, dim=128, cached=16383, shortest=3000, keep=4096, first=4, last=512),
        # one user, four drafted tokens
        dict(name="verify_one", op="verify", batch=1, drafts=4, ragged=False, vocab=GPTJ_VOCAB, dtype="float32", known=True, temp=0.8),
        # drafts looked up in the prompt, greedy or not, half-width logits
        dict(name="verify_looked_up", op="verify", batch=8, drafts=5, ragged=True, vocab=GPTJ_VOCAB, dtype="bfloat16", known=False, temp=1.0),
        # a full batch
        dict(name="verify_batch", op="verify", batch=64, drafts=7, ragged=True, vocab=GPTJ_VOCAB, dtype="float32", known=True, temp=1.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    while True:
        op = rng.choice(["attend", "attend", "prompt", "evict", "verify"])
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        if op == "verify":
            case = dict(op="verify", batch=spread(1, 64), drafts=rng.randint(1, 8), ragged=rng.random() < 0.5,
                        vocab=rng.choice([512, spread(300, 60000), GPTJ_VOCAB]), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                        known=rng.random() < 0.7, temp=rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]))
        elif op == "evict":
            cached = spread(100, 16000)
            keep = max(3, int(cached * rng.uniform(0.1, 1.1)))
            first = rng.randint(0, min(16, keep // 3))
            case = dict(op="evict", batch=spread(1, 16), kv_heads=kv_heads, dim=dim, cached=cached, shortest=max(1, int(cached * rng.uniform(0.2, 1.0))),
                        keep=keep, first=first, last=rng.randint(0, keep // 2 - first // 2))
        else:
            few = op == "attend"
            cached = spread(1, 16000) if few else spread(70, 8000)
            tokens = min(cached, rng.choice([1, 1, 1, 2, 4, 5, 8])) if few else max(33, int(cached * rng.choice([1.0, 1.0, rng.uniform(0.1, 1.0)])))
            heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
            case = dict(op="attend", batch=spread(1, 40) if few else spread(1, 6), heads=heads, kv_heads=kv_heads, dim=dim, tokens=tokens,
                        ragged=rng.random() < 0.5, cached=cached, shortest=max(tokens, int(cached * rng.uniform(0.2, 1.0))),
                        window=spread(1, 2 * cached), sinks=rng.choice([0, 1, 4, 16, 70]),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]) if few else "bfloat16", weighed=few and rng.random() < 0.4)
            if heads > 64:
                continue
            # all pairs of queries and slots, which the plain form fills in
            if case["batch"] * heads * tokens * -(-cached // PAGE) * PAGE > 2.2e9 or case["batch"] * kv_heads * cached * dim > 5.4e8:
                continue
        cost = work(case)
        if cost["bytes"] <= MOST_BYTES and cost["flops"] <= MOST_FLOPS:
            return case


def _evenly(batch, most, least):
    """Lengths from the longest to the shortest, the same for every seed."""
    return [most - (most - least) * i // max(1, batch - 1) for i in range(batch)]


def _lengths(case):
    return _evenly(case["batch"], case["cached"], case["shortest"])


def _new(case):
    """How many tokens of each sequence are new."""
    most = case["tokens"]
    return [1 + (most - 1) * (3 * i + 2) % most if case["ragged"] else most for i in range(case["batch"])]


def _drafted(case):
    most = case["drafts"]
    return [(5 * i + most) % (most + 1) if case["ragged"] else most for i in range(case["batch"])]


def _pages(case):
    return -(-case["cached"] // PAGE)


def work(case):
    if case["op"] == "verify":
        size = 4 if case["dtype"] == "float32" else 2
        rows = sum((2 if case["known"] else 1) * n + 1 for n in _drafted(case))
        sampled = 0 if case["temp"] == 0 else case["batch"]
        return {"bytes": rows * case["vocab"] * size + sampled * case["vocab"] * 4, "flops": 5.0 * rows * case["vocab"]}
    kv_row = case["kv_heads"] * case["dim"] * 2 * 2
    if case["op"] == "evict":
        moved = sum(min(n, case["keep"]) for n in _lengths(case) if n > case["keep"])
        seen = sum(_lengths(case)) * case["kv_heads"] * 4
        return {"bytes": 2.0 * moved * kv_row + seen + 2 * case["batch"] * case["kv_heads"] * min(case["keep"], case["cached"]) * 4, "flops": 0.0}
    size = 4 if case["dtype"] == "float32" else 2
    window, sinks = case["window"], case["sinks"]
    pairs = read = rows = 0
    for length, n in zip(_lengths(case), _new(case)):
        first = length - n
        low = max(0, first - window + 1)                      # of the window of the first new token
        read += length - low + min(sinks, low)
        rows += n
        for p in range(first, length):
            lo = max(0, p - window + 1)
            pairs += p - lo + 1 + min(sinks, lo)
    bytes_ = read * kv_row + 2.0 * rows * case["heads"] * case["dim"] * size + 2.0 * rows * case["kv_heads"] * case["dim"] * size
    if case["weighed"]:
        bytes_ += 8.0 * sum(_lengths(case)) * case["kv_heads"]
    return {"bytes": bytes_, "flops": 4.0 * pairs * case["heads"] * case["dim"]}


def _inputs(case, seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed * 7919 + 17)
    host = torch.Generator()
    host.manual_seed(seed * 104729 + 3)
    batch = case["batch"]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)

    if case["op"] == "verify":
        vocab, drafts = case["vocab"], case["drafts"]
        dtype = getattr(torch, case["dtype"])
        # a few entries stand out of a broad rest, and the draft model agrees with the target roughly
        target = normal(batch, drafts + 1, vocab, scale=2.5)
        draft = target[:, :drafts] + normal(batch, drafts, vocab, scale=0.7)
        race = torch.rand((batch, drafts, vocab), generator=g, device=device).clamp_(min=1e-30)
        temp = case["temp"] if case["temp"] > 0 else 0.2
        tokens = (draft / temp - torch.log(-torch.log(race))).argmax(-1).to(torch.int32)
        del race
        tiny = torch.finfo(torch.float32).tiny
        return dict(target=target.to(dtype), draft=draft.to(dtype) if case["known"] else None, tokens=tokens,
                    accept=torch.rand((batch, drafts), generator=g, device=device).clamp_(min=tiny),
                    noise=torch.rand((batch, vocab), generator=g, device=device).clamp_(min=tiny),
                    count=torch.tensor(_drafted(case), dtype=torch.int32, device=device),
                    temp=torch.full((batch,), case["temp"], device=device))
    pages, kv_heads, dim = _pages(case), case["kv_heads"], case["dim"]
    spare = -(-case["keep"] // PAGE) if case["op"] == "evict" else 0
    n_pages = batch * (pages + spare)
    order = torch.randperm(n_pages, generator=host).to(torch.int32)
    s = dict(kpool=normal(n_pages, kv_heads, PAGE, dim, dtype=torch.bfloat16), vpool=normal(n_pages, kv_heads, PAGE, dim, dtype=torch.bfloat16),
             page_table=order[:batch * pages].reshape(batch, pages).to(device).contiguous(),
             lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=device))
    if case["op"] == "evict":
        s["spare"] = order[batch * pages:].reshape(batch, spare).to(device).contiguous()
        # few slots hold most of the weight; the newest have had little time to gain any
        s["weights"] = torch.rand((batch, kv_heads, pages * PAGE), generator=g, device=device).pow_(-0.7)
        return s
    dtype, heads, tokens = getattr(torch, case["dtype"]), case["heads"], case["tokens"]
    s["q"] = normal(batch, tokens, heads, dim, dtype=dtype, scale=1.5)
    s["k"] = normal(batch, tokens, kv_heads, dim, dtype=dtype)
    s["v"] = normal(batch, tokens, kv_heads, dim, dtype=dtype)
    s["new"] = torch.tensor(_new(case), dtype=torch.int32, device=device)
    s["weights"] = s["weights_out"] = None
    if case["weighed"]:
        s["weights"] = torch.rand((batch, kv_heads, pages * PAGE), generator=g, device=device)
        s["weights_out"] = torch.zeros_like(s["weights"])
    return s


def prepare(case, seed):
    return dict(_inputs(case, seed, torch.device("cuda")), case=case)


def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["op"]](state, case)
    return _RUN_PLAIN[case["op"]](state, case)


# ---- the framework's calls -------------------------------------------------------------------------------------------------------

def _package():
    path = os.path.join(os.getcwd(), "mesh-transformer-jax_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_attend(s, case):
    _package()
    from mesh_transformer.cache import cache_attention
    out = cache_attention(s["q"], s["k"], s["v"], s["kpool"], s["vpool"], s["page_table"], s["lengths"], new=s["new"],
                          window=case["window"], sinks=case["sinks"], weights=s["weights"], weights_out=s["weights_out"])
    return [out, s["kpool"], s["vpool"]] + ([s["weights_out"]] if case["weighed"] else [])


def _own_evict(s, case):
    _package()
    from mesh_transformer.cache import cache_evict
    kept, lengths, weights, table = cache_evict(s["kpool"], s["vpool"], s["page_table"], s["lengths"], s["weights"], s["spare"],
                                                case["keep"], first=case["first"], last=case["last"])
    return [kept, lengths, weights, table, s["kpool"], s["vpool"]]


def _own_verify(s, case):
    _package()
    from mesh_transformer.sampling import verify_drafts
    tokens, accepted, logprobs = verify_drafts(s["target"], s["draft"], s["tokens"], s["accept"], s["noise"],
                                               count=s["count"], temp=s["temp"])
    return [tokens, accepted, logprobs]


_RUN_OWN = {"attend": _own_attend, "evict": _own_evict, "verify": _own_verify}


# ---- their plain form ------------------------------------------------------------------------------------------------------------

def _append(pool, rows, table, lengths, new):
    """Row t of ``rows`` [batch, tokens, heads, dim] becomes slot lengths - new + t; rows from ``new`` on are not used."""
    batch, tokens = rows.shape[:2]
    t = torch.minimum(torch.arange(tokens, device=rows.device)[None], (new - 1).clamp(min=0)[:, None])    # the last one again
    slot = ((lengths - new)[:, None] + t).clamp(min=0).long()
    page = table.gather(1, slot // PAGE).long()
    old = pool[page, :, slot % PAGE]
    value = rows.gather(1, t[:, :, None, None].expand_as(rows).long()).to(pool.dtype)
    pool[page, :, slot % PAGE] = torch.where((new > 0)[:, None, None, None], value, old)


def _plain_attend(s, case):
    lengths, new, table = s["lengths"], s["new"], s["page_table"]
    batch, tokens, heads, dim = s["q"].shape
    kv_heads = case["kv_heads"]
    group = heads // kv_heads
    _append(s["kpool"], s["k"], table, lengths, new)
    _append(s["vpool"], s["v"], table, lengths, new)
    keys = s["kpool"][table.long()].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, dim).float()
    values = s["vpool"][table.long()].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, dim).float()
    slot = torch.arange(keys.shape[2], device=keys.device)
    place = (lengths - new)[:, None] + torch.arange(tokens, device=keys.device)[None]
    place = place[:, :, None]
    seen = (slot <= place) & ((slot < case["sinks"]) | (place - slot < case["window"])) & (place < lengths[:, None, None])
    seen = seen[:, None, None]                                                       # [batch, 1, 1, tokens, slots]
    q = s["q"].float().reshape(batch, tokens, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(batch, kv_heads, group * tokens, dim) @ keys.transpose(2, 3) * dim ** -0.5).reshape(batch, kv_heads, group, tokens, -1)
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    share = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    del scores
    total = share.sum(-1, keepdim=True)
    share = share / torch.where(total == 0, 1.0, total)
    values = torch.where((slot < lengths[:, None])[:, None, :, None], values, 0.0)
    out = (share.reshape(batch, kv_heads, group * tokens, -1) @ values).reshape(batch, kv_heads, group, tokens, dim)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, tokens, heads, dim).to(s["q"].dtype)
    if not case["weighed"]:
        return [out, s["kpool"], s["vpool"]]
    before = torch.where(slot < (lengths - new)[:, None], 1.0, 0.0)[:, None] * s["weights"]
    s["weights_out"].copy_(torch.where((slot < lengths[:, None])[:, None], before + share.sum((2, 3)), s["weights_out"]))
    return [out, s["kpool"], s["vpool"], s["weights_out"]]


def _plain_evict(s, case):
    keep, first, last = case["keep"], case["first"], case["last"]
    lengths, table, spare, weights = s["lengths"], s["page_table"], s["spare"], s["weights"]
    batch, kv_heads, slots = weights.shape
    slot = torch.arange(slots, device=weights.device)
    length = lengths[:, None, None]
    held = slot < length
    safe = held & ((slot < first) | (slot >= length - last))
    rank = torch.where(safe, float("inf"), torch.where(held, weights, float("-inf")))
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(torch.arange(order.shape[-1], device=weights.device) < length, order, slots)
    kept = order.sort(-1).values                                                     # ``slots``: nothing
    kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=slots)
    some = kept < slots
    weights_out = torch.where(some, weights.gather(-1, kept.clamp(max=slots - 1)), 0.0)
    weights_out = torch.nn.functional.pad(weights_out, (0, max(0, slots - keep)))[..., :slots]
    moves = (lengths > keep)[:, None, None]
    weights_out = torch.where(moves, weights_out, torch.where(held, weights, 0.0))
    # kept rows go to the spare pages of the sequences that give something up
    source = kept.clamp(max=slots - 1)
    from_page = table.long().gather(1, (source // PAGE).reshape(batch, -1)).reshape(source.shape)
    place = torch.arange(keep, device=weights.device)
    to_page = spare.long()[:, place // PAGE][:, None].expand_as(source)
    head = torch.arange(kv_heads, device=weights.device)[None, :, None].expand_as(source)
    to_row = (place % PAGE).expand_as(source)
    s["kpool"][to_page, head, to_row] = torch.where(moves[..., None], s["kpool"][from_page, head, source % PAGE], s["kpool"][to_page, head, to_row])
    s["vpool"][to_page, head, to_row] = torch.where(moves[..., None], s["vpool"][from_page, head, source % PAGE], s["vpool"][to_page, head, to_row])
    table_out = torch.nn.functional.pad(spare, (0, max(0, table.shape[1] - spare.shape[1])), value=-1)[:, :table.shape[1]]
    table_out = torch.where(moves[:, :, 0], table_out, table)
    return [torch.where(some, kept, -1).to(torch.int32), lengths.clamp(max=keep), weights_out, table_out, s["kpool"], s["vpool"]]


def _shares(logits, temp):
    """softmax(logits / temp) in 64 bits; temp 0: all of it at the first largest entry."""
    logits = logits.double()
    greedy = (temp <= 0)[:, None, None]
    t = torch.where(greedy, 1.0, temp.double()[:, None, None])
    e = torch.exp((logits - logits.amax(-1, keepdim=True)) / t)
    one = torch.zeros_like(e).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
    return torch.where(greedy, one, e / e.sum(-1, keepdim=True))


def _plain_verify(s, case):
    target, tokens, temp, count = s["target"], s["tokens"].long(), s["temp"], s["count"]
    batch, drafts = tokens.shape
    p = _shares(target, temp)
    if s["draft"] is not None:
        q = _shares(s["draft"], temp)
        # a greedy target takes its own choice whatever the draft's shares are
        q = torch.where((temp <= 0)[:, None, None], torch.zeros_like(q).scatter_(-1, tokens[..., None], 1.0), q)
    else:
        q = torch.zeros_like(p[:, :drafts]).scatter_(-1, tokens[..., None], 1.0)
    k = torch.arange(drafts, device=tokens.device)
    good = s["accept"].double() * q.gather(-1, tokens[..., None])[..., 0] < p[:, :drafts].gather(-1, tokens[..., None])[..., 0]
    good = good & (k < count[:, None])
    accepted = good.long().cumprod(1).sum(1)
    row = accepted[:, None, None].expand(-1, 1, p.shape[-1])
    p_row = p.gather(1, row)[:, 0]
    q_row = torch.nn.functional.pad(q, (0, 0, 0, 1)).gather(1, row)[:, 0]
    q_row = torch.where((accepted < count)[:, None], q_row, 0.0)
    rest = (p_row - q_row).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p_row)
    chosen = (rest / -torch.log(s["noise"].double())).argmax(-1)
    place = torch.arange(drafts + 1, device=tokens.device)
    padded = torch.nn.functional.pad(tokens, (0, 1), value=-1)
    out = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], chosen[:, None], -1))
    share = p.gather(-1, out.clamp(min=0)[..., None])[..., 0]
    logprobs = torch.where(out >= 0, torch.log(share), 0.0)
    return [out.to(torch.int32), accepted.to(torch.int32), logprobs.to(torch.float32)]


_RUN_PLAIN = {"attend": _plain_attend, "evict": _plain_evict, "verify": _plain_verify}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed, torch.device("cuda"))
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "evict":
        return _exact_evict(case, s)
    return _exact_verify(case, s)


def _exact_attend(case, s):
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    weights = None if s["weights_out"] is None else s["weights_out"].double()
    for b, (length, n) in enumerate(zip(_lengths(case), _new(case))):
        pages = s["page_table"][b].tolist()
        for t in range(n):
            at = length - n + t
            s["kpool"][pages[at // PAGE], :, at % PAGE] = s["k"][b, t].to(torch.bfloat16)
            s["vpool"][pages[at // PAGE], :, at % PAGE] = s["v"][b, t].to(torch.bfloat16)
        place = torch.arange(length - n, length, device=out.device)
        slot = torch.arange(length, device=out.device)
        back = place[:, None] - slot[None]
        hidden = (back < 0) | ((back >= case["window"]) & (slot[None] >= case["sinks"]))
        for h in range(case["kv_heads"]):
            keys = torch.cat([s["kpool"][p, h] for p in pages])[:length].double()
            values = torch.cat([s["vpool"][p, h] for p in pages])[:length].double()
            received = torch.zeros(length, dtype=torch.float64, device=out.device)
            for i in range(h * group, (h + 1) * group):
                scores = (s["q"][b, :n, i].double() @ keys.T) / case["dim"] ** 0.5
                share = torch.softmax(scores.masked_fill_(hidden, float("-inf")), -1)
                out[b, :n, i] = share @ values
                received += share.sum(0)
            if weights is not None:
                weights[b, h, :length] = received
                weights[b, h, :length - n] += s["weights"][b, h, :length - n].double()
    return [out, s["kpool"].double(), s["vpool"].double()] + ([weights] if weights is not None else [])


def _exact_evict(case, s):
    keep = case["keep"]
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device=s["weights"].device)
    for b, length in enumerate(_lengths(case)):
        pages, spare = s["page_table"][b].tolist(), s["spare"][b].tolist()
        for h in range(case["kv_heads"]):
            w = s["weights"][b, h, :length].double()
            if length <= keep:
                weights[b, h, :length] = w
                continue
            middle = w[case["first"]:length - case["last"]].tolist()
            take = sorted(range(len(middle)), key=lambda i: (-middle[i], i))[:keep - case["first"] - case["last"]]
            kept = list(range(case["first"])) + sorted(case["first"] + i for i in take) + list(range(length - case["last"], length))
            at = torch.tensor(kept, device=w.device)
            weights[b, h, :keep] = w[at]
            for pool in (s["kpool"], s["vpool"]):
                rows = torch.cat([pool[p, h] for p in pages])[at]
                for i, page in enumerate(spare):
                    part = rows[i * PAGE:(i + 1) * PAGE]
                    pool[page, h, :len(part)] = part
    return [None, None, weights, None, s["kpool"].double(), s["vpool"].double()]


def _exact_verify(case, s):
    """The logarithms; tokens and counts are whole numbers."""
    logprobs = torch.zeros((case["batch"], case["drafts"] + 1), dtype=torch.float64, device=s["target"].device)
    for b, count in enumerate(_drafted(case)):
        def shares(row):
            row = row.double()
            if case["temp"] == 0:
                return (torch.arange(len(row), device=row.device) == int((row == row.max()).nonzero()[0])).double()
            return torch.softmax(row / float(s["temp"][b]), -1)

        k = 0
        while k < count:
            token = int(s["tokens"][b, k])
            p = shares(s["target"][b, k])
            drawn = 1.0 if s["draft"] is None else float(shares(s["draft"][b, k])[token])
            if case["temp"] == 0 and float(p[token]) == 0:
                break
            if case["temp"] != 0 and not float(s["accept"][b, k]) * drawn < float(p[token]):
                break
            logprobs[b, k] = torch.log(p[token])
            k += 1
        p = shares(s["target"][b, k])
        rest = p.clone()
        if k < count and case["temp"] != 0:
            if s["draft"] is None:
                rest[int(s["tokens"][b, k])] = 0
            else:
                rest = (p - shares(s["draft"][b, k])).clamp_(min=0)
        if not float(rest.sum()) > 0:
            rest = p
        logprobs[b, k] = torch.log(p[int((rest / -torch.log(s["noise"][b].double())).argmax())])
    return [None, None, logprobs]
