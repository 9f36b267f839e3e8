"""Plain NumPy forms, in 64 bits, of the operators over caller-owned paged caches and of the verification of drafts.

They follow the definitions in include/mtj_b200.h (mtj_k_cache_attn, mtj_k_cache_evict, mtj_verify_drafts), one sequence at a time,
and share no code with the kernels.  Test infrastructure only."""
import numpy as np

PAGE = 64


def slots_of(pool, table_row, n):
    """The first n slots of one sequence: [n, kv_heads, d_head] from a pool [pages, kv_heads, 64, d_head]."""
    rows = [pool[table_row[i // PAGE], :, i % PAGE] for i in range(n)]
    return np.stack(rows).astype(np.float64) if rows else np.zeros((0, pool.shape[1], pool.shape[3]))


def attention(q, keys, values, length, fresh, window, sinks, scale):
    """q [fresh, heads, d], keys and values [length, kv_heads, d] with the new tokens in place -> (out [fresh, heads, d], the
    weight that every slot received [kv_heads, length])."""
    heads, kv_heads = q.shape[1], keys.shape[1]
    group = heads // kv_heads
    out = np.zeros((fresh, heads, keys.shape[2]))
    received = np.zeros((kv_heads, length))
    for t in range(fresh):
        p = length - fresh + t
        seen = [j for j in range(p + 1) if j < sinks or p - j < window]
        for h in range(heads):
            k, v = keys[seen, h // group], values[seen, h // group]
            s = scale * (k @ q[t, h].astype(np.float64))
            a = np.exp(s - s.max())
            a /= a.sum()
            out[t, h] = a @ v
            received[h // group, seen] += a
    return out, received


def evict(weights, length, keep, first, last):
    """The slots that one key head keeps, ascending; weights [slots]."""
    if length <= keep:
        return list(range(length))
    middle = range(first, length - last)
    heaviest = sorted(middle, key=lambda i: (-float(weights[i]), i))[:keep - first - last]
    return sorted([*range(first), *heaviest, *range(length - last, length)])


def shares(logits, temp):
    logits = logits.astype(np.float64)
    if not temp > 0:
        p = np.zeros(len(logits))
        p[int(np.argmax(logits))] = 1.0
        return p
    e = np.exp((logits - logits.max()) / temp)
    return e / e.sum()


def verify(target, draft, tokens, accept, noise, temp):
    """One sequence: target [n + 1, vocab], draft [n, vocab] or None, tokens and accept [n], noise [vocab] ->
    (tokens that come out, number taken, log p of them)."""
    out, logs = [], []
    for k, x in enumerate(tokens):
        p = shares(target[k], temp)
        inside = 0 <= x < len(p)
        if not temp > 0:
            take, rest = inside and p[x] == 1.0, p
        else:
            q = np.zeros(len(p))
            if draft is not None:
                q = shares(draft[k], temp)
            elif inside:
                q[x] = 1.0
            take = inside and float(accept[k]) * q[x] < p[x]
            rest = np.maximum(p - q, 0.0)
        if not take:
            break
        out.append(int(x))
        logs.append(np.log(p[x]))
    else:
        p = rest = shares(target[len(tokens)], temp)
    if not rest.sum() > 0:
        rest = p
    nxt = int(np.argmax(rest / -np.log(noise.astype(np.float64)))) if temp > 0 else int(np.argmax(p))
    return [*out, nxt], len(out), [*logs, np.log(p[nxt])]
