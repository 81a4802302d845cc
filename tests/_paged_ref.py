"""Plain restatements of the paged operators: attention in 64 bits with the error bound of each
output, and the block tables, slot writes and kept drafts as a host program does them."""

import math

import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative


def parts(cache):
    return (cache[0], cache[1]) if cache.shape[0] == 2 else (cache[:, 0], cache[:, 1])


def visible(n, t, mask_rows, device):
    """[t, n] truth values: what each of the last t queries sees of n positions."""
    pos = torch.arange(n, device=device) - (n - t)
    i = torch.arange(t, device=device).unsqueeze(1)
    if mask_rows is None:
        return pos.unsqueeze(0) <= i
    seen = (pos < 0).unsqueeze(0).expand(t, n).clone()
    for j in range(t):
        if n - t + j >= 0 and j // 64 < mask_rows.shape[1]:
            seen[:, n - t + j] = ((mask_rows[:, j // 64] >> (j % 64)) & 1).bool()
    return seen


def attention(query, cache, tables, lengths, starts, mask=None, scale=None):
    """(out, lse, bound) in 64 bits.  `bound` is how far a kernel's output may be off that takes
    exact products, sums in 32 bits, rounds each weight to the type once, and the result once:
      weights     u * A with A = sum p |v| / sum p, and in fp16, where a weight below 2^-14 of the
                  largest is held in steps of 2^-24, 2^-25 sum |v| / sum p on top
      result      u |o| (fp16: at least 2^-25)
      scores      a sum of D products is off by (D + 8) 2^-24 sum |q k| scale; with exp and the
                  scaling, each weight by that and 2^-20, numerator and denominator both: 2 A times
      sums        (n + 64) 2^-24, numerator and denominator both: 2 A times
    """
    keys, values = parts(cache)
    S, H, D = keys.shape[1:]
    G = query.shape[1] // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, half = U[query.dtype], query.dtype == torch.float16
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    bound = torch.zeros_like(out)
    lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float64, device=query.device)
    begin = starts.tolist()
    for r, n in enumerate(lengths.tolist()):
        a, b = begin[r], begin[r + 1]
        t = b - a
        if t == 0 or n == 0:
            continue
        p = torch.arange(n, device=query.device)
        block = tables[r].long()[p // S]
        seen = visible(n, t, None if mask is None else mask[a:b], query.device).repeat_interleave(G, 0)
        for h in range(H):
            q = query[a:b, h * G:(h + 1) * G].double().reshape(t * G, D)
            k, v = keys[block, p % S, h].double(), values[block, p % S, h].double()
            x = (q @ k.t()) * scale
            size = (q.abs() @ k.abs().t()) * scale
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            size = torch.where(seen, size, torch.zeros_like(size)).amax(1, keepdim=True)
            top = x.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            w = torch.exp(x - top)
            w = torch.where(seen, w, torch.zeros_like(w))
            total = w.sum(1, keepdim=True)
            safe = torch.where(total == 0, torch.ones_like(total), total)
            o, A = w @ v, w @ v.abs()
            # a position that a row does not see has no part in it, whatever it holds
            odd = ~torch.isfinite(v).all(1)
            if odd.any():
                clean = torch.where(odd.unsqueeze(1), torch.zeros_like(v), v)
                o, A = w @ clean, w @ clean.abs()
                for j in torch.nonzero(odd).flatten().tolist():
                    hit = seen[:, j].unsqueeze(1)
                    o = o + torch.where(hit, w[:, j:j + 1] * v[j:j + 1], torch.zeros_like(o))
            o, A = o / safe, A / safe
            e = u * (A + o.abs()) + 2 * A * (size * (D + 8) * 2.0**-24 + 2.0**-20 + (n + 64) * 2.0**-24)
            if half:
                e = e + 2.0**-25 * (1 + (seen.double() @ torch.where(torch.isfinite(v), v, torch.zeros_like(v)).abs())
                                    / safe)
            out[a:b, h * G:(h + 1) * G] = o.reshape(t, G, D)
            bound[a:b, h * G:(h + 1) * G] = e.reshape(t, G, D)
            lse[a:b, h * G:(h + 1) * G] = (top + torch.log(total)).reshape(t, G)
    return out, lse, bound


def build_tables(lengths, new_lengths, tables, free, state, S, max_tokens):
    """The update one request after the other, on lists; returns
    (tables, lengths, state, slots, starts, free, refused, bad)."""
    rows, ring = [list(r) for r in tables], list(free)
    head, count = state
    N, C = len(ring), len(rows[0]) if rows else 0
    asked, taken, returned = 0, 0, []
    after, slots, starts, refused, bad = [], [], [0], False, False
    for row, a, b in zip(rows, lengths, new_lengths):
        if not (0 <= a <= C * S and 0 <= b <= C * S):
            bad = True
            after.append(a)
            starts.append(len(slots))
            n = min(max(-(-a // S), 0), C)
            row[n:] = [-1] * (C - n)
            continue
        have, want = -(-a // S), -(-b // S)
        asked += max(0, want - have)
        if want > have and asked > count:
            refused = True
            row[have:] = [-1] * (C - have)
            after.append(a)
            slots += [-1] * (b - a)
        else:
            old = row[:have]
            if want > have:
                taken = asked
            fresh = [ring[(head + asked - (want - have) + i) % N] for i in range(max(0, want - have))]
            returned += old[want:]
            row[:] = (old[:want] + fresh + [-1] * C)[:C]
            after.append(b)
            slots += [row[p // S] * S + p % S for p in range(a, b)]
        starts.append(len(slots))
    # requests behind a refused one may still fit only if they ask for nothing, so `taken` is the
    # asked-for sum up to the last that fits
    for i, block in enumerate(returned):
        ring[(head + count + i) % N] = block
    bad = bad or len(slots) > max_tokens
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return rows, after, [(head + taken) % N, count - taken + len(returned)], slots, starts, ring, refused, bad
