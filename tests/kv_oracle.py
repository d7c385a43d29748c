"""Plain 64-bit forms of the cache's operators, for the tests: the code table written out, requests one after the other."""
import math

import numpy as np


def e4m3_values():
    """Value of each of the 256 codes: sign, four exponent bits (bias 7), three mantissa bits; 0x7f and 0xff are NaN."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if c & 127 == 127 else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(-v if c & 128 else v)
    return np.array(out)


VALUES = e4m3_values()


def encode(x):
    """Nearest code of each value, ties to the even code, beyond 448 saturated, NaN to 0x7f."""
    x = np.asarray(x, np.float64)
    grid = VALUES[:127]
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=1e300, neginf=-1e300)), 448.0)
    hi = np.searchsorted(grid, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - grid[lo], grid[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    pick = np.where(grid[hi] == a, hi, pick)
    code = pick | np.where(np.signbit(x), 128, 0)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def scale_for(amax):
    """Smallest 2^e, e in [-32, 64], with amax / 2^e <= 448."""
    if not amax > 0:
        return 2.0 ** -32
    e = -32
    while e < 64 and amax / 2.0 ** e > 448:
        e += 1
    return 2.0 ** e


def write(x, slots, codes, scale):
    """x [tokens, heads, dim] float64 into codes [blocks, heads, bs, dim] and scale [blocks, heads] (changed in place)."""
    blocks, heads, bs, dim = codes.shape
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if not 0 <= s < blocks * bs:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) // bs == s // bs:
            n += 1
        b, off = s // bs, s % bs
        for h in range(heads):
            part = x[t:t + n, h]
            size = np.abs(part[np.isfinite(part)])
            new = scale_for(size.max() if size.size else 0.0)
            if off:
                old = float(scale[b, h])
                new = max(new, old)
                if new != old:
                    codes[b, h, :off] = encode(VALUES[codes[b, h, :off]] * (old / new))
            codes[b, h, off:off + n] = encode(part / new)
            scale[b, h] = new
        t += n


def attend(q, k_codes, v_codes, k_scale, v_scale, table, starts, lens, scale, causal, heads_per_key):
    """(out, lse, sum p|v|) in float64; rows behind the last request are NaN."""
    rows, heads, dim = q.shape
    blocks, _, bs, _ = k_codes.shape
    out, lse, mag = np.full(q.shape, np.nan), np.full((rows, heads), np.nan), np.full(q.shape, np.nan)
    for r in range(len(lens)):
        n, length = int(starts[r + 1] - starts[r]), int(min(lens[r], table.shape[1] * bs))
        ids = table[r, :-(-length // bs)].astype(np.int64)
        good = (ids >= 0) & (ids < blocks)
        at = np.where(good, ids, 0)
        held = np.repeat(good, bs)[:length]
        for h in range(k_codes.shape[1]):
            k = (VALUES[k_codes[at, h]] * k_scale[at, h].astype(np.float64)[:, None, None]).reshape(-1, dim)[:length]
            v = (VALUES[v_codes[at, h]] * v_scale[at, h].astype(np.float64)[:, None, None]).reshape(-1, dim)[:length]
            for i in range(n):
                seen = held.copy()
                if causal:
                    seen[max(0, length - n + i + 1):] = False
                for g in range(heads_per_key):
                    hq, row = h * heads_per_key + g, int(starts[r]) + i
                    if not seen.any():
                        out[row, hq], lse[row, hq], mag[row, hq] = 0.0, -np.inf, 0.0
                        continue
                    s = (k[seen] @ q[row, hq]) * scale
                    m = s.max()
                    p = np.exp(s - m)
                    out[row, hq] = p @ v[seen] / p.sum()
                    mag[row, hq] = p @ np.abs(v[seen]) / p.sum()
                    lse[row, hq] = m + np.log(p.sum())
    return out, lse, mag


def plan(context, new, free, count, table, bs, num_blocks, max_tokens):
    """The step's arrays as a dict, table changed in place; None when it cannot be planned."""
    R, width = table.shape
    if any(c < 0 or n < 0 for c, n in zip(context, new)) or any(c + n > width * bs for c, n in zip(context, new)):
        return None
    need = [-(-(c + n) // bs) - -(-c // bs) for c, n in zip(context, new)]
    if sum(new) > max_tokens or sum(need) > count:
        return None
    used, slots, pos, req = 0, [], [], []
    for r in range(R):
        have = -(-context[r] // bs)
        for j in range(need[r]):
            table[r, have + j] = free[count - 1 - used]
            used += 1
        for p in range(context[r], context[r] + new[r]):
            b = int(table[r, p // bs])
            slots.append(b * bs + p % bs if 0 <= b < num_blocks else -1)
            pos.append(p)
            req.append(r)
    pad = max_tokens - len(slots)
    return dict(query_start=np.cumsum([0] + list(new)), seq_lens=np.add(context, new), slot_map=np.array(slots + [-1] * pad),
                positions=np.array(pos + [0] * pad), token_request=np.array(req + [-1] * pad), taken=used, free_count=count - used)


def scores(x, tokens, k):
    """(logprob, entropy, lse, top ids, top logprobs) of logits [rows, vocab] in float64."""
    x = np.asarray(x, np.float64)
    rows, vocab = x.shape
    lp, ent, lse, ids, top = np.zeros(rows), np.zeros(rows), np.zeros(rows), np.zeros((rows, k), np.int64), np.zeros((rows, k))
    for r in range(rows):
        t = int(tokens[r])
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            lp[r] = ent[r] = lse[r] = np.nan
            ids[r], top[r] = -1, np.nan
            continue
        order = np.lexsort((np.arange(vocab), -(x[r] + 0.0)))[:k]
        ids[r] = order
        m = x[r].max()
        if m == -np.inf:
            lp[r], lse[r], top[r] = (-np.inf if 0 <= t < vocab else 0.0), -np.inf, -np.inf
            continue
        e = np.exp(x[r] - m)
        lse[r] = m + np.log(e.sum())
        p = e / e.sum()
        ent[r] = np.log(e.sum()) - np.sum(p[p > 0] * (x[r][p > 0] - m))      # not with lse, which may have lost log s beside a huge m
        lp[r] = (x[r, t] - m) - np.log(e.sum()) if 0 <= t < vocab else 0.0
        top[r] = (x[r, order] - m) - np.log(e.sum())
    return lp, ent, lse, ids, top


def score_gradient(x, tokens, lse, ent, u, w):
    x = np.asarray(x, np.float64)
    out = np.zeros(x.shape)
    for r in range(x.shape[0]):
        t = int(tokens[r])
        given = 0 <= t < x.shape[1]
        if lse[r] == -np.inf:
            continue
        l = x[r] - lse[r]
        p = np.exp(l)
        l = np.where(p > 0, l, 0.0)
        out[r] = -p * ((u[r] if given else 0.0) + w[r] * (l + ent[r]))
        if given:
            out[r, t] += u[r]
    return out
