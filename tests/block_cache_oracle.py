"""Plain 64-bit definitions of the block-scaled cache operators and of draft
verification (CPU, loops), for the tests."""
import math

import torch

D = 128


def e4m3_values(x):
    """Nearest e4m3 value of a float64 tensor, ties to even, saturating at 448."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def power_of_two_scale(amax):
    """Smallest 2^e, e in [-64, 100], with amax <= 448 * 2^e."""
    if amax == 0:
        return 2.0 ** -64
    e = -64
    while e < 100 and amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate32(x, cos_sin):
    """Neox rotation in fp32, products rounded before the sum (the operator's
    arithmetic: its codes are one rounding of this value)."""
    x, c, s = x.float(), cos_sin[..., :D // 2], cos_sin[..., D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def append(qkv, cos_sin, k, v, ks, vs, cu, lens, table, hq):
    """k, v: float64 code values [NB, BS, HKV, D], ks, vs float64 [NB, HKV], updated
    in place; returns the rotated q in fp32."""
    hkv, bs = k.shape[2], k.shape[1]
    x = qkv.view(qkv.shape[0], hq + 2 * hkv, D)
    q = torch.zeros(qkv.shape[0], hq, D)
    for s, total in enumerate(lens):
        n = cu[s + 1] - cu[s]
        begin = total - n
        for i in range(n):
            pos = min(max(begin + i, 0), cos_sin.shape[0] - 1)
            q[cu[s] + i] = rotate32(x[cu[s] + i, :hq], cos_sin[pos])
        page = begin // bs
        while n and page * bs < total:
            lo, hi = max(begin, page * bs), min(total, (page + 1) * bs)
            blk = table[s][page] if 0 <= page < len(table[s]) else -1
            if 0 <= blk < k.shape[0]:
                rows = slice(cu[s] + lo - begin, cu[s] + hi - begin)
                pos = torch.arange(lo, hi).clamp(0, cos_sin.shape[0] - 1)
                kn = rotate32(x[rows, hq:hq + hkv], cos_sin[pos][:, None])
                for cache, scales, new in ((k, ks, kn.double()), (v, vs, x[rows, hq + hkv:].double())):
                    for h in range(hkv):
                        vals = new[:, h]
                        fin = vals[torch.isfinite(vals)].abs()
                        scale = power_of_two_scale(fin.max().item() if len(fin) else 0.0)
                        kept = lo - page * bs
                        if kept:
                            old = scales[blk, h].item()
                            scale = max(scale, old)
                            if scale != old:
                                cache[blk, :kept, h] = e4m3_values(cache[blk, :kept, h] * (old / scale))
                        scales[blk, h] = scale
                        cache[blk, kept:kept + hi - lo, h] = e4m3_values(vals / scale)
            page += 1
    return q


def attention(q, k, v, ks, vs, cu, lens, table, sm_scale, window=0, sinks=0):
    """float64 [T, HQ, D]; k, v code values."""
    hkv, bs = k.shape[2], k.shape[1]
    group = q.shape[1] // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    for s, total in enumerate(lens):
        n = cu[s + 1] - cu[s]
        if n == 0 or total <= 0:
            continue
        blocks = torch.tensor(table[s][:-(-total // bs)], dtype=torch.long)
        keys = (k[blocks].double() * ks[blocks][:, None, :, None].double()).reshape(-1, hkv, D)[:total]
        vals = (v[blocks].double() * vs[blocks][:, None, :, None].double()).reshape(-1, hkv, D)[:total]
        for i in range(n):
            pos = total - n + i
            sees = [j for j in range(0, pos + 1) if not window or j > pos - window or j < sinks]
            if not sees:
                continue
            for h in range(q.shape[1]):
                x = keys[sees, h // group] @ q[cu[s] + i, h].double() * sm_scale
                p = torch.exp(x - x.max())
                out[cu[s] + i, h] = (p / p.sum()) @ vals[sees, h // group]
    return out


def probabilities(row, temperature):
    row = row.double()
    row = torch.where(torch.isnan(row), -math.inf, row).clamp_max(torch.finfo(torch.float32).max)
    p = torch.zeros_like(row)
    if row.max() == -math.inf:
        return p
    if temperature <= 0:
        p[int((row == row.max()).nonzero()[0])] = 1
        return p
    p = torch.exp((row - row.max()) / temperature)
    return p / p.sum()


def verify(logits, tokens, cu, uniforms, noise, temperature=None, draft=None):
    vocab = logits.shape[1]
    out, accepted = torch.full((logits.shape[0],), -1, dtype=torch.int64), []
    for s in range(len(cu) - 1):
        heat = 1.0 if temperature is None else float(temperature[s])
        for r in range(cu[s], cu[s + 1]):
            p, last = probabilities(logits[r], heat), r == cu[s + 1] - 1
            q = torch.zeros(vocab, dtype=torch.float64)
            if not last:
                d = int(tokens[r + 1])
                if draft is not None:
                    q = draft[r].double()
                elif 0 <= d < vocab:
                    q[d] = 1
                if 0 <= d < vocab and float(uniforms[r]) * q[d] < p[d]:
                    out[r] = d
                    continue
            w = (p - q).clamp_min(0)
            w = w if w.max() > 0 else p
            race = w / noise[s].double()
            out[r] = int((race == race.max()).nonzero()[0])
            accepted.append(r - cu[s])
            break
        else:
            accepted.append(0)
    return out, torch.tensor(accepted, dtype=torch.int32)
