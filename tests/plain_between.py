"""Plain 64-bit forms of the operators between two steps: attention that keeps its weights, eviction, verification of drafts.
Tensors on the CPU, one row and one head at a time."""
import math

import torch

PAGE = 64


def gather(pages, table_row, head, length):
    """[length, ...] rows of one sequence and head, in order; None where the table names no page."""
    return [pages[table_row[p // PAGE], head, p % PAGE] if 0 <= table_row[p // PAGE] < pages.shape[0] else None for p in range(length)]


def weights(q, k, v, scores, table, row0, start, new, heads, scale):
    """(out, scores', out's tolerance, scores' tolerance) with the tolerances of a float32 computation: a score is off by
    (D + 8) 2^-24 of the sum of its products' sizes, a weight by twice that and by the rounding of its sums."""
    k, q = k.double(), q.double()
    v = v.double() if v is not None else None
    n_pages, kvh, _, dim = k.shape
    vd = v.shape[-1] if v is not None else 0
    group = heads // kvh
    out = torch.zeros(q.shape[0], heads * vd, dtype=torch.float64)
    out_tol = torch.zeros_like(out)
    got, tol = scores.double().clone(), torch.zeros(scores.shape, dtype=torch.float64)
    u = 2.0 ** -24
    for i, (r0, s0, n) in enumerate(zip(row0, start, new)):
        length = s0 + n
        row = table[i]
        ok = [p for p in range(length) if 0 <= row[p // PAGE] < n_pages]
        if n == 0:
            continue
        pages = torch.tensor([row[p // PAGE] for p in ok], dtype=torch.long)
        at = torch.tensor([p % PAGE for p in ok], dtype=torch.long)
        place = torch.tensor(ok, dtype=torch.long)
        for h in range(kvh):
            keys = k[pages, h, at]
            gained = torch.zeros(len(ok), dtype=torch.float64)
            wrong = torch.zeros(len(ok), dtype=torch.float64)
            for j in range(n):
                seen = place <= s0 + j
                if not bool(seen.any()):
                    continue
                for g in range(group):
                    x = q[r0 + j, (h * group + g) * dim:(h * group + g + 1) * dim]
                    s = (keys[seen] @ x) * scale
                    size = (keys[seen].abs() @ x.abs()) * abs(scale)
                    w = torch.softmax(s, 0)
                    off = w * (2 * (dim + 8) * u * float(size.max()) + (length + 32) * u)
                    gained[seen] += w
                    wrong[seen] += off
                    if v is not None:
                        vals = v[pages, h, at][seen]
                        sl = slice((h * group + g) * vd, (h * group + g + 1) * vd)
                        out[r0 + j, sl] = w @ vals
                        out_tol[r0 + j, sl] = off @ vals.abs()
            old = torch.where(place < s0, got[pages, h, at], torch.zeros((), dtype=torch.float64))
            got[pages, h, at] = old + gained
            tol[pages, h, at] = wrong + (n * group + 4) * u * (old.abs() + gained)
    return out, got, out_tol, tol


def choose(scores, length, keep, first, recent):
    """The places that stay, in order, of one unit's scores (a list of floats)."""
    keep = max(0, min(keep, length))
    first = min(first, keep)
    recent = min(recent, keep - first)
    middle = list(range(first, length - recent))
    middle.sort(key=lambda p: (-(scores[p] if scores[p] == scores[p] else -math.inf), scores[p] != scores[p], p))
    return sorted(list(range(first)) + middle[:keep - first - recent] + list(range(length - recent, length)))


def turn(key, move, inv_freq, interleaved):
    """A key (64 bits) turned by the angle of ``move`` places."""
    n = len(inv_freq)
    out = key.clone()
    angle = move * inv_freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = (key[0:2 * n:2], key[1:2 * n:2]) if interleaved else (key[:n], key[n:2 * n])
    x, y = a * c - b * s, b * c + a * s
    if interleaved:
        out[0:2 * n:2], out[1:2 * n:2] = x, y
    else:
        out[:n], out[n:2 * n] = x, y
    return out


def target(logits, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """The target's probabilities of one row of logits (64 bits)."""
    x = logits.double()
    if temperature == 0.0:
        p = torch.zeros_like(x)
        p[int(torch.argmax(x))] = 1.0
        return p
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))        # noqa: E731
    values, order = torch.sort(x / f32(temperature), descending=True, stable=True)
    p = torch.softmax(values, 0)
    if top_k:
        p = p[:top_k] / p[:top_k].sum()
    if min_p > 0.0:
        p = p[p >= p[0] * f32(min_p)]
        p = p / p.sum()
    if top_p < 1.0:
        n = int((torch.cumsum(p, 0) < f32(top_p)).sum()) + 1
        p = p[:n] / p[:n].sum()
    full = torch.zeros_like(x)
    full[order[:p.numel()]] = p
    return full


def verify(logits, row0, n_drafts, drafts, probs, accept, draw, temperature, **filters):
    """(accepted drafts, the token behind them) of one sequence; ``probs`` [drafts, vocabulary] or None."""
    for j in range(n_drafts + 1):
        p = target(logits[row0 + j], temperature, **filters)
        if j == n_drafts:
            break
        x = int(drafts[j])
        if probs is not None:
            q = probs[j].double()
        else:
            q = torch.zeros_like(p)
            if 0 <= x < p.numel():
                q[x] = 1.0
        if 0 <= x < p.numel() and float(accept[j]) * float(q[x]) < float(p[x]):
            continue
        rest = torch.clamp(p - q, min=0.0)
        p = rest if float(rest.sum()) > 0.0 else p
        break
    over = torch.nonzero(torch.cumsum(p, 0) > float(draw) * float(p.sum()))
    return j, int(over[0]) if over.numel() else int(torch.nonzero(p)[-1])
