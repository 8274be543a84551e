"""Plain 64-bit forms of the paged-cache operators, for their tests: one request, head and query at a time over the
keys that it sees, and a plan request by request."""
import math

import torch


def visible(pos, window, sinks):
    """The keys a query at ``pos`` sees, as a list of positions."""
    return [j for j in range(pos + 1) if window == 0 or j > pos - window or j < sinks]


def attend(q, k_cache, v_cache, table, pos_of, group, window, sinks, scale):
    """Attention of rows q [n, heads, dim] at positions ``pos_of`` (one request each row of ``table``: a list
    of page lists): float64 (out, sum of p |v|)."""
    n, heads, dim = q.shape
    pages, _, page, _ = k_cache.shape
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(n):
        keys = [j for j in visible(pos_of[i], window, sinks) if 0 <= table[i][j // page] < pages]
        if not keys:
            continue
        pg = torch.tensor([table[i][j // page] for j in keys], device=q.device)
        at = torch.tensor([j % page for j in keys], device=q.device)
        k, v = k_cache[pg, :, at].double(), v_cache[pg, :, at].double()       # [keys, kv_heads, dim]
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = (q[i].double()[None] * k).sum(-1) * scale                          # [keys, heads]
        p = torch.softmax(s, 0)
        out[i] = (p[..., None] * v).sum(0)
        mag[i] = (p[..., None] * v.abs()).sum(0)
    return out, mag


def norm_rope(x, gain, cos, sin, eps):
    """x [n, heads, dim], cos / sin [n, dim / 2] (float64): RMSNorm (gain None: none), then the rotation of halves."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gain.double()
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def plan(new, lengths, table, free, count, page, total):
    """The plan by its definition; ``table`` (lists) is changed in place. Returns a dict of lists."""
    width = len(table[0])
    stack, short, end = list(free[:count]), False, 0
    r = dict(slots=[], positions=[], cu=[0], kv=[], held=[], status=[])
    for b, (a, n) in enumerate(zip(lengths, new)):
        a, n = max(a, 0), max(n, 0)
        end += n
        room, full = end <= total, a + n > width * page
        want = range(0) if full or not room else range(math.ceil(a / page), math.ceil((a + n) / page))
        short = short or len(want) > len(stack)
        ok = room and not full and not (short and len(want))
        for i in want if ok else ():
            table[b][i] = stack.pop()
        for p in range(a, a + n):
            r["slots"].append(table[b][p // page] * page + p % page if ok else -1)
            r["positions"].append(p)
        r["cu"].append(end)
        r["kv"].append(a + n if ok else 0)
        r["held"].append(a + n if ok else a)
        r["status"].append(3 if not room else 2 if full else 0 if ok else 1)
    r["slots"] = (r["slots"] + [-1] * total)[:total]
    r["positions"] = (r["positions"] + [0] * total)[:total]
    r["count"] = len(stack)
    return r
