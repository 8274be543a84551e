"""Timed operators of the paged key-value cache: what serving many streams from one page pool calls.

A layer's cache is ``[pages, kv_heads, page_size, head_dim]`` for K and for V; ``block_table[r, i]`` is the page
of request r's tokens ``i * page_size ...``. Four operators work on it:

* ``plan``: pages for new tokens, and the slot and position of each (block table and slot map);
* ``store``: RMSNorm of every query and key head, rotation, K and V into their slots;
* ``decode``: attention of one new token per request over its pages, with an optional sliding window and
  first tokens that stay visible;
* ``prefill``: the same for the new tokens of prompts, packed one request after the other.

Head counts 16 / 8 with 128 channels are the talker's; the others are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
SECTION = 20          # channels below 3 * SECTION rotate by (t, h, w) in turn, the others by t


def _pkg():
    import __graft_entry__
    return __graft_entry__.import_package()


def listed():
    return [
        # one step of a serving batch: a new token for each of 64 streams; latency alone
        dict(name="plan_step_64", op="plan", requests=64, prompts=0, longest=1, context=3000, page=64, ragged=1),
        # a burst of admissions between running streams: prompts up to 1500 tokens, single tokens, idle rows
        dict(name="plan_admit_400", op="plan", requests=400, prompts=60, longest=1500, context=2500, page=16, ragged=2),
        # the new tokens of 40 streams with (t, h, w) positions
        dict(name="store_40_mrope", op="store", tokens=40, hq=16, hkv=8, dim=128, page=64, mrope=True, dtype="bf16"),
        # prompts of a voice-cloning batch, packed
        dict(name="store_6001", op="store", tokens=6001, hq=16, hkv=8, dim=128, page=64, mrope=False, dtype="bf16"),
        # another head layout, in half precision
        dict(name="store_1777_fp16", op="store", tokens=1777, hq=24, hkv=4, dim=64, page=16, mrope=False, dtype="fp16"),
        # one stream in the middle of an utterance
        dict(name="decode_1_at_700", op="decode", requests=1, shortest=700, longest=700, hq=16, hkv=8, dim=128, page=64,
             window=0, sinks=0, dtype="bf16", ragged=3),
        # a serving batch with ragged contexts
        dict(name="decode_64", op="decode", requests=64, shortest=129, longest=4090, hq=16, hkv=8, dim=128, page=64,
             window=0, sinks=0, dtype="bf16", ragged=4),
        # long-running streams that attend a window and the prompt's first tokens
        dict(name="decode_24_window", op="decode", requests=24, shortest=3001, longest=20011, hq=16, hkv=8, dim=128, page=64,
             window=1024, sinks=16, dtype="bf16", ragged=5),
        # few requests with very long contexts, grouped heads, half precision
        dict(name="decode_3_long", op="decode", requests=3, shortest=40007, longest=60001, hq=32, hkv=4, dim=64, page=128,
             window=0, sinks=0, dtype="fp16", ragged=6),
        # short prompts and pieces appended to running contexts, in one call
        dict(name="prefill_12_short", op="prefill", requests=12, shortest=5, longest=300, context=900, hq=16, hkv=8, dim=128,
             page=64, window=0, sinks=0, dtype="bf16", ragged=7),
        # one long prompt
        dict(name="prefill_4096", op="prefill", requests=1, shortest=4096, longest=4096, context=0, hq=16, hkv=8, dim=128,
             page=64, window=0, sinks=0, dtype="bf16", ragged=8),
        # long prompts under a window, another head layout, half precision
        dict(name="prefill_3_window", op="prefill", requests=3, shortest=1111, longest=3500, context=700, hq=32, hkv=4, dim=64,
             page=32, window=777, sinks=5, dtype="fp16", ragged=9),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["plan", "store", "decode", "decode", "prefill", "prefill"])
    page = rng.choice([16, 32, 64, 128, 256])
    ragged = rng.randint(10, 10 ** 6)
    if op == "plan":
        n = log_int(1, 400)
        return dict(op=op, requests=n, prompts=rng.randint(0, n // 6), longest=log_int(2, 1500), context=log_int(1, 3000), page=page,
                    ragged=ragged)
    hq, hkv, dim = rng.choice([(16, 8, 128), (16, 8, 128), (8, 8, 64), (32, 4, 64), (16, 1, 128), (12, 4, 128), (20, 4, 64)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "store":
        return dict(op=op, tokens=log_int(1, 4000), hq=hq, hkv=hkv, dim=dim, page=page, mrope=dim == 128 and rng.random() < 0.4, dtype=dtype)
    window, sinks = (log_int(1, 2000), rng.choice([0, 1, 4, 16, 50])) if rng.random() < 0.4 else (0, 0)
    base = dict(op=op, hq=hq, hkv=hkv, dim=dim, page=page, window=window, sinks=sinks, dtype=dtype, ragged=ragged)
    if op == "decode":
        longest = log_int(1, 20000)
        return dict(base, requests=log_int(1, max(1, min(64, 120000 // longest))), shortest=rng.randint(1, longest), longest=longest)
    longest = log_int(1, 2000)
    n = log_int(1, max(1, min(16, 4000 // longest)))
    return dict(base, requests=n, shortest=rng.randint(1, longest), longest=longest, context=rng.choice([0, log_int(1, 2000)]))


# ---- inputs --------------------------------------------------------------------------------------


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _sizes(case):
    """(tokens held before the call, new tokens) per request: a property of the case, not of the seed."""
    rng = random.Random(case["ragged"])
    n = case["requests"]
    if case["op"] == "plan":
        held = [rng.randint(0, case["context"]) for _ in range(n)]
        new = [1 if rng.random() < 0.9 or case["prompts"] == 0 else 0 for _ in range(n)]
        for r in rng.sample(range(n), case["prompts"]):
            held[r], new[r] = 0, rng.randint(1, case["longest"])
        return held, new
    between = [rng.randint(case["shortest"], case["longest"]) for _ in range(n)]
    between[0] = case["longest"]
    if case["op"] == "decode":
        return [x - 1 for x in between], [1] * n
    return [rng.randint(0, case["context"]) for _ in range(n)], between


def _pages(n, page):
    return -(-n // page)


def _tables(g, held, width, page, spare):
    """A block table over pages in random order, and the stack of pages that are free."""
    total = sum(_pages(x, page) for x in held)
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, x in enumerate(held):
        n = _pages(x, page)
        table[r, :n] = order[at:at + n]
        at += n
    return table, order[total:].contiguous(), total + spare


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "plan":
        held, new = _sizes(case)
        page = case["page"]
        width = _pages(case["context"] + case["longest"] + 1, page)
        wanted = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(held, new))
        s["table"], s["free"], _ = _tables(g, held, width, page, wanted + 37)
        s["count"], s["lengths"], s["new"], s["tokens"] = _ints([s["free"].numel()]), _ints(held), _ints(new), sum(new)
        s["lengths_out"], s["count_out"] = torch.empty_like(s["lengths"]), torch.empty_like(s["count"])
        return s
    hq, hkv, dim, page, dt = case["hq"], case["hkv"], case["dim"], case["page"], _type(case)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)
    if case["op"] == "store":
        n = case["tokens"]
        rows = 8192
        angle = torch.outer(torch.arange(rows, dtype=torch.float64), THETA ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2)))
        angle = torch.cat((angle, angle), -1)
        s["cos"], s["sin"] = angle.cos().to("cuda", dt), angle.sin().to("cuda", dt)
        s["qkv"] = randn(n, (hq + 2 * hkv) * dim)       # one projection's output
        s["wq"], s["wk"] = (1 + 0.1 * randn(dim).float()).to(dt), (1 + 0.1 * randn(dim).float()).to(dt)
        pos = torch.randint(0, rows, (3 if case["mrope"] else 1, n), generator=g, device="cuda", dtype=torch.int32)
        s["pos"] = pos if case["mrope"] else pos[0].contiguous()
        pages = _pages(n, page) + 3
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:n].to(torch.int32)
        s["k"], s["v"] = randn(pages, hkv, page, dim), randn(pages, hkv, page, dim)
        return s
    held, new = _sizes(case)
    full = [a + b for a, b in zip(held, new)]
    s["longest"] = max(full)
    s["table"], _, pages = _tables(g, full, _pages(max(full), page), page, 3)
    s["lens"] = _ints(full)
    s["new"] = new
    s["cu"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
    s["q"] = randn(sum(new), hq, dim)
    s["k"], s["v"] = randn(pages, hkv, page, dim), randn(pages, hkv, page, dim)
    return s


# ---- plain forms ---------------------------------------------------------------------------------


def _plan(s):
    page, total = s["case"]["page"], s["tokens"]
    held, new, table, free = s["lengths"].long(), s["new"].long(), s["table"].long(), s["free"].long()
    count = s["count"].long()
    n, width = table.shape
    cu = torch.cat((torch.zeros(1, dtype=torch.long, device="cuda"), new.cumsum(0)))
    fits = (held + new <= width * page) & (cu[1:] <= total)
    have = (held + page - 1) // page
    need = torch.where(fits, (held + new + page - 1) // page - have, 0)
    taken = need.cumsum(0)
    ok = fits & ((need == 0) | (taken <= count))
    col = torch.arange(width, device="cuda")
    fresh = ok[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    at = count - 1 - ((taken - need)[:, None] + col - have[:, None])
    table = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table)
    t = torch.arange(total, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    p = held[r] + t - cu[r]
    real = t < cu[-1]
    slot = table[r, (p // page).clamp(max=width - 1)] * page + p % page
    i32 = torch.int32
    return dict(slots=torch.where(real & ok[r], slot, -1).to(i32), positions=torch.where(real, p, 0).to(i32), cu=cu.to(i32),
                lens=torch.where(ok, held + new, 0).to(i32), status=torch.where(cu[1:] > total, 3, torch.where(~fits, 2, torch.where(ok, 0, 1))).to(i32),
                held=torch.where(ok, held + new, held).to(i32), count=(count - torch.where(ok, need, 0).sum()).to(i32),
                table=table.to(i32))


def _rotation(s):
    """cos and sin of every token, f32 [tokens, 1, dim]."""
    cos, sin, pos, dim = s["cos"].float(), s["sin"].float(), s["pos"].long(), s["case"]["dim"]
    if pos.dim() == 1:
        return cos[pos][:, None], sin[pos][:, None]
    d = torch.arange(dim, device="cuda") % (dim // 2)
    which = torch.where(d < 3 * SECTION, d % 3, 0)
    at = pos[which].T                                     # [tokens, dim]
    d = torch.arange(dim, device="cuda")
    return cos[at, d][:, None], sin[at, d][:, None]


def _split(s):
    c = s["case"]
    n, hq, hkv, dim = c["tokens"], c["hq"], c["hkv"], c["dim"]
    q, k, v = s["qkv"].split([hq * dim, hkv * dim, hkv * dim], 1)
    return q.view(n, hq, dim), k.view(n, hkv, dim), v.view(n, hkv, dim)


def _store(s):
    q, k, v = _split(s)
    cos, sin = _rotation(s)

    def head(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y.chunk(2, -1)
        return (y * cos + torch.cat((-b, a), -1) * sin).to(s["qkv"].dtype)
    page, slots = s["case"]["page"], s["slots"].long()
    s["k"][slots // page, :, slots % page] = head(k, s["wk"])
    s["v"][slots // page, :, slots % page] = v
    return dict(q=head(q, s["wq"]), k=s["k"], v=s["v"])


def _attend(s):
    """Attention of padded query rows over padded contexts: decode and prefill."""
    c = s["case"]
    hq, hkv, dim, page = c["hq"], c["hkv"], c["dim"], c["page"]
    n, width = s["table"].shape
    cu, lens = s["cu"].long(), s["lens"].long()
    most, total = max(s["new"]), s["q"].shape[0]
    keys = width * page
    i = torch.arange(most, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=total - 1)                                   # [n, most]
    q = s["q"][row].float().view(n, most, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)
    at = s["table"].long().clamp(min=0)
    k = s["k"][at].permute(0, 2, 1, 3, 4).reshape(n, hkv, keys, dim).float()
    v = s["v"][at].permute(0, 2, 1, 3, 4).reshape(n, hkv, keys, dim).float()
    pos = (lens - (cu[1:] - cu[:-1]))[:, None] + i                                   # [n, most]
    j = torch.arange(keys, device="cuda")
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    seen &= (j < lens[:, None, None])
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, hkv, hq // hkv, most, keys) * dim ** -0.5
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, keys), v).view(n, hkv, hq // hkv, most, dim)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, hq, dim).to(s["q"].dtype)
    t = torch.arange(total, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o[r, t - cu[r]]


def run(s):
    c = s["case"]
    if not own:
        return _plan(s) if c["op"] == "plan" else _store(s) if c["op"] == "store" else _attend(s)
    pkg = _pkg()
    if c["op"] == "plan":
        p = pkg.paged_plan(s["new"], s["lengths"], s["table"], s["free"], s["count"], c["page"], s["tokens"],
                           lengths_out=s["lengths_out"], free_count_out=s["count_out"])
        return dict(slots=p.slots, positions=p.positions, cu=p.cu_tokens, lens=p.kv_lens, status=p.status, held=s["lengths_out"],
                    count=s["count_out"], table=s["table"])
    if c["op"] == "store":
        q, k, v = _split(s)
        out = pkg.qk_norm_rope_store(q, k, v, s["wq"], s["wk"], s["cos"], s["sin"], s["pos"], s["slots"], s["k"], s["v"], eps=EPS)
        return dict(q=out, k=s["k"], v=s["v"])
    if c["op"] == "decode":
        return pkg.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], window=c["window"], sinks=c["sinks"],
                                          max_len=s["longest"])
    return pkg.paged_attention_prefill(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], window=c["window"], sinks=c["sinks"],
                                       max_len=s["longest"])


# ---- work and exact values -----------------------------------------------------------------------


def _seen(c, pos):
    """How many keys a query at `pos` sees, and the first of its window."""
    lo = max(0, pos + 1 - c["window"]) if c["window"] else 0
    return pos + 1 - lo + min(lo, c["sinks"]), lo


def work(case):
    if case["op"] == "plan":
        held, new = _sizes(case)
        page = case["page"]
        fresh = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(held, new))
        n = len(held)
        return {"bytes": 4 * (2 * n + 1 + fresh) + 4 * (2 * sum(new) + 4 * n + 2 + fresh), "flops": 0}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["op"] == "store":
        n = case["tokens"]
        # a token's heads in and out, its table rows (half of each: both halves hold the same), its position and slot
        return {"bytes": n * (4 * (hq + 2 * hkv) * dim + 2 * dim + (16 if case["mrope"] else 8)) + 4 * dim, "flops": n * (hq + hkv) * dim * 7}
    held, new = _sizes(case)
    pairs = sum(_seen(case, a + i)[0] for a, b in zip(held, new) for i in range(b))
    keys = 0
    for a, b in zip(held, new):
        lo = _seen(case, a)[1]                             # the first query's window reaches furthest back
        keys += a + b - lo + min(lo, case["sinks"])
    return {"bytes": 4 * keys * hkv * dim + 4 * sum(new) * hq * dim + 4 * sum(_pages(a + b, case["page"]) for a, b in zip(held, new)),
            "flops": 4 * pairs * hq * dim}


def _planned(s):
    """The plan by its definition, request after request: the first that finds too few pages ends the giving."""
    page, table, free, short = s["case"]["page"], s["table"].tolist(), s["free"].tolist(), False
    slots, positions, cu, lens, status, held = [], [], [0], [], [], []
    for r, (a, b) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
        fits = a + b <= len(table[r]) * page
        want = range(_pages(a, page), _pages(a + b, page)) if fits else range(0)
        short = short or len(want) > len(free)
        ok = fits and not (short and len(want))
        for i in want if ok else ():
            table[r][i] = free.pop()
        slots += [table[r][p // page] * page + p % page if ok else -1 for p in range(a, a + b)]
        positions += range(a, a + b)
        cu.append(cu[-1] + b)
        lens.append(a + b if ok else 0)
        held.append(a + b if ok else a)
        status.append(0 if ok else 1 if fits else 2)
    return {k: _ints(x) for k, x in dict(slots=slots, positions=positions, cu=cu, lens=lens, status=status, held=held,
                                         count=[len(free)], table=table).items()}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "plan":
        return _planned(s)
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["op"] == "store":
        n, half = case["tokens"], dim // 2
        x = s["qkv"].to(f64).view(n, hq + 2 * hkv, dim)
        gain = torch.stack([s["wq"].to(f64)] * hq + [s["wk"].to(f64)] * hkv)
        y = x[:, :hq + hkv] / torch.sqrt(x[:, :hq + hkv].square().sum(-1, keepdim=True) / dim + EPS) * gain
        pos = s["pos"].long()
        cos, sin = torch.empty(n, half, dtype=f64, device="cuda"), torch.empty(n, half, dtype=f64, device="cuda")
        for d in range(half):
            p = pos if not case["mrope"] else pos[d % 3 if d < 3 * SECTION else 0]
            cos[:, d], sin[:, d] = s["cos"][p, d].to(f64), s["sin"][p, d].to(f64)
        a, b = y[..., :half], y[..., half:]
        c, si = cos[:, None], sin[:, None]
        z = torch.cat((a * c - b * si, b * c + a * si), -1)
        k, v = s["k"].to(f64), s["v"].to(f64)
        slots = s["slots"].long()
        k.permute(0, 2, 1, 3)[slots // page, slots % page] = z[:, hq:]
        v.permute(0, 2, 1, 3)[slots // page, slots % page] = x[:, hq + hkv:]
        return dict(q=z[:, :hq], k=k, v=v)
    held, new = _sizes(case)
    if sum(_seen(case, a + i)[0] for a, b in zip(held, new) for i in range(b)) * hq * dim > 2e11:
        return None
    out = torch.zeros(sum(new), hq, dim, dtype=f64, device="cuda")
    at = 0
    for r, (a, b) in enumerate(zip(held, new)):
        pages = s["table"][r, :_pages(a + b, page)].long()
        for h in range(hkv):
            k = s["k"][pages, h].reshape(-1, dim)[:a + b].to(f64)
            v = s["v"][pages, h].reshape(-1, dim)[:a + b].to(f64)
            for i in range(0, b, 512):                     # 512 queries at a time
                m = min(512, b - i)
                p = torch.arange(a + i, a + i + m, device="cuda")[:, None]
                j = torch.arange(a + b, device="cuda")[None]
                hidden = j > p
                if case["window"]:
                    hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
                for x in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    z = (s["q"][at + i:at + i + m, x].to(f64) @ k.T.contiguous()) / math.sqrt(dim)
                    z[hidden] = -math.inf
                    out[at + i:at + i + m, x] = torch.softmax(z, -1) @ v
        at += b
    return out
