"""The paged 8-bit key/value cache's operators, measured: plain forms in torch and the framework's calls.

Four operators serve a batch of requests from a cache in pages.  ``page_step`` gives requests
pages and says where their new rows go; ``rope_kv_pages`` rotates a step's q and k and writes k
and v into the pages as e4m3 codes under one power-of-two scale a (page, KV head, key or value);
``mha_decode_pages`` is one query a request over its pages; ``mha_prefill_pages`` is the ragged
rows of prompt chunks over them.

The layout both sides share: ``pool`` (pages, G, 2, page, D) e4m3 holds keys [.., 0, ..] and
values [.., 1, ..]; ``scales`` (pages, G, 2) float32; a cached value is its code times its scale.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BF16, F8, F32, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of a serving batch: every request one token further, some cross into a new page
        dict(name="pages: decode step, 64 requests", op="step", B=64, page=64, max_pages=128, rows=64, ended=0.0,
             lo=1, hi=8000, new_lo=1, new_hi=1),
        # a step of a large batch that mixes decode rows, prompt chunks and requests that ended
        dict(name="pages: mixed step, 509 requests", op="step", B=509, page=16, max_pages=1024, rows=16384, ended=0.1,
             lo=1, hi=12000, new_lo=1, new_hi=150),
        # one token for each of 64 sequences, the decode batch of this repository's benchmark
        dict(name="write: 64 tokens, D 64", op="write", B=64, page=16, H=40, G=8, D=64, lo=1, hi=2047, new_lo=1, new_hi=1),
        # one prompt chunk of 2048 tokens that starts inside a page
        dict(name="write: prompt of 2048, D 128", op="write", B=1, page=64, H=32, G=8, D=128, lo=37, hi=37,
             new_lo=2048, new_hi=2048),
        # prompts and decode rows of one step
        dict(name="write: 6111 ragged rows", op="write", B=48, page=32, H=32, G=4, D=128, lo=1, hi=5000,
             new_lo=1, new_hi=813),
        # a single short conversation: latency
        dict(name="decode: 1 x 500, D 64", op="decode", B=1, page=16, H=32, G=8, D=64, lo=500, hi=500, window=-1),
        # the decode batch of this repository's benchmark: 64 sequences of context 2048
        dict(name="decode: 64 x 2048, D 64", op="decode", B=64, page=64, H=32, G=8, D=64, lo=2048, hi=2048, window=-1),
        # one long document: the keys have to be split over the machine
        dict(name="decode: 1 x 120001, D 128", op="decode", B=1, page=64, H=32, G=8, D=128, lo=120001, hi=120001,
             window=-1),
        # a ragged serving batch, a few tokens to thousands
        dict(name="decode: 128 x 3..8191, D 128", op="decode", B=128, page=32, H=32, G=4, D=128, lo=3, hi=8191,
             window=-1),
        # a prompt's first chunk, the benchmark's prompt of 2048 tokens
        dict(name="prompt: 1 x 2048, D 64", op="prompt", B=1, page=64, H=32, G=8, D=64, lo=2048, hi=2048,
             new_lo=2048, new_hi=2048, window=-1, causal=True),
        # a few tokens for each sequence (a draft to verify): latency and cache bytes
        dict(name="prompt: 16 x 7 on 4096, D 128", op="prompt", B=16, page=64, H=32, G=8, D=128, lo=4096, hi=4096,
             new_lo=7, new_hi=7, window=-1, causal=True),
        # ragged chunks on contexts of other lengths
        dict(name="prompt: 8 ragged chunks, D 128", op="prompt", B=8, page=32, H=32, G=8, D=128, lo=900, hi=9001,
             new_lo=61, new_hi=1433, window=-1, causal=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["step", "write", "decode", "decode", "prompt", "prompt"])
    page = rng.choice([16, 32, 64, 128])
    if op == "step":
        B = _log(rng, 1, 509)
        hi = _log(rng, 16, 12000)
        new_hi = rng.choice([1, _log(rng, 2, 400)])
        rows = B * new_hi if rng.random() < 0.7 else max(1, B * new_hi // 3)   # sometimes too few rows for everyone
        return dict(op=op, B=B, page=page, max_pages=max(1, (hi + new_hi) // page + rng.randint(0, 2)),
                    rows=min(rows, 16384), ended=rng.choice([0.0, 0.1, 0.3]), lo=1, hi=hi, new_lo=1, new_hi=new_hi)
    D = rng.choice([64, 128])
    G = rng.choice([1, 2, 3, 4, 8])
    H = G * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    H = H if H <= 64 else G * 4
    if op == "write":
        new_hi = rng.choice([1, _log(rng, 2, 800)])
        B = _log(rng, 1, max(1, min(256, 7000 // new_hi)))
        return dict(op=op, B=B, page=page, H=H, G=G, D=D, lo=1, hi=_log(rng, 2, 5000), new_lo=1, new_hi=new_hi)
    window = rng.choice([-1, -1, -1, _log(rng, 1, 2000)])
    if op == "decode":
        hi = _log(rng, 2, 60000)
        B = _log(rng, 1, max(1, min(256, 250000 // hi)))
        return dict(op=op, B=B, page=page, H=H, G=G, D=D, lo=rng.choice([1, hi]), hi=hi, window=window)
    hi = _log(rng, 2, 9000)
    new_hi = _log(rng, 1, min(hi, 1400))
    B = _log(rng, 1, max(1, min(64, 12000000 * 8 // (hi * new_hi * max(H, 8)))))
    return dict(op=op, B=B, page=page, H=H, G=G, D=D, lo=max(new_hi, hi // rng.choice([1, 5])), hi=hi,
                new_lo=rng.choice([1, new_hi]), new_hi=new_hi, window=window,
                causal=True if window >= 0 else rng.random() < 0.9)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced on a log scale."""
    if n == 1 or lo == hi:
        return [hi] * n
    return [max(lo, min(hi, int(round(lo * (hi / lo) ** (i / (n - 1)))))) for i in range(n)]


def _new(case):
    """Each request's new rows, paired with the lengths by a fixed stride so that long meets short."""
    n = _spread(case["new_lo"], case["new_hi"], case["B"])
    step = next(s for s in (7, 11, 13, 17, 19, 23) if case["B"] % s)
    return [n[(i * step + 3) % case["B"]] for i in range(case["B"])]


def _step_lists(case):
    """(lengths, new tokens) of a page_step case; -1 ends a request."""
    lengths, new = _spread(case["lo"], case["hi"], case["B"]), _new(case)
    every = round(1 / case["ended"]) if case["ended"] else 0
    return lengths, [-1 if every and i % every == every - 1 else n for i, n in enumerate(new)]


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prefix(counts):
    return [0] + [int(x) for x in np.cumsum(counts)]


def _pages_for(lengths, page, seed, spare=3):
    """Block tables over a shuffled pool: (tables, number of pages)."""
    need = [-(-n // page) for n in lengths]
    total, width = sum(need) + spare, max(1, max(need))
    order = np.random.RandomState(seed % (1 << 31)).permutation(total).astype(np.int32)
    tables = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(tables).cuda(), total


def _pool(pages, G, page, D, seed):
    """A filled cache: normal keys and values of each head's own size, page by page under a scale."""
    g = _gen(seed)
    size = torch.rand((1, G, 2, 1, 1), generator=g, device="cuda") * 1.5 + 0.5
    pool = torch.empty((pages, G, 2, page, D), dtype=F8, device="cuda")
    scales = torch.empty((pages, G, 2), dtype=F32, device="cuda")
    step = max(1, (1 << 27) // (G * 2 * page * D))
    for lo in range(0, pages, step):
        x = torch.randn((min(step, pages - lo), G, 2, page, D), generator=g, device="cuda") * size
        s = _scale_of(x.abs().amax((-1, -2)))
        pool[lo:lo + step] = (x / s[..., None, None]).to(F8)
        scales[lo:lo + step] = s
    return pool, scales


def prepare(case, seed):
    B, page = case["B"], case["page"]
    rs = np.random.RandomState(seed % (1 << 31))
    order = rs.permutation(B)
    g = _gen(seed + 1)
    s = dict(case, seed=seed)
    if case["op"] == "step":
        lengths, new = _step_lists(case)
        lengths, new = [lengths[i] for i in order], [new[i] for i in order]
        # what earlier steps left: every request holds the pages of its tokens
        lengths = [min(n, case["max_pages"] * page) for n in lengths]
        held = [-(-n // page) for n in lengths]
        total = sum(held) + sum(-(-max(n, 0) // page) + 1 for n in new)
        ids = rs.permutation(total).astype(np.int32)
        tables = np.full((B, case["max_pages"]), -1, np.int32)
        for b, at in enumerate(_prefix(held)[:-1]):
            tables[b, :held[b]] = ids[at:at + held[b]]
        free = ids[sum(held):]
        head = int(rs.randint(total))
        ring = np.full(total, -1, np.int32)
        ring[(head + np.arange(len(free))) % total] = free
        s.update(lengths=_ints(lengths), new=_ints(new), tables=torch.from_numpy(tables).cuda(),
                 pages=torch.from_numpy(ring).cuda(), ring=_ints([head, len(free), 0, 0]))
        return s
    if case["op"] == "write":
        before, new = _spread(case["lo"], case["hi"], B), _new(case)
        before, new = [before[i] for i in order], [new[i] for i in order]
        # the pool is the pages that the step writes; the earlier pages do not take part
        first = [n // page for n in before]
        count = [-(-(n + m) // page) - f for n, m, f in zip(before, new, first)]
        ids = rs.permutation(sum(count))
        slots, positions = [], []
        for b, at in enumerate(_prefix(count)[:-1]):
            t = np.arange(before[b], before[b] + new[b])
            slots.append(ids[at + t // page - first[b]] * page + t % page)
            positions.append(t)
        H, G, D = case["H"], case["G"], case["D"]
        rows, S = sum(new), case["hi"] + case["new_hi"] + 1
        s["pool"], s["scales"] = _pool(sum(count), G, page, D, seed + 2)
        # only a request's last page of earlier steps holds anything, up to where the step goes on
        held = np.zeros(sum(count), np.int64)
        held[ids[_prefix(count)[:-1]]] = [n % page for n in before]
        empty = torch.arange(page, device="cuda")[None, :] >= torch.from_numpy(held).cuda()[:, None]
        s["pool"].view(torch.uint8).masked_fill_(empty[:, None, None, :, None], 0)
        s["qkv"] = torch.randn((rows, (H + 2 * G) * D), generator=g, device="cuda").mul_(1.3).to(BF16)
        # the angle table of a decoder: (cos, sin) pairs, position by position
        t = torch.arange(S, device="cuda", dtype=F64)[:, None]
        a = t * 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=F64) / D)
        s["angles"] = torch.stack((a.cos(), a.sin()), -1).reshape(S, D).to(BF16)
        s["slots"], s["positions"] = _ints(np.concatenate(slots)), _ints(np.concatenate(positions))
        s["q"] = torch.empty((rows, H, D), dtype=BF16, device="cuda")
        return s
    lengths = [_spread(case["lo"], case["hi"], B)[i] for i in order]
    s["tables"], total = _pages_for(lengths, page, seed)
    s["pool"], s["scales"] = _pool(total, case["G"], page, case["D"], seed + 2)
    s["lengths"] = _ints(lengths)
    rows = B
    if case["op"] == "prompt":
        new = [min(_new(case)[i], n) for i, n in zip(order, lengths)]
        rows = sum(new)
        s["row_start"] = _ints(_prefix(new))
    s["q"] = torch.randn((rows, case["H"], case["D"]), generator=g, device="cuda").mul_(1.3).to(BF16)
    s["out"] = torch.empty_like(s["q"])
    return s


# ---------------------------------------------------------------------------- plain forms
def _scale_of(amax):
    """2^e, e the smallest whole number with amax <= 448 * 2^e (448 = 0.875 * 2^9); 2^-60 at least."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -60)).clamp(min=-60))


def _values(pool, scales):
    """The cached values (exact in bf16: four significant bits and a power of two)."""
    return pool.to(BF16) * scales.to(BF16)[..., None, None]


def _plain_step(s):
    page, rows = s["page"], s["rows"]
    tables, lengths, new, pages, ring = s["tables"], s["lengths"].long(), s["new"].long(), s["pages"], s["ring"]
    B, width, P = tables.shape[0], tables.shape[1], pages.numel()
    dev = tables.device
    head, count = ring[0].long(), ring[1].long()
    ended, n = new < 0, new.clamp(min=0)
    row_end = n.cumsum(0)
    held = (lengths + page - 1) // page
    want = (lengths + n + page - 1) // page
    fits = ~ended & (want <= width) & (row_end <= rows)
    need = torch.where(fits, want - held, 0)
    taken_end = need.cumsum(0)
    served = fits & ((need == 0) | (taken_end <= count))
    need = torch.where(served, need, 0)
    first = taken_end - torch.where(fits, want - held, 0)      # where a served request's pages begin
    used = need.sum()
    j = torch.arange(width, device=dev)
    k = j[None, :] - held[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    tables_out = torch.where(fresh, pages[(head + first[:, None] + k) % P], tables)
    back = torch.where(ended, held, 0)
    back_first = back.cumsum(0) - back
    giving = ended[:, None] & (j[None, :] < held[:, None])
    at = torch.where(giving, (head + count + back_first[:, None] + j[None, :]) % P, P)
    pages_out = torch.cat((pages, pages[:1])).scatter(0, at.reshape(-1), tables.reshape(-1))[:P]
    lengths_out = torch.where(ended, 0, torch.where(served, lengths + n, lengths))
    ring_out = torch.stack(((head + used) % P, count - used + back.sum(), (~ended & ~served).sum(), row_end[-1]))
    r = torch.arange(rows, device=dev)
    b = torch.searchsorted(row_end, r, right=True).clamp(max=B - 1)
    position = lengths[b] + r - (row_end[b] - n[b])
    live = (r < row_end[-1]) & served[b]
    entry = tables_out[b, torch.where(live, position // page, 0)].long()
    slots = torch.where(live, entry * page + position % page, -1)
    row_start = torch.cat((torch.zeros(1, dtype=torch.int64, device=dev), row_end))
    small = [x.int() for x in (slots, torch.where(live, position, 0), row_start, lengths_out, ring_out)]
    return dict(zip(("slots", "positions", "row_start", "lengths", "ring"), small), tables=tables_out, pages=pages_out)


def _rotated(x, cs):
    """x (rows, heads, D) with its halves turned by the (cos, sin) rows."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, n = cs[:, None, 0::2], cs[:, None, 1::2]
    return torch.cat((a * c - b * n, b * c + a * n), -1)


def _plain_write(s):
    H, G, D, page = s["H"], s["G"], s["D"], s["page"]
    rows = s["qkv"].shape[0]
    x = s["qkv"].float().reshape(rows, H + 2 * G, D)
    cs = s["angles"].float()[s["positions"].long()]
    turned = _rotated(x[:, :H + G], cs)
    q = turned[:, :H].to(BF16)
    kv = torch.stack((turned[:, H:], x[:, H + G:]), 2)                      # (rows, G, 2, D)
    slot = s["slots"].long()
    at, off = slot // page, slot % page
    P = s["pool"].shape[0]
    index = at[:, None, None].expand(rows, G, 2)
    amax = torch.zeros((P, G, 2), device=x.device).scatter_reduce(0, index, kv.abs().amax(-1), "amax")
    low = torch.full((P,), page, device=x.device, dtype=torch.int64).scatter_reduce(0, at, off, "amin")
    # a page that starts in this step takes its own scale; one that goes on keeps the larger
    scale = _scale_of(amax)
    scale = torch.where((low == 0)[:, None, None], scale, torch.maximum(scale, s["scales"]))
    scale = torch.where((low < page)[:, None, None], scale, s["scales"])
    held = torch.arange(page, device=x.device)[None, :] < low[:, None]
    kept = (s["pool"].float() * (s["scales"] / scale)[..., None, None]).to(F8)
    pool = torch.where(held[:, None, None, :, None], kept.view(torch.uint8), s["pool"].view(torch.uint8))
    pool[at, :, :, off] = (kv / scale[at][..., None]).to(F8).view(torch.uint8)
    return dict(q=q, kv=_values(pool.view(F8), scale), scales=scale)


def _gathered(s):
    """Keys and values of every request in order, f32, padded: (B, G, S, D) twice; zeros past the length."""
    tables, page = s["tables"].long().clamp(min=0), s["page"]
    B, width = tables.shape
    x = s["pool"][tables].float() * s["scales"][tables][..., None, None]     # (B, width, G, 2, page, D)
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, B, s["G"], width * page, s["D"])
    live = torch.arange(width * page, device=x.device)[None, :] < s["lengths"][:, None]
    return torch.where(live[None, :, None, :, None], x, 0.0), live


def _softmax_product(scores, seen, v):
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total > 0, total, 1.0)


def _plain_decode(s):
    H, G, D = s["H"], s["G"], s["D"]
    (k, v), live = _gathered(s)
    B, S = live.shape
    q = s["q"].float().reshape(B, G, H // G, D)
    if s["window"] >= 0:
        live = live & (torch.arange(S, device=live.device)[None, :] >= s["lengths"][:, None] - 1 - s["window"])
    scores = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    return _softmax_product(scores, live[:, None, None, :], v).reshape(B, H, D).to(BF16)


def _plain_prompt(s):
    H, G, D = s["H"], s["G"], s["D"]
    (k, v), live = _gathered(s)
    B, S = live.shape
    rows = s["q"].shape[0]
    start = s["row_start"].long()
    n = start[1:] - start[:-1]
    r = torch.arange(rows, device=live.device)
    b = torch.searchsorted(start[1:], r, right=True)
    i = r - start[b]
    N = s["new_hi"]
    q = torch.zeros((B, N, H, D), device=live.device)
    q[b, i] = s["q"].float()
    q = q.reshape(B, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, (H // G) * N, D)
    key = torch.arange(S, device=live.device)[None, None, :]
    position = (s["lengths"].long() - n)[:, None, None] + torch.arange(N, device=live.device)[None, :, None]
    seen = live[:, None, :] & ((key <= position) if s["causal"] else torch.ones_like(key <= position))
    if s["window"] >= 0:
        seen = seen & (key >= position - s["window"])
    seen = seen[:, None, None].expand(B, 1, H // G, N, S).reshape(B, 1, (H // G) * N, S)
    out = _softmax_product((q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D)), seen, v)
    out = out.reshape(B, G, H // G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)
    return out[b, i].to(BF16)


# ---------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if not own:
        return dict(step=_plain_step, write=_plain_write, decode=_plain_decode, prompt=_plain_prompt)[op](s)
    from iron_b200 import kernels as K

    window = None if s.get("window", -1) < 0 else s["window"]
    if op == "step":
        # the new lengths and ring go to buffers of their own, so the same step can be taken again
        got = K.page_step(s["tables"], s["lengths"], s["new"], s["pages"], s["ring"], page_size=s["page"], rows=s["rows"])
        return dict(zip(("slots", "positions", "row_start", "lengths", "ring"), got), tables=s["tables"], pages=s["pages"])
    if op == "write":
        K.rope_kv_pages(s["qkv"], s["angles"], s["q"], s["pool"], s["scales"], s["slots"], s["positions"],
                        H=s["H"], G=s["G"], D=s["D"])
        return dict(q=s["q"], kv=_values(s["pool"], s["scales"]), scales=s["scales"])
    if op == "decode":
        return K.mha_decode_pages(s["q"], s["pool"], s["scales"], s["tables"], s["lengths"], s["out"], window=window)
    return K.mha_prefill_pages(s["q"], s["pool"], s["scales"], s["tables"], s["lengths"], s["row_start"], s["out"],
                               causal=s["causal"], window=window)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    B, page = case["B"], case["page"]
    if case["op"] == "step":
        lengths, new = _step_lists(case)
        lengths = [min(n, case["max_pages"] * page) for n in lengths]
        rows = min(case["rows"], sum(max(n, 0) for n in new))
        taken = sum(-(-(a + n) // page) - -(-a // page) for a, n in zip(lengths, new) if n > 0)
        back = sum(-(-a // page) for a, n in zip(lengths, new) if n < 0)
        # lengths, new and row starts; a table entry and its ring entry for each page; slot and position of each row
        return dict(bytes=4 * (4 * B + 1) + 8 * (taken + back) + 8 * rows + 32, flops=8.0 * B + 4.0 * rows)
    H, G, D = case["H"], case["G"], case["D"]
    if case["op"] == "write":
        rows = sum(_new(case))
        pages = sum(-(-(a + n) // page) - a // page for a, n in zip(_spread(case["lo"], case["hi"], B), _new(case)))
        # q, k, v rows in, q out in bf16, k and v out in 8 bits, angles, slots and positions, scales
        return dict(bytes=rows * (2 * (H + 2 * G) * D + 2 * H * D + 2 * G * D + 2 * D + 8) + 8 * G * pages,
                    flops=rows * (3.0 * (H + G) * D + 4.0 * G * D))
    lengths = _spread(case["lo"], case["hi"], B)
    w = case["window"]
    if case["op"] == "decode":
        keys = sum(n if w < 0 else min(n, w + 1) for n in lengths)
        rows, pairs, read = B, keys, keys
    else:
        new = [min(m, n) for m, n in zip(_new(case), lengths)]
        rows = sum(new)
        pairs = read = 0
        for n, m in zip(lengths, new):
            position = np.arange(n - m, n)
            lo = np.maximum(position - w, 0) if w >= 0 else np.zeros(m, np.int64)
            hi = position if case["causal"] else np.full(m, n - 1)
            pairs += int((hi - lo + 1).sum())
            read += n - int(lo[0])
    # keys and values in 8 bits, a pair of scales a page and head, table entries, q in and out
    return dict(bytes=read * G * 2 * D + (-(-read // page)) * (8 * G + 4) + 4 * rows * H * D,
                flops=4.0 * H * D * pairs)


# ---------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    if case["op"] == "step":
        return None   # whole numbers
    s = prepare(case, seed)
    H, G, D, page = s["H"], s["G"], s["D"], s["page"]
    if case["op"] == "write":
        x = s["qkv"].double().reshape(-1, H + 2 * G, D)
        table = s["angles"].double()[s["positions"].long()]
        z = torch.complex(x[:, :H + G, :D // 2], x[:, :H + G, D // 2:]) * torch.complex(table[:, 0::2], table[:, 1::2])[:, None]
        turned = torch.cat((z.real, z.imag), -1)
        kv = torch.stack((turned[:, H:], x[:, H + G:]), 2)
        old = s["pool"].double() * s["scales"].double()[..., None, None]
        scales = s["scales"].double().clone()
        slot = s["slots"].long()
        order = torch.argsort(slot)
        pages, counts = torch.unique_consecutive(slot[order] // page, return_counts=True)
        for p, idx in zip(pages.tolist(), torch.split(order, counts.tolist())):
            off = int(slot[idx[0]]) % page
            amax = kv[idx].abs().amax((0, -1))
            e = torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(min=-60)
            new = torch.exp2(e)
            if off:
                new = torch.maximum(new, scales[p])
            scales[p] = new
            old[p, :, :, :off] = _e4m3(old[p, :, :, :off], new)
            old[p, :, :, off:off + len(idx)] = _e4m3(kv[idx].permute(1, 2, 0, 3), new)
        return dict(q=turned[:, :H], kv=old, scales=scales)
    lengths = s["lengths"].tolist()
    start = s["row_start"].tolist() if case["op"] == "prompt" else list(range(case["B"] + 1))
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for b, n in enumerate(lengths):
        m = start[b + 1] - start[b]
        if not m or not n:
            continue
        ids = s["tables"][b, :-(-n // page)].long()
        kv = s["pool"][ids].double() * s["scales"][ids].double()[..., None, None]
        kv = kv.permute(2, 1, 0, 3, 4).reshape(2, G, -1, D)[:, :, :n]
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        seen = (key <= pos) if case.get("causal", True) else (key <= n)
        if case["window"] >= 0:
            seen = seen & (key >= pos - case["window"])
        for h in range(H):
            z = s["q"][start[b]:start[b + 1], h].double() @ kv[0, h * G // H].T / math.sqrt(D)
            out[start[b]:start[b + 1], h] = torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ kv[1, h * G // H]
    return out


def _e4m3(x, scale):
    """x rounded to the nearest e4m3 multiple of ``scale`` ((G, 2), ties to even), as the value it stands for."""
    scale = scale[:, :, None, None]
    y = (x / scale).clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale
