"""Plain restatements of the paged 8-bit cache's operators, request by request, in 64 bits."""

import math

import numpy as np
import torch

E4M3_MAX = 448.0


def page_step(tables, lengths, new, pages, ring, page, rows):
    """``iron_page_step`` as a loop over the requests (lists and numpy arrays, copies returned)."""
    tables, pages = tables.copy(), pages.copy()
    B, width = tables.shape
    P, head, count = len(pages), int(ring[0]), int(ring[1])
    row, needed, taken, refused = 0, 0, 0, 0
    slots, positions, starts, out, back = np.full(rows, -1), np.zeros(rows, int), [0], [], []
    for b in range(B):
        n, held = int(new[b]), -(-int(lengths[b]) // page)
        if n < 0:
            back += list(tables[b, :held])
            out.append(0)
            starts.append(row)
            continue
        want = -(-(int(lengths[b]) + n) // page)
        fits = want <= width and row + n <= rows
        needed += want - held if fits else 0
        if fits and (want == held or needed <= count):
            for j in range(held, want):
                tables[b, j] = pages[(head + taken) % P]
                taken += 1
            for i in range(n):
                t = int(lengths[b]) + i
                slots[row + i], positions[row + i] = tables[b, t // page] * page + t % page, t
            out.append(int(lengths[b]) + n)
        else:
            refused += 1
            out.append(int(lengths[b]))
        row += n
        starts.append(row)
    for j, p in enumerate(back):
        pages[(head + count + j) % P] = p
    return dict(tables=tables, pages=pages, slots=slots, positions=positions, row_start=np.array(starts),
                lengths=np.array(out), ring=np.array([(head + taken) % P, count - taken + len(back), refused, row]))


def e4m3(x):
    """f64 -> the nearest e4m3 value (ties to even), as f64; magnitudes past 448 do not come here."""
    y = np.abs(x)
    step = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    return np.where(np.isfinite(x), np.round(np.where(np.isfinite(x), x, 0) / step) * step, np.nan)


def scale_of(x):
    """The page scale of new values ``x``: the smallest power of two with max <= 448 times it, 2^-60 at least."""
    y = np.abs(x[np.isfinite(x)])
    top = y.max() if y.size else 0.0
    return 2.0 ** max(-60, math.ceil(math.log2(top / E4M3_MAX))) if top > 0 else 2.0 ** -60


def rotate(x, cs):
    """(heads, D) f32 by one (cos, sin) row, every product and sum rounded to f32."""
    h = x.shape[-1] // 2
    a, b, c, s = x[:, :h], x[:, h:], cs[0::2], cs[1::2]
    return np.concatenate((a * c - b * s, b * c + a * s), -1, dtype=np.float32)


def write(qkv, angles, pool, scales, slots, positions, H, G, D):
    """``iron_rope_kv_pages_e4m3``: (q f32, pool as f64 codes, scales f64); ``pool`` (P, G, 2, page, D) f64 codes."""
    pool, scales = pool.copy(), scales.astype(np.float64).copy()
    page = pool.shape[3]
    rows = len(slots)
    x = qkv.astype(np.float32).reshape(rows, H + 2 * G, D)
    q = np.empty((rows, H, D), np.float32)
    runs = []
    kv = np.empty((rows, G, 2, D), np.float32)
    for r in range(rows):
        cs = angles[min(max(int(positions[r]), 0), len(angles) - 1)].astype(np.float32)
        turned = rotate(x[r, :H + G], cs)
        q[r], kv[r, :, 0], kv[r, :, 1] = turned[:H], turned[H:], x[r, H + G:]
        s = int(slots[r])
        if s < 0 or s >= pool.shape[0] * page:
            continue
        if runs and runs[-1][0] + runs[-1][1] == r and s % page and int(slots[r - 1]) == s - 1:
            runs[-1][1] += 1
        else:
            runs.append([r, 1])
    for r, n in runs:
        p, off = int(slots[r]) // page, int(slots[r]) % page
        for g in range(G):
            for k in range(2):
                new = kv[r:r + n, g, k].astype(np.float64)
                s = scale_of(new)
                if off:
                    s = max(s, scales[p, g, k])
                    pool[p, g, k, :off] = e4m3(pool[p, g, k, :off] * (scales[p, g, k] / s))
                scales[p, g, k] = s
                pool[p, g, k, off:off + n] = e4m3(new / s)
    return q, pool, scales


def attention(q, pool, scales, tables, lengths, row_start, causal=True, window=None, scale=None):
    """(out, weight): attention in f64 and sum(p |v|) / sum(p), the size that a rounding of p multiplies.

    All tensors on one device; pages outside the pool count as absent."""
    rows, H, D = q.shape
    P, G, _, page, _ = pool.shape
    out = torch.zeros((rows, H, D), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b in range(len(lengths)):
        n, r0, r1 = int(lengths[b]), int(row_start[b]), int(row_start[b + 1])
        if r1 <= r0 or n <= 0:
            continue
        ids = tables[b, :-(-n // page)].long()
        there = (ids >= 0) & (ids < P)
        ids = ids.clamp(0, P - 1)
        kv = pool[ids].double() * scales[ids].double()[..., None, None]
        kv = kv.permute(2, 1, 0, 3, 4).reshape(2, G, -1, D)[:, :, :n]
        pos = torch.arange(n - (r1 - r0), n, device=q.device)[:, None]
        key = torch.arange(n, device=q.device)[None, :]
        seen = there.repeat_interleave(page)[:n][None, :] & ((key <= pos) if causal else (key >= 0))
        if window is not None:
            seen = seen & (key >= pos - window)
        for h in range(H):
            k, v = kv[0, h * G // H], kv[1, h * G // H]
            s = (q[r0:r1, h].double() @ k.T) * scale
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            bad = torch.isnan(v)
            o = p @ torch.where(bad, 0.0, v)
            hit = seen.double() @ bad.double() > 0            # a NaN reaches the rows that see it
            out[r0:r1, h] = torch.where(hit, math.nan, o)
            size[r0:r1, h] = p @ torch.where(bad, 0.0, v).abs()
    return out, size


def cache(pages, G, page, D, seed, device="cuda", spread=4):
    """A random cache: codes of every size, a power-of-two scale a page, head and kind."""
    g = torch.Generator(device=device).manual_seed(seed)
    pool = (torch.randn((pages, G, 2, page, D), generator=g, device=device) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = torch.randint(-7 - spread // 2, -7 + spread - spread // 2, (pages, G, 2), generator=g, device=device)
    return pool, torch.exp2(e.float())


def tables_for(lengths, page, seed, width=0, spare=2):
    """Shuffled block tables for ``lengths``: (int32 numpy (B, width), pages of the pool)."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    ids = np.random.RandomState(seed).permutation(total).astype(np.int32)
    tables = np.full((len(lengths), max(width, max(need, default=0), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at:at + n]
        at += n
    return tables, total
