"""The paged 8-bit cache on a B200: every operator against its plain form, and a run of them together."""

import math

import numpy as np
import pytest
import torch

from tests import pages_ref as R
from tests.util import to_numpy

pytestmark = pytest.mark.gpu

BF16, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=I32).cuda()


# ---------------------------------------------------------------------------- page_step
def step_inputs(B, width, page, seed, free, ended, new_hi, full=False):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, width * page + 1, B) if full else rng.integers(0, max(1, width * page - new_hi), B)
    new = np.where(rng.random(B) < ended, -1, rng.integers(0, new_hi + 1, B))
    held = -(-lengths // page)
    P = int(held.sum()) + free + 3
    ids = rng.permutation(P)
    tables = np.full((B, width), -1)
    at = 0
    for b in range(B):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    head = int(rng.integers(P))
    pages = np.full(P, -1)
    pages[(head + np.arange(free)) % P] = ids[at:at + free]
    return tables, lengths, new, pages, np.array([head, free, 0, 0])


def check_step(got, tables, pages, want):
    slots, positions, row_start, lengths, ring = (t.cpu().numpy() for t in got)
    for name, x in dict(slots=slots, positions=positions, row_start=row_start, lengths=lengths, ring=ring,
                        tables=tables.cpu().numpy(), pages=pages.cpu().numpy()).items():
        assert np.array_equal(x, want[name]), name


@pytest.mark.parametrize("B, width, page, free, ended, new_hi, rows", [
    (1, 1, 16, 1, 0.0, 1, 1),
    (3, 4, 16, 0, 0.3, 5, 20),               # nothing free
    (64, 9, 64, 200, 0.1, 3, 128),
    (65, 33, 16, 7, 0.2, 30, 2000),          # the ring runs out
    (300, 17, 32, 900, 0.1, 90, 4000),       # the rows run out (and the cluster form)
    (1025, 5, 128, 1500, 0.1, 2, 1500),      # more than one round of requests
    (2500, 3, 256, 100, 0.5, 600, 100000),
])
@pytest.mark.parametrize("full", [False, True], ids=["room", "full tables"])
def test_page_step(B, width, page, free, ended, new_hi, rows, full):
    from iron_b200 import kernels as K

    tables, lengths, new, pages, ring = step_inputs(B, width, page, B + page, free, ended, new_hi, full)
    want = R.page_step(tables, lengths, new, pages, ring, page, rows)
    t, l, n, p, r = map(ints, (tables, lengths, new, pages, ring))
    got = K.page_step(t, l, n, p, r, page_size=page, rows=rows)
    check_step(got, t, p, want)
    assert np.array_equal(l.cpu().numpy(), lengths) and np.array_equal(r.cpu().numpy(), ring)
    # in place
    t, p = ints(tables), ints(pages)
    got = K.page_step(t, l, n, p, r, page_size=page, rows=rows, lengths_out=l, ring_out=r)
    assert got[3] is l and got[4] is r
    check_step(got, t, p, want)


def test_page_step_without_requests_or_rows():
    from iron_b200 import kernels as K

    pages, ring = ints(np.arange(5)), ints([3, 2, 9, 9])
    slots, _, row_start, _, out = K.page_step(ints(np.zeros((0, 4))), ints([]), ints([]), pages, ring, page_size=16, rows=3)
    assert slots.tolist() == [-1, -1, -1] and row_start.tolist() == [0] and out.tolist() == [3, 2, 0, 0]
    # no room for rows: a request that brings none is served, one that brings some is not
    t = ints(np.full((2, 2), -1))
    _, _, row_start, lengths, out = K.page_step(t, ints([0, 0]), ints([0, 4]), pages, ring, page_size=16, rows=0)
    assert lengths.tolist() == [0, 0] and out.tolist() == [3, 2, 1, 4] and row_start.tolist() == [0, 0, 4]


def test_pages_are_never_held_twice():
    """Many steps in place: every page is free once or held once, and the tables say what the plain loop says."""
    from iron_b200 import kernels as K

    rng = np.random.default_rng(3)
    B, width, page, P, rows = 40, 12, 16, 150, 300
    tables, lengths, pages, ring = np.full((B, width), -1), np.zeros(B, int), np.arange(P), np.array([0, P, 0, 0])
    t, l, p, r = map(ints, (tables, lengths, pages, ring))
    for _ in range(60):
        new = np.where(rng.random(B) < 0.1, -1, rng.integers(0, 12, B))
        want = R.page_step(tables, lengths, new, pages, ring, page, rows)
        got = K.page_step(t, l, ints(new), p, r, page_size=page, rows=rows, lengths_out=l, ring_out=r)
        check_step(got, t, p, want)
        tables, lengths, pages, ring = want["tables"], want["lengths"], want["pages"], want["ring"]
        held = [x for b in range(B) for x in tables[b, :-(-lengths[b] // page)]]
        free = [pages[(ring[0] + i) % P] for i in range(ring[1])]
        assert sorted(held + free) == list(range(P))


def test_page_step_survives_a_ring_that_says_nonsense():
    """Counts and ids outside their ranges are wrong answers at most: everything stays inside its buffer."""
    from iron_b200 import kernels as K

    t, l, n, p = ints(np.full((3, 4), 77)), ints([5, 1 << 30, -4]), ints([100, -1, 20]), ints([-9, 1 << 30, 3])
    before = t.clone()
    got = K.page_step(t, l, n, p, ints([-7, 99, 0, 0]), page_size=16, rows=40)
    assert got[2].tolist() == [0, 100, 100, 120] and got[4][1].item() >= 0
    assert t.shape == before.shape and torch.cuda.synchronize() is None


def test_page_step_of_as_many_requests_as_it_takes():
    from iron_b200 import _lib
    from iron_b200 import kernels as K

    B, width, page, rows = _lib.load().iron_page_step_max_requests(), 7, 16, 30000
    tables, lengths, new, pages, ring = step_inputs(B, width, page, 1, 9000, 0.2, 6)
    want = R.page_step(tables, lengths, new, pages, ring, page, rows)
    t, l, n, p, r = map(ints, (tables, lengths, new, pages, ring))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):                          # a stream other than the one that made the inputs
        got = K.page_step(t, l, n, p, r, page_size=page, rows=rows, lengths_out=l, ring_out=r)
    stream.synchronize()
    check_step(got, t, p, want)


# ---------------------------------------------------------------------------- rope_kv_pages
def write_case(H, G, D, page, before, new, seed, wild=False):
    """Requests with ``before`` tokens bring ``new`` rows; the pool holds the pages the step touches."""
    rng = np.random.default_rng(seed)
    first = [b // page for b in before]
    count = [-(-(b + n) // page) - f for b, n, f in zip(before, new, first)]
    P = sum(count) + 2
    ids = rng.permutation(P)
    slots, positions, at = [], [], 0
    for b, n, f, c in zip(before, new, first, count):
        t = np.arange(b, b + n)
        slots += list(ids[at + t // page - f] * page + t % page)
        positions += list(t)
        at += c
    rows = len(slots)
    qkv = rng.standard_normal((rows, (H + 2 * G) * D)).astype(np.float32)
    qkv *= np.exp2(rng.integers(-6, 7, (rows, 1)))          # scales that grow from step to step
    if wild and rows:
        flat = qkv.reshape(-1)
        flat[rng.integers(0, flat.size, 40)] = rng.choice([np.inf, -np.inf, np.nan, 3e38, 1e-40, 0.0], 40)
        qkv[rows // 2, H * D:] = 0
    S = max(positions, default=0) + 3
    a = np.arange(S)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    angles = np.stack((np.cos(a), np.sin(a)), -1).reshape(S, D)
    qkv, angles = (torch.from_numpy(x.astype(np.float32)).to(BF16) for x in (qkv, angles))
    pool, scales = R.cache(P, G, page, D, seed, device="cpu")
    return qkv, angles, pool, scales, np.array(slots, int), np.array(positions, int)


def check_write(q_out, pool, scales, want):
    q, codes, sc = want
    assert torch.equal(q_out.cpu().view(torch.int16), torch.from_numpy(q).to(BF16).view(torch.int16)) or np.array_equal(
        q_out.cpu().float().numpy(), torch.from_numpy(q).to(BF16).float().numpy(), equal_nan=True)
    assert np.array_equal(scales.cpu().double().numpy(), sc)
    assert np.array_equal(pool.cpu().double().numpy(), codes, equal_nan=True)


@pytest.mark.parametrize("H, G, D, page, before, new", [
    (1, 1, 64, 16, [0], [1]),
    (4, 2, 64, 16, [15, 0, 31, 7], [1, 1, 1, 1]),
    (8, 8, 128, 16, [3], [50]),
    (5, 1, 128, 32, [0, 31, 5, 100], [40, 2, 9, 8]),           # runs of eight and nine rows
    (6, 3, 64, 64, [70, 1, 0], [200, 64, 63]),
    (12, 4, 128, 128, [100, 127], [29, 130]),
    (2, 2, 64, 256, [17], [600]),
])
@pytest.mark.parametrize("wild", [False, True], ids=["normal", "with infinities and NaN"])
def test_rope_kv_pages(H, G, D, page, before, new, wild):
    from iron_b200 import kernels as K

    qkv, angles, pool, scales, slots, positions = write_case(H, G, D, page, before, new, page + H, wild)
    with np.errstate(all="ignore"):
        want = R.write(qkv.float().numpy(), angles.float().numpy(), pool.double().numpy(), scales.numpy(), slots, positions, H, G, D)
    pool, scales = pool.cuda(), scales.cuda()
    q = torch.full((len(slots), H, D), 7.0, dtype=BF16, device="cuda")
    assert K.rope_kv_pages(qkv.cuda(), angles.cuda(), q, pool, scales, ints(slots), ints(positions), H=H, G=G, D=D) is q
    check_write(q, pool, scales, want)
    # the same step once more finds its own rows and scales there: nothing changes
    K.rope_kv_pages(qkv.cuda(), angles.cuda(), q, pool, scales, ints(slots), ints(positions), H=H, G=G, D=D)
    check_write(q, pool, scales, want)


def test_rows_without_a_slot_and_positions_past_the_table():
    from iron_b200 import kernels as K

    H, G, D, page = 4, 2, 64, 16
    qkv, angles, pool, scales, slots, positions = write_case(H, G, D, page, [14, 3, 0], [20, 5, 9], 5)
    slots[21:25] = [-1, 1 << 30, len(pool) * page, -7]          # rows of the second request
    slots[-3:] = -1
    positions[-1] = 10 ** 6                                      # clamped to the last angle row
    want = R.write(qkv.float().numpy(), angles.float().numpy(), pool.double().numpy(), scales.numpy(), slots, positions, H, G, D)
    pool, scales = pool.cuda(), scales.cuda()
    # rows farther apart than their width
    wide = torch.zeros((len(slots), (H + 2 * G) * D + 24), dtype=BF16, device="cuda")
    wide[:, :-24] = qkv.cuda()
    q = torch.empty((len(slots), H, D), dtype=BF16, device="cuda")
    K.rope_kv_pages(wide[:, :-24], angles.cuda(), q, pool, scales, ints(slots), ints(positions), H=H, G=G, D=D)
    check_write(q, pool, scales, want)


def test_a_page_filled_token_by_token_keeps_its_values():
    """Forty steps of one token whose size grows: every stored value stays within half a step of
    its last code, plus what each change of scale lost below the smallest code."""
    from iron_b200 import kernels as K

    G, D, page, n = 2, 64, 64, 40
    g = torch.Generator().manual_seed(1)
    x = torch.randn((n, 4 * G, D), generator=g) * torch.exp2(torch.arange(n) / 4 - 6)[:, None, None]
    qkv = x[:, : 3 * G].reshape(n, -1).to(BF16).cuda()
    angles = torch.zeros((64, D), dtype=BF16, device="cuda")
    angles[:, 0::2] = 1                                          # no rotation
    pool, scales = torch.zeros((1, G, 2, page, D), dtype=F8, device="cuda"), torch.ones((1, G, 2), device="cuda")
    q = torch.empty((1, G, D), dtype=BF16, device="cuda")
    for t in range(n):
        K.rope_kv_pages(qkv[t:t + 1], angles, q, pool, scales, ints([t]), ints([t]), H=G, G=G, D=D)
    want = qkv.double().reshape(n, 3 * G, D)[:, G:].reshape(n, 2, G, D).permute(2, 1, 0, 3)   # (G, 2, n, D)
    got = (pool.double() * scales.double()[..., None, None])[0, :, :, :n]
    # a normal code is off by half a step (2^-4); the smallest code is 2^-9 of the scale, and the halves of it lost
    # under every earlier scale (each at most half the next) sum to no more than one such step
    bound = want.abs() * 2.0 ** -4 + scales.double()[0, :, :, None, None] * 2.0 ** -9
    assert (got - want).abs().le(bound).all()


# ---------------------------------------------------------------------------- attention
def tolerance(want, size):
    """Half a bf16 step of the output, a half's half step for each probability (2^-11 of sum p |v| / sum p) twice
    over for the f32 exponentials, sums and scores, and the smallest bf16 numbers."""
    return want.abs() * 2.0 ** -8 + size * 2.0 ** -10 + 1e-30


def check_attention(out, want, size):
    out = out.double()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    ok = torch.isnan(want) | ((out - want).abs() <= tolerance(want, size))
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} beyond the bound, worst {float((out - want).abs().nan_to_num().max()):.3g}"


def queries(rows, H, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, H, D), generator=g, device="cuda") * torch.exp2(
        torch.randint(-3, 3, (rows, H, 1), generator=g, device="cuda").float())).to(BF16)


def poison(pool, scales, tables, lengths, page):
    """NaN codes wherever no request has a token."""
    used = torch.zeros(pool.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for t in range(0, n, page):
            used[int(tables[b, t // page]), : min(page, n - t)] = True
    pool.view(torch.uint8).masked_fill_(~used[:, None, None, :, None].cuda(), 0x7F)


@pytest.mark.parametrize("H, G, D", [(4, 4, 64), (8, 1, 64), (6, 2, 128), (32, 8, 64), (9, 1, 128), (16, 1, 128), (40, 2, 64), (7, 7, 128)])
@pytest.mark.parametrize("page, lengths", [
    (16, [1]), (64, [0, 1, 15, 16, 17, 64, 65]), (32, [700, 33, 0, 129]), (128, [3001]), (256, [255, 256, 257, 5])])
def test_decode(H, G, D, page, lengths):
    from iron_b200 import kernels as K

    tables, P = R.tables_for(lengths, page, H + page, width=14 if page == 256 else 0)
    pool, scales = R.cache(P, G, page, D, H * D + page)
    poison(pool, scales, tables, lengths, page)
    q = queries(len(lengths), H, D, 5)
    t, l = ints(tables), ints(lengths)
    for window in (None, 0, 40):
        out = K.mha_decode_pages(q, pool, scales, t, l, window=window)
        want, size = R.attention(q, pool, scales, t, lengths, range(len(lengths) + 1), window=window)
        check_attention(out, want, size)


def test_decode_many_short_and_a_few_long():
    """Segments of very different lengths over every CTA's share, and shares that cut them."""
    from iron_b200 import kernels as K

    lengths = [1, 20000, 5, 0, 333, 4097] + [17 * i % 500 for i in range(90)]
    H, G, D, page = 12, 4, 128, 32
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    q, t, l = queries(len(lengths), H, D, 3), ints(tables), ints(lengths)
    workspace = K.pages_workspace(D).fill_(0xFF)             # a workspace needs no clearing
    out = K.mha_decode_pages(q, pool, scales, t, l, scale=0.03, workspace=workspace)
    check_attention(out, *R.attention(q, pool, scales, t, lengths, range(len(lengths) + 1), scale=0.03))
    again = K.mha_decode_pages(q, pool, scales, t, l, scale=0.03, workspace=workspace)
    assert torch.equal(out, again)                           # the order of the sums is fixed


@pytest.mark.parametrize("H, G, D, page, lengths, new", [
    (4, 4, 64, 16, [1], [1]),
    (8, 2, 64, 64, [100, 7, 64, 0, 300], [5, 7, 1, 0, 130]),
    (6, 2, 128, 32, [257, 128, 129, 1], [128, 128, 129, 1]),
    (16, 1, 128, 128, [1500], [333]),
    (5, 5, 64, 16, [40, 700], [0, 650]),
    (24, 8, 128, 64, [513, 2, 77], [512, 2, 76]),
    (12, 1, 64, 256, [300, 900], [300, 11]),
    (3, 3, 128, 32, [1000], [1000]),
    (8, 2, 128, 64, [1000, 129, 2500, 128, 256, 257], [3, 1, 9, 32, 32, 33]),   # one half of an item's columns or fewer
    (32, 2, 64, 16, [4000, 130, 385], [8, 5, 9]),
])
@pytest.mark.parametrize("mask", ["causal", "window 0", "window 50", "all"])
def test_prefill(H, G, D, page, lengths, new, mask):
    from iron_b200 import kernels as K

    kw = dict(causal=mask != "all", window=int(mask.split()[1]) if " " in mask else None)
    tables, P = R.tables_for(lengths, page, H + page)
    pool, scales = R.cache(P, G, page, D, H * D + page)
    poison(pool, scales, tables, lengths, page)
    start = np.concatenate(([0], np.cumsum(new)))
    q = queries(int(start[-1]) + 3, H, D, 5)
    out = torch.full_like(q, 9.0)
    t, l = ints(tables), ints(lengths)
    assert K.mha_prefill_pages(q, pool, scales, t, l, ints(start), out, **kw) is out
    want, size = R.attention(q, pool, scales, t, lengths, start, **kw)
    n = int(start[-1])
    check_attention(out[:n], want[:n], size[:n])
    assert (out[n:] == 9).all()                              # rows of no request stay as they were


@pytest.mark.parametrize("D", [64, 128])
def test_more_rows_than_keys_and_rows_that_see_nothing(D):
    from iron_b200 import kernels as K

    lengths, start, page = [3, 0, 40], [0, 10, 14, 60], 16
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, 2, page, D, 3)
    q, t = queries(60, 4, D, 1), ints(tables)
    out = K.mha_prefill_pages(q, pool, scales, t, ints(lengths), ints(start))
    check_attention(out, *R.attention(q, pool, scales, t, lengths, start))
    assert (out[:7] == 0).all() and (out[10:14] == 0).all()
    out = K.mha_prefill_pages(q, pool, scales, t, ints(lengths), ints(start), causal=False)
    check_attention(out, *R.attention(q, pool, scales, t, lengths, start, causal=False))


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 30, 2**33, 80])
def test_a_window_wider_than_the_cache_is_none(window):
    """Rows before the first key and a window near the largest integer: no difference of the two wraps."""
    from iron_b200 import kernels as K

    lengths, start, page = [3, 40], [0, 50, 120], 16
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, 2, page, 64, 3)
    q, t, l = queries(120, 4, 64, 1), ints(tables), ints(lengths)
    check_attention(K.mha_prefill_pages(q, pool, scales, t, l, ints(start), window=window),
                    *R.attention(q, pool, scales, t, lengths, start))
    check_attention(K.mha_decode_pages(q[:2], pool, scales, t, l, window=window),
                    *R.attention(q[:2], pool, scales, t, lengths, range(3)))


@pytest.mark.parametrize("H, G, D", [(8, 2, 64), (10, 2, 128)])
def test_many_requests_most_of_which_bring_nothing(H, G, D):
    """Hundreds of requests: more than a CTA has threads, rows of some of them far apart, lengths past the table."""
    from iron_b200 import kernels as K

    rng = np.random.default_rng(4)
    B, page, width = 700, 16, 6
    lengths = np.where(rng.random(B) < 0.3, 0, rng.integers(1, width * page + 1, B))
    new = np.where(rng.random(B) < 0.9, 0, np.minimum(lengths, rng.integers(0, 90, B)))
    new[:200] = new[400:600] = 0
    tables, P = R.tables_for(lengths, page, 1, width=width)
    pool, scales = R.cache(P, G, page, D, 3)
    start, t = np.concatenate(([0], np.cumsum(new))), ints(tables)
    told = ints(np.where(lengths == width * page, lengths + 1000, lengths))
    q = queries(max(B, int(start[-1])), H, D, 1)
    n = int(start[-1])
    out = K.mha_prefill_pages(q[:n], pool, scales, t, told, ints(start))
    check_attention(out, *R.attention(q[:n], pool, scales, t, lengths, start))
    out = K.mha_decode_pages(q[:B], pool, scales, t, told)
    check_attention(out, *R.attention(q[:B], pool, scales, t, lengths, range(B + 1)))


@pytest.mark.parametrize("H, G, D, page", [(8, 2, 64, 16), (32, 2, 128, 64), (5, 5, 128, 32)])
@pytest.mark.parametrize("lengths, new", [
    ([700], [1]), ([0], [1]), ([5, 300, 1], [1, 1, 1]), ([0, 40, 1000, 17, 2000, 64], [1, 1, 300, 1, 0, 2]),
    ([100 + 7 * i for i in range(70)], [1 if i % 3 else 0 for i in range(70)]),
    ([3000] + [0] * 100 + [64, 4097], [1] + [0] * 100 + [64, 1])])
@pytest.mark.parametrize("kw", [dict(), dict(window=33), dict(causal=False)], ids=str)
def test_single_rows_among_others(H, G, D, page, lengths, new, kw):
    """A step of prompts' rows and of requests that bring one row each."""
    from iron_b200 import kernels as K

    tables, P = R.tables_for(lengths, page, 5)
    pool, scales = R.cache(P, G, page, D, 6)
    poison(pool, scales, tables, lengths, page)
    start = np.concatenate(([0], np.cumsum(new)))
    n = int(start[-1])
    for spare in (0, 2):
        q = queries(n + spare, H, D, 5)
        out = torch.full_like(q, 9.0)
        K.mha_prefill_pages(q, pool, scales, ints(tables), ints(lengths), ints(start), out, **kw)
        want, size = R.attention(q, pool, scales, ints(tables), lengths, start, **kw)
        check_attention(out[:n], want[:n], size[:n])
        assert (out[n:] == 9).all()


@pytest.mark.parametrize("prompt", [False, True])
def test_queries_that_are_not_finite(prompt):
    """An infinite or NaN query spoils its own row and head, and no other."""
    from iron_b200 import kernels as K

    n, page, G, H, D = 200, 16, 2, 8, 64
    tables, P = R.tables_for([n], page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    m = 150 if prompt else 1
    q, t, l = queries(m, H, D, 1), ints(tables), ints([n])
    want, size = R.attention(q, pool, scales, t, [n], [0, m])
    bad = q.clone()
    bad[0, 1, 3], bad[m - 1, 6, 0] = float("nan"), float("nan")
    out = K.mha_prefill_pages(bad, pool, scales, t, l, ints([0, m])) if prompt else K.mha_decode_pages(bad, pool, scales, t, l)
    want[0, 1], want[m - 1, 6] = float("nan"), float("nan")
    check_attention(out, want, size)


@pytest.mark.parametrize("D", [64, 128])
def test_nan_reaches_only_the_rows_that_see_it(D):
    """NaN keys and values of single tokens inside a chunk, where earlier rows share the tile."""
    from iron_b200 import kernels as K

    n, page, G, H = 300, 32, 2, 6
    tables, P = R.tables_for([n], page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    raw = pool.view(torch.uint8)
    for token, kind, d in ((150, 1, 5), (151, 1, 0), (260, 1, D - 1), (200, 0, 7), (299, 1, 33)):
        raw[int(tables[0, token // page]), token % G, kind, token % page, d] = 0xFF if token % 2 else 0x7F
    q, t, l = queries(n, H, D, 1), ints(tables), ints([n])
    for kw in (dict(), dict(window=30)):
        out = K.mha_prefill_pages(q, pool, scales, t, l, ints([0, n]), **kw)
        want, size = R.attention(q, pool, scales, t, [n], [0, n], **kw)
        assert torch.isnan(want).any() and not torch.isnan(want).all()
        check_attention(out, want, size)
    out = K.mha_decode_pages(q[-1:], pool, scales, t, l, window=30)
    check_attention(out, *R.attention(q[-1:], pool, scales, t, [n], [0, 1], window=30))


@pytest.mark.parametrize("D", [64, 128])
def test_pages_outside_the_pool_count_as_absent(D):
    from iron_b200 import kernels as K

    lengths, new, page = [500, 70, 200], [200, 3, 1], 16
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, 2, page, D, 3)
    tables[0, 3], tables[0, 20], tables[1, :5], tables[2, 4] = -1, P, 1 << 30, -5
    start, t, l = np.concatenate(([0], np.cumsum(new))), ints(tables), ints(lengths)
    q = queries(sum(new), 4, D, 1)
    out = K.mha_prefill_pages(q, pool, scales, t, l, ints(start))
    check_attention(out, *R.attention(q, pool, scales, t, lengths, start))
    out = K.mha_decode_pages(q[:3], pool, scales, t, l)
    check_attention(out, *R.attention(q[:3], pool, scales, t, lengths, range(4)))


@pytest.mark.parametrize("prompt", [False, True])
def test_scales_far_apart_and_scores_far_out(prompt):
    """Page scales from 2^-30 to 2^20 that are no powers of two, queries of 2^-20 and 2^20, one key that takes all."""
    from iron_b200 import kernels as K

    n, page, G, H, D = 600, 16, 2, 4, 64
    tables, P = R.tables_for([n, n], page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    g = torch.Generator(device="cuda").manual_seed(8)
    scales[..., 1] *= torch.exp2(torch.rand(scales.shape[:2], generator=g, device="cuda") * 50 - 30)
    scales[..., 0] *= 1.37
    m = 200 if prompt else 1
    q = queries(2 * m, H, D, 1)
    q[:m] *= 2.0 ** -20
    q[m:] *= 2.0 ** 5
    start, t, l = [0, m, 2 * m], ints(tables), ints([n, n])
    out = K.mha_prefill_pages(q, pool, scales, t, l, ints(start)) if prompt else K.mha_decode_pages(q, pool, scales, t, l)
    want, size = R.attention(q, pool, scales, t, [n, n], start)
    # scores of some thousands carry their f32 rounding (2^-24 each, of sums and of the product with log2 e) into the exponent
    s = (q.double().abs().amax() * 448 * scales[..., 0].max().double() * math.sqrt(D))
    size = size * (1 + float(s) * 2.0 ** -24 * 4 * 2 ** 10)
    check_attention(out, want, size)


def test_a_cache_past_four_gigabytes():
    """Page offsets past 2^32 bytes: the pages in use are the pool's last."""
    from iron_b200 import kernels as K

    G, page, D, H = 8, 64, 128, 16
    P = (5 << 30) // (G * 2 * page * D)
    pool, scales = torch.zeros((P, G, 2, page, D), dtype=F8, device="cuda"), torch.ones((P, G, 2), device="cuda")
    few, few_scales = R.cache(6, G, page, D, 1)
    pool[-6:], scales[-6:] = few, few_scales
    lengths, new = [200, 130], [90, 130]
    local = np.array([[3, 0, 5, 1], [2, 4, 1, 0]])
    q, l, start = queries(sum(new), H, D, 2), ints(lengths), [0, 90, 220]
    want, size = R.attention(q, few, few_scales, ints(local), lengths, start)
    check_attention(K.mha_prefill_pages(q, pool, scales, ints(local + P - 6), l, ints(start)), want, size)
    want, size = R.attention(q[:2], few, few_scales, ints(local), lengths, [0, 1, 2])
    check_attention(K.mha_decode_pages(q[:2], pool, scales, ints(local + P - 6), l), want, size)
    # and the write: the last page, from its second half on
    qkv, angles = queries(20, H + 2 * G, D, 4).reshape(20, -1), torch.ones((300, D), dtype=BF16, device="cuda")
    slots, pos = np.arange(20) + (P - 1) * page + 40, np.arange(20)
    ref = R.write(to_numpy(qkv.float()), np.ones((300, D), np.float32), few[-1:].double().cpu().numpy(),
                  few_scales[-1:].cpu().numpy(), slots - (P - 1) * page, pos, H, G, D)
    out = torch.empty((20, H, D), dtype=BF16, device="cuda")
    K.rope_kv_pages(qkv, angles, out, pool, scales, ints(slots), ints(pos), H=H, G=G, D=D)
    check_write(out, pool[-1:], scales[-1:], ref)
    assert (pool[:1].view(torch.uint8) == 0).all()


# ---------------------------------------------------------------------------- together
def test_a_serving_run():
    """Requests come, grow and end over many captured steps; each step's attention is held to the plain
    form on the cache as it lies, and the cache to the rows that were written."""
    from iron_b200 import kernels as K

    rng = np.random.default_rng(11)
    B, width, page, P, rows, H, G, D = 6, 10, 16, 40, 96, 8, 2, 64
    tables, lengths, new = ints(np.full((B, width), -1)), ints(np.zeros(B)), ints(np.zeros(B))
    pages, ring = ints(np.arange(P)), ints([0, P, 0, 0])
    pool, scales = torch.zeros((P, G, 2, page, D), dtype=F8, device="cuda"), torch.ones((P, G, 2), device="cuda")
    a = np.arange(width * page)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    angles = torch.from_numpy(np.stack((np.cos(a), np.sin(a)), -1).reshape(-1, D)).to(BF16).cuda()
    qkv = torch.zeros((rows, (H + 2 * G) * D), dtype=BF16, device="cuda")
    slots, positions, row_start = ints(np.zeros(rows)), ints(np.zeros(rows)), ints(np.zeros(B + 1))
    q, out = torch.zeros((rows, H, D), dtype=BF16, device="cuda"), torch.zeros((rows, H, D), dtype=BF16, device="cuda")

    def step():
        K.page_step(tables, lengths, new, pages, ring, page_size=page, rows=rows, lengths_out=lengths, ring_out=ring,
                    slots=slots, positions=positions, row_start=row_start)
        K.rope_kv_pages(qkv, angles, q, pool, scales, slots, positions, H=H, G=G, D=D)
        K.mha_prefill_pages(q, pool, scales, tables, lengths, row_start, out)

    step()                                                   # nobody brings anything
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    history = [np.zeros((0, 2 * G, D)) for _ in range(B)]
    for _ in range(40):
        n = np.where(rng.random(B) < 0.12, -1, np.where(rng.random(B) < 0.3, rng.integers(0, 40, B), 1))
        new.copy_(ints(n))
        qkv.copy_(torch.from_numpy(rng.standard_normal(qkv.shape)).to(BF16))
        was = lengths.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        # a refused request's rows may be past the buffer: what there is of them is computed on what it had
        now, start, x = lengths.cpu().numpy(), np.minimum(row_start.cpu().numpy(), rows), qkv.cpu().float().numpy().reshape(rows, -1, D)
        for b in range(B):
            if n[b] < 0:
                assert now[b] == 0
                history[b] = history[b][:0]
            elif now[b] == was[b] + n[b]:
                cs = angles.cpu().float().numpy()
                fresh = [np.concatenate((R.rotate(x[start[b] + i], cs[was[b] + i])[H:H + G], x[start[b] + i, H + G:]))
                         for i in range(n[b])]
                history[b] = np.concatenate([history[b]] + [f[None] for f in fresh])
            else:
                assert now[b] == was[b]                      # refused: its rows went nowhere
        served = int(start[-1])
        want, size = R.attention(q, pool, scales, tables, now, start)
        check_attention(out[:served], want[:served], size[:served])
        for b in np.nonzero(now)[0]:
            ids = tables[b, : -(-now[b] // page)].long()
            got = (pool[ids].double() * scales[ids].double()[..., None, None]).permute(0, 3, 2, 1, 4).reshape(-1, 2 * G, D)
            err = np.abs(got[: now[b]].cpu().numpy() - history[b])
            sc = scales[ids].double().permute(0, 2, 1).reshape(-1, 1, 2 * G, 1).repeat(1, page, 1, 1).reshape(-1, 2 * G, 1)
            # half a step of each of at most four scales a page goes through here (normal codes move exactly)
            assert (err <= np.abs(history[b]) * 2.0 ** -4 + 2.0 ** -9 * sc[: now[b]].cpu().numpy()).all()


def test_two_streams_and_two_graphs():
    """Calls without a workspace of the caller's own may overlap: each has one, captured ones too."""
    from iron_b200 import kernels as K

    lengths, H, G, D, page = [9000, 37, 2500, 1], 8, 2, 128, 32
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    t, l = ints(tables), ints(lengths)
    qs = [queries(4, H, D, i) for i in range(4)]
    want = [R.attention(q, pool, scales, t, lengths, range(5)) for q in qs]
    K.mha_decode_pages(qs[0], pool, scales, t, l)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(4)], [], [torch.empty_like(q) for q in qs]
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            K.mha_decode_pages(qs[i], pool, scales, t, l, outs[i])
    for _ in range(20):
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    graphs[i].replay()
                else:
                    K.mha_decode_pages(qs[i], pool, scales, t, l, outs[i])
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        check_attention(out, *w)


def test_a_tensor_of_another_kind_of_memory_is_refused():
    from iron_b200 import kernels as K

    pool, scales = R.cache(4, 1, 16, 64, 1)
    q, t, l = queries(1, 1, 64, 1), ints([[0, 1]]), ints([20])
    with pytest.raises(RuntimeError):
        K.mha_decode_pages(q, pool, scales, t.cpu(), l)
    with pytest.raises(ValueError):
        K.mha_decode_pages(q, pool[:, :, :, ::2], scales, t, l)


# ---------------------------------------------------------------------------- bad page ids
def guarded(x):
    """``x`` as int32 inside a larger buffer: (the tensor, a check that what lies around it is as it was)."""
    x = np.asarray(x)
    buffer = torch.full((x.size + 128,), 0x5A5A5A5A, dtype=I32, device="cuda")
    inner = buffer[64:64 + x.size].view(x.shape)
    inner.copy_(ints(x))
    return inner, lambda: bool((buffer[:64] == 0x5A5A5A5A).all() and (buffer[64 + x.size:] == 0x5A5A5A5A).all())


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("bad", [-1, 12, 1 << 28, (1 << 28) + 5, 1 << 30, -(1 << 28), (1 << 24) + 3, -(1 << 31), (1 << 31) - 1])
def test_page_ids_outside_the_pool_give_no_slots(page, bad):
    """Held or taken from the ring, an id that is no page's is never turned into a slot, not even where
    its product with the page size wraps into the pool: the rows' slots are -1 and a write changes
    nothing but the pages of the others."""
    from iron_b200 import kernels as K

    P, H, G, D = 12, 2, 1, 64
    t, t_ok = guarded([[bad, 1], [-1, -1], [7, -1], [2, bad]])
    l, n = ints([5, 0, 3, page]), ints([4, 3, 2, 1])
    p, p_ok = guarded([bad] + [9] * (P - 1))
    slots, s_ok = guarded(np.zeros(12))
    positions, pos_ok = guarded(np.zeros(12))
    K.page_step(t, l, n, p, ints([0, P, 0, 0]), page_size=page, rows=12, lengths_out=l, slots=slots, positions=positions)
    assert slots.tolist() == [-1] * 7 + [7 * page + 3, 7 * page + 4, 9 * page, -1, -1]
    assert positions.tolist() == [5, 6, 7, 8, 0, 1, 2, 3, 4, page, 0, 0] and l.tolist() == [9, 3, 5, page + 1]
    assert t.tolist() == [[bad, 1], [bad, -1], [7, -1], [2, 9]]
    assert t_ok() and p_ok() and s_ok() and pos_ok()
    pool, scales = R.cache(P, G, page, D, 1)
    before, scales_before = pool.view(torch.uint8).clone(), scales.clone()
    qkv, angles = queries(12, H + 2 * G, D, 2).reshape(12, -1), torch.ones((8, D), dtype=BF16, device="cuda")
    K.rope_kv_pages(qkv, angles, torch.empty((12, H, D), dtype=BF16, device="cuda"), pool, scales, slots, positions, H=H, G=G, D=D)
    others = [i for i in range(P) if i not in (7, 9)]
    assert torch.equal(pool.view(torch.uint8)[others], before[others]) and torch.equal(scales[others], scales_before[others])
    assert not torch.equal(pool.view(torch.uint8)[7], before[7]) and not torch.equal(pool.view(torch.uint8)[9], before[9])


@pytest.mark.parametrize("head, count", [(-7, 99), (2, -4), (1 << 30, 3), (-(1 << 31), (1 << 31) - 1)])
def test_a_ring_that_says_nonsense_serves_inside_its_buffers(head, count):
    """A ring's head and count outside their ranges, bad ids in it, lengths below zero and past the
    table: requests are served, nothing around the buffers changes, and every slot is -1 or a page's."""
    from iron_b200 import kernels as K

    B, width, page, P, rows = 6, 4, 16, 5, 90
    t, t_ok = guarded(np.full((B, width), 1 << 29))
    l, l_ok = guarded([5, -4, 1 << 30, 20, 0, (1 << 31) - 1])
    p, p_ok = guarded([-9, 1 << 28, 3, 1 << 30, 4])
    outs = [guarded(np.zeros(k)) for k in (rows, rows, B + 1, 4)]
    slots, positions, row_start, ring = (o[0] for o in outs)
    ring.copy_(torch.tensor([head, count, 0, 0], dtype=I32))
    K.page_step(t, l, ints([20, -1, 20, 3, 9, 1]), p, ring, page_size=page, rows=rows, lengths_out=l, ring_out=ring,
                slots=slots, positions=positions, row_start=row_start)
    assert t_ok() and l_ok() and p_ok() and all(ok() for _, ok in outs)
    assert row_start.tolist() == [0, 20, 20, 40, 43, 52, 53]
    got = slots.tolist()
    assert all(s == -1 or 0 <= s < P * page for s in got) and got[53:] == [-1] * 37
    assert got[:11] == [-1] * 11                             # the request's first page is 1 << 29, which wraps to 0
    free = max(0, min(count, P))
    assert l.tolist() == [25 if free >= 1 else 5, 0, 1 << 30, 23, 9 if free >= 2 else 0, (1 << 31) - 1]
    assert 0 <= ring[0].item() < P and ring.tolist()[1:] == [free - min(free, 2), 2 if free else 4, 53]
    assert any(s >= 0 for s in got) == (free > 0)            # one of the ring's next two ids is a page's


# ---------------------------------------------------------------------------- queries that are not finite
@pytest.mark.parametrize("form", ["decode", "prompt", "single rows among others"])
@pytest.mark.parametrize("D, page", [(64, 16), (128, 64), (64, 256)])
@pytest.mark.parametrize("kw", [dict(), dict(window=70), dict(causal=False)], ids=str)
def test_infinite_and_nan_queries_over_present_and_absent_pages(form, D, page, kw):
    """An absent token is not there for a query of any value: rows all of whose present scores are
    -infinity, and rows that see no present token, are zeros; a NaN or +infinity in a score is NaN."""
    from iron_b200 import kernels as K

    if form == "decode" and "causal" in kw:
        kw = dict(window=0)                                  # a decode step has no mask to drop
    H, G = 8, 2
    lengths, new = [700, 400, 300, 40], [150, 130, 200, 5]
    if form != "prompt":
        new = [1, 1, 1, 1]
    if form == "single rows among others":
        lengths, new = lengths + [9] * 20, new + [0] * 19 + [3]
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    poison(pool, scales, tables, lengths, page)
    pool[:, :, 0, :, 7] = torch.where(torch.isnan(pool[:, :, 0, :, 7].float()), 0.0, 2.0).to(F8)   # every key's element 7 is there
    tables[0, ::3] = -1
    tables[1, :] = P + 5                                     # a request none of whose pages is there
    start = np.concatenate(([0], np.cumsum(new)))
    q, inf, nan = queries(int(start[-1]), H, D, 5), math.inf, math.nan
    for b in range(4):
        for r in {start[b], (start[b] + start[b + 1]) // 2, start[b + 1] - 1}:
            q[r, 0, 7], q[r, 1, 7], q[r, 3, 2], q[r, 5, :], q[r, 6, 7] = -inf, inf, nan, -inf, -inf
            q[r, 6, 3] = 3e38
    t, l = ints(tables), ints(lengths)
    if form == "decode":
        out = K.mha_decode_pages(q, pool, scales, t, l, **kw)
    else:
        out = K.mha_prefill_pages(q, pool, scales, t, l, ints(start), **kw)
    want, size = R.attention(q, pool, scales, t, lengths, start, **kw)
    zero = (want[start[0]:start[1]] == 0).all(-1)
    assert zero.any() and torch.isnan(want).any() and (want[start[1]:start[2]] == 0).all()
    check_attention(out, want, size)
    assert (out[start[1]:start[2]] == 0).all()


# ---------------------------------------------------------------------------- status words
@pytest.mark.parametrize("prompt", [False, True])
def test_status_words(prompt):
    """A wait that gives up is reported to the call's word, or to the device's own, never to nobody; calls
    that end well touch neither, and what a word holds stays until it is cleared.  (No wait of these
    kernels can be made to give up without breaking one, so the report itself is not run here.)"""
    from iron_b200 import kernels as K

    H, G, D, page, lengths = 4, 2, 64, 16, [40, 3]
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    q, t, l = queries(2, H, D, 1), ints(tables), ints(lengths)
    call = (lambda **kw: K.mha_prefill_pages(q, pool, scales, t, l, ints([0, 1, 2]), **kw)) if prompt else (
        lambda **kw: K.mha_decode_pages(q, pool, scales, t, l, **kw))
    word = K.pages_status()
    assert word.dtype is I32 and word.shape == (1,) and word.is_cuda and int(word) == 0
    assert K.pages_status(q.device).data_ptr() == K.pages_status("cuda").data_ptr() == word.data_ptr()
    own = torch.zeros(1, dtype=I32, device="cuda")
    for value in (0, -6):
        own.fill_(value), word.fill_(value)
        assert torch.equal(call(), call(status=own)) and int(own) == int(word) == value
    word.zero_()


# ---------------------------------------------------------------------------- scores of any size
@pytest.mark.parametrize("H, G, D", [(8, 1, 64), (4, 2, 128), (24, 2, 64)])
@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_one_key_takes_all_at_any_size_of_its_score(form, H, G, D):
    """A row that sees a single token gives that token's value, be its score 2^-90 or 2^110, of either sign."""
    from iron_b200 import kernels as K

    B, page = 8, 16
    lengths = [1] * B if form == "decode" else [2] * B
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    t, l, first = ints(tables), ints(lengths), torch.arange(0, 2 * B, 2, device="cuda")
    value = pool[t[:, 0].long(), :, 1, 0].double() * scales[t[:, 0].long(), :, 1].double()[..., None]
    want = value.repeat_interleave(H // G, 1)
    for power in range(-100, 101):
        q = queries(2 * B if form == "prompt" else B, H, D, power + 200) * 2.0 ** power
        if form == "decode":
            out = K.mha_decode_pages(q, pool, scales, t, l)
        else:
            out = K.mha_prefill_pages(q, pool, scales, t, l, ints(np.arange(B + 1) * 2))[first]
        assert ((out.double() - want).abs() <= tolerance(want, want.abs())).all(), f"queries times 2^{power}"


@pytest.mark.parametrize("form", ["decode", "prompt"])
@pytest.mark.parametrize("power", [20, 60, -60])
def test_queries_of_very_large_and_very_small_size(form, power):
    """Queries times 2^20 and 2^60: one key takes all, and the output is its value to half a bf16 step;
    times 2^-60: all present keys weigh the same."""
    from iron_b200 import kernels as K

    n, page, G, H, D = 600, 16, 2, 4, 64
    tables, P = R.tables_for([n], page, 1)
    pool, scales = R.cache(P, G, page, D, 3)
    m = 200 if form == "prompt" else 1
    q = queries(m, H, D, 1) * 2.0 ** power
    t, l = ints(tables), ints([n])
    out = K.mha_prefill_pages(q, pool, scales, t, l, ints([0, m])) if form == "prompt" else K.mha_decode_pages(q, pool, scales, t, l)
    want, size = R.attention(q, pool, scales, t, [n], [0, m])
    ids = t[0].long()
    k = (pool[ids, :, 0].double() * scales[ids, :, 0].double()[..., None, None]).permute(1, 0, 2, 3).reshape(G, -1, D)[:, :n]
    k = k.repeat_interleave(H // G, 0)
    s = torch.einsum("rhd,hkd->rhk", q.double(), k) / math.sqrt(D)
    seen = (torch.arange(n, device="cuda")[None] <= torch.arange(n - m, n, device="cuda")[:, None])[:, None]
    top = torch.where(seen, s, -math.inf).topk(2, -1).values
    # f32 products and sums of D terms are off by at most D roundings of the terms' sum (2^-23 each, for sums that
    # truncate), on either key; e^-40 of weight is far below a half's
    error = 2 * D * 2.0 ** -23 * (torch.einsum("rhd,hkd->rhk", q.double().abs(), k.abs()).amax(-1) / math.sqrt(D))
    clear = (top[..., 0] - top[..., 1] > error + 40) if power > 0 else torch.full_like(top[..., 0], True, dtype=torch.bool)
    assert clear.double().mean() > 0.9
    check_attention(out[clear], want[clear], size[clear])


# ---------------------------------------------------------------------------- writes of more than 1024 rows
def runs_around_looks(page, rows, seed):
    """(before, new) of requests whose page runs begin at the last row, the first row and the second row
    of a look of 32 rows, of one, eight, nine and a page's rows, and then of random lengths, ``rows`` in all."""
    rng = np.random.default_rng(seed)
    before, new = [], []

    def bring(n, b=0):
        before.append(b), new.append(n)

    for n in (1, 8, 9, page, page + 1):
        for first in (31, 32, 33):
            while (sum(new) + 1) % 32 != (first + 1) % 32:           # single rows up to the place
                bring(1, int(rng.integers(0, 3 * page)))
            bring(n)
            bring(n, page - 1)
    while sum(new) < rows:
        n = int(rng.choice([1, 2, 7, 8, 9, page - 1, page, 3 * page]))
        bring(min(n, rows - sum(new)), int(rng.integers(0, 2 * page)))
    return before, new


@pytest.mark.parametrize("H, G, D, page, rows", [(4, 2, 64, 16, 1025), (2, 2, 128, 16, 1100), (6, 1, 128, 64, 1503),
                                                 (2, 1, 64, 256, 3000), (3, 3, 128, 256, 2947), (1, 1, 64, 32, 1056)])
@pytest.mark.parametrize("kind", ["mixed", "mixed, with infinities and NaN", "rows without slots", "one prompt", "single rows"])
def test_rope_kv_pages_of_many_rows(H, G, D, page, rows, kind):
    from iron_b200 import kernels as K

    if kind == "one prompt":
        before, new = [37], [rows]
    elif kind == "single rows":
        before, new = [(5 * i) % (2 * page) for i in range(1100)], [1] * 1100
    else:
        before, new = runs_around_looks(page, rows, page + rows)
    qkv, angles, pool, scales, slots, positions = write_case(H, G, D, page, before, new, page + H, "NaN" in kind)
    assert len(slots) == sum(new) > 1024
    if kind == "rows without slots":
        slots[::97] = -1                                     # holes end a run where they lie in one
        slots[[31, 32, 63, 64, 65, 96]] = -1
        # what follows a hole inside a page would share the page with what lies before it: those rows go nowhere
        for b, n in zip(np.cumsum([0] + new[:-1]), new):
            hole = False
            for r in range(b, b + n):
                hole = (hole or slots[r] < 0) and not (slots[r] >= 0 and slots[r] % page == 0)
                if hole:
                    slots[r] = -1
    with np.errstate(all="ignore"):
        want = R.write(qkv.float().numpy(), angles.float().numpy(), pool.double().numpy(), scales.numpy(), slots, positions, H, G, D)
    pool, scales = pool.cuda(), scales.cuda()
    q = torch.full((len(slots), H, D), 7.0, dtype=BF16, device="cuda")
    for _ in range(2):                                       # the second finds its own rows and scales there
        K.rope_kv_pages(qkv.cuda(), angles.cuda(), q, pool, scales, ints(slots), ints(positions), H=H, G=G, D=D)
        check_write(q, pool, scales, want)


# ---------------------------------------------------------------------------- repeats, overlap, mixed steps
@pytest.mark.parametrize("H, G, D", [(32, 8, 64), (16, 2, 128)])
@pytest.mark.parametrize("lengths, new", [([2048], [2048]), ([4096] * 16, [7] * 16), ([900, 9001, 3000], [900, 61, 1433]),
                                          ([300 + 17 * i for i in range(40)], [1] * 38 + [64, 300])])
def test_the_prompt_form_repeats_itself_bit_for_bit(H, G, D, lengths, new):
    """Partial results join in a fixed order, whatever the workspace held."""
    from iron_b200 import kernels as K

    page = 64
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    start = ints(np.concatenate(([0], np.cumsum(new))))
    q, t, l = queries(sum(new), H, D, 3), ints(tables), ints(lengths)
    workspace = K.pages_workspace(D, True)
    outs = []
    for fill in (0, 0xFF, 0x3C, 0xFF):
        outs.append(K.mha_prefill_pages(q, pool, scales, t, l, start, workspace=workspace.fill_(fill)))
    assert all(torch.equal(outs[0], x) for x in outs[1:])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("singles", [0, 20], ids=["prompts", "prompts and single rows"])
def test_ragged_calls_on_two_streams_and_in_two_graphs(D, singles):
    """As for the decode form: calls without a workspace of the caller's own have one each."""
    from iron_b200 import kernels as K

    H, G, page = 8, 2, 32
    lengths, new = [9000, 37, 2500, 300] + [100 + i for i in range(singles)], [200, 37, 5, 64] + [1] * singles
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    start = np.concatenate(([0], np.cumsum(new)))
    t, l, r = ints(tables), ints(lengths), ints(start)
    qs = [queries(int(start[-1]), H, D, i) for i in range(4)]
    want = [R.attention(q, pool, scales, t, lengths, start) for q in qs]
    K.mha_prefill_pages(qs[0], pool, scales, t, l, r)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(4)], [], [torch.empty_like(q) for q in qs]
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            K.mha_prefill_pages(qs[i], pool, scales, t, l, r, outs[i])
    for _ in range(20):
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    graphs[i].replay()
                else:
                    K.mha_prefill_pages(qs[i], pool, scales, t, l, r, outs[i])
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        check_attention(out, *w)


@pytest.mark.parametrize("B, H, G, D, page, width, P, rows", [(24, 8, 2, 128, 32, 12, 150, 320), (40, 16, 1, 64, 64, 9, 170, 1400),
                                                             (17, 6, 3, 128, 16, 40, 300, 160)])
def test_a_mixed_serving_run(B, H, G, D, page, width, P, rows):
    """More than sixteen requests, most of which bring one row a step and some a prompt's chunk, end, or
    find no room: every captured step's bookkeeping, cache and outputs against the plain forms."""
    from iron_b200 import kernels as K

    rng = np.random.default_rng(B)
    tables, lengths, new = ints(np.full((B, width), -1)), ints(np.zeros(B)), ints(np.zeros(B))
    pages, ring = ints(rng.permutation(P)), ints([0, P, 0, 0])
    pool, scales = torch.zeros((P, G, 2, page, D), dtype=F8, device="cuda"), torch.ones((P, G, 2), device="cuda")
    a = np.arange(width * page)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    angles = torch.from_numpy(np.stack((np.cos(a), np.sin(a)), -1).reshape(-1, D)).to(BF16).cuda()
    qkv = torch.zeros((rows, (H + 2 * G) * D), dtype=BF16, device="cuda")
    slots, positions, row_start = ints(np.zeros(rows)), ints(np.zeros(rows)), ints(np.zeros(B + 1))
    q, out = torch.zeros((rows, H, D), dtype=BF16, device="cuda"), torch.zeros((rows, H, D), dtype=BF16, device="cuda")

    def step():
        K.page_step(tables, lengths, new, pages, ring, page_size=page, rows=rows, lengths_out=lengths, ring_out=ring,
                    slots=slots, positions=positions, row_start=row_start)
        K.rope_kv_pages(qkv, angles, q, pool, scales, slots, positions, H=H, G=G, D=D)
        K.mha_prefill_pages(q, pool, scales, tables, lengths, row_start, out)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    refused = 0
    for i in range(16):
        n = np.where(rng.random(B) < 0.08, -1, np.where(rng.random(B) < (0.5 if i == 0 else 0.1), rng.integers(2, rows // 6, B), 1))
        new.copy_(ints(n))
        qkv.copy_(torch.from_numpy(rng.standard_normal(qkv.shape)).to(BF16))
        before = [x.cpu().numpy() for x in (tables, lengths, pages, ring)]
        old_pool, old_scales = pool.cpu().double().numpy(), scales.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        step_want = R.page_step(before[0], before[1], n, before[2], before[3], page, rows)
        check_step((slots, positions, row_start, lengths, ring), tables, pages, step_want)
        check_write(q, pool, scales, R.write(qkv.cpu().float().numpy(), angles.cpu().float().numpy(), old_pool, old_scales,
                                             step_want["slots"], step_want["positions"], H, G, D))
        start = np.minimum(step_want["row_start"], rows)
        want, size = R.attention(q, pool, scales, tables, step_want["lengths"], start)
        check_attention(out[: start[-1]], want[: start[-1]], size[: start[-1]])
        refused += int(step_want["ring"][2])
    assert (refused > 0) == (B > 17) and int(K.pages_status()) == 0      # the smallest batch finds room for all


@pytest.mark.parametrize("starts", [[0, 40, -(1 << 31), 60], [30, -(1 << 31), (1 << 31) - 1, -5], [-7, 20, (1 << 31) - 1, -(1 << 31)]])
@pytest.mark.parametrize("others", [0, 20], ids=["few", "more than sixteen"])
def test_row_starts_out_of_order_or_out_of_range_stay_inside_the_buffers(starts, others):
    """Row starts that no step hands out: a request has the rows from its start to the next one, both
    brought into the buffer, and none where they run backwards."""
    from iron_b200 import kernels as K

    H, G, D, page, rows = 4, 2, 64, 16, 50
    lengths = [60, 70, 80] + [5] * others
    starts = starts + [rows] * others
    tables, P = R.tables_for(lengths, page, 1)
    pool, scales = R.cache(P, G, page, D, 2)
    q, t = queries(rows, H, D, 1), ints(tables)
    buffer = torch.full((rows + 20, H, D), 9.0, dtype=BF16, device="cuda")
    out = K.mha_prefill_pages(q, pool, scales, t, ints(lengths), ints(starts), buffer[10:-10])
    assert (buffer[:10] == 9).all() and (buffer[-10:] == 9).all()
    mine = [(min(max(a, 0), rows), max(min(max(a, 0), rows), min(max(b, 0), rows))) for a, b in zip(starts, starts[1:])]
    for b, (r0, r1) in enumerate(mine):
        if r1 > r0 and not any(c != b and x < r1 and r0 < y for c, (x, y) in enumerate(mine)):    # its rows are no other's too
            want, size = R.attention(q[r0:r1], pool, scales, t[b:b + 1], lengths[b:b + 1], [0, r1 - r0])
            check_attention(out[r0:r1], want, size)
