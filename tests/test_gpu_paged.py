"""The paged serving operators against plain implementations in 64 bits.

Tolerances are derived, first order, from the roundings that a correct f32
kernel makes (u = 2^-24, half a step), with the sums' length as the factor of
an accumulation in any order.
"""
import math

import numpy as np
import pytest

import myos
from myos import _lib

pytestmark = pytest.mark.gpu

U = 2.0**-24
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from myos import dev as m

    return m


def cache(rng, pages, heads, page, d, kv, nhd=False, fill=float("nan")):
    """A cache whose every slot holds `fill` until a test writes it."""
    t = torch.float32 if kv == "f32" else torch.bfloat16
    shape = (pages, page, heads, d) if nhd else (pages, heads, page, d)
    k, v = (torch.full(shape, fill, dtype=t, device="cuda") for _ in range(2))
    return (k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)) if nhd else (k, v)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


# ---------------------------------------------------------------- attention
def fill_cache(rng, k, v, lens, page, spare=2):
    """Random K and V in the slots that the lengths use, pages in random order.
    Returns the table (unused entries -1) and the values as f64 [b][heads, len, d]."""
    pages, heads, _, d = k.shape
    blocks = max(1, -(-max(lens) // page))
    table = np.full((len(lens), blocks + spare), -1)
    order, at, ks, vs = rng.permutation(pages), 0, [], []
    for b, n in enumerate(lens):
        held = -(-n // page)
        table[b, :held] = order[at:at + held]
        at += held
        kb, vb = (torch.randn(heads, n, d, device="cuda").to(k.dtype) for _ in range(2))
        j = np.arange(n)
        if n:
            pg, sl = torch.from_numpy(table[b, j // page]).cuda(), torch.from_numpy(j % page).cuda()
            k[pg, :, sl] = kb.transpose(0, 1)
            v[pg, :, sl] = vb.transpose(0, 1)
        ks.append(kb.double().cpu().numpy())
        vs.append(vb.double().cpu().numpy())
    return table, ks, vs


def plain_attention(q, ks, vs, scale, keep):
    """(out, lse, tolerance of out, tolerance of lse) in f64; keep[b]: the keys
    attended to."""
    n, hq, d = q.shape
    out, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    tol, ltol = np.zeros((n, hq, d)), np.zeros((n, hq))
    for b in range(n):
        group = hq // ks[b].shape[0]
        j = np.nonzero(keep[b])[0]
        if j.size == 0:
            continue
        for h in range(hq):
            k, v = ks[b][h // group][j], vs[b][h // group][j]
            s = k @ q[b, h] * scale
            top = s.max()
            p = np.exp(s - top)
            out[b, h] = p @ v / p.sum()
            lse[b, h] = top + np.log(p.sum())
            # a score: d products added (d + 2 roundings of at most the sum of magnitudes), the scale, and
            # its distance to the maximum in exp's argument; exp itself within 2 steps
            es = (d + 4) * U * (np.abs(k) @ np.abs(q[b, h]) * abs(scale)).max() + 4 * U * np.abs(s).max() + 4 * U
            # numerator and denominator: every weight off by es (twice: its own and the maximum's), j.size
            # additions and as many rescalings
            rel = 2 * (2 * es + (2 * j.size + 16) * U)
            tol[b, h] = rel * (p @ np.abs(v)) / p.sum() + 1e-30
            ltol[b, h] = rel + 4 * U * abs(lse[b, h])
    return out, lse, tol, ltol


def kept(lens, window=0, bad=()):
    return [np.array([(not window or j >= n - window) and (b, j) not in bad for j in range(n)], bool)
            for b, n in enumerate(lens)]


def attend(dev, q, kv, table, lens, work=None, **kw):
    out = torch.full(q.shape, float("nan"), device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda") if work is None else work
    dev.paged_attention(out, q, kv, table, lens, work, lse=lse, **kw)
    return out, lse


def check_attention(out, lse, want):
    o, l, tol, ltol = want
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(out).all()
    assert (np.abs(out - o) <= tol).all(), (np.abs(out - o) / np.maximum(tol, 1e-300)).max()
    empty = np.isneginf(l)
    assert (np.isneginf(lse) == empty).all() and (out[empty] == 0).all()
    assert (np.abs(lse[~empty] - l[~empty]) <= ltol[~empty]).all()


ATTN = [
    # hq, hkv, d, page, kv, lengths, window, nhd
    (12, 2, 128, 16, "bf16", [0, 1, 15, 16, 17, 63, 64, 65, 200], 0, False),
    (12, 2, 128, 16, "f32", [0, 1, 15, 16, 17, 63, 64, 65, 200], 0, False),
    (40, 8, 128, 32, "bf16", [700, 1, 2049], 0, True),
    (40, 8, 128, 32, "f32", [700, 1, 2049], 0, True),
    (8, 8, 64, 1, "bf16", [5, 130], 0, False),          # pages of one slot
    (8, 8, 64, 3, "f32", [5, 130, 0], 0, True),         # pages that end inside every tile
    (5, 1, 80, 16, "bf16", [33, 127, 128, 129], 0, False),
    (7, 1, 8, 24, "f32", [33, 127, 128, 129], 0, False),
    (14, 2, 256, 64, "bf16", [1000, 77], 0, False),
    (8, 1, 256, 64, "f32", [1000, 77], 0, True),
    (3, 1, 72, 16, "bf16", [1], 0, False),
    (12, 2, 128, 16, "bf16", [1000, 100, 101, 99, 0, 164], 100, False),
    (28, 4, 128, 16, "f32", [1000, 1, 65], 1, False),   # a window of the newest key alone
    (32, 4, 64, 16, "bf16", [640] * 70, 0, False),      # more sequences than SMs / heads
    (16, 2, 128, 16, "bf16", [5000], 0, False),         # one long sequence over many blocks
    (12, 2, 128, 16, "bf16", [700, 650, 690, 10] * 3, 0, False),  # several shares an item, some left empty
    (4, 2, 256, 16, "f32", [300, 290, 280], 0, False),
    (2, 1, 64, 512, "bf16", [70001, 3], 0, False),
    (2, 2, 64, 512, "f32", [70001, 3], 50000, True),
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(x) for x in c[:5]) + f"-n{len(c[5])}-w{c[6]}")
def test_attention(dev, case):
    hq, hkv, d, page, kvt, lens, window, nhd = case
    rng = np.random.default_rng(hq * 1000 + d + page)
    torch.manual_seed(hq + d)
    pages = sum(-(-n // page) for n in lens) + 3
    k, v = cache(rng, pages, hkv, page, d, kvt, nhd)
    table, ks, vs = fill_cache(rng, k, v, lens, page)
    q = torch.randn(len(lens), hq, d, device="cuda") * 2
    out, lse = attend(dev, q, dev.PagedKV(k, v), i32(table), i32(lens), window=window)
    scale = 1 / math.sqrt(d)
    check_attention(out, lse, plain_attention(q.double().cpu().numpy(), ks, vs, scale, kept(lens, window)))


@pytest.mark.parametrize("kvt", ["f32", "bf16"])
def test_attention_of_strided_rows_and_bad_pages(dev, kvt):
    """q inside q|k|v rows, out inside wider rows, a strided table; pages out
    of range are left out, lengths past the table end at it, negative ones are
    empty."""
    rng = np.random.default_rng(5)
    torch.manual_seed(5)
    hq, hkv, d, page, lens = 12, 2, 128, 16, [100, 40, 7]
    k, v = cache(rng, 20, hkv, page, d, kvt)
    table, ks, vs = fill_cache(rng, k, v, lens, page, spare=0)
    wide = i32(np.concatenate([table, np.full((3, 5), 10**9)], 1))[:, : table.shape[1]]
    bad = {(0, j) for j in range(16, 32)} | {(1, j) for j in range(32, 40)}
    wide[0, 1], wide[1, 2] = 20, -7
    rows = torch.randn(3, (hq + 2 * hkv) * d, device="cuda")
    q = rows[:, : hq * d].view(3, hq, d)
    buf = torch.full((3, hq * d + 64), 7.0, device="cuda")
    out = buf[:, 32 : 32 + hq * d].view(3, hq, d)
    lse = torch.zeros(3, hq, device="cuda")
    work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
    scale = 0.3
    dev.paged_attention(out, q, dev.PagedKV(k, v), wide, i32(lens), work, scale=scale, lse=lse)
    want = plain_attention(q.double().cpu().numpy(), ks, vs, scale, kept(lens, 0, bad))
    check_attention(out, lse, want)
    assert (buf[:, :32] == 7).all() and (buf[:, 32 + hq * d :] == 7).all()
    # past the table: the same keys as a length of exactly the table (all of row 0's pages)
    full = table.shape[1] * page
    k[:], v[:] = torch.randn_like(k), torch.randn_like(v)
    wide[:, :] = i32(rng.permutation(20)[: table.shape[1]])[None]
    a, la = attend(dev, q, dev.PagedKV(k, v), wide, i32([full, 2**31 - 1, -5]))
    assert torch.equal(a[2], torch.zeros_like(a[2])) and torch.isneginf(la[2]).all()
    q2 = q.clone()
    q2[1] = q[0]
    b, _ = attend(dev, q2, dev.PagedKV(k, v), wide, i32([full, 2**31 - 1, -5]))
    torch.testing.assert_close(b[1], b[0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("kvt", ["f32", "bf16"])
@pytest.mark.parametrize("d", [136, 192, 256])
@pytest.mark.parametrize("lens", [[2500] + [30, 0, 41, 7] * 30, [400] * 40, [900, 3]], ids=["pieces", "items", "few"])
def test_attention_of_long_heads(dev, kvt, d, lens):
    """Heads past 128 dims: shares of many pieces, whole items, a few long ones."""
    test_attention(dev, (10, 2, d, 16, kvt, lens, 0, False))


def test_attention_far_into_a_large_cache(dev):
    """Element offsets past 32 bits: the pages lie behind 2^32 elements."""
    rng = np.random.default_rng(6)
    torch.manual_seed(6)
    d, page, hkv, hq, lens = 128, 64, 8, 40, [130, 700]
    pages = (1 << 32) // (hkv * page * d) + 40
    k = torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda")
    table = np.stack([np.arange(11), np.arange(11) + 20]) + (1 << 32) // (hkv * page * d)
    ks, vs = [], []
    for b, n in enumerate(lens):
        x = torch.randn(hkv, 11 * page, d, device="cuda").bfloat16()
        for i, p in enumerate(table[b]):
            k[p] = x[:, i * page : (i + 1) * page]
        ks.append(x[:, :n].double().cpu().numpy())
    q = torch.randn(2, hq, d, device="cuda")
    out, lse = attend(dev, q, dev.PagedKV(k, k), i32(table), i32(lens))
    check_attention(out, lse, plain_attention(q.double().cpu().numpy(), ks, ks, d**-0.5, kept(lens)))


def test_attention_over_more_tiles_than_a_product_of_32_bits_holds(dev):
    """592 shares of 7.5 million tiles: three pages, over and over in the table.

    A share's warp adds up one part of 8 keys of about 7.5e6 / 592 tiles, one
    rounding (a whole step at most, in the tensor core) each, and one for each
    share that is joined: (12670 + 592 + 64) 2 U of the sum of the weights, and
    of that of the weighted values.
    """
    torch.manual_seed(14)
    d, page, blocks = 8, 1024, 234375
    k, v = (torch.randn(3, 1, page, d, device="cuda") for _ in range(2))
    q = torch.randn(1, 2, d, device="cuda")
    order = np.arange(blocks) % 3
    n = blocks * page - 100
    out, lse = attend(dev, q, dev.PagedKV(k, v), i32(order[None]), i32([n]))
    times = np.bincount(order, minlength=3)[:, None] * np.ones((3, page))
    times[order[-1], page - 100 :] -= 1
    w = times.reshape(-1)
    k64, v64 = (x.double().cpu().numpy().reshape(-1, d) for x in (k, v))
    s = q[0].double().cpu().numpy() @ k64.T * d**-0.5
    e = w * np.exp(s - s.max(1, keepdims=True))
    want = e @ v64 / e.sum(1, keepdims=True)
    tol = (12670 + 592 + 64) * 2 * U
    most = e @ np.abs(v64) / e.sum(1, keepdims=True)
    assert (np.abs(out[0].double().cpu().numpy() - want) <= tol * (most + np.abs(want)) * 1.01).all()
    assert (np.abs(lse[0].double().cpu().numpy() - np.log(e.sum(1)) - s.max(1)) <= tol * 1.01 + 1e-5).all()


def test_attention_of_many_short_sequences(dev):
    """More sequences than a block has threads, many of them empty."""
    rng = np.random.default_rng(12)
    torch.manual_seed(12)
    hq, hkv, d, page, n = 2, 2, 64, 4, 3000
    lens = rng.integers(0, 6, n) * (rng.random(n) < 0.7)
    k, v = cache(rng, int((-(-lens // page)).sum()) + 1, hkv, page, d, "bf16")
    table, ks, vs = fill_cache(rng, k, v, lens.tolist(), page)
    q = torch.randn(n, hq, d, device="cuda")
    out, lse = attend(dev, q, dev.PagedKV(k, v), i32(table), i32(lens))
    check_attention(out, lse, plain_attention(q.double().cpu().numpy(), ks, vs, d**-0.5, kept(lens.tolist())))


def test_attention_on_two_streams_at_once(dev):
    """Calls that run at the same time, each with a work buffer of its own."""
    rng = np.random.default_rng(13)
    torch.manual_seed(13)
    hq, hkv, d, page = 12, 2, 128, 16
    lens = [[4000, 300, 1], [2500, 2501, 17]]
    sets = []
    for n in lens:
        k, v = cache(rng, sum(-(-m // page) for m in n), hkv, page, d, "bf16")
        table, ks, vs = fill_cache(rng, k, v, n, page)
        q = torch.randn(3, hq, d, device="cuda")
        work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
        want = plain_attention(q.double().cpu().numpy(), ks, vs, d**-0.5, kept(n))
        sets.append((q, dev.PagedKV(k, v), i32(table), i32(n), work, want, torch.cuda.Stream()))
    outs = [torch.zeros(50, 3, hq, d, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    for i in range(50):
        for (q, kv, table, n, work, _, st), o in zip(sets, outs):
            dev.paged_attention(o[i], q, kv, table, n, work, stream=st)
    torch.cuda.synchronize()
    for (q, kv, table, n, work, want, st), o in zip(sets, outs):
        assert (np.abs(o[0].double().cpu().numpy() - want[0]) <= want[2]).all()
        assert (o.view(torch.int32) == o[0].view(torch.int32)).all()
        assert not work[: 16 * 1024].any()  # the arrival counts are back at zero


def test_attention_extremes(dev):
    """Scores far apart (one key takes all the weight) and large equal ones."""
    hq, hkv, d, page = 8, 1, 64, 16
    for kvt in ("f32", "bf16"):
        k, v = cache(None, 8, hkv, page, d, kvt)
        table = np.arange(8)[None]
        kb = np.zeros((hkv, 100, d))
        kb[0, :, 0] = -100.0
        kb[0, 77, 0] = 100.0
        vb = np.tile(np.arange(100.0)[:, None], (1, d))[None]
        j = torch.arange(100, device="cuda")
        k[j // page, 0, j % page] = torch.from_numpy(kb[0]).cuda().to(k.dtype)
        v[j // page, 0, j % page] = torch.from_numpy(vb[0]).cuda().to(k.dtype)
        q = torch.zeros(1, hq, d, device="cuda")
        q[0, :, 0] = torch.tensor([0.0, 1.0, 10.0, 100.0, -1.0, -10.0, -100.0, 1e4], device="cuda")
        out, lse = attend(dev, q, dev.PagedKV(k, v), i32(table), i32([100]), scale=1.0)
        check_attention(out, lse, plain_attention(q.double().cpu().numpy(), [kb], [vb], 1.0, kept([100])))


def test_attention_replayed_with_other_lengths_and_a_shared_buffer(dev):
    """One captured launch serves every length the table can hold; the work
    buffer goes from one shape to the next; the same inputs give the same
    bits, on another stream as well."""
    rng = np.random.default_rng(8)
    torch.manual_seed(8)
    hq, hkv, d, page = 12, 2, 128, 16
    most = [3000, 900, 0, 1]
    k, v = cache(rng, 260, hkv, page, d, "bf16")
    table, ks, vs = fill_cache(rng, k, v, most, page)
    table, lens, q = i32(table), i32(most), torch.randn(4, hq, d, device="cuda")
    work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
    kv = dev.PagedKV(k, v)
    out, lse = attend(dev, q, kv, table, lens, work)
    k2, v2 = cache(rng, 80, 8, 16, 64, "f32")
    t2, ks2, vs2 = fill_cache(rng, k2, v2, [1200], 16)
    q2 = torch.randn(1, 16, 64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dev.paged_attention(out, q, kv, table, lens, work, lse=lse)
    for now in ([3000, 900, 0, 1], [17, 0, 0, 0], [0, 0, 0, 0], [2999, 1, 0, 1]):
        lens.copy_(i32(now))
        out.fill_(float("nan"))
        o2, l2 = attend(dev, q2, dev.PagedKV(k2, v2), i32(t2), i32([1200]), work)
        g.replay()
        check_attention(o2, l2, plain_attention(q2.double().cpu().numpy(), ks2, vs2, 0.125, kept([1200])))
        keep = [np.arange(m) < n for n, m in zip(now, most)]
        check_attention(out, lse, plain_attention(q.double().cpu().numpy(), ks, vs, d**-0.5, keep))
        first = out.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        o3 = torch.empty_like(out)
        dev.paged_attention(o3, q, kv, table, lens, work, stream=s)
        s.synchronize()
        assert torch.equal(first.view(torch.int32), o3.view(torch.int32))


# ---------------------------------------------------------------- tables
def plain_tables(table, ctx, new, free, page, num_pages, rows):
    n, blocks = table.shape
    table = table.copy()
    slots, pos, seq = np.full(rows, -1, np.int64), np.zeros(rows, np.int64), np.full(rows, -1, np.int64)
    lens, starts, taken, asked, refused, at = np.zeros(n, np.int64), np.zeros(n + 1, np.int64), 0, 0, 0, 0
    for b in range(n):
        c, a = max(int(ctx[b]), 0), max(int(new[b]), 0)
        lens[b] = c
        end = at + a
        starts[b + 1] = min(end, rows)
        seq[min(at, rows) : min(end, rows)] = b
        if a > 0:
            held = -(-c // page)
            need = -(-(c + a) // page) - held
            fits = c + a <= blocks * page and end <= rows
            if fits and (need == 0 or asked + need <= len(free)):
                for j in range(need):
                    table[b, held + j] = free[len(free) - 1 - asked - j]
                lens[b] = c + a
                for i in range(a):
                    p = table[b, (c + i) // page]
                    pos[at + i] = c + i
                    slots[at + i] = p * page + (c + i) % page if 0 <= p < num_pages else -1
                taken = max(taken, asked + need) if need else taken
            else:
                refused += 1
            asked += need if fits else 0
        at = end
    return table, slots, pos, seq, lens, starts, np.array([len(free) - taken, refused])


def run_tables(dev, table, ctx, new, free, page, num_pages, rows, num_free=None):
    i = lambda *n: torch.full(n, 99, dtype=torch.int32, device="cuda")  # noqa: E731
    t, n = i32(table), len(ctx)
    slots = torch.full((rows,), 99, dtype=torch.int64, device="cuda")
    out = (slots, i(rows), i(rows), i(n), i(n + 1), i(2))
    dev.paged_tables(t, i32(ctx), i32(new), i32(free), i32([len(free) if num_free is None else num_free]),
                     page, num_pages, *out)
    return [x.cpu().numpy() for x in (t, *out)]


def same(got, want):
    for g, w, name in zip(got, want, ("table", "slots", "positions", "row_seq", "kv_lens", "seq_starts", "result")):
        np.testing.assert_array_equal(g, w, err_msg=name)


@pytest.mark.parametrize("n,page,most,chunk,short", [
    (1, 16, 64, 1, 0), (1, 16, 64, 40, 0), (1, 16, 64, 40, 1), (7, 1, 9, 3, 0), (64, 16, 640, 1, 2),
    (300, 32, 900, 200, 0), (300, 24, 900, 200, 17), (1500, 16, 300, 60, 40), (5000, 8, 64, 9, 3),
    (16384, 16, 64, 2, 0)])
def test_tables(dev, n, page, most, chunk, short):
    rng = np.random.default_rng(n + page)
    ctx = rng.integers(0, most + 1, n)
    new = rng.integers(0, chunk + 1, n)
    new[rng.random(n) < 0.3] = min(1, chunk)
    over = rng.random(n) < 0.03  # some do not fit their row of the table
    new = np.where(over, new, np.minimum(new, most - ctx))
    blocks = -(-most // page)
    held = np.minimum(-(-ctx // page), blocks)
    need = int((-(-(ctx + new) // page) - -(-ctx // page)).sum())
    free_n = max(0, need - short)
    num_pages = int(held.sum()) + free_n + 2
    pages = rng.permutation(num_pages)
    table = np.full((n, blocks), -1)
    table[np.arange(blocks)[None, :] < held[:, None]] = pages[: held.sum()]
    free = pages[held.sum() : held.sum() + free_n]
    rows = int(new.sum()) + int(rng.integers(0, 7))
    args = (table, ctx, new, free, page, num_pages, max(rows, 1))
    same(run_tables(dev, *args), plain_tables(*args))
    # a row buffer that ends inside a request's rows
    if rows > 3:
        args = args[:-1] + (int(rows * 0.7),)
        same(run_tables(dev, *args), plain_tables(*args))


def test_tables_edges(dev):
    table = np.array([[5, 1, -1, -1], [3, -1, -1, -1], [-1, -1, -1, -1], [900, -1, -1, -1]])
    # negative lengths, a page out of range, a free page out of range, a request far too long
    args = (table, [17, -4, -1, 3], [3, 2, 0, 2], [7, 900, 2], 16, 10, 12)
    got = run_tables(dev, *args)
    same(got, plain_tables(*args))
    assert list(got[1][:3]) == [17, 18, 19] and list(got[1][5:7]) == [-1, -1]
    args = (table, [2**31 - 1, 2, 0, 0], [2**31 - 1, 1, 2**31 - 1, 0], [7, 8, 2], 16, 10, 12)
    same(run_tables(dev, *args)[3:], plain_tables_far(*args))
    # more free pages named than the list holds, and a negative count
    t = np.full((1, 2), -1)
    assert list(run_tables(dev, t, [0], [20], [4, 6], 16, 10, 20, num_free=100)[0][0]) == [6, 4]
    got = run_tables(dev, t, [0], [20], [4, 6], 16, 10, 20, num_free=-3)
    assert list(got[0][0]) == [-1, -1] and list(got[6]) == [0, 1] and (got[1] == -1).all()
    # no rows to map: everything that adds tokens is refused
    got = run_tables(dev, t, [3], [1], [4], 16, 10, 0)
    assert list(got[6]) == [1, 1] and list(got[4]) == [3]


def plain_tables_far(table, ctx, new, free, page, num_pages, rows):
    """Lengths whose sums pass 32 bits: every request with rows behind the
    first one's end is refused."""
    seq = np.zeros(rows, np.int64)
    return [seq, np.array([2**31 - 1, 2, 0, 0]), np.array([0, rows, rows, rows, rows]), np.array([3, 3])]


def test_tables_step_after_step(dev):
    """A decode loop: lengths and the free count of one step are the next
    step's, both steps in one captured graph."""
    rng = np.random.default_rng(3)
    n, page, blocks, num_pages = 9, 4, 12, 60
    table, free = np.full((n, blocks), -1), rng.permutation(num_pages)
    t, f = i32(table), i32(free)
    lens = [i32(np.zeros(n)), i32(np.zeros(n))]
    res = [i32([num_pages, 0]), i32([0, 0])]
    add, rows = i32(rng.integers(0, 2, n)), 12
    slots = torch.zeros(rows, dtype=torch.int64, device="cuda")
    pos, seq, starts = i32(np.zeros(rows)), i32(np.zeros(rows)), i32(np.zeros(n + 1))

    def step(a, b):
        dev.paged_tables(t, lens[a], add, f, res[a][:1], page, num_pages, slots, pos, seq, lens[b], starts, res[b])

    step(0, 1)  # the first call, outside the capture; its effects are undone
    t.copy_(i32(table))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(0, 1)
        step(1, 0)
    cur, left = np.zeros(n, np.int64), num_pages
    for _ in range(20):
        a = rng.integers(0, 2, n)
        add.copy_(i32(a))
        g.replay()
        for _ in range(2):
            table, *rest = plain_tables(table, cur, a, free[:left], page, num_pages, rows)
            cur, left = rest[3], int(rest[5][0])
        np.testing.assert_array_equal(t.cpu().numpy(), table)
        np.testing.assert_array_equal(slots.cpu().numpy(), rest[0])
        np.testing.assert_array_equal(lens[0].cpu().numpy(), cur)
        assert res[0].tolist() == list(rest[5])


# ---------------------------------------------------------------- norm, rotate, store
STORE = [
    # rows, hq, hkv, d, rot, norm, kv, page, nhd
    (1, 12, 2, 128, 128, (False, False), "f32", 16, False),
    (1, 40, 8, 128, 128, (True, True), "bf16", 16, False),
    (67, 40, 8, 128, 128, (True, True), "f32", 16, True),
    (67, 12, 2, 128, 64, (True, False), "bf16", 3, False),
    (33, 8, 8, 64, 64, (False, True), "bf16", 1, True),
    (5, 5, 1, 80, 40, (True, True), "f32", 16, False),
    (19, 3, 1, 8, 8, (True, True), "bf16", 7, False),
    (19, 16, 4, 256, 256, (True, True), "bf16", 64, False),
    (130, 7, 7, 72, 0, (True, True), "f32", 16, True),
    (2000, 12, 2, 128, 128, (False, False), "bf16", 16, False),
]


def plain_head(x, gamma, cos, sin, eps):
    """(f64 value, tolerance) of heads x [.., d] in f64, cos/sin [.., rot / 2]."""
    d, y, size = x.shape[-1], x, np.zeros_like(x)
    if gamma is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma
        size = (d / 2 + 6) * U * np.abs(y)  # the sum of squares, halved by the root; root, divisions, two products
    half = cos.shape[-1]
    a, b, ea, eb = y[..., :half], y[..., half : 2 * half], size[..., :half], size[..., half : 2 * half]
    c, s = np.abs(cos), np.abs(sin)
    out = np.concatenate([a * cos - b * sin, a * sin + b * cos, y[..., 2 * half :]], -1)
    tol = np.concatenate([ea * c + eb * s + 2 * U * (np.abs(a) * c + np.abs(b) * s),
                          ea * s + eb * c + 2 * U * (np.abs(a) * s + np.abs(b) * c), size[..., 2 * half :]], -1)
    return out, tol


@pytest.mark.parametrize("case", STORE, ids=lambda c: "-".join(str(x) for x in c[:5]) + f"-{c[6]}-p{c[7]}")
@pytest.mark.parametrize("in_place", [False, True])
def test_store(dev, case, in_place):
    rows, hq, hkv, d, rot, norm, kvt, page, nhd = case
    rng = np.random.default_rng(rows + d)
    torch.manual_seed(rows + d)
    pages, npos = rows // page + 4, 500
    k, v = cache(rng, pages, hkv, page, d, kvt, nhd, fill=5.0)
    wide = torch.randn(rows, (hq + 2 * hkv) * d + 8, device="cuda")
    qkv = wide[:, : (hq + 2 * hkv) * d]
    host = qkv.double().cpu().numpy().reshape(rows, -1, d)
    slots = rng.permutation(pages * page)[:rows]
    pos = rng.integers(0, npos, rows)
    if rows > 4:  # padding, a slot past the cache, positions outside the tables
        slots[1], slots[2], pos[3], pos[4] = -1, pages * page, npos, -1
    qg, kg = ((1 + 0.3 * torch.randn(d, device="cuda")).bfloat16() if on else None for on in norm)
    cs, sn = dev.rope_table(npos, rot, 1e4) if rot else (np.zeros((npos, 0)), np.zeros((npos, 0)))
    tables = (torch.from_numpy(cs).cuda(), torch.from_numpy(sn).cuda()) if rot else (None, None)
    q = qkv[:, : hq * d].view(rows, hq, d) if in_place else torch.zeros(rows, hq, d, device="cuda")
    dev.qk_norm_rope_store(q, qkv, dev.PagedKV(k, v), i32(pos), torch.from_numpy(slots).cuda(), *tables,
                           q_gamma=qg, k_gamma=kg, eps=1e-5)
    good = (pos >= 0) & (pos < npos) if rot else np.ones(rows, bool)
    at = np.clip(pos, 0, npos - 1)
    c, s = (x.astype(np.float64)[at][:, None] for x in (cs, sn))
    gam = [g.double().cpu().numpy() if g is not None else None for g in (qg, kg)]
    want, tol = plain_head(host[:, :hq], gam[0], c, s, 1e-5)
    got = q.double().cpu().numpy()
    assert (np.abs(got - want) <= tol)[good].all()
    assert np.isnan(got[~good]).all()
    want, tol = plain_head(host[:, hq : hq + hkv], gam[1], c, s, 1e-5)
    step = 0 if kvt == "f32" else 2.0**-8
    tol = tol + step * (np.abs(want) + tol)
    kc, vc = (x.double().cpu().numpy() for x in (k, v))
    used = np.zeros((pages, page), bool)
    for r in range(rows):
        if not good[r] or not 0 <= slots[r] < pages * page:
            continue
        p, o = divmod(int(slots[r]), page)
        used[p, o] = True
        assert (np.abs(kc[p, :, o] - want[r]) <= tol[r]).all()
        plain = qkv[r].view(-1, d)[hq + hkv :].to(v.dtype).double().cpu().numpy()
        assert (vc[p, :, o] == plain).all()  # values are stored as they are, or rounded once
    free = ~used[:, None, :, None] & np.ones_like(kc, bool)
    assert (kc[free] == 5).all() and (vc[free] == 5).all()
    if not in_place:
        assert (qkv.double().cpu().numpy().reshape(rows, -1, d) == host).all()


# ---------------------------------------------------------------- logits
def plain_logits(x, hist, plen, hlen, rep, freq, pres, bias, mask):
    """f64 controlled logits and their tolerance; bias: per row [(id, value)],
    mask: per row bool [vocab] or None."""
    y, tol = x.astype(np.float64), np.zeros(x.shape)
    n, vocab = x.shape
    for r in range(n):
        said = [t for t in hist[r][: max(0, hlen[r])]]
        for t in set(t for t in said if 0 <= t < vocab):
            if rep is not None:
                y[r, t] = y[r, t] / rep[r] if x[r, t] > 0 else y[r, t] * rep[r]
                tol[r, t] += U * abs(y[r, t])
            times = sum(1 for i, u in enumerate(said) if u == t and i >= plen[r])
            if freq is not None:
                y[r, t] -= float(freq[r]) * times
                tol[r, t] += U * (abs(float(freq[r])) * times + abs(y[r, t]) * 1.01)
            if pres is not None and times:
                y[r, t] -= float(pres[r])
                tol[r, t] += U * abs(y[r, t]) * 1.01
        for t, b in dict(bias[r]).items():
            if 0 <= t < vocab:
                y[r, t] += b
                tol[r, t] += U * abs(y[r, t]) * 1.01 + U * abs(b) * 1e-3
        if mask is not None and mask[r] is not None:
            y[r, ~mask[r]] = -np.inf
            tol[r, ~mask[r]] = 0
    return y, tol * 1.01 + 1e-37


def check_logits(out, ids, want, tol):
    o = out.double().cpu().numpy()
    inf = ~np.isfinite(want)
    assert (o[inf] == want[inf]).all()
    assert (np.abs(o[~inf] - want[~inf]) <= tol[~inf]).all()
    check_ids(out, ids)


def check_ids(out, ids):
    o = out.cpu().numpy().copy()
    o[np.isnan(o)] = -np.inf
    np.testing.assert_array_equal(ids.cpu().numpy(), o.argmax(1))  # numpy: the first maximum


@pytest.mark.parametrize("rows,vocab,width,nbias", [
    (1, 1, 1, 1), (1, 151936, 300, 0), (3, 152064, 500, 40), (5, 8192, 64, 9), (4, 8193, 700, 9),
    (70, 1001, 33, 5), (2, 33, 0, 0), (300, 97, 50, 3), (2, 262147, 2000, 100),
    (250, 70001, 40, 3),     # a block's ids in several passes
    (2, 5003, 20000, 9),     # more tokens than the table has room for: chunk by chunk
    (3, 9001, 50, 4000)])    # more biases
@pytest.mark.parametrize("strided", [False, True])
def test_logits(dev, rows, vocab, width, nbias, strided):
    rng = np.random.default_rng(rows + vocab)
    pad = 3 if strided else 0  # rows at every alignment
    buf = torch.from_numpy(rng.standard_normal((rows, vocab + pad)).astype(np.float32) * 5).cuda()
    logits, x = buf[:, :vocab], buf[:, :vocab].cpu().numpy()
    wide = max(width, 1)
    hist = (np.minimum(vocab * rng.random((rows, wide + pad)) ** 4, vocab - 1)).astype(np.int64)
    if width > 10:
        hist[:, 3], hist[:, 5], hist[:, 7] = -1, vocab, -(2**31)  # no tokens of this vocabulary
    hlen = rng.integers(0, width + 1, rows)
    hlen[0] = width
    plen = rng.integers(-1, width + 2, rows)
    rep, freq, pres = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.6), (-0.5, 0.7), (0, 0.9)))
    bias = [[(int(t), float(np.float32(rng.uniform(-9, 9)))) for t in rng.integers(-1, vocab + 1, rng.integers(0, nbias + 1))]
            for _ in range(rows)]
    for r in range(rows):  # the same token twice: the last entry counts
        if len(bias[r]) > 1:
            bias[r][-1] = (bias[r][0][0], bias[r][-1][1])
    starts = np.cumsum([0] + [len(b) for b in bias])
    flat = [e for b in bias for e in b] + [(0, 0.0)]
    bits = rng.random((rows // 2 + 1, vocab)) < 0.3
    which = rng.integers(-1, bits.shape[0] + 1, rows)  # -1 and one past the masks: none
    words = np.packbits(np.pad(bits, ((0, 0), (0, -vocab % 32))), axis=1, bitorder="little").view(np.int32)
    mask = [bits[g] if 0 <= g < len(bits) else None for g in which]
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    args = dict(history=i32(hist)[:, :wide], prompt_lens=i32(plen), hist_lens=i32(hlen), repetition=f(rep),
                frequency=f(freq), presence=f(pres), bias_starts=i32(starts), bias_ids=i32([t for t, _ in flat]),
                bias_vals=f([b for _, b in flat]), mask=torch.from_numpy(words).cuda(), mask_rows=i32(which))
    want, tol = plain_logits(x, hist[:, :wide], plen, hlen, rep, freq, pres, bias, mask)
    out = torch.full((rows, vocab + 2 * pad), 3.0, device="cuda")[:, pad : pad + vocab]
    ids = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    dev.logit_controls(out, logits, ids=ids, **args)
    check_logits(out, ids, want, tol)
    if strided:
        whole = out._base if out._base is not None else out
        assert (whole[:, :pad] == 3).all() and (whole[:, pad + vocab :] == 3).all()
    only = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    dev.logit_controls(None, logits, ids=only, **args)
    assert torch.equal(only, ids)
    first = out.clone()
    dev.logit_controls(logits, logits, **args)  # in place, no ids
    assert torch.equal(logits, first)


def test_logits_parts_alone(dev):
    """Each control without the others, and none at all."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 500)).astype(np.float32)
    hist, plen, hlen = rng.integers(0, 40, (3, 60)), [0, 10, 60], [60, 60, 60]
    t, h = torch.from_numpy(x).cuda(), i32(hist)
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    one = np.array([1.3, 0.5, 2.0], np.float32)
    none = [[], [], []]
    for name, at in (("repetition", 4), ("frequency", 5), ("presence", 6)):
        a = [x, hist, plen, hlen, None, None, None, none, None]
        a[at] = one
        out, ids = torch.empty_like(t), torch.zeros(3, dtype=torch.uint32, device="cuda")
        dev.logit_controls(out, t, history=h, prompt_lens=i32(plen), hist_lens=i32(hlen), ids=ids, **{name: f(one)})
        check_logits(out, ids.view(torch.int32), *plain_logits(*a))
    # no lengths: the whole width, all of it output
    out = torch.empty_like(t)
    dev.logit_controls(out, t, history=h, frequency=f(one))
    want, tol = plain_logits(x, hist, [0] * 3, [60] * 3, None, one, None, none, None)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    out, ids = torch.empty_like(t), torch.zeros(3, dtype=torch.int32, device="cuda")
    dev.logit_controls(out, t, ids=ids)
    assert torch.equal(out, t)
    check_ids(out, ids)
    with pytest.raises(myos.MyosError) as e:
        dev.logit_controls(out, t, mask=torch.zeros(3, 15, dtype=torch.int32, device="cuda"))
    assert e.value.code == _lib.ERR_SHAPE


@pytest.mark.parametrize("rows,vocab,width,most,nbias", [
    (64, 100003, 3000, 90, 5),   # a row's tokens all in one run of ids: chunk by chunk in one of its blocks
    (160, 30011, 200, 30011, 3000),  # one row with nearly all the biases
    (333, 24577, 1, 24577, 0), (75, 60000, 0, 1, 0)])
@pytest.mark.parametrize("pad", [0, 3])
def test_logits_of_long_slices(dev, rows, vocab, width, most, nbias, pad):
    rng = np.random.default_rng(rows + vocab)
    buf = torch.from_numpy(rng.standard_normal((rows, vocab + pad)).astype(np.float32) * 5).cuda()
    logits, x = buf[:, pad:], buf[:, pad:].cpu().numpy()
    hist, hlen = rng.integers(0, most, (rows, max(width, 1))), [width] * rows
    plen = rng.integers(0, width + 1, rows)
    rep, freq, pres = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.6), (-0.5, 0.7), (0, 0.9)))
    bias = [[(int(t), 1.5) for t in rng.permutation(vocab)[: nbias if r == 1 else min(nbias, 3)]] for r in range(rows)]
    bits = rng.random((rows, vocab)) < 0.7
    words = np.packbits(np.pad(bits, ((0, 0), (0, -vocab % 32))), axis=1, bitorder="little").view(np.int32)
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    flat = [e for b in bias for e in b] + [(0, 0.0)]
    args = dict(history=i32(hist), prompt_lens=i32(plen), hist_lens=i32(hlen), repetition=f(rep), frequency=f(freq),
                presence=f(pres), bias_starts=i32(np.cumsum([0] + [len(b) for b in bias])),
                bias_ids=i32([t for t, _ in flat]), bias_vals=f([b for _, b in flat]),
                mask=torch.from_numpy(words).cuda())
    want, tol = plain_logits(x, hist, plen, hlen, rep, freq, pres, bias, list(bits))
    out, ids = torch.full((rows, vocab), 3.0, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    dev.logit_controls(out, logits, ids=ids, **args)
    check_logits(out, ids, want, tol)
    ends = buf[:, :pad].clone()
    again = torch.zeros_like(ids)
    dev.logit_controls(logits, logits, ids=again, **args)  # in place
    assert torch.equal(logits, out) and torch.equal(again, ids) and torch.equal(buf[:, :pad], ends)


def test_logits_rows_far_apart(dev):
    """Rows more than 2^31 elements apart."""
    rng = np.random.default_rng(4)
    far, vocab = (1 << 31) + 64, 1000
    buf = torch.empty(far + vocab, device="cuda")
    x = buf.as_strided((2, vocab), (far, 1))
    host = rng.standard_normal((2, vocab)).astype(np.float32)
    x.copy_(torch.from_numpy(host).cuda())
    hist, ids = rng.integers(0, vocab, (2, 30)), torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.tensor([0.5, 0.25], device="cuda")
    dev.logit_controls(x, x, history=i32(hist), presence=f, ids=ids)
    want, tol = plain_logits(host, hist, [0, 0], [30, 30], None, None, f.cpu().numpy(), [[], []], None)
    check_logits(x, ids, want, tol)


@pytest.mark.parametrize("vocab", [5, 40000])
def test_logits_rows_without_a_choice(dev, vocab):
    """Masked out altogether, all NaN, NaN and infinities in and out of masked
    places, ties: greedy_token's rule."""
    x = torch.zeros(8, vocab, device="cuda")
    x[1] = float("nan")
    x[2, 3] = float("nan")
    x[2, 4] = 1
    x[3] = -math.inf
    x[4, 2] = math.inf
    x[4, 4] = math.inf
    x[5, 1] = float("nan")
    x[5, 2] = math.inf
    x[6, vocab - 1] = 2
    x[7] = torch.finfo(torch.float32).min
    words = np.zeros((3, -(-vocab // 32)), np.uint32)
    words[1, 0], words[2] = 0b11000, 0xFFFFFFFF  # none; tokens 3 and 4; all
    which = i32([0, 2, -1, 2, 2, 1, 1, 2])
    out, ids = torch.empty_like(x), torch.full((8,), 9, dtype=torch.int32, device="cuda")
    dev.logit_controls(out, x, mask=torch.from_numpy(words.view(np.int32)).cuda(), mask_rows=which, ids=ids)
    # row 6: its 2 stands at the last token, which the mask of tokens 3 and 4 allows when there are five
    assert ids.tolist() == [0, 0, 4, 0, 2, 3, 4 if vocab == 5 else 3, 0]
    assert torch.isneginf(out[0]).all() and torch.isnan(out[1]).all() and torch.isnan(out[2, 3])
    assert torch.isneginf(out[5, :3]).all() and (out[5, 3:5] == 0).all()


# ---------------------------------------------------------------- together
def test_a_serving_loop(dev):
    """Prompts, then decode steps of a batch through two layers' caches, each
    decode step one captured graph: tables, store, attention, a projection to
    logits, controls with the greedy id fed back; against the same loop in
    64 bits over plain lists."""
    rng = np.random.default_rng(11)
    torch.manual_seed(11)
    hq, hkv, d, page, vocab, layers, n, steps = 8, 2, 64, 8, 320, 2, 5, 12
    prompts = [rng.integers(0, vocab, m) for m in (3, 8, 17, 1, 30)]
    width, pages, blocks, hmax = (hq + 2 * hkv) * d, 40, 6, 48
    emb = torch.randn(vocab, hq * d, device="cuda") / 8
    wqkv = [torch.randn(hq * d, width, device="cuda") / 16 for _ in range(layers)]
    head = torch.randn(hq * d, vocab, device="cuda") / 4
    qg, kg = ((1 + 0.2 * torch.randn(d, device="cuda")).bfloat16() for _ in range(2))
    cs, sn = (torch.from_numpy(x).cuda() for x in dev.rope_table(blocks * page, d, 1e4))
    kvs = [dev.PagedKV(*cache(rng, pages, hkv, page, d, "f32")) for _ in range(layers)]
    table, free = i32(np.full((n, blocks), -1)), i32(rng.permutation(pages))
    lens, res = [i32(np.zeros(n)), i32(np.zeros(n))], [i32([pages, 0]), i32([0, 0])]
    hist, hlen = i32(np.zeros((n, hmax))), i32([len(p) for p in prompts])
    for b, p in enumerate(prompts):
        hist[b, : len(p)] = i32(p)
    plen = hlen.clone()
    rep, pres = (torch.full((n,), x, device="cuda") for x in (1.2, 0.4))
    words = np.full((1, vocab // 32), 0xFFFFFFFF, np.uint32)
    words[0, 0] = 0xFFFF0000  # tokens 0..15 are out for sequence 2
    mask, which = torch.from_numpy(words.view(np.int32)).cuda(), i32([-1, -1, 0, -1, -1])
    work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    out, logits = torch.zeros(n, hq, d, device="cuda"), torch.zeros(n, vocab, device="cuda")
    last = {}

    def forward(tokens, add, a, rows, pick):
        """One step of `rows` token rows (n requests); a: which lengths are old."""
        slots = torch.zeros(rows, dtype=torch.int64, device="cuda")
        pos, seq, starts = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (rows, rows, n + 1))
        dev.paged_tables(table, lens[a], add, free, res[a][:1], page, pages, slots, pos, seq, lens[1 - a], starts, res[1 - a])
        x = emb[tokens.long()]
        for i in range(layers):
            q = torch.empty(rows, hq, d, device="cuda")
            dev.qk_norm_rope_store(q, x @ wqkv[i], kvs[i], pos, slots, cs, sn, q_gamma=qg, k_gamma=kg)
            if pick:
                dev.paged_attention(out, q, kvs[i], table, lens[1 - a], work)
                x = x + out.view(n, -1)
        if pick:
            torch.matmul(x, head, out=logits)
            dev.logit_controls(logits, logits, history=hist, prompt_lens=plen, hist_lens=hlen, repetition=rep,
                               presence=pres, mask=mask, mask_rows=which, ids=ids)
            hist.scatter_(1, hlen.long()[:, None], ids[:, None])
            hlen.add_(1)

    # the prompts, all but their last tokens, in one packed step (their K and V only: with two layers the
    # second's input is the embedding, here and in the plain loop), then the last tokens as the first decode step
    flat = np.concatenate([p[:-1] for p in prompts])
    forward(i32(np.concatenate([flat, [0, 0]])), i32([len(p) - 1 for p in prompts]), 0, len(flat) + 2, False)
    ids.copy_(i32([p[-1] for p in prompts]))
    one = i32(np.ones(n))
    torch.backends.cuda.matmul.allow_tf32 = False
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    keep = [x.clone() for x in (table, *lens, *res, hist, hlen, ids)]
    with torch.cuda.stream(s):  # warm-up; its effects are undone (the cache slots are written again)
        forward(ids.clone(), one, 1, n, True)
    torch.cuda.current_stream().wait_stream(s)
    for x, y in zip((table, *lens, *res, hist, hlen, ids), keep):
        x.copy_(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        forward(ids, one, 1, n, True)
        forward(ids, one, 0, n, True)
    got = []
    for _ in range(steps // 2):
        g.replay()
        got.append((ids.cpu().numpy(), logits.double().cpu().numpy()))
    assert res[1].tolist()[1] == 0
    said = hist.cpu().numpy()

    # the same in 64 bits, fed the ids that were picked
    E, W, H = emb.double().cpu().numpy(), [w.double().cpu().numpy() for w in wqkv], head.double().cpu().numpy()
    G = [x.double().cpu().numpy() for x in (qg, kg)]
    C, S = cs.double().cpu().numpy(), sn.double().cpu().numpy()
    for b, p in enumerate(prompts):
        K, V = [[] for _ in range(layers)], [[] for _ in range(layers)]
        for t in range(len(p) + steps - 1):
            tok, pick = said[b, t], t >= len(p) - 1
            x = E[tok].copy()
            for i in range(layers):
                y = (x @ W[i]).reshape(-1, d)
                c, sn_ = C[t][None], S[t][None]
                qh, _ = plain_head(y[:hq], G[0], c, sn_, 1e-6)
                kh, _ = plain_head(y[hq : hq + hkv], G[1], c, sn_, 1e-6)
                K[i].append(kh)
                V[i].append(y[hq + hkv :])
                if pick:
                    o, *_ = plain_attention(qh[None], [np.stack(K[i], 1)], [np.stack(V[i], 1)], d**-0.5, [np.ones(t + 1, bool)])
                    x = x + o[0].reshape(-1)
            if not pick:
                continue
            step = t - (len(p) - 1)
            m = np.ones(vocab, bool)
            m[:16] = b != 2
            want, _ = plain_logits((x @ H)[None], said[b : b + 1], [len(p)], [t + 1], np.array([1.2], np.float32), None,
                                   np.array([0.4], np.float32), [[]], [m])
            # f32 roundings of sums of at most 512 terms through two layers: 1e-3 of the logits' size is over a
            # hundred times their first-order sum (2 (512 + 64) u per layer)
            close = 2e-3 * np.abs(x @ H).max()
            picked = said[b, t + 1]
            assert want[0, picked] >= want[0].max() - close
            if step % 2 == 1:
                assert got[step // 2][0][b] == picked
                fine = np.isfinite(want[0])
                assert (np.isneginf(got[step // 2][1][b]) == ~fine).all()
                assert (np.abs(got[step // 2][1][b][fine] - want[0][fine]) <= close).all()
