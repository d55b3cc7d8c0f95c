"""Calls of the paged serving operators at the edges of what their documentation
allows: histories of no or few tokens, lengths and rows near 2^31, tables near
the shared-memory limit, caches whose tensors got other memory, NaN queries.

Tolerances as in test_gpu_paged.py (u = 2^-24, half a step of f32).
"""
import os
import subprocess
import sys

import numpy as np
import pytest

import myos
from myos import _lib

torch = pytest.importorskip("torch")

from test_gpu_paged import (U, attend, cache, check_attention, check_logits, dev, fill_cache,  # noqa: E402,F401
                            i32, kept, plain_attention, plain_logits)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- logits
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (12, 151936), (16, 152064), (18, 152064), (40, 152064),
                                        (64, 152064), (100, 65537), (333, 32003)])
@pytest.mark.parametrize("width", [1, 2, 3, 8])
def test_penalties_of_short_histories_without_biases(dev, rows, vocab, width):
    """The first decode steps: a row's few tokens are the work of one or two of
    its blocks, whose lists hold them."""
    rng = np.random.default_rng(rows * 10 + width)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 5
    hist = rng.integers(0, vocab, (rows, width))
    hist[0, 0], hist[-1, -1] = vocab - 1, x[-1].argmax()
    plen, hlen = rng.integers(0, width + 1, rows), rng.integers(0, width + 1, rows)
    hlen[0] = hlen[-1] = width
    rep, freq, pres = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((1.1, 1.6), (0.1, 0.7), (0.1, 0.9)))
    t, f = torch.from_numpy(x).cuda(), lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    args = dict(history=i32(hist), prompt_lens=i32(plen), hist_lens=i32(hlen), repetition=f(rep), frequency=f(freq),
                presence=f(pres))
    out, ids = torch.full_like(t, 3.0), torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    dev.logit_controls(out, t, ids=ids, **args)
    check_logits(out, ids, *plain_logits(x, hist, plen, hlen, rep, freq, pres, [[]] * rows, None))
    only = torch.full_like(ids, 77)
    dev.logit_controls(None, t, ids=only, **args)
    assert torch.equal(only, ids)
    dev.logit_controls(t, t, **args)  # in place
    assert torch.equal(t, out)


# ---------------------------------------------------------------- tables
def test_tables_of_as_many_rows_as_are_allowed(dev):
    """One prompt that fills a row buffer of 2^31 - 1 rows (34 GB of outputs): the
    threads' strides from row to row go past 2^31 at its end."""
    rows, page = 2**31 - 1, 65536
    blocks = 2**31 // page
    torch.cuda.empty_cache()
    free = torch.from_numpy(np.random.default_rng(1).permutation(blocks).astype(np.int32)).cuda()
    table = torch.full((1, blocks), -1, dtype=torch.int32, device="cuda")
    slots = torch.full((rows,), -9, dtype=torch.int64, device="cuda")
    pos, seq = (torch.full((rows,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    lens, starts, result = (torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (1, 2, 2))
    dev.paged_tables(table, i32([0]), i32([rows]), free, i32([blocks]), page, blocks, slots, pos, seq, lens, starts, result)
    assert torch.equal(table[0], free.flip(0))
    assert lens.tolist() == [rows] and starts.tolist() == [0, rows] and result.tolist() == [0, 0]
    step = 1 << 27
    for r0 in range(0, rows, step):
        r = torch.arange(r0, min(rows, r0 + step), device="cuda")
        assert (pos[r0 : r0 + step] == r).all() and (seq[r0 : r0 + step] == 0).all()
        assert (slots[r0 : r0 + step] == table[0, r // page].long() * page + r % page).all()
    del table, slots, pos, seq, r
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [3900, 3978, 3979, 4000, 4096, 4097])
def test_tables_of_batches_near_48_kb_of_shared_memory(n):
    """Each batch as a process's first call: the kernel's own shared memory and
    the requests' together pass the limit that holds unless it is raised."""
    code = f"""if 1:
        import torch
        from myos import dev
        n, page, blocks = {n}, 16, 2
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        table, free = i32(n, blocks) - 1, torch.arange(n, dtype=torch.int32, device="cuda")
        slots, out = torch.zeros(n, dtype=torch.int64, device="cuda"), [i32(n), i32(n), i32(n), i32(n + 1), i32(2)]
        dev.paged_tables(table, i32(n), i32(n) + 1, free, i32(1) + n, page, n, slots, *out)
        r = torch.arange(n, device="cuda")
        assert torch.equal(table[:, 0].long(), n - 1 - r) and (table[:, 1] == -1).all()
        assert torch.equal(slots, (n - 1 - r) * page) and (out[0] == 0).all() and torch.equal(out[1].long(), r)
        assert (out[2] == 1).all() and torch.equal(out[3][1:].long(), r + 1) and out[4].tolist() == [0, 0]
    """
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": os.path.dirname(os.path.dirname(myos.__file__))})
    assert r.returncode == 0, r.stderr[-2000:]


def test_tables_of_lengths_that_reach_31_bits(dev):
    """A table row with room for more than 2^31 - 1 tokens: a request grows to that
    length, and past it is refused like one that its row has no room for."""
    page, blocks, top = 65536, 32769, 2**31 - 1
    num_pages = 2 * blocks
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").repeat(6, 1)
    ctx, new = [top, top - 1, top - 3, top - 2, 5, top], [1, 1, 3, 3, top, 0]
    rows = 10
    i = lambda n: torch.full((n,), 99, dtype=torch.int32, device="cuda")  # noqa: E731
    slots, pos, seq = torch.full((rows,), 99, dtype=torch.int64, device="cuda"), i(rows), i(rows)
    lens, starts, result = i(6), i(7), i(2)
    dev.paged_tables(table, i32(ctx), i32(new), i32([0]), i32([0]), page, num_pages, slots, pos, seq, lens, starts, result)
    assert lens.tolist() == [top, top, top, top - 2, 5, top]
    assert starts.tolist() == [0, 1, 2, 5, 8, 10, 10] and result.tolist() == [0, 3]
    assert pos.tolist() == [0, top - 1, top - 3, top - 2, top - 1] + [0] * 5
    assert slots.tolist() == [-1, top - 1, top - 3, top - 2, top - 1] + [-1] * 5
    assert seq.tolist() == [0, 1, 2, 2, 2, 3, 3, 3, 4, 4]


# ---------------------------------------------------------------- the cache object
def test_a_cache_goes_by_its_tensors_as_they_are_at_the_call(dev):
    """PagedKV holds its tensors: memory, strides and shape are theirs at each
    call, also after they were given other ones."""
    torch.manual_seed(3)
    pages, hkv, page, d, hq, rows = 4, 2, 16, 64, 4, 10
    shape = (pages, hkv, page, d)
    k, v = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    kv = dev.PagedKV(k, v)
    qkv, q = torch.randn(rows, (hq + 2 * hkv) * d, device="cuda"), torch.zeros(rows, hq, d, device="cuda")
    pos, slots = i32(np.arange(rows)), torch.arange(rows, device="cuda")
    table, lens, work = i32([[0, 1, 2, 3]]), i32([rows]), torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")

    def attention():
        out = torch.zeros(1, hq, d, device="cuda")
        dev.paged_attention(out, q[:1], kv, table, lens, work)
        return out

    dev.qk_norm_rope_store(q, qkv, kv, pos, slots)
    first = attention()
    olds = k.data, v.data  # the old memory stays allocated
    before = [t.clone() for t in olds]
    k.data, v.data = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    assert not attention().any()
    dev.qk_norm_rope_store(q, qkv * 2, kv, pos, slots)
    assert torch.equal(k, before[0] * 2) and torch.equal(v, before[1] * 2)
    assert torch.equal(olds[0], before[0]) and torch.equal(olds[1], before[1])
    # other strides, a larger cache, another dtype
    nhd = [torch.zeros(pages + 3, page, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k.data, v.data = (t.permute(0, 2, 1, 3) for t in nhd)
    dev.qk_norm_rope_store(q, qkv, kv, pos, slots + (pages + 2) * page)
    assert torch.equal(nhd[0][pages + 2, :rows], before[0][0, :, :rows].transpose(0, 1).bfloat16())
    table.fill_(pages + 2)
    torch.testing.assert_close(attention(), first, rtol=2**-6, atol=2**-6)  # K and V rounded to bf16
    # k alone was changed: refused, nothing is written
    kept = nhd[1].clone()
    k.data = torch.zeros(shape, device="cuda")
    for call in (attention, lambda: dev.qk_norm_rope_store(q, qkv, kv, pos, slots)):
        with pytest.raises(myos.MyosError) as e:
            call()
        assert e.value.code == _lib.ERR_ARG
    assert not k.any() and torch.equal(nhd[1], kept)


def test_a_cache_without_memory_is_refused(dev):
    k, v = (torch.zeros(4, 2, 16, 64, device="cuda") for _ in range(2))
    kv = dev.PagedKV(k, v)
    k.untyped_storage().resize_(0)
    out, work = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
    with pytest.raises(myos.MyosError) as e:
        dev.paged_attention(out, out, kv, i32([[0]]), i32([1]), work)
    assert e.value.code == _lib.ERR_ARG


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("kvt", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_nan_query_has_a_nan_lse(dev, kvt, d):
    """The store marks a row whose position has no angles with a NaN query: its
    attention is NaN in out and lse, not that of an empty sequence, however its
    keys are split; the other rows and heads do not see it."""
    rng = np.random.default_rng(d)
    torch.manual_seed(d)
    hq, hkv, page, lens = 6, 2, 16, [5000, 5000, 40, 40, 0, 1, 1]
    k, v = cache(rng, sum(-(-n // page) for n in lens), hkv, page, d, kvt)
    table, ks, vs = fill_cache(rng, k, v, lens, page)
    q = torch.randn(len(lens), hq, d, device="cuda")
    q[1], q[3], q[4], q[6, 2] = float("nan"), float("nan"), float("nan"), float("nan")
    nan = torch.isnan(q[:, :, 0])
    nan[4] = False  # no keys: zeros and -inf
    out, lse = attend(dev, q, dev.PagedKV(k, v), i32(table), i32(lens))
    assert torch.isnan(out[nan]).all() and torch.isnan(lse[nan]).all()
    assert not torch.isnan(out[~nan]).any() and not torch.isnan(lse[~nan]).any()
    clean = torch.nan_to_num(q)
    want = plain_attention(clean.double().cpu().numpy(), ks, vs, d**-0.5, kept(lens))
    for x, y in ((out, want[0]), (lse, want[1])):
        x[nan] = torch.from_numpy(y).cuda()[nan].float()
    check_attention(out, lse, want[:2] + tuple(t + 2 * U * np.abs(np.nan_to_num(w, neginf=0)) for t, w in zip(want[2:], want)))


@pytest.mark.parametrize("view", [False, True])
def test_penalties_of_a_history_without_columns(dev, view):
    """No token so far: the penalties change nothing, biases still count."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((3, 20001)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    hist = i32(np.zeros((3, 5)))[:, :0] if view else torch.empty(3, 0, dtype=torch.int32, device="cuda")
    two = torch.full((3,), 2.0, device="cuda")
    out, ids = torch.zeros_like(t), torch.zeros(3, dtype=torch.int32, device="cuda")
    zero = i32([0, 0, 0])
    dev.logit_controls(out, t, history=hist, prompt_lens=zero, hist_lens=zero, repetition=two, frequency=two,
                       presence=two, ids=ids)
    assert torch.equal(out, t) and ids.tolist() == x.argmax(1).tolist()
    dev.logit_controls(out, t, history=hist, repetition=two, bias_starts=i32([0, 1, 1, 2]), bias_ids=i32([20000, 7]),
                       bias_vals=torch.tensor([50.0, 50.0], device="cuda"), ids=ids)
    assert ids.tolist() == [20000, int(x[1].argmax()), 7]


def test_a_mask_tensor_of_too_few_rows_is_refused(dev):
    """Row r uses mask r where mask_rows is not given: also where there is none."""
    t, out = torch.zeros(3, 100, device="cuda"), torch.full((3, 100), 5.0, device="cuda")
    for n in (0, 1, 2):
        with pytest.raises(myos.MyosError) as e:
            dev.logit_controls(out, t, mask=torch.zeros(n, 4, dtype=torch.int32, device="cuda"))
        assert e.value.code == _lib.ERR_SHAPE and (out == 5).all()
    # named, a mask outside them is none
    dev.logit_controls(out, t, mask=torch.zeros(0, 4, dtype=torch.int32, device="cuda"), mask_rows=i32([0, -1, 2]))
    assert torch.equal(out, t)


@pytest.mark.parametrize("kvt", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_score_leaves_the_tensor_core_after_four_steps(dev, kvt, d):
    """The tensor core cuts its f32 sums off: one product of 1 and, in each other
    step, one a little below a step of 1 (2 u), which a sum that holds the 1
    loses. The score of a single key is its log-sum-exp.

    Four steps lose three of them (6 u); the sums are joined with roundings of u
    each, at most 4; the products with log2 e and ln 2 round twice, and the two
    constants are off by 0.25 u together: 12.25 u.
    """
    first, step = 2.0**-12, 8 if kvt == "f32" else 16
    small = (2 - 2.0 ** (-10 if kvt == "f32" else -7)) * first  # one term of a key
    q, k = torch.zeros(1, 1, d, device="cuda"), torch.zeros(d)
    # a step of an f32 cache takes values 4 c and 4 c + 1, or 4 c + 2 and 4 c + 3, of 16
    at = torch.arange(0, d, step) if kvt == "bf16" else torch.tensor([16 * (s // 2) + 2 * (s % 2) for s in range(d // 8)])
    q[0, 0, at.cuda()], k[at] = first, small
    q[0, 0, 0], k[0] = 1, 1
    kc, vc = cache(None, 1, 1, 16, d, kvt, fill=0.0)
    kc[0, 0, 0] = k.cuda().to(kc.dtype)
    vc[0, 0, 0] = 1
    out, lse = attend(dev, q, dev.PagedKV(kc, vc), i32([[0]]), i32([1]), scale=1.0)
    exact = 1 + (len(at) - 1) * first * small
    assert (out == 1).all()
    off = abs(lse.double().item() - exact) / U
    assert off <= 12.25, off


@pytest.mark.parametrize("kvt", ["f32", "bf16"])
@pytest.mark.parametrize("d", [8, 64, 128, 256])
def test_a_single_key_gives_its_value_exactly(dev, kvt, d):
    """One key has the weight 1: out is V, all 24 bits of it, also where the other
    keys of a window or of a table are left out."""
    torch.manual_seed(d)
    n, hkv, page = 40, 2, 16
    k, v = (torch.randn(n, hkv, page, d, device="cuda").to(torch.float32 if kvt == "f32" else torch.bfloat16) for _ in range(2))
    v[0], v[1, :, 0], v[2, :, 0] = v[0] * 1e30, v[1, :, 0] * 1e-30, 1 - 2.0**-24
    q = torch.randn(n, 8, d, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    kv = dev.PagedKV(k, v)
    out, _ = attend(dev, q, kv, table, i32([1] * n))
    assert torch.equal(out, v[:, :, 0].float().repeat_interleave(4, 1))
    out, _ = attend(dev, q, kv, table, i32([7] * n), window=1)
    assert torch.equal(out, v[:, :, 6].float().repeat_interleave(4, 1))
