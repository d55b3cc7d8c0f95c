"""The 8-bit projections in use: a layer of the serving step over pages, far offsets,
calls on tensors that they refuse."""
import numpy as np
import pytest

import myos
from myos import _lib
from test_gpu_i8 import ints, norm64, np64, product, rows_of, same, some, stepped, swiglu64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from myos import dev as m

    return m


def quantised(dev, rng, channels, k):
    """A weight, its channels in 8 bits, and what they stand for."""
    w = torch.from_numpy((rng.standard_normal((channels, k)) / np.sqrt(k)).astype(np.float32)).cuda().bfloat16()
    q, s = rows_of(channels, k, torch.int8, -k % 16), torch.zeros(channels, device="cuda")
    dev.quant_rows(q, s, w)
    same(q, s, stepped(np64(w)))
    return q, s


@pytest.mark.parametrize("rows,out", [(1, torch.float32), (5, torch.bfloat16), (70, torch.float32), (300, torch.bfloat16)])
def test_a_layer_over_pages(dev, rows, out):
    """Norm, q|k|v, store, attention, o_proj, norm, gate|up, SwiGLU, down_proj of `rows` sequences that
    each add a token: every 8-bit step bit for bit from its own inputs, and the layer against the
    same layer in 64 bits with the same 8-bit weights."""
    rng = np.random.default_rng(rows)
    hidden, hq, hkv, d, inner, page, ctx = 640, 4, 2, 64, 1000, 16, 40
    wide = (hq + 2 * hkv) * d
    weights = {n: quantised(dev, rng, *s) for n, s in
               {"qkv": (wide, hidden), "o": (hidden, hq * d), "gate_up": (2 * inner, hidden), "down": (hidden, inner)}.items()}
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    gammas = [(1 + 0.1 * f(hidden)).bfloat16() for _ in range(2)]
    bias, x, residual = f(wide), f(rows, hidden), 2 * f(rows, hidden)
    lens = torch.from_numpy(rng.integers(0, ctx, rows).astype(np.int32)).cuda()
    blocks = -(-ctx // page)
    pages = rows * blocks + 3
    k, v = (torch.from_numpy(rng.standard_normal((pages, hkv, page, d)).astype(np.float32)).cuda() for _ in range(2))
    table = torch.from_numpy(rng.permutation(pages)[: rows * blocks].reshape(rows, blocks).astype(np.int32)).cuda()
    slots = table[torch.arange(rows), (lens // page).long()].long() * page + lens % page
    cos, sin = (torch.from_numpy(t).cuda() for t in dev.rope_table(ctx, d, 1e4))

    # ---- the layer
    i8 = lambda n: (rows_of(rows, n, torch.int8, -n % 16), torch.zeros(rows, device="cuda"))  # noqa: E731
    new = lambda n, t=out: torch.zeros(rows, n, dtype=t, device="cuda")  # noqa: E731
    total1, total2, qkv, attn = new(hidden, torch.float32), new(hidden, torch.float32), new(wide, torch.float32), new(hq * d, torch.float32)
    o, gate_up, down = new(hidden), new(2 * inner), new(hidden)
    a1, a2, a3, a4 = i8(hidden), i8(hq * d), i8(hidden), i8(inner)
    before = k.clone(), v.clone()
    kv = dev.PagedKV(k, v)
    dev.add_norm_quant(*a1, x, gammas[0], residual=residual, total=total1)
    dev.matmul_i8(qkv, *a1, *weights["qkv"], bias=bias)
    q = new(hq * d, torch.float32).view(rows, hq, d)
    dev.qk_norm_rope_store(q, qkv, kv, lens, slots, cos, sin)
    work = torch.zeros(dev.WORK_BYTES, dtype=torch.uint8, device="cuda")
    dev.paged_attention(attn.view(rows, hq, d), q, kv, table, lens + 1, work)
    dev.quant_rows(*a2, attn)
    dev.matmul_i8(o, *a2, *weights["o"])
    dev.add_norm_quant(*a3, o, gammas[1], residual=total1, total=total2)
    dev.matmul_i8(gate_up, *a3, *weights["gate_up"])
    dev.swiglu_quant(*a4, gate_up)
    dev.matmul_i8(down, *a4, *weights["down"])

    # ---- each step from its own inputs
    assert torch.equal(total1, x + residual) and torch.equal(total2, o.float() + total1)
    same(*a1, stepped(norm64(np64(total1), np64(gammas[0]), 1e-6)))
    assert torch.equal(qkv.cpu(), product(*a1, *weights["qkv"], bias, torch.float32))
    same(*a2, stepped(np64(attn)))
    assert torch.equal(o.cpu(), product(*a2, *weights["o"], None, out))
    same(*a3, stepped(norm64(np64(total2), np64(gammas[1]), 1e-6)))
    assert torch.equal(gate_up.cpu(), product(*a3, *weights["gate_up"], None, out))
    same(*a4, stepped(swiglu64(np64(gate_up))))
    assert torch.equal(down.cpu(), product(*a4, *weights["down"], None, out))
    dev.matmul_i8_status()

    # ---- the whole in 64 bits, its activations in 8 bits too but no step of f32 or bf16 between
    w64 = {n: np64(q_) * np64(s)[:, None] for n, (q_, s) in weights.items()}

    def held(y):
        q_, s = stepped(y)
        return q_.astype(np.float64) * s.astype(np.float64)[:, None]

    t1 = np64(x) + np64(residual)
    y = held(norm64(t1, np64(gammas[0]), 1e-6)) @ w64["qkv"].T + np64(bias)
    y = y.reshape(rows, hq + 2 * hkv, d)
    c, s_ = np64(cos)[lens.cpu().numpy()][:, None], np64(sin)[lens.cpu().numpy()][:, None]
    turn = lambda h: np.concatenate([h[..., :d // 2] * c - h[..., d // 2:] * s_, h[..., :d // 2] * s_ + h[..., d // 2:] * c], -1)  # noqa: E731
    qs, ks, vs = turn(y[:, :hq]), turn(y[:, hq:hq + hkv]), y[:, hq + hkv:]
    att = np.zeros((rows, hq, d))
    for b in range(rows):
        n = int(lens[b])
        at = [(int(table[b, j // page]), j % page) for j in range(n)]
        for h in range(hq):
            g = h // (hq // hkv)
            kk = np.array([np64(before[0][p, g, i]) for p, i in at] + [ks[b, g]])
            vv = np.array([np64(before[1][p, g, i]) for p, i in at] + [vs[b, g]])
            e = kk @ qs[b, h] / np.sqrt(d)
            e = np.exp(e - e.max())
            att[b, h] = e @ vv / e.sum()
    oo = held(att.reshape(rows, -1)) @ w64["o"].T
    t2 = t1 + oo
    gu = held(norm64(t2, np64(gammas[1]), 1e-6)) @ w64["gate_up"].T
    want = held(swiglu64(gu)) @ w64["down"].T
    # A value near a border may land a step away where its inputs differ by a rounding. A step is 1/127 of
    # its row's largest value, at most 5 standard deviations here: 1/25 of one. bf16 rounds o and gate|up by
    # 2^-8 of a value, 1/10 of a step of it, so up to a fifth of the values move by a step: 1/25 sqrt(1/5) < 0.02
    # of the products' 2-norm twice over (the second SwiGLU doubles what comes in); f32's roundings, 2^-24
    # by some hundred, move one value in 10^4: a hundredth of that.
    rel = np.linalg.norm(np64(down) - want) / np.linalg.norm(want)
    assert rel < (0.08 if out == torch.bfloat16 else 2e-3), rel


def test_offsets_past_32_bits(dev):
    """Rows whose elements lie past 2^31 and 2^32 of their buffers: rows, weights, results."""
    rng = np.random.default_rng(0)
    far = 1 << 26
    for rows in (40, 16, 70):  # 40 rows of 2^26: the last begins past 2^31
        x = torch.zeros(rows, far, dtype=torch.bfloat16, device="cuda")[:, :640]
        x.copy_(torch.from_numpy(some(rng, rows, 640)))
        q, s = rows_of(rows, 640, torch.int8), torch.zeros(rows, device="cuda")
        dev.quant_rows(q, s, x)
        same(q, s, stepped(np64(x)))
        del x
        a = torch.zeros(rows, far, dtype=torch.int8, device="cuda")[:, :640]
        a.copy_(q)
        w = torch.zeros(130, 1 << 25, dtype=torch.int8, device="cuda")[:, :640]
        w.copy_(ints(rng, 130, 640))
        w_s = torch.rand(130, device="cuda") + 0.1
        out = torch.zeros(rows, far, dtype=torch.bfloat16, device="cuda")[:, :130]
        dev.matmul_i8(out, a, s, w, w_s)
        want = product(a, s, w, w_s, None, torch.bfloat16)
        assert torch.equal(out.cpu().nan_to_num(7), want.nan_to_num(7))
        del a, w, out


def test_many_rows_and_few_channels(dev):
    rng = np.random.default_rng(3)
    a, w = ints(rng, 70001, 64), ints(rng, 3, 64)
    a_s, w_s = torch.rand(70001, device="cuda"), torch.rand(3, device="cuda")
    out = torch.zeros(70001, 3, device="cuda")
    dev.matmul_i8(out, a, a_s, w, w_s)
    assert torch.equal(out.cpu(), product(a, a_s, w, w_s, None, torch.float32))
    x = torch.from_numpy(some(rng, 70001, 40)).cuda()
    q, s = rows_of(70001, 40, torch.int8), torch.zeros(70001, device="cuda")
    dev.quant_rows(q, s, x)
    same(q, s, stepped(np64(x)))


def test_columns_of_one_buffer(dev):
    """q, scales and results at every offset that their type allows: values that do not begin at 16 bytes."""
    rng = np.random.default_rng(4)
    for off in (1, 2, 3, 4, 8):
        for width in (129, 1024, 5000):
            x = rows_of(6, width + 16, torch.float32)[:, off:off + width]
            r, t = (rows_of(6, width + 16, torch.float32)[:, off:off + width] for _ in range(2))
            x.copy_(torch.from_numpy(some(rng, 6, width)))
            r.copy_(torch.from_numpy(some(rng, 6, width)))
            g = torch.ones(width + 8, device="cuda").bfloat16()[off:off + width]
            q, s = rows_of(6, width + 16, torch.int8)[:, off:off + width], torch.zeros(6 + off, device="cuda")[off:]
            dev.add_norm_quant(q, s, x, g, residual=r, total=t)
            assert torch.equal(t, x + r)
            same(q, s, stepped(norm64(np64(t), np64(g), 1e-6)))
        for rows in (3, 50, 300):
            a, w = ints(rng, rows, 300, 4), ints(rng, 77, 300, 4)
            a_s, w_s, b = (torch.rand(n + off, device="cuda")[off:] for n in (rows, 77, 77))
            for dtype in (torch.float32, torch.bfloat16):
                out = torch.zeros(rows, 96, dtype=dtype, device="cuda")[:, off:off + 77]
                dev.matmul_i8(out, a, a_s, w, w_s, bias=b)
                assert torch.equal(out.cpu(), product(a, a_s, w, w_s, b, dtype))


def test_refused_tensors_are_left_alone(dev):
    f = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    i8, bf = torch.int8, torch.bfloat16
    q, s, x, out = torch.full((4, 64), 9, dtype=i8, device="cuda"), torch.full((4,), 9.0, device="cuda"), f(4, 64), torch.full((4, 5), 9.0, device="cuda")
    w, w_s, g = f(5, 64, t=i8), f(5), f(64, t=bf)
    calls = [
        (lambda: dev.quant_rows(q, s, x.half()), _lib.ERR_ARG), (lambda: dev.quant_rows(q, s, x.double()), _lib.ERR_ARG),
        (lambda: dev.quant_rows(q.int(), s, x), _lib.ERR_ARG), (lambda: dev.quant_rows(q, s, f(4, 65)), _lib.ERR_SHAPE),
        (lambda: dev.quant_rows(q, f(5), x), _lib.ERR_SHAPE), (lambda: dev.quant_rows(q, s.double(), x), _lib.ERR_ARG),
        (lambda: dev.quant_rows(q, s, x.cpu()), _lib.ERR_ARG), (lambda: dev.quant_rows(q[0], s, x), _lib.ERR_SHAPE),
        (lambda: dev.quant_rows(q, s, f(64, 4).T), _lib.ERR_ARG), (lambda: dev.quant_rows(q[:, ::2], s, x[:, ::2]), _lib.ERR_ARG),
        (lambda: dev.quant_rows(f(64, 4, t=i8).T, s, x), _lib.ERR_ARG), (lambda: dev.quant_rows(q, f(8)[::2], x), _lib.ERR_ARG),
        (lambda: dev.swiglu_quant(q, s, x), _lib.ERR_SHAPE), (lambda: dev.swiglu_quant(q, s, f(4, 129)), _lib.ERR_SHAPE),
        (lambda: dev.add_norm_quant(q, s, x, g.float()), _lib.ERR_ARG), (lambda: dev.add_norm_quant(q, s, x, g[:63]), _lib.ERR_SHAPE),
        (lambda: dev.add_norm_quant(q, s, x, g, residual=x.bfloat16()), _lib.ERR_ARG),
        (lambda: dev.add_norm_quant(q, s, x, g, residual=f(4, 63)), _lib.ERR_SHAPE), (lambda: dev.add_norm_quant(q, s, x, g, total=f(3, 64)), _lib.ERR_SHAPE),
        (lambda: dev.add_norm_quant(q, s, x, g, eps=-1.0), _lib.ERR_ARG), (lambda: dev.add_norm_quant(q, s, x, None), _lib.ERR_ARG),
        (lambda: dev.add_norm_quant(q, s, x, g, total=x.as_strided((4, 64), (32, 1)), residual=f(4, 64)), _lib.ERR_SHAPE),
        (lambda: dev.matmul_i8(out, q.float(), s, w, w_s), _lib.ERR_ARG), (lambda: dev.matmul_i8(out.half(), q, s, w, w_s), _lib.ERR_ARG),
        (lambda: dev.matmul_i8(out, q, s, f(5, 63, t=i8), w_s), _lib.ERR_SHAPE), (lambda: dev.matmul_i8(f(4, 6), q, s, w, w_s), _lib.ERR_SHAPE),
        (lambda: dev.matmul_i8(out, q, f(3), w, w_s), _lib.ERR_SHAPE), (lambda: dev.matmul_i8(out, q, s, w, f(4)), _lib.ERR_SHAPE),
        (lambda: dev.matmul_i8(out, q, s, w, w_s, bias=f(4)), _lib.ERR_SHAPE), (lambda: dev.matmul_i8(out, q, s, w, w_s, bias=f(5, t=bf)), _lib.ERR_ARG),
        (lambda: dev.matmul_i8(out, q, s, f(64, 5, t=i8).T, w_s), _lib.ERR_ARG),
        (lambda: dev.matmul_i8(out, q[:, 1:], s, w[:, 1:], w_s), _lib.ERR_ARG),                     # rows that do not begin at 16 bytes
        (lambda: dev.matmul_i8(out, q[:, :60].contiguous(), s, w[:, :60], w_s), _lib.ERR_ARG),        # nor go on at 16
        (lambda: dev.matmul_i8(out, q[:, :0], s, w[:, :0], w_s), _lib.ERR_ARG),                            # no k: an empty tensor has no address
    ]
    for i, (call, code) in enumerate(calls):
        with pytest.raises(myos.MyosError) as e:
            call()
        assert e.value.code == code, (i, e.value)
    with pytest.raises(TypeError):
        dev.matmul_i8(out, q, s, w)
    with pytest.raises(TypeError):
        dev.quant_rows(q, s, x, scale=1.0)
    assert bool((q == 9).all()) and bool((s == 9).all()) and bool((out == 9).all())


def test_rows_behind_the_last_are_left(dev):
    """Results and 8-bit rows end with the rows and channels that were asked for."""
    rng = np.random.default_rng(6)
    for rows in (1, 9, 33, 100, 257):
        a, w = ints(rng, rows, 256), ints(rng, 131, 256)
        a_s, w_s = torch.rand(rows, device="cuda"), torch.rand(131, device="cuda")
        buf = torch.full((rows + 300, 300), 5.0, device="cuda")
        dev.matmul_i8(buf[:rows, :131], a, a_s, w, w_s)
        assert bool((buf[rows:] == 5).all()) and bool((buf[:, 131:] == 5).all())
        x = torch.from_numpy(some(rng, rows, 500)).cuda()
        q, s = torch.full((rows + 5, 512), 5, dtype=torch.int8, device="cuda"), torch.full((rows + 5,), 5.0, device="cuda")
        dev.quant_rows(q[:rows, :500], s[:rows], x)
        assert bool((q[rows:] == 5).all()) and bool((q[:, 500:] == 5).all()) and bool((s[rows:] == 5).all())


def test_the_same_call_again_gives_the_same_bits(dev):
    rng = np.random.default_rng(7)
    for rows, k, n in ((3, 5120, 1000), (64, 8960, 1536), (300, 5120, 2000)):
        a, w = ints(rng, rows, k), ints(rng, n, k)
        a_s, w_s = torch.rand(rows, device="cuda"), torch.rand(n, device="cuda")
        outs = [torch.zeros(rows, n, device="cuda") for _ in range(20)]
        for o in outs:
            dev.matmul_i8(o, a, a_s, w, w_s)
        assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("width", [129, 1025, 1520, 2047, 2056, 5000, 5120, 8192, 13824, 16383, 16384, 16392])
def test_many_rows(dev, width, x):
    """The forms that keep several rows on their way at once: 515 rows, some of them marked, zero or alike."""
    dtype = torch.float32 if x == "f32" else torch.bfloat16
    rng = np.random.default_rng(width)
    rows, half = 515, width // 2
    a = some(rng, rows, width)
    a[7, width // 3], a[511, width - 1] = np.nan, -np.inf
    a[100], a[101] = 3.0, -a[102]
    pad = -width % 8
    t = rows_of(rows, width, dtype, pad)
    t.copy_(torch.from_numpy(a))
    q, s = rows_of(rows, width, torch.int8, pad), torch.zeros(rows, device="cuda")
    dev.quant_rows(q, s, t)
    same(q, s, stepped(np64(t)))
    res = rows_of(rows, width, torch.float32, pad)
    res.copy_(torch.from_numpy(some(rng, rows, width)))
    want = t.float() + res
    g = torch.from_numpy(rng.standard_normal(width)).cuda().bfloat16()
    dev.add_norm_quant(q, s, t, g, residual=res, total=res)
    assert torch.equal(res.nan_to_num(1.0), want.nan_to_num(1.0))
    same(q, s, stepped(norm64(np64(want), np64(g), 1e-6)))
    if width % 2 == 0:
        q2 = rows_of(rows, half, torch.int8, -half % 8)
        dev.swiglu_quant(q2, s, t)
        same(q2, s, stepped(swiglu64(np64(t))))
    if width <= 8192:  # gate and up of this width each
        gu = torch.cat([t, t.flip(1)], 1)
        dev.swiglu_quant(q, s, gu)
        same(q, s, stepped(swiglu64(np64(gu))))


@pytest.mark.parametrize("rows,k,channels", [(4097, 13824, 700), (1300, 4100, 3000), (20000, 260, 300), (515, 1000, 20000)])
def test_row_tiles_in_groups(dev, rows, k, channels):
    """Row tiles that pass the weights in more than one group, ragged last tiles among them."""
    rng = np.random.default_rng(rows)
    a, w = ints(rng, rows, k, -k % 16), ints(rng, channels, k, -k % 16)
    a_s, w_s = torch.rand(rows, device="cuda"), torch.rand(channels, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.zeros(rows, channels, dtype=dtype, device="cuda")
        dev.matmul_i8(out, a, a_s, w, w_s)
        assert torch.equal(out.cpu(), product(a, a_s, w, w_s, None, dtype))


def test_calls_on_two_streams_at_once(dev):
    """Large and small products and rows interleaved on two streams: each its own results, again and again."""
    rng = np.random.default_rng(9)
    jobs = []
    for rows, k, n in ((300, 2048, 4000), (64, 8960, 1536), (3, 5120, 7168), (1024, 640, 2000)):
        a, w = ints(rng, rows, k), ints(rng, n, k)
        a_s, w_s = torch.rand(rows, device="cuda"), torch.rand(n, device="cuda")
        x = torch.from_numpy(some(rng, rows, k)).cuda()
        q, s = rows_of(rows, k, torch.int8), torch.zeros(rows, device="cuda")
        dev.quant_rows(q, s, x)
        want = torch.zeros(rows, n, device="cuda")
        dev.matmul_i8(want, a, a_s, w, w_s)
        assert torch.equal(want.cpu(), product(a, a_s, w, w_s, None, torch.float32))
        jobs.append((a, a_s, w, w_s, x, want, q.clone(), s.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        a, a_s, w, w_s, x, want, q, s = jobs[i % 4 if i % 2 else 3 - i % 4]
        o, q2, s2 = torch.empty_like(want), torch.empty_like(q), torch.empty_like(s)
        outs.append((o, want, q2, q, s2, s))
    torch.cuda.synchronize()
    for i, (o, want, q2, q, s2, s) in enumerate(outs):
        a, a_s, w, w_s, x = jobs[i % 4 if i % 2 else 3 - i % 4][:5]
        dev.matmul_i8(o, a, a_s, w, w_s, stream=streams[i % 2])
        dev.quant_rows(q2, s2, x, stream=streams[i % 2])
    torch.cuda.synchronize()
    for o, want, q2, q, s2, s in outs:
        assert torch.equal(o, want) and torch.equal(q2, q) and torch.equal(s2, s)
