"""The 8-bit projections at the ends of f32's range: gates below the normal numbers,
rows past the largest, borders between steps. Bit for bit against 64 bits, as in test_gpu_i8.
The status, and kernels one after another."""
import numpy as np
import pytest

from test_gpu_i8 import norm64, np64, rows_of, same, stepped, swiglu64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
T = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    from myos import dev as m

    return m


def checked_swiglu(dev, x, want=stepped):
    """swiglu_quant of x [rows, 2 width], its rows 16 bytes apart from their like, against `want` of y."""
    rows, width = x.shape[0], x.shape[1] // 2
    q, s = rows_of(rows, width, torch.int8, -width % 16), torch.zeros(rows, device="cuda")
    dev.swiglu_quant(q, s, x)
    same(q, s, want(swiglu64(np64(x))))


# a warp a row, a block, values in shared memory (from 512 rows on), one value at a time
@pytest.mark.parametrize("rows,width", [(3, 2), (6, 96), (6, 101), (6, 1536), (5, 8200), (515, 2600), (515, 101), (3, 40000)])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_subnormal_gates(dev, x, rows, width):
    """Gates below f32's normal numbers, brought back by large up values; a large gate and such an up value."""
    rng = np.random.default_rng(width)
    unit, most = (2.0**-149, 2**12) if x == "f32" else (2.0**-133, 2**6)
    gate = rng.integers(1, most, (rows, width)) * unit * rng.choice([-1, 1], (rows, width))
    up = np.exp2(rng.uniform(100, 127, (rows, width)))
    gate[0], up[0] = 3 * unit, 2.0**100 * rng.choice([0.5, 0.75, 1.0], width)  # a row of one gate
    other = rng.random((rows, width)) < 0.5  # the other rows: half of them ordinary values of the same size
    other[:2] = False
    size = 0.5 * np.abs(gate * up).max(1, keepdims=True)
    gate = np.where(other, rng.standard_normal((rows, width)), gate)
    up = np.where(other, size * rng.standard_normal((rows, width)), up)
    far = rng.random((rows, width)) < 0.1
    far[:2] = False
    gate, up = np.where(far, np.exp2(rng.uniform(100, 127, (rows, width))), gate), np.where(far, rng.integers(1, most, (rows, width)) * unit, up)
    t = torch.from_numpy(np.concatenate([gate, up], 1)).cuda().to(T[x])
    assert bool((t[:2, :width].abs() < 2.0**-126).all() and (t[:, :width] != 0).all())
    checked_swiglu(dev, t)


def test_gates_whose_products_f32_loses(dev):
    for g, u, q, s in (((1, 1), (2.0**127, 2.0**126), (127, 64), 2.0**-23 / 127), ((3, 4), (2.0**100, 0.9 * 2.0**100), (106, 127), 2.0**-47 * 0.9 / 127)):
        x = torch.tensor([[g[0] * 2.0**-149, g[1] * 2.0**-149, *u]], dtype=torch.float64).float().cuda()
        got, scale = torch.zeros(1, 2, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
        dev.swiglu_quant(got, scale, x)
        assert got.tolist() == [list(q)] and scale.item() == pytest.approx(s, rel=2.0**-23)


# ---------------------------------------------------------------- past f32
PAST = 2.0**128 - 2.0**103  # from here on f32 has no finite number


def marked(y):
    """`stepped`, a row with a y past f32 marked."""
    q, s = stepped(y)
    bad = ~(np.abs(y) < PAST).all(1)
    q[bad], s[bad] = 0, np.nan
    return q, s


@pytest.mark.parametrize("width", [96, 101, 1536, 8200, 40000])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_norms_past_f32(dev, x, width):
    """y past f32 where gamma * total is not: such rows are marked, those that end just below are not."""
    rows, at = 60, width // 3
    ratio = np.concatenate([np.linspace(0.1, 9, 30), 2 * (1 + np.arange(-15, 15) * 2.0**-9)])  # y at the column, in 2^127
    t = np.full((rows, width), 2.0**-10)
    t[:, at] *= np.sqrt(ratio**2 * (width - 1) / (width - ratio**2))
    t = torch.from_numpy(t).cuda().to(T[x])
    g = torch.ones(width, device="cuda").bfloat16()
    g[at] = 2.0**127
    y = norm64(np64(t), np64(g), 0.0)
    past = ~(np.abs(y) < PAST).all(1)
    assert 10 < past.sum() < 50 and np.isfinite(y).all() and bool((t.float() * g.float()).isfinite().all())
    q, s = rows_of(rows, width, torch.int8, -width % 16), torch.zeros(rows, device="cuda")
    dev.add_norm_quant(q, s, t, g, eps=0.0)
    same(q, s, marked(y))
    total = torch.zeros(rows, width, device="cuda")
    dev.add_norm_quant(q, s, t, g, residual=torch.zeros(rows, width, device="cuda"), total=total, eps=0.0)
    assert torch.equal(total, t.float())
    same(q, s, marked(y))


@pytest.mark.parametrize("rows", [300, 3000])
@pytest.mark.parametrize("width", [64, 101, 1536, 2600])
def test_swiglu_next_to_the_largest_number(dev, rows, width):
    """y on either side of f32's end, closer to it than an f32 product is to y."""
    rng = np.random.default_rng(rows + width)
    gate, up = rng.standard_normal((rows, width)), 1e37 * rng.standard_normal((rows, width))
    at = rng.integers(0, width, rows)
    g = rng.uniform(1.3, 4, rows).astype(np.float32).astype(np.float64)
    u = (PAST / (g / (1 + np.exp(-g)))).astype(np.float32)
    u = (u.view(np.int32) + rng.integers(-2, 3, rows).astype(np.int32)).view(np.float32)
    gate[np.arange(rows), at], up[np.arange(rows), at] = g, u * rng.choice([-1, 1], rows)
    t = torch.from_numpy(np.concatenate([gate, up], 1).astype(np.float32)).cuda()
    y = np.abs(swiglu64(np64(t))).max(1)
    assert 0.3 < (y < PAST).mean() < 0.7 and (np.abs(y / PAST - 1) < 2.0**-20).all()
    checked_swiglu(dev, t, marked)


# ---------------------------------------------------------------- on a border
@pytest.mark.parametrize("width", [96, 101, 1536, 8200, 40000])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_norms_on_a_border(dev, x, width):
    """Rows whose factor is 1/5, which f64 does not hold, and whose y in f64 is on a border all the same: each
    product is rounded, so a tie is one, and goes to the even step."""
    rng = np.random.default_rng(width)
    t = np.full((4, width), 5.0)
    pairs = rng.permutation(width - 1)[: (width - 1) // 2 * 2] + 1
    t[:, pairs[::2]], t[:, pairs[1::2]] = 1.0, 7.0  # 1 + 49 = 25 + 25
    t *= rng.choice([-1, 1], (4, width))
    g = 5.0 * rng.integers(0, 26, width) * rng.choice([-1, 1], width) / np.where(t[0] == 5, 5, 1)
    g[0] = 254.0  # of a total of 5: the scale is 2
    g = np.where(np.abs(g) * np.abs(t[0]) > 1270, 5.0, g)
    t, g = torch.from_numpy(t).cuda().to(T[x]), torch.from_numpy(g).cuda().bfloat16()
    y = norm64(np64(t), np64(g), 0.0)
    assert (np.abs(y).max(1) == 254).all() and ((np.abs(y) % 2) == 1).sum() > width // 4
    q, s = rows_of(4, width, torch.int8, -width % 16), torch.zeros(4, device="cuda")
    dev.add_norm_quant(q, s, t, g, eps=0.0)
    same(q, s, stepped(y))


# ---------------------------------------------------------------- the status
def test_the_status_waits_for_every_stream(dev):
    """A product on a stream that the default stream does not wait for is over when the status is known."""
    a = torch.ones(4096, 4096, dtype=torch.int8, device="cuda")
    one, out = torch.ones(4096, device="cuda"), torch.zeros(4096, 4096, device="cuda")
    dev.matmul_i8(out, a, one, a, one)
    dev.matmul_i8_status()
    side = torch.cuda.Stream()
    for _ in range(1000):
        dev.matmul_i8(out, a, one, a, one, stream=side)
    dev.matmul_i8_status()
    assert side.query()
    assert bool((out == 4096).all())


# ---------------------------------------------------------------- one kernel after another
@pytest.mark.parametrize("rows", [1, 5, 8, 12, 16, 40, 300])
@pytest.mark.parametrize("k,channels", [(100, 600), (1000, 333), (640, 1024), (4090, 512)])
def test_products_of_what_the_kernel_before_wrote(dev, rows, k, channels):
    """Weights and rows in 8 bits, then their product, again and again over the same buffers: each product
    reads what the calls before it have just written."""
    rng = np.random.default_rng(rows + k)
    n = 12
    x, w = (torch.from_numpy(rng.standard_normal((n, m, k)).astype(np.float32)).cuda() for m in (rows, channels))
    q, s = rows_of(rows, k, torch.int8, -k % 16), torch.zeros(rows, device="cuda")
    wq, ws = rows_of(channels, k, torch.int8, -k % 16), torch.zeros(channels, device="cuda")
    out = torch.zeros(n, rows, channels, device="cuda")
    want = []
    for i in range(n):
        a, b = stepped(np64(x[i])), stepped(np64(w[i]))
        y = (a[0].astype(np.int64) @ b[0].astype(np.int64).T).astype(np.float32) * a[1][:, None] * b[1][None, :]
        want.append(torch.from_numpy(y))

    def chain(order):
        for i in order:
            dev.quant_rows(wq, ws, w[i])
            dev.quant_rows(q, s, x[i])
            dev.matmul_i8(out[i], q, s, wq, ws)
            dev.quant_rows(q, s, x[(i + 1) % n])  # the rows alone anew, the weights as they are
            dev.quant_rows(q, s, x[i])
            dev.matmul_i8(out[i], q, s, wq, ws)

    chain(range(n))
    for i in range(n):
        assert torch.equal(out[i].cpu(), want[i])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain(reversed(range(n)))
    for _ in range(3):
        out.zero_()
        for _ in range(5):
            g.replay()
        for i in range(n):
            assert torch.equal(out[i].cpu(), want[i])
