"""Calls of the paged serving operators at the edges of what their documentation
allows: histories of few tokens.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged import check_logits, dev, i32, plain_logits  # noqa: E402,F401

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
