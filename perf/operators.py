"""The operators of one serving step over a paged key-value cache, as they are timed.

tables   block tables, slot maps and row positions from the requests' lengths
store    per-head norm and rotation of q and k, K and V stored into the cache's pages
attn     attention of one new token per sequence over the pages
logits   penalties for repeated tokens, biases and grammar masks on logits, and the greedy id

`run` computes them in plain torch (own = False) or with myos.dev (own = True).
"""
import math
import sys

import numpy as np
import torch

own = False

PKG = "an-operating-system-for-ai-models-and-tensor-inference_b200"
WORK_BYTES = 16 << 20  # MYOS_PAGED_WORK_BYTES


def _dev():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from myos import dev

    return dev


# ---------------------------------------------------------------- cases
def listed():
    qwen, large = {"hq": 12, "hkv": 2, "d": 128}, {"hq": 40, "hkv": 8, "d": 128}
    return [
        # one chat request in decode: every launch is latency
        {"name": "tables 1 decode", "op": "tables", "nseq": 1, "page": 16, "max_len": 4352, "prompts": 0.0, "new": 1},
        # a decode step of the batched workload, 64 x (512 + 128)
        {"name": "tables 64 decode", "op": "tables", "nseq": 64, "page": 16, "max_len": 640, "prompts": 0.0, "new": 1},
        # a busy server: decode rows between chunks of prompts
        {"name": "tables 1021 mixed", "op": "tables", "nseq": 1021, "page": 32, "max_len": 8192, "prompts": 0.3, "new": 777},
        # one token of the 1.5B heads, f32 cache, no per-head norm
        {"name": "store 1 row f32", "op": "store", "rows": 1, "pad": 0, **qwen, "rot": 128, "norm": False, "kv": "f32", "page": 16, "nhd": False},
        # a decode step of 64 sequences of the 14B heads with per-head norms, three of the rows padding
        {"name": "store 64 rows bf16", "op": "store", "rows": 64, "pad": 3, **large, "rot": 128, "norm": True, "kv": "bf16", "page": 16, "nhd": False},
        # prompts of many requests in one chunk
        {"name": "store 16001 rows bf16", "op": "store", "rows": 16001, "pad": 0, **large, "rot": 128, "norm": True, "kv": "bf16", "page": 32, "nhd": False},
        # one long chat: 4096 prompt tokens and the first generated one
        {"name": "attn 1 x 4097 bf16", "op": "attn", "nseq": 1, "min_len": 4097, "max_len": 4097, **qwen, "kv": "bf16", "page": 16, "window": 0, "nhd": False},
        # the batched workload at its end, f32 cache
        {"name": "attn 64 x 640 f32", "op": "attn", "nseq": 64, "min_len": 512, "max_len": 640, **qwen, "kv": "f32", "page": 16, "window": 0, "nhd": False},
        # long and short contexts side by side, 14B heads
        {"name": "attn 32 ragged bf16", "op": "attn", "nseq": 32, "min_len": 0, "max_len": 32768, **large, "kv": "bf16", "page": 16, "window": 0, "nhd": False},
        # one sequence, penalties and the greedy id
        {"name": "logits 1", "op": "logits", "rows": 1, "vocab": 151936, "history": 256, "bias": 0, "mask": False},
        # a batch with every control in use
        {"name": "logits 64 all", "op": "logits", "rows": 64, "vocab": 152064, "history": 4096, "bias": 300, "mask": True},
        # a small odd vocabulary, many rows
        {"name": "logits 333 odd", "op": "logits", "rows": 333, "vocab": 32003, "history": 1000, "bias": 5, "mask": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "store", "attn", "attn", "logits"])
    page = rng.choice([8, 16, 16, 32, 64])
    hq, hkv, d = rng.choice([(12, 2, 128), (40, 8, 128), (28, 4, 128), (8, 8, 64), (32, 8, 64), (5, 1, 80), (16, 4, 256)])
    kv = rng.choice(["f32", "bf16"])
    nhd = rng.random() < 0.3
    if op == "tables":
        return {"op": op, "nseq": _log(rng, 1, 1021), "page": page, "max_len": _log(rng, 64, 8192), "prompts": round(rng.uniform(0, 0.3), 3), "new": _log(rng, 1, 777)}
    if op == "store":
        rows = _log(rng, 1, 16001 * 40 // max(40, hq) // (2 if d > 128 else 1))
        return {"op": op, "rows": rows, "pad": min(rows - 1, rng.randrange(4)), "hq": hq, "hkv": hkv, "d": d, "rot": rng.choice([d, d, d // 2 // 8 * 8]), "norm": rng.random() < 0.5, "kv": kv, "page": page, "nhd": nhd}
    if op == "attn":
        nseq = _log(rng, 1, 128)
        most = 32 * 32768 * 8 * 128 * 4 // 5 // (nseq * hkv * d * (4 if kv == "f32" else 2))
        max_len = _log(rng, 1, max(1, min(32768, most)))
        return {"op": op, "nseq": nseq, "min_len": rng.choice([0, max_len // 2]), "max_len": max_len, "hq": hq, "hkv": hkv, "d": d, "kv": kv, "page": page, "window": rng.choice([0, 0, 0, 1000]), "nhd": nhd}
    rows = _log(rng, 1, 333)
    vocab = _log(rng, 500, min(152064, 152064 * 64 // rows))
    return {"op": op, "rows": rows, "vocab": vocab, "history": _log(rng, 1, 4096), "bias": rng.choice([0, 5, min(300, vocab // 2)]), "mask": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _lens(rng, n, lo, hi):
    """Lengths between lo and hi; a wide range is filled evenly over its logarithm and its values."""
    if hi < 2 * max(1, lo):
        v = rng.integers(lo, hi + 1, n)
    else:
        a = np.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 0.5), n)).astype(np.int64)
        v = np.where(rng.random(n) < 0.4, a, rng.integers(max(lo, 1), hi + 1, n))
        if lo == 0 and n > 4:
            v[rng.integers(0, n)] = 0  # an empty row of a padded batch
    v[rng.integers(0, n)] = hi
    return v


def _rows(case):
    """Rows of a step: one for each request, 0.55 of the longest chunk for each prompt, and some to spare (a launch of fixed size)."""
    return case["nseq"] + int(0.55 * case["new"] * int(case["nseq"] * case["prompts"])) + 5


def _cache(gen, case, num_pages):
    shape = (num_pages, case["page"], case["hkv"], case["d"]) if case["nhd"] else (num_pages, case["hkv"], case["page"], case["d"])
    t = torch.float32 if case["kv"] == "f32" else torch.bfloat16
    k, v = (torch.empty(shape, dtype=t, device="cuda").normal_(generator=gen) for _ in range(2))
    return (k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)) if case["nhd"] else (k, v)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    zeros = lambda *n, t=torch.int32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    op, s = case["op"], {"case": case}
    if op == "tables":
        n, p, most = case["nseq"], case["page"], case["max_len"]
        ctx = rng.integers(1, most + 1, n)
        new, rows = np.ones(n, np.int64), _rows(case)
        chunk = rng.permutation(n) < int(n * case["prompts"])
        new[chunk] = rng.integers(1, case["new"] + 1, n)[chunk]
        ctx[chunk] = (ctx[chunk] // 2) * (rng.random(n)[chunk] < 0.5)
        new[rng.random(n) < 0.02] = 0
        new[0] = max(1, new[0])
        new = np.minimum(new, most)
        new = np.clip(rows - (np.cumsum(new) - new), 0, new)  # a step's token budget
        ctx = np.minimum(ctx, most - new)
        held = -(-ctx // p)
        blocks = -(-most // p)
        need = int((-(-(ctx + new) // p) - held).sum())
        free = need + int(rng.integers(0, n + 1)) if rng.random() < 0.7 else max(0, need - int(rng.integers(0, 4)))
        num_pages = int(held.sum()) + free
        pages = rng.permutation(num_pages)
        table = np.full((n, blocks), -1)
        table[np.arange(blocks)[None, :] < held[:, None]] = pages[: int(held.sum())]
        s.update(table=i32(table), ctx=i32(ctx), new=i32(new), free=i32(pages[int(held.sum()) :] if free else [0]), num_free=i32([free]), num_pages=num_pages)
        s.update(slots=zeros(rows, t=torch.int64), positions=zeros(rows), token_seq=zeros(rows), kv_lens=zeros(n), seq_starts=zeros(n + 1), result=zeros(2))
    elif op == "store":
        t, hq, hkv, d, p = case["rows"], case["hq"], case["hkv"], case["d"], case["page"]
        num_pages = -(-t // p) + 5
        live = t - case["pad"]
        slots = np.full(t, -1, np.int64)
        pages = rng.permutation(num_pages)
        slots[:live] = pages[np.arange(live) // p] * p + np.arange(live) % p  # prompts fill their pages in order
        positions = np.zeros(t, np.int64)
        positions[:live] = (int(rng.integers(0, 2000)) + np.arange(live)) % 32768
        half = case["rot"] // 2
        angle = torch.arange(32768, dtype=torch.float64, device="cuda")[:, None] * (1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half))[None, :]
        s["k"], s["v"] = _cache(gen, case, num_pages)
        s.update(qkv=torch.randn(t, (hq + 2 * hkv) * d, device="cuda", generator=gen), q_out=torch.zeros(t, hq, d, device="cuda"))
        s.update(positions=i32(positions), slots=torch.from_numpy(slots).cuda(), cos=angle.cos().float(), sin=angle.sin().float(), q_gamma=None, k_gamma=None)
        if case["norm"]:
            s["q_gamma"], s["k_gamma"] = ((1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).bfloat16() for _ in range(2))
    elif op == "attn":
        n, hq, hkv, d, p = case["nseq"], case["hq"], case["hkv"], case["d"], case["page"]
        lens = _lens(rng, n, case["min_len"], case["max_len"])
        held, blocks = -(-lens // p), -(-case["max_len"] // p)
        num_pages = int(held.sum()) + 3
        table = np.full((n, blocks), -1)
        table[np.arange(blocks)[None, :] < held[:, None]] = rng.permutation(num_pages)[: int(held.sum())]
        s["k"], s["v"] = _cache(gen, case, num_pages)
        s.update(q=torch.randn(n, hq, d, device="cuda", generator=gen) * 1.5, table=i32(table), lens=i32(lens))
        s.update(out=torch.zeros(n, hq, d, device="cuda"), lse=torch.zeros(n, hq, device="cuda"), work=torch.zeros(WORK_BYTES, dtype=torch.uint8, device="cuda"))
    else:
        n, vocab, most = case["rows"], case["vocab"], case["history"]
        total = rng.integers(1, most + 1, n)
        total[rng.integers(0, n)] = most
        history = np.minimum(vocab * rng.random((n, most)) ** 3, vocab - 1)  # common tokens come often
        f32 = lambda lo, hi: torch.from_numpy(rng.uniform(lo, hi, n).astype(np.float32)).cuda()  # noqa: E731
        s.update(logits=torch.randn(n, vocab, device="cuda", generator=gen) * 4, out=torch.zeros(n, vocab, device="cuda"), ids=zeros(n))
        s.update(history=i32(history), prompt_lens=i32(rng.integers(0, total + 1)), hist_lens=i32(total), repetition=f32(1.0, 1.5), frequency=f32(0.0, 0.6), presence=f32(0.0, 0.6))
        s.update(bias_starts=None, bias_ids=None, bias_vals=None, mask=None, mask_rows=None)
        if case["bias"]:
            each = rng.integers(0, case["bias"] + 1, n)
            ids = np.concatenate([rng.choice(vocab, e, replace=False) for e in each] + [np.zeros(1, np.int64)])
            s.update(bias_starts=i32(np.concatenate([[0], np.cumsum(each)])), bias_ids=i32(ids), bias_vals=torch.from_numpy(rng.uniform(-8, 8, ids.size).astype(np.float32)).cuda())
        if case["mask"]:
            groups = max(1, n // 2)
            words = rng.integers(0, 1 << 32, (groups, -(-vocab // 32)), dtype=np.uint64).astype(np.uint32)
            words[rng.random(words.shape) < 0.5] = 0  # a grammar state allows a part of the vocabulary
            s.update(mask=torch.from_numpy(words.view(np.int32)).cuda(), mask_rows=i32(rng.integers(-1, groups, n)))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _run_own(s, op)
    return {"tables": _tables, "store": _store, "attn": _attn, "logits": _logits}[op](s)


def _run_own(s, op):
    dev, c = _dev(), s["case"]
    if op == "tables":
        dev.paged_tables(s["table"], s["ctx"], s["new"], s["free"], s["num_free"], c["page"], s["num_pages"], s["slots"], s["positions"], s["token_seq"], s["kv_lens"], s["seq_starts"], s["result"])
        return {n: s[n] for n in ("table", "slots", "positions", "token_seq", "kv_lens", "seq_starts", "result")}
    if op == "store":
        kv = dev.PagedKV(s["k"], s["v"])
        dev.qk_norm_rope_store(s["q_out"], s["qkv"], kv, s["positions"], s["slots"], s["cos"], s["sin"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=1e-6)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if op == "attn":
        kv = dev.PagedKV(s["k"], s["v"])
        dev.paged_attention(s["out"], s["q"], kv, s["table"], s["lens"], s["work"], window=c["window"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    dev.logit_controls(
        s["out"], s["logits"], history=s["history"], prompt_lens=s["prompt_lens"], hist_lens=s["hist_lens"], repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
        bias_starts=s["bias_starts"], bias_ids=s["bias_ids"], bias_vals=s["bias_vals"], mask=s["mask"], mask_rows=s["mask_rows"], ids=s["ids"])  # fmt: skip
    return {"logits": s["out"], "ids": s["ids"]}


def _tables(s):
    c, table = s["case"], s["table"]
    p, (n, blocks), rows = c["page"], table.shape, s["slots"].numel()
    ctx, new = s["ctx"].long(), s["new"].long()
    end = torch.cumsum(new, 0)
    start = end - new
    held = (ctx + p - 1) // p
    need = torch.where(new > 0, (ctx + new + p - 1) // p - held, 0)
    fits = (new == 0) | ((ctx + new <= blocks * p) & (end <= rows))
    need = torch.where(fits, need, 0)
    upto = torch.cumsum(need, 0)
    free = s["num_free"].long()
    ok = fits & ((need == 0) | (upto <= free))
    need = torch.where(ok, need, 0)
    before = upto - need  # of an admitted request: the pages taken by those in front of it
    col = torch.arange(blocks, device="cuda")[None, :]
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    at = (free - 1 - before[:, None] - (col - held[:, None])).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(end, r, right=True)
    live = b < n
    b = b.clamp(max=n - 1)
    good = live & ok[b]
    pos = torch.where(good, ctx[b] + r - start[b], 0)
    page = table[b, (pos // p).clamp(max=blocks - 1)].long()
    slots = torch.where(good & (page >= 0) & (page < s["num_pages"]), page * p + pos % p, -1)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), end]).clamp(max=rows)
    result = torch.cat([free - need.sum(), (~ok).sum()[None]])
    i = torch.int32
    return {"table": table, "slots": slots, "positions": pos.to(i), "token_seq": torch.where(live, b, -1).to(i), "kv_lens": torch.where(ok, ctx + new, ctx).to(i), "seq_starts": starts.to(i), "result": result.to(i)}


def _turned(x, gamma, cos, sin):
    """x [T, H, d] f32 -> norm over d (with a gamma), then the rotation of the first 2 * cos.shape[-1] values."""
    if gamma is not None:
        x = gamma.float() * (x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)))
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half : 2 * half]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half :]], -1)


def _store(s):
    c = s["case"]
    t, hq, hkv, d, p = c["rows"], c["hq"], c["hkv"], c["d"], c["page"]
    q, k, v = s["qkv"].view(t, hq + 2 * hkv, d).split([hq, hkv, hkv], 1)
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    live = t - c["pad"]
    page, at = s["slots"][:live] // p, s["slots"][:live] % p
    s["k"][page, :, at] = _turned(k, s["k_gamma"], cos, sin)[:live].to(s["k"].dtype)
    s["v"][page, :, at] = v[:live].to(s["v"].dtype)
    return {"q": _turned(q, s["q_gamma"], cos, sin), "k": s["k"], "v": s["v"]}


def _attn(s):
    c = s["case"]
    n, hq, hkv, d, p = c["nseq"], c["hq"], c["hkv"], c["d"], c["page"]
    pages = s["table"].clamp(min=0).long()
    k, v = (x[pages].transpose(1, 2).reshape(n, hkv, -1, d).float() for x in (s["k"], s["v"]))
    j, lens = torch.arange(k.shape[2], device="cuda")[None, :], s["lens"].long()[:, None]
    ok = j < lens
    if c["window"]:
        ok &= j >= lens - c["window"]
    q = s["q"].view(n, hkv, hq // hkv, d)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~ok[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(n, hq, d), "lse": (top + torch.log(total)).reshape(n, hq)}


def _logits(s):
    x, h = s["logits"], s["history"].long()
    n, vocab = x.shape
    at = torch.arange(h.shape[1], device="cuda")[None, :]
    used, made = at < s["hist_lens"][:, None], (at >= s["prompt_lens"][:, None]) & (at < s["hist_lens"][:, None])
    seen = torch.zeros(n, vocab, device="cuda").scatter_add_(1, h, used.float()) > 0
    count = torch.zeros(n, vocab, device="cuda").scatter_add_(1, h, made.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0).float()
    if s["bias_ids"] is not None:
        e = torch.arange(s["bias_ids"].numel(), device="cuda")
        row = torch.searchsorted(s["bias_starts"][1:].long(), e, right=True)
        bias = torch.zeros(n + 1, vocab, device="cuda")
        bias[row, s["bias_ids"].long()] = s["bias_vals"]
        x = x + bias[:n]
    if s["mask"] is not None:
        bits = ((s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).view(s["mask"].shape[0], -1)[:, :vocab]
        allowed = (bits[s["mask_rows"].clamp(min=0).long()] != 0) | (s["mask_rows"] < 0)[:, None]
        x = x.masked_fill(~allowed, -math.inf)
    top = x.amax(1, keepdim=True)
    ids = torch.where(x == top, torch.arange(vocab, device="cuda")[None, :], vocab).amin(1)
    return {"logits": x, "ids": ids.to(torch.int32)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "tables":
        n, rows = case["nseq"], _rows(case)
        return {"bytes": 4 * (2 * n + 1) + 4 * (2 * n + 3) + 16 * rows + 8 * rows / case["page"], "flops": 0}
    if op == "store":
        t, hq, hkv, d = case["rows"], case["hq"], case["hkv"], case["d"]
        size = 4 if case["kv"] == "f32" else 2
        return {"bytes": t * (4 * d * (2 * hq + 2 * hkv) + size * d * 2 * hkv + 4 * case["rot"] + 12), "flops": t * d * (hq + hkv) * (7 if case["norm"] else 3)}
    if op == "attn":
        total, size = _keys(case), 4 if case["kv"] == "f32" else 2
        return {"bytes": 2 * total * case["hkv"] * case["d"] * size + 8 * case["nseq"] * case["hq"] * case["d"] + 4 * total / case["page"], "flops": 4 * total * case["hq"] * case["d"]}
    n, v = case["rows"], case["vocab"]
    return {"bytes": n * (8 * v + 2 * case["history"] + 4 * case["bias"]) + (n // 2 * v / 8 if case["mask"] else 0), "flops": 4 * n * v}


def _keys(case):
    """The mean over seeds of the keys that a pass attends to."""
    rng = np.random.default_rng(0)
    lens = [_lens(rng, case["nseq"], case["min_len"], case["max_len"]) for _ in range(64)]
    lens = np.stack(lens) if not case["window"] else np.minimum(np.stack(lens), case["window"])
    return float(lens.sum(1).mean())


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if op == "store":
        t, hq, hkv, d, p = case["rows"], case["hq"], case["hkv"], case["d"], case["page"]
        x = s["qkv"].double().reshape(t, -1, d)
        half = case["rot"] // 2
        at = s["positions"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None, :]

        def head(y, gamma):
            if gamma is not None:
                y = y / torch.sqrt(y.pow(2).sum(2, keepdim=True) / d + 1e-6) * gamma.double()
            z = torch.complex(y[:, :, :half], y[:, :, half : 2 * half]) * turn
            return torch.cat([z.real, z.imag, y[:, :, 2 * half :]], 2)

        k, v = s["k"].double().clone(), s["v"].double().clone()
        keys = head(x[:, hq : hq + hkv], s["k_gamma"])
        live = torch.nonzero(s["slots"] >= 0)[:, 0]
        for h in range(hkv):
            k[:, h][s["slots"][live] // p, s["slots"][live] % p] = keys[live, h]
            v[:, h][s["slots"][live] // p, s["slots"][live] % p] = x[live, hq + hkv + h]
        return {"q": head(x[:, :hq], s["q_gamma"]), "k": k, "v": v}
    if op == "attn":
        out = torch.zeros(case["nseq"], case["hq"], case["d"], dtype=torch.float64, device="cuda")
        lse = torch.full((case["nseq"], case["hq"]), -math.inf, dtype=torch.float64, device="cuda")
        group = case["hq"] // case["hkv"]
        for b, n in enumerate(s["lens"].tolist()):
            j = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
            if j.numel() == 0:
                continue
            page, at = s["table"][b].long()[j // case["page"]], j % case["page"]
            for h in range(case["hkv"]):
                k, v = s["k"][page, h, at].double(), s["v"][page, h, at].double()
                x = s["q"][b, h * group : (h + 1) * group].double() @ k.T / math.sqrt(case["d"])
                lse[b, h * group : (h + 1) * group] = torch.logsumexp(x, 1)
                out[b, h * group : (h + 1) * group] = torch.softmax(x, 1) @ v
        return {"out": out, "lse": lse}
    rows = []
    host = {n: (x.cpu().numpy() if x is not None else None) for n, x in s.items() if n not in ("case", "out", "logits", "ids")}
    for b in range(case["rows"]):
        x = s["logits"][b].double().cpu().numpy()
        said = host["history"][b, : host["hist_lens"][b]]
        seen = np.unique(said)
        r = float(host["repetition"][b])
        x[seen] = np.where(x[seen] > 0, x[seen] / r, x[seen] * r)
        tokens, times = np.unique(said[host["prompt_lens"][b] :], return_counts=True)
        x[tokens] -= float(host["frequency"][b]) * times + float(host["presence"][b])
        if host["bias_ids"] is not None:
            part = slice(host["bias_starts"][b], host["bias_starts"][b + 1])
            x[host["bias_ids"][part]] += host["bias_vals"][part].astype(np.float64)
        if host["mask"] is not None and host["mask_rows"][b] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_rows"][b]].view(np.uint8), bitorder="little")[: x.size]
            x[bits == 0] = -math.inf
        rows.append(x)
    return {"logits": torch.from_numpy(np.stack(rows)), "ids": None}
