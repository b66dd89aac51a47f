"""Operators of a batched serving step over a paged 8-bit K/V cache, and what a pass through each costs.

  plan       kv_plan_dev: pages, block tables and slot maps of a step from the requests' lengths.
  rope       rope_rows_dev: rotary positions of q and k rows (half or interleaved pairs, part of the head,
             frequencies scaled for long contexts).
  append     kv8_append_dev: K and V rows into int8 pages with one scale for each page and KV head.
  attention  attention_kv8_dev: causal GQA attention of a ragged batch over such pages.
  logprobs   logprobs_dev: log probability of given tokens, entropy and top alternatives of logit rows.

A page holds `page` tokens of every KV head as 1 KiB blocks of 32 tokens x 32 dimensions, in the order
of the matrix instructions' operands: the codes of K's block are [dim / 8][token % 16][token / 16][dim % 8],
those of V's [token / 4 % 4][dim % 16][dim / 16][token / 16][token % 4]. A code c stands for c * scale.

Inputs are made from the seed on the GPU. Where `own` is false `run` computes in elementary torch
operations; where it is true it makes the library's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
HEADS = [(14, 2, 64), (16, 8, 64), (12, 12, 64), (32, 4, 128), (24, 8, 128)]     # query / KV heads, head size
VOCAB = 151936


def listed():
    return [
        # one decode step of 64 requests: a token each, now and then a new page, some requests ending
        {"name": "plan_decode_64", "kind": "plan", "requests": 64, "page": 64, "max_len": 8192, "max_new": 1},
        # a busy server's step: 1024 requests, prompt chunks among the single tokens
        {"name": "plan_mixed_1024", "kind": "plan", "requests": 1024, "page": 32, "max_len": 4096, "max_new": 96},
        # q and k of 8 sequences decoding together, a small model's heads: bound by the launch
        {"name": "rope_decode_8", "kind": "rope", "rows": 8, "heads": 16, "hd": 64, "rot": 64, "interleaved": False,
         "scaling": "none", "max_pos": 2048},
        # q and k of a long prompt's chunk far into the context, half of each head, interleaved, YaRN
        {"name": "rope_prefill_8192", "kind": "rope", "rows": 8192, "heads": 36, "hd": 128, "rot": 64,
         "interleaved": True, "scaling": "yarn", "max_pos": 131072},
        # one token of each of 64 sequences into pages that are partly full
        {"name": "append_decode_64", "kind": "append", "requests": 64, "max_rows": 1, "page": 64, "kv_heads": 4,
         "hd": 128, "max_len": 8192},
        # two prompts' chunks of up to 6000 tokens, ragged, after earlier ones
        {"name": "append_prefill_6000", "kind": "append", "requests": 2, "max_rows": 6000, "page": 64, "kv_heads": 8,
         "hd": 128, "max_len": 12000},
        # one user's decode step on a short conversation, a small model: bound by latency
        {"name": "attention_decode_1", "kind": "attention", "requests": 1, "max_rows": 1, "max_len": 211, "page": 32,
         "heads": 14, "kv_heads": 2, "hd": 64, "window": 0},
        # a decode step of 64 conversations of 1 .. 16384 tokens
        {"name": "attention_decode_64", "kind": "attention", "requests": 64, "max_rows": 1, "max_len": 16384,
         "page": 64, "heads": 32, "kv_heads": 4, "hd": 128, "window": 0},
        # a decode step at the end of one very long document
        {"name": "attention_long_1", "kind": "attention", "requests": 1, "max_rows": 1, "max_len": 131071,
         "page": 64, "heads": 24, "kv_heads": 8, "hd": 128, "window": 0},
        # chunks of four prompts behind what their conversations already hold
        {"name": "attention_prefill_4", "kind": "attention", "requests": 4, "max_rows": 1000, "max_len": 5000,
         "page": 64, "heads": 32, "kv_heads": 4, "hd": 128, "window": 0},
        # one sampled token's log probability with five alternatives, a whole vocabulary
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "top": 5},
        # scoring a 961-token prompt, twenty alternatives each
        {"name": "logprobs_961", "kind": "logprobs", "rows": 961, "vocab": VOCAB, "top": 20},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "append", "attention", "attention", "attention", "logprobs"])
    if kind == "plan":
        return {"kind": kind, "requests": _log(rng, 1, 1024), "page": rng.choice([32, 64, 128]),
                "max_len": _log(rng, 100, 8192), "max_new": _log(rng, 1, 96)}
    if kind == "rope":
        hd = rng.choice([32, 64, 96, 128, 256])
        heads = rng.randint(1, 36)
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        return {"kind": kind, "rows": _log(rng, 1, 8192 * 36 * 64 // max(36 * 64, heads * rot)), "heads": heads,
                "hd": hd, "rot": rot, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "bands"]), "max_pos": _log(rng, 1, 131072)}
    heads, kv, hd = rng.choice(HEADS)
    if kind == "append":
        c = {"kind": kind, "requests": _log(rng, 1, 64), "max_rows": _log(rng, 1, 4000),
             "page": rng.choice([32, 64, 128]), "kv_heads": kv, "hd": rng.choice([32, 64, 96, 128, 256])}
        while c["requests"] * c["max_rows"] * kv * c["hd"] > 2 * 6000 * 8 * 128:
            c["max_rows"] = max(1, c["max_rows"] * 2 // 3)
            c["requests"] = max(1, c["requests"] * 5 // 6)
        return {**c, "max_len": c["max_rows"] + _log(rng, 1, 4096)}
    if kind == "attention":
        if rng.random() < 0.5:          # a decode step
            c = {"requests": _log(rng, 1, 64), "max_rows": rng.choice([1, 1, 1, 2, 4]), "max_len": _log(rng, 4, 16384)}
            c["requests"] = min(c["requests"], 64 * 4 * 128 // (kv * hd))
        else:                           # prompts, or their chunks
            rows = _log(rng, 5, 1000)
            c = {"requests": _log(rng, 1, 4), "max_rows": rows, "max_len": rows + _log(rng, 1, 4000)}
        return {"kind": kind, **c, "page": rng.choice([32, 64, 128]), "heads": heads, "kv_heads": kv,
                "hd": rng.choice([32, 64, 96, 128, 128, 256]) if c["max_rows"] < 5 and c["requests"] < 8 else hd,
                "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)])}
    vocab = _log(rng, 100, VOCAB)
    return {"kind": kind, "rows": _log(rng, 1, min(4096, 961 * VOCAB // vocab)), "vocab": vocab,
            "top": rng.randint(0, 20)}


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 6007 + 11)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a, np.int32), device="cuda")


def _frequencies(theta, rot, scaling, factor=8.0, trained=4096.0):
    """Radians per position of each pair, and the factor of the rotated vector, in 64 bits."""
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk" and rot > 2:
        return (theta * factor ** (rot / (rot - 2.0))) ** (-2.0 * i / rot), 1.0
    if scaling == "yarn":               # fast pairs as trained, slow ones interpolated, a ramp between
        at = [rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    if scaling == "bands":              # by the number of turns over the trained context: 1 .. 4
        smooth = np.clip((trained * f / (2 * math.pi) - 1.0) / 3.0, 0.0, 1.0)
        return f * smooth + f / factor * (1 - smooth), 1.0
    return f, 1.0


def _sizes(case):
    """New rows and cached tokens (the new ones counted) of each request: by the case alone, so that shapes are."""
    rng, n = np.random.default_rng([case["requests"], case["max_rows"], case["max_len"]]), case["requests"]
    rows = rng.integers(max(1, case["max_rows"] // 2), case["max_rows"] + 1, n)
    rest = np.exp(rng.uniform(0, math.log(max(1, case["max_len"] - case["max_rows"]) + 1), n)).astype(np.int64) - 1
    rows[n // 2], rest[n // 2] = case["max_rows"], case["max_len"] - case["max_rows"]   # the longest is there
    return rows, rows + rest


def _steps(case):
    """New tokens (-1: the request has ended) and cached ones of a step's requests, by the case alone."""
    rng, n = np.random.default_rng([case["requests"], case["max_new"], case["max_len"]]), case["requests"]
    new = rng.integers(1, case["max_new"] + 1, n)
    new[rng.random(n) < 0.6] = 1
    new[rng.random(n) < 0.04] = -1
    new[0] = case["max_new"]
    return new, rng.integers(0, case["max_len"] + 1, n)


def _batch(case, rng):
    """A ragged batch: its sizes and its pages, in a shuffled pool with room for all and a few more."""
    n = case["requests"]
    rows, lens = _sizes(case)
    need = -(-lens // case["page"])
    ld = int(need.max())
    pages = int(need.sum()) + 3
    order = rng.permutation(pages)
    table = np.full((n, ld), -1, np.int64)
    at = np.concatenate([[0], np.cumsum(need)])
    for b in range(n):
        table[b, :need[b]] = order[at[b]:at[b + 1]]
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    seq = np.repeat(np.arange(n), rows)
    pos = np.arange(total) - start[seq] + lens[seq] - rows[seq]
    return {"rows": total, "ld": ld, "pages": pages, "table": _i32(table), "start": _i32(start[:n]),
            "count": _i32(rows), "len": _i32(lens), "seq": _i32(seq), "pos": _i32(pos),
            "host": {"rows": rows, "lens": lens, "table": table, "start": start, "seq": seq, "pos": pos}}


def _pages(case, g, pages):
    """Codes of about normal values and the scales of page and head that such values have."""
    shape = (pages, case["kv_heads"], case["page"] // 32, case["hd"] // 32, 1024)
    codes = [(36.0 * _randn(g, *shape)).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp(0.3 * _randn(g, *shape[:2])) / 36.0 for _ in range(2)]
    return codes, scales


def prepare(case, seed):
    g, rng, kind = _gen(seed), np.random.default_rng(seed * 6007 + 11), case["kind"]
    s = {"case": case}
    if kind == "plan":
        n, page = case["requests"], case["page"]
        new, lens = (rng.permutation(v) for v in _steps(case))
        ld = -(-(case["max_len"] + case["max_new"]) // page)
        held = -(-lens // page)
        spare = max(1, int(np.maximum(new, 0).sum()) // page)          # now and then too few
        pages = int(held.sum()) + spare
        order = rng.permutation(pages)
        table = np.full((n, ld), -1, np.int64)
        mask = np.arange(ld)[None] < held[:, None]
        table[mask] = order[:int(held.sum())]
        free = np.full(pages, -1, np.int64)
        free[:spare] = order[int(held.sum()):]
        cap = int(np.maximum(new, 0).sum()) + 5             # the step's rows, padded
        s.update(new=_i32(new), len=_i32(lens), table=_i32(table), free=_i32(free), nfree=_i32([spare]), ld=ld,
                 pages=pages, cap=cap)
        s["out"] = {"len": torch.empty_like(s["len"]), "nfree": torch.empty_like(s["nfree"]),
                    "start": torch.empty_like(s["len"]), "count": torch.empty_like(s["len"]),
                    **{k: torch.empty(cap, device="cuda", dtype=torch.int32) for k in ("seq", "pos", "slot")},
                    "status": torch.empty(2, device="cuda", dtype=torch.int32)}
    elif kind == "rope":
        f, s["mscale"] = _frequencies(1e6, case["rot"], case["scaling"])
        s["freqs"] = torch.as_tensor(f, device="cuda")
        s["pos"] = torch.randint(0, case["max_pos"] + 1, (case["rows"],), generator=g, device="cuda",
                                 dtype=torch.int32)
        s["in"] = _randn(g, case["rows"], case["heads"], case["hd"])
        s["x"] = torch.empty_like(s["in"])
    elif kind == "append":
        s.update(_batch(case, rng))
        s["codes"], s["scales"] = _pages(case, g, s["pages"])
        s["k"], s["v"] = (_randn(g, s["rows"], case["kv_heads"], case["hd"])
                          * torch.exp(0.3 * _randn(g, s["rows"], 1, 1)) for _ in range(2))
    elif kind == "attention":
        s.update(_batch(case, rng))
        s["codes"], s["scales"] = _pages(case, g, s["pages"])
        s["q"] = 2.0 * _randn(g, s["rows"], case["heads"], case["hd"])
        s["ctx"] = torch.zeros_like(s["q"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["x"] = 2.5 * _randn(g, rows, vocab)
        s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["logprob"], s["entropy"] = (torch.empty(rows, device="cuda") for _ in range(2))
        s["ids"] = torch.empty(rows, case["top"], device="cuda", dtype=torch.int32)
        s["top"] = torch.empty(rows, case["top"], device="cuda")
    return s


# ---- the library's calls -------------------------------------------------------------------------
def _rehip():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rusty-engine_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rehip
    return rehip


def _work(s, nbytes):
    """The workspace that the program keeps for these calls, of the size that the library asks for."""
    if s.get("work") is None or s["work"].numel() < nbytes:
        s["work"] = torch.empty(max(nbytes, 16), device="cuda", dtype=torch.uint8)
    return s["work"].data_ptr()


def _plan_own(s, c):
    o = s["out"]
    _rehip().kv_plan_dev(c["requests"], c["page"], s["new"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(),
                         s["ld"], s["free"].data_ptr(), s["pages"], s["nfree"].data_ptr(), o["len"].data_ptr(),
                         o["nfree"].data_ptr(), o["start"].data_ptr(), o["count"].data_ptr(), s["cap"],
                         o["seq"].data_ptr(), o["pos"].data_ptr(), o["slot"].data_ptr(), o["status"].data_ptr())
    return {**o, "table": s["table"], "free": s["free"]}


def _rope_own(s, c):
    r = _rehip()
    r.rope_rows_dev(s["in"].data_ptr(), c["heads"] * c["hd"], c["rows"], c["heads"], c["hd"], c["rot"],
                    r.ROPE_INTERLEAVED if c["interleaved"] else r.ROPE_HALF, s["freqs"].data_ptr(), s["mscale"],
                    s["pos"].data_ptr(), s["x"].data_ptr(), c["heads"] * c["hd"])
    return s["x"]


def _cache_args(s, c):
    (kc, vc), (ks, vs) = s["codes"], s["scales"]
    return (c["requests"], s["start"].data_ptr(), s["count"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(),
            s["ld"], c["page"], s["pages"], kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr())


def _append_own(s, c):
    w = c["kv_heads"] * c["hd"]
    _rehip().kv8_append_dev(s["k"].data_ptr(), w, s["v"].data_ptr(), w, s["rows"], *_cache_args(s, c), c["kv_heads"],
                            c["hd"])
    return {"codes": s["codes"], "scales": s["scales"]}


def _attention_own(s, c):
    r = _rehip()
    w = c["heads"] * c["hd"]
    nbytes = r.attention_kv8_work_bytes(s["rows"], c["requests"], c["max_rows"], c["max_len"], c["heads"],
                                        c["kv_heads"], c["hd"])
    r.attention_kv8_dev(s["q"].data_ptr(), w, s["rows"], *_cache_args(s, c), c["max_rows"], c["max_len"], c["heads"],
                        c["kv_heads"], c["hd"], c["hd"] ** -0.5, c["window"], s["ctx"].data_ptr(), _work(s, nbytes),
                        nbytes)
    return s["ctx"]


def _logprobs_own(s, c):
    r = _rehip()
    nbytes = r.logprobs_work_bytes(c["rows"], c["vocab"], c["top"])
    top = c["top"] > 0
    r.logprobs_dev(s["x"].data_ptr(), c["vocab"], c["rows"], c["vocab"], s["targets"].data_ptr(), c["top"],
                   s["logprob"].data_ptr(), s["entropy"].data_ptr(), s["ids"].data_ptr() if top else None,
                   s["top"].data_ptr() if top else None, _work(s, nbytes), nbytes)
    return {"logprob": s["logprob"], "entropy": s["entropy"], "ids": s["ids"], "top": s["top"]}


# ---- the plain forms -----------------------------------------------------------------------------
def _plan_plain(s, c):
    n, page, ld, pages, cap = c["requests"], c["page"], s["ld"], s["pages"], s["cap"]
    new, lens, table, free = s["new"].long(), s["len"].long(), s["table"], s["free"]
    held = (lens + page - 1) // page
    back = torch.where(new < 0, held, 0)                    # pages of ended requests, pushed in order
    first = torch.cumsum(back, 0) - back
    j = torch.arange(ld, device="cuda")
    at = torch.where(j < back[:, None], s["nfree"].long() + first[:, None] + j, pages)
    free = torch.cat([free, free[:1]]).scatter(0, at.reshape(-1), table.reshape(-1))[:pages]
    total = s["nfree"].long() + back.sum()
    rows = new.clamp(min=0)
    after = lens + rows
    fits = after <= ld * page
    need = torch.where(fits & (new > 0), (after + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0)
    ok = fits & (new >= 0) & ((need == 0) | (upto <= total))
    take = torch.where(ok, need, 0)
    mine = (j >= held[:, None]) & (j < (held + take)[:, None])
    at = (total - 1 - (upto - need)[:, None] - (j - held[:, None])).clamp(0, pages - 1)
    table = torch.where(mine, free[at], table)
    out_len = torch.where(ok, after, torch.where(new < 0, 0, lens))
    start = torch.cumsum(rows, 0) - rows
    count = torch.where(ok, rows, 0)
    t = torch.arange(cap, device="cuda")
    b = torch.searchsorted(torch.cumsum(rows, 0), t, right=True).clamp(max=n - 1)
    i = t - start[b]
    live = (i >= 0) & (i < count[b])
    pos = out_len[b] - count[b] + i
    slot = table[b, (pos // page).clamp(0, ld - 1)].long() * page + pos % page
    given = lambda v: torch.where(live, v, -1).int()  # noqa: E731
    s["table"].copy_(table)
    s["free"].copy_(free)
    return {"len": out_len.int(), "nfree": (total - take.sum()).int(), "start": start.int(), "count": count.int(),
            "seq": given(b), "pos": given(pos), "slot": given(slot),
            "status": torch.stack([((new > 0) & ~ok).sum(), rows.sum()]).int(), "table": s["table"], "free": s["free"]}


def _rope_plain(s, c):
    x, rot = s["in"], c["rot"]
    a = s["pos"].double()[:, None] * s["freqs"]
    cos, sin = ((f(a) * s["mscale"]).float()[:, None] for f in (torch.cos, torch.sin))
    if c["interleaved"]:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    else:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _k_rows(blocks):
    """K's codes (.., page / 32, hd / 32, 1024) as (.., page, hd)."""
    *lead, p, d, _ = blocks.shape
    v = blocks.reshape(-1, p, d, 4, 16, 2, 8).permute(0, 1, 5, 4, 2, 3, 6)
    return v.reshape(*lead, 32 * p, 32 * d)


def _v_rows(blocks):
    *lead, p, d, _ = blocks.shape
    v = blocks.reshape(-1, p, d, 4, 16, 2, 2, 4).permute(0, 1, 6, 3, 7, 2, 5, 4)
    return v.reshape(*lead, 32 * p, 32 * d)


def _k_blocks(rows):
    *lead, p, d = rows.shape
    v = rows.reshape(-1, p // 32, 2, 16, d // 32, 4, 8).permute(0, 1, 4, 5, 3, 2, 6)
    return v.reshape(*lead, p // 32, d // 32, 1024)


def _v_blocks(rows):
    *lead, p, d = rows.shape
    v = rows.reshape(-1, p // 32, 2, 4, 4, d // 32, 2, 16).permute(0, 1, 5, 3, 7, 6, 2, 4)
    return v.reshape(*lead, p // 32, d // 32, 1024)


def _quantise_into(x, blocks, scale, to_rows, to_blocks, s, c):
    """Rows x of the batch into their pages: a page's scale is the largest magnitude / 127 of what it
    holds; where new rows raise it, the codes that were there are rounded to the new scale."""
    page, pos, seq = c["page"], s["pos"].long(), s["seq"].long()
    pid = s["table"].long()[seq, pos // page]
    amax = torch.where(torch.isfinite(x), x, 0).abs().amax(-1)
    top = torch.zeros_like(scale).scatter_reduce(0, pid[:, None].expand_as(amax), amax, "amax")
    lens, count = s["len"].long(), s["count"].long()
    old = (lens - count) % page                             # earlier rows in each request's first page
    b = torch.arange(c["requests"], device="cuda")
    p0 = s["table"].long()[b, (lens - count) // page]
    kept = torch.where(old[:, None] > 0, scale[p0], 0)
    want = top * torch.tensor(1 / 127, device="cuda", dtype=torch.float32)
    want = torch.where(want < torch.finfo(torch.float32).tiny, 0, want)
    fresh = torch.zeros_like(scale, dtype=torch.bool)
    fresh[pid] = True
    new = torch.where(fresh, want, scale)
    new[p0] = torch.maximum(kept, want[p0])
    codes = to_rows(blocks)
    here = codes[p0]
    r = torch.where(kept < new[p0], kept / torch.where(new[p0] > 0, new[p0], 1), 1)[..., None, None]
    early = (torch.arange(page, device="cuda") < old[:, None])[:, None, :, None]
    codes[p0] = torch.where(early, torch.round(here.float() * r).to(torch.int8), here)
    q = torch.round(x / torch.where(new[pid] > 0, new[pid], 1)[..., None])
    q = torch.where(new[pid][..., None] > 0, q, 0).nan_to_num(0, 127, -127).clamp(-127, 127).to(torch.int8)
    codes[pid, :, pos % page] = q
    blocks.copy_(to_blocks(codes))
    scale.copy_(new)


def _append_plain(s, c):
    _quantise_into(s["k"], s["codes"][0], s["scales"][0], _k_rows, _k_blocks, s, c)
    _quantise_into(s["v"], s["codes"][1], s["scales"][1], _v_rows, _v_blocks, s, c)
    return {"codes": s["codes"], "scales": s["scales"]}


def _attention_plain(s, c):
    n, top, hd, kv = c["requests"], c["max_rows"], c["hd"], c["kv_heads"]
    grp = c["heads"] // kv
    table = s["table"].long().clamp(min=0)
    k, v = (rows(codes[table]).float() * scale[table][..., None, None] for rows, codes, scale in
            zip((_k_rows, _v_rows), s["codes"], s["scales"]))               # (n, pages, kv, page, hd)
    k, v = (t.transpose(1, 2).reshape(n, kv, -1, hd) for t in (k, v))
    i = torch.arange(top, device="cuda")
    count, lens = s["count"].long()[:, None], s["len"].long()[:, None]
    row = (s["start"].long()[:, None] + i).clamp(max=s["rows"] - 1)         # (n, top)
    q = s["q"][row].reshape(n, top, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, top * grp, hd)
    x = (q @ k.transpose(-1, -2).contiguous()).reshape(n, kv, top, grp, -1) * hd ** -0.5
    j, pos = torch.arange(k.shape[2], device="cuda"), (lens - count + i)[..., None]
    seen = (j <= pos) & (j > pos - c["window"] if c["window"] else j >= 0)
    x = x.masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(n, kv, top * grp, -1)
    y = (p @ v).reshape(n, kv, top, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, top, c["heads"], hd)
    at = s["seq"].long()
    return y[at, torch.arange(s["rows"], device="cuda") - s["start"].long()[at]]


def _logprobs_plain(s, c):
    x = s["x"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    logz = torch.log(z)
    out = {"logprob": (d.gather(1, s["targets"].long()[:, None]) - logz)[:, 0],
           "entropy": (logz - (e * torch.where(e > 0, d, 0)).sum(-1, keepdim=True) / z)[:, 0]}
    bits = x.view(torch.int32).long()                       # ordered as the values, then the lower index first
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * 2 ** 20 - torch.arange(c["vocab"], device="cuda")
    ids = torch.topk(key, c["top"], -1)[1]
    return {**out, "ids": ids.int(), "top": d.gather(1, ids) - logz}


PLAIN = {"plan": _plan_plain, "rope": _rope_plain, "append": _append_plain, "attention": _attention_plain,
         "logprobs": _logprobs_plain}
OWN = {"plan": _plan_own, "rope": _rope_own, "append": _append_own, "attention": _attention_own,
       "logprobs": _logprobs_own}


def run(s):
    return (OWN if own else PLAIN)[s["case"]["kind"]](s, s["case"])


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "plan":                  # lengths in and out, new pages, and three numbers for each row
        n, rows = case["requests"], int(np.maximum(_steps(case)[0], 0).sum())
        return {"bytes": 4 * (5 * n + 2 * (rows // case["page"]) + 3 * rows), "flops": 10 * n + 4 * rows}
    if kind == "rope":
        n = case["rows"] * case["heads"]
        out = n * (case["hd"] + case["hd"])                 # rows in, rows out
        return {"bytes": 4 * out + 4 * case["rows"], "flops": 3 * n * case["rot"] + 40 * case["rows"] * case["rot"]}
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    rows, lens = _sizes(case)
    total, kv = int(rows.sum()), case["kv_heads"] * case["hd"]
    if kind == "append":
        pages = int((-(-lens // case["page"]) - (lens - rows) // case["page"]).sum())
        return {"bytes": 10 * total * kv + 8 * case["kv_heads"] * pages, "flops": 6 * total * kv}
    w = case["window"] or 1 << 40
    seen = sum(int(np.minimum(np.arange(n - r, n) + 1, w).sum()) for r, n in zip(rows, lens))
    keys = int(np.minimum(lens, w + rows).sum())
    width = case["heads"] * case["hd"]
    return {"bytes": 8 * total * width + 2 * keys * kv, "flops": 4 * seen * width}


# ---- the same in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None
    s = prepare(case, seed)
    if kind == "rope":
        x = s["in"].double()
        turn = torch.polar(torch.full_like(s["freqs"], s["mscale"]).expand(case["rows"], -1).contiguous(),
                           s["pos"].double()[:, None] * s["freqs"])[:, None]
        rot, part = case["rot"], x[..., :case["rot"]]
        pairs = part.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, rot // 2)).mT
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = y.flatten(-2) if case["interleaved"] else y.mT.flatten(-2)
        return torch.cat([y, x[..., rot:]], -1)
    if kind == "append":                # the scales: the largest of each page's rows
        h, page = s["host"], case["page"]
        scales = [t.double() for t in s["scales"]]
        for x, scale in zip((s["k"], s["v"]), scales):
            a = x.double().abs().amax(-1) / 127
            for b in range(case["requests"]):
                n, to, r = int(h["rows"][b]), int(h["lens"][b]), int(h["start"][b])
                for p in range((to - n) // page, -(-to // page)):
                    lo, hi = max(p * page, to - n), min((p + 1) * page, to)
                    most, at = a[r + lo - to + n:r + hi - to + n].amax(0), int(h["table"][b, p])
                    scale[at] = torch.maximum(most, scale[at]) if lo % page else most
        return {"codes": [None, None], "scales": scales}
    if kind == "attention":
        h, hd, kv = s["host"], case["hd"], case["kv_heads"]
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        for b in range(case["requests"]):
            n, to, r = int(h["rows"][b]), int(h["lens"][b]), int(h["start"][b])
            pages = torch.as_tensor(h["table"][b, :-(-to // case["page"])], device="cuda")
            t, d = torch.arange(32, device="cuda")[:, None], torch.arange(32, device="cuda")[None]
            where = [d // 8 * 256 + t % 16 * 16 + t // 16 * 8 + d % 8,
                     t // 4 % 4 * 256 + d % 16 * 16 + d // 16 * 8 + t // 16 * 4 + t % 4]
            k, v = (torch.cat([codes[pages, g][..., w].double().transpose(-3, -2).reshape(-1, case["page"], hd)
                               * scale[pages, g].double()[:, None, None] for g in range(kv)])
                    .reshape(kv, -1, hd)[:, :to] for codes, scale, w in zip(s["codes"], s["scales"], where))
            pos = torch.arange(to - n, to, device="cuda")[:, None]
            j = torch.arange(to, device="cuda")[None]
            hide = (j > pos) | (j <= pos - (case["window"] or to + 1))
            for i in range(case["heads"]):
                g = i // (case["heads"] // kv)
                x = s["q"][r:r + n, i].double() @ k[g].T.contiguous() / math.sqrt(hd)
                out[r:r + n, i] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v[g]
        return out
    at = torch.arange(case["rows"], device="cuda")
    result = {"logprob": [], "entropy": [], "top": []}
    for i in at.split(64):
        y = torch.log_softmax(s["x"][i].double(), -1)
        result["logprob"].append(y[torch.arange(len(i)), s["targets"][i].long()])
        result["entropy"].append(-(y.exp() * y).sum(-1))
        result["top"].append(y.topk(case["top"], -1)[0])
    return {**{k: torch.cat(v) for k, v in result.items()}, "ids": None}
