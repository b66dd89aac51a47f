"""Operators of a batched serving step whose conversations outgrow their pages and which decodes several tokens a step, and
what a pass through each costs.

  attention  attention_kv8_sinks_dev: causal GQA attention of a ragged batch over int8 pages, a sliding window and a few
             first tokens that stay visible; the context rows and the log of each row's sum of exponentials.
  mass       kv8_mass_dev: the attention weight that each cached token gets from a step's rows, added to what it has.
  evict      kv_evict_plan_dev and kv8_evict_dev: requests longer than a limit are cut to the first, the last and the
             heaviest tokens, which move to fresh pages in order, head by head.
  verify     draft_verify_dev: drafted tokens against the target's probabilities from given random numbers: how many are
             accepted, and the token behind them.
  rewind     kv_rewind_dev: rejected tokens are taken off the lengths, pages behind the ends go back to the stack.

A page holds `page` tokens of every KV head as 1 KiB blocks of 32 tokens x 32 dimensions, in the order of the matrix
instructions' operands: the codes of K's block are [dim / 8][token % 16][token / 16][dim % 8], those of V's
[token / 4 % 4][dim % 16][dim / 16][token / 16][token % 4]. A code c stands for c * scale, a scale for each page and head.

Inputs are made from the seed on the GPU. Where `own` is false `run` computes in elementary torch operations; where it is
true it makes the library's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
HEADS = [(14, 2, 64), (16, 8, 64), (12, 12, 64), (32, 4, 128), (32, 8, 128)]     # query / KV heads, head size
VOCAB = 151936


def listed():
    return [
        # one user's step far into a conversation, a small model with a short window: bound by latency
        {"name": "attention_decode_1", "kind": "attention", "requests": 1, "max_rows": 1, "max_len": 2900, "page": 32,
         "heads": 14, "kv_heads": 2, "hd": 64, "window": 1024, "sinks": 4},
        # a decode step of 64 conversations of up to 65536 tokens
        {"name": "attention_decode_64", "kind": "attention", "requests": 64, "max_rows": 1, "max_len": 65536,
         "page": 64, "heads": 32, "kv_heads": 4, "hd": 128, "window": 4096, "sinks": 4},
        # 32 conversations with up to four drafted tokens each
        {"name": "attention_drafts_32", "kind": "attention", "requests": 32, "max_rows": 5, "max_len": 20000,
         "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "window": 2048, "sinks": 16},
        # chunks of two long prompts
        {"name": "attention_prefill_2", "kind": "attention", "requests": 2, "max_rows": 2000, "max_len": 12000,
         "page": 64, "heads": 32, "kv_heads": 4, "hd": 128, "window": 2048, "sinks": 4},
        # weights of a decode step of 64 conversations
        {"name": "mass_decode_64", "kind": "mass", "requests": 64, "max_rows": 1, "max_len": 8192, "page": 64,
         "heads": 32, "kv_heads": 4, "hd": 128, "window": 0, "sinks": 0},
        # weights of two prompts' chunks
        {"name": "mass_prefill_2", "kind": "mass", "requests": 2, "max_rows": 1000, "max_len": 5000, "page": 64,
         "heads": 16, "kv_heads": 8, "hd": 64, "window": 0, "sinks": 0},
        # one conversation over its limit
        {"name": "evict_1", "kind": "evict", "requests": 1, "limit": 2100, "max_len": 2101, "keep": 1050, "first": 4,
         "recent": 256, "page": 32, "kv_heads": 2, "hd": 64},
        # a server after a burst of long prompts: most of 32 conversations over the limit
        {"name": "evict_32", "kind": "evict", "requests": 32, "limit": 4096, "max_len": 8192, "keep": 2048, "first": 4,
         "recent": 512, "page": 64, "kv_heads": 8, "hd": 128},
        # four tokens drafted by lookup for one user
        {"name": "verify_1", "kind": "verify", "requests": 1, "drafts": 4, "vocab": VOCAB, "probs": False},
        # up to four tokens drafted by a small model for each of 64 requests, some of them greedy
        {"name": "verify_64", "kind": "verify", "requests": 64, "drafts": 4, "vocab": VOCAB, "probs": True},
        # their rejected tokens taken back
        {"name": "rewind_64", "kind": "rewind", "requests": 64, "drafts": 4, "page": 64, "max_len": 8192},
        # the most requests, long drafts, small pages
        {"name": "rewind_4096", "kind": "rewind", "requests": 4096, "drafts": 16, "page": 16, "max_len": 1024},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "mass", "mass", "evict", "evict", "verify", "verify", "rewind"])
    heads, kv, hd = rng.choice(HEADS)
    if kind in ("attention", "mass"):
        if rng.random() < 0.6:          # a decode step, some of them with drafts
            c = {"requests": _log(rng, 1, 64), "max_rows": rng.choice([1, 1, 1, 2, 3, 5]),
                 "max_len": _log(rng, 4, 65536 if kind == "attention" else 8192)}
            c["requests"] = min(c["requests"], 64 * 4 * 128 // (kv * hd))
            w = rng.choice([0, 1, 1, 1, 1]) * _log(rng, 1, 4096)
            if w == 0:
                c["max_len"] = min(c["max_len"], 8192)
        else:                           # prompts, or their chunks
            rows, w = _log(rng, 5, 1000), rng.choice([0, 1, 1]) * _log(rng, 1, 2048)
            c = {"requests": _log(rng, 1, 3), "max_rows": rows, "max_len": rows + _log(rng, 1, 4000 if w else 1000)}
        hd = rng.choice([32, 64, 96, 128, 128, 256]) if c["max_rows"] < 5 and c["requests"] < 8 else hd
        return {"kind": kind, **c, "page": rng.choice([32, 64, 128]), "heads": heads, "kv_heads": kv, "hd": hd,
                "window": w, "sinks": rng.choice([0, 1, 4, 4, 16, 100]) if w else 0}
    if kind == "evict":
        keep = _log(rng, 1, 2048)
        first = min(rng.choice([0, 1, 4, 16]), keep)
        limit = keep + _log(rng, 1, 2048) - 1
        return {"kind": kind, "requests": _log(rng, 1, 32), "limit": limit, "max_len": limit + _log(rng, 1, 4000),
                "keep": keep, "first": first, "recent": rng.randint(0, keep - first), "page": rng.choice([32, 64, 128]),
                "kv_heads": kv, "hd": rng.choice([32, 64, 96, 128])}
    if kind == "verify":
        vocab = _log(rng, 100, VOCAB)
        return {"kind": kind, "requests": _log(rng, 1, 64), "drafts": rng.randint(0, 4), "vocab": vocab,
                "probs": rng.random() < 0.5}
    return {"kind": kind, "requests": _log(rng, 1, 4096), "drafts": _log(rng, 1, 16), "page": rng.choice([16, 32, 64, 128]),
            "max_len": _log(rng, 20, 1024)}


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 6007 + 11)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a, np.int32), device="cuda")


def _sizes(case):
    """New rows and cached tokens (the new ones counted) of each request: by the case alone, so that shapes are."""
    rng, n = np.random.default_rng([case["requests"], case["max_rows"], case["max_len"]]), case["requests"]
    rows = rng.integers(max(1, case["max_rows"] // 2), case["max_rows"] + 1, n)
    rest = np.exp(rng.uniform(0, math.log(max(1, case["max_len"] - case["max_rows"]) + 1), n)).astype(np.int64) - 1
    rows[n // 2], rest[n // 2] = case["max_rows"], max(0, case["max_len"] - case["max_rows"])   # the longest is there
    return rows, rows + rest


def _long(case):
    """Lengths of the requests of an eviction: most of them over the limit, by the case alone."""
    rng, n = np.random.default_rng([case["requests"], case["limit"], case["max_len"]]), case["requests"]
    lens = rng.integers(case["limit"] + 1, case["max_len"] + 1, n)
    lens[rng.random(n) < 0.2] = case["limit"]
    lens[n // 2] = case["max_len"]
    return lens


def _drafts(case):
    """Drafted tokens of each request, by the case alone."""
    rng = np.random.default_rng([case["requests"], case["drafts"]])
    n = rng.integers(0, case["drafts"] + 1, case["requests"])
    n[case["requests"] // 2] = case["drafts"]
    return n


def _tables(lens, page, rng, spare, ld=None):
    """Page numbers of requests of these lengths, from a shuffled pool with `spare` pages more: (table, pages, the rest)."""
    need = -(-lens // page)
    ld = ld or int(need.max())
    pages = int(need.sum()) + spare
    order = rng.permutation(pages)
    table = np.full((len(lens), ld), -1, np.int64)
    table[np.arange(ld)[None] < need[:, None]] = order[:int(need.sum())]
    return table, pages, order[int(need.sum()):]


def _codes(case, g, pages):
    """Codes of about normal values and the scales of page and head that such values have."""
    shape = (pages, case["kv_heads"], case["page"] // 32, case["hd"] // 32, 1024)
    codes = [(36.0 * _randn(g, *shape)).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp(0.3 * _randn(g, *shape[:2])) / 36.0 for _ in range(2)]
    return codes, scales


def prepare(case, seed):
    g, rng, kind = _gen(seed), np.random.default_rng(seed * 6007 + 11), case["kind"]
    s = {"case": case}
    if kind in ("attention", "mass"):
        rows, lens = _sizes(case)
        table, pages, _ = _tables(lens, case["page"], rng, 3)
        start = np.concatenate([[0], np.cumsum(rows)])
        seq = np.repeat(np.arange(len(rows)), rows)
        s.update(rows=int(start[-1]), ld=table.shape[1], pages=pages, table=_i32(table), start=_i32(start[:-1]),
                 count=_i32(rows), len=_i32(lens), seq=_i32(seq),
                 host={"rows": rows, "lens": lens, "table": table, "start": start})
        s["codes"], s["scales"] = _codes(case, g, pages)
        s["q"] = 2.0 * _randn(g, s["rows"], case["heads"], case["hd"])
        s["ctx"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros(s["rows"], case["heads"], device="cuda")
        if kind == "mass":              # what the step's attention gave, and what earlier steps left
            s["lse"] = _attention_plain(s, case)["lse"]
            s["mass"] = torch.exp(_randn(g, pages, case["kv_heads"], case["page"]) - 2.0)
    elif kind == "evict":
        lens, page, n = rng.permutation(_long(case)), case["page"], case["requests"]
        fresh = -(-case["keep"] // page)
        cuts = int((lens > case["limit"]).sum())
        spare = fresh * max(1, cuts - n // 16) + 1           # now and then too few for the last of them
        table, pages, rest = _tables(lens, page, rng, spare, -(-case["max_len"] // page) + 1)
        free = np.full(pages, -1, np.int64)
        free[:spare] = rest
        s.update(ld=table.shape[1], pages=pages, table=_i32(table), len=_i32(lens), free=_i32(free), nfree=_i32([spare]),
                 host={"lens": lens, "table": table, "free": free, "spare": spare})
        s["codes"], s["scales"] = _codes(case, g, pages)
        # weights of which some are equal
        s["mass"] = torch.round(256.0 * torch.exp(_randn(g, pages, case["kv_heads"], page) - 2.0)) / 256.0
        s["kept"] = torch.full((n, case["kv_heads"], case["keep"]), -1, device="cuda", dtype=torch.int32)
        s["out"] = {**{k: torch.empty_like(s[k]) for k in ("len", "nfree", "table")}, "free": s["free"].clone(),
                    "from_len": torch.empty_like(s["len"]), "status": torch.empty(2, device="cuda", dtype=torch.int32)}
        s["dropped"] = torch.zeros_like(s["len"])
    elif kind == "verify":
        drafts, vocab, n = _drafts(case), case["vocab"], case["requests"]
        start = np.concatenate([[0], np.cumsum(drafts + 1)])
        rows = int(start[-1])
        seq = _i32(np.repeat(np.arange(n), drafts + 1)).long()
        s.update(rows=rows, start=_i32(start[:-1]), count=_i32(drafts + 1))
        x = 1.5 * _randn(g, rows, vocab)
        likely = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        at = torch.arange(rows, device="cuda")
        x[at, likely] += math.log(vocab) + 2.0 + 2.0 * _randn(g, rows)     # a row's mode has about half of it and more
        t = 0.5 + 0.75 * torch.rand(n, generator=g, device="cuda")
        t[torch.rand(n, generator=g, device="cuda") < 0.2] = 0.0
        s.update(x=x, t=t, u=torch.rand(rows, generator=g, device="cuda"), r=torch.rand(n, generator=g, device="cuda"))
        if case["probs"]:               # a draft model that differs a little
            s["q"] = torch.softmax((x + 0.7 * _randn(g, rows, vocab)) / t.clamp(min=0.3)[seq][:, None], -1)
            chosen = torch.multinomial(s["q"], 1, generator=g)[:, 0]
        else:
            chosen = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, likely,
                                 torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
        s["tokens"] = torch.roll(chosen, 1).int()           # row i's judges the token of row i + 1
        s["out"] = {"accepted": torch.empty(n, device="cuda", dtype=torch.int32),
                    "back": torch.empty(n, device="cuda", dtype=torch.int32),
                    "tokens": torch.empty(rows, device="cuda", dtype=torch.int32)}
    else:
        n, page = case["requests"], case["page"]
        back = _drafts(case)
        lens = back + 1 + np.random.default_rng([n, case["max_len"]]).integers(0, case["max_len"], n)
        shuffled = rng.permutation(n)
        lens, back = lens[shuffled], back[shuffled]
        spare = 7
        table, pages, rest = _tables(lens, page, rng, spare, -(-(case["max_len"] + case["drafts"] + 1) // page))
        free = np.full(pages, -1, np.int64)
        free[:spare] = rest
        s.update(ld=table.shape[1], pages=pages, table=_i32(table), len=_i32(lens), back=_i32(back), free=_i32(free),
                 nfree=_i32([spare]))
        s["out"] = {"len": torch.empty_like(s["len"]), "nfree": torch.empty_like(s["nfree"])}
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


def _batch_args(s, c):
    return (s["rows"], c["requests"], s["start"].data_ptr(), s["count"].data_ptr(), s["len"].data_ptr(),
            s["table"].data_ptr(), s["ld"], c["page"], s["pages"])


def _attention_own(s, c):
    r = _rehip()
    (kc, vc), (ks, vs) = s["codes"], s["scales"]
    nbytes = r.attention_kv8_work_bytes(s["rows"], c["requests"], c["max_rows"], c["max_len"], c["heads"], c["kv_heads"],
                                        c["hd"])
    r.attention_kv8_sinks_dev(s["q"].data_ptr(), c["heads"] * c["hd"], *_batch_args(s, c), kc.data_ptr(), vc.data_ptr(),
                              ks.data_ptr(), vs.data_ptr(), c["max_rows"], c["max_len"], c["heads"], c["kv_heads"],
                              c["hd"], c["hd"] ** -0.5, c["window"], c["sinks"], s["ctx"].data_ptr(),
                              s["lse"].data_ptr(), _work(s, nbytes), nbytes)
    return {"ctx": s["ctx"], "lse": s["lse"]}


def _mass_own(s, c):
    _rehip().kv8_mass_dev(s["q"].data_ptr(), c["heads"] * c["hd"], s["lse"].data_ptr(), *_batch_args(s, c),
                          s["codes"][0].data_ptr(), s["scales"][0].data_ptr(), c["max_rows"], c["max_len"], c["heads"],
                          c["kv_heads"], c["hd"], c["hd"] ** -0.5, c["window"], c["sinks"], s["mass"].data_ptr())
    return s["mass"]


def _evict_own(s, c):
    r, o = _rehip(), s["out"]
    (kc, vc), (ks, vs) = s["codes"], s["scales"]
    r.kv_evict_plan_dev(c["requests"], c["page"], c["limit"], c["keep"], s["len"].data_ptr(), s["table"].data_ptr(), s["ld"],
                        s["free"].data_ptr(), s["pages"], s["nfree"].data_ptr(), o["len"].data_ptr(),
                        o["table"].data_ptr(), o["free"].data_ptr(), o["nfree"].data_ptr(), o["from_len"].data_ptr(),
                        s["table"].data_ptr(), s["dropped"].data_ptr(), o["status"].data_ptr())
    r.kv8_evict_dev(c["requests"], o["from_len"].data_ptr(), s["table"].data_ptr(), o["table"].data_ptr(), s["ld"], c["page"],
                    s["pages"], kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), s["mass"].data_ptr(),
                    c["kv_heads"], c["hd"], c["keep"], c["first"], c["recent"], c["max_len"], s["kept"].data_ptr())
    return {**o, "dropped": s["dropped"], "kept": s["kept"], "codes": s["codes"], "scales": s["scales"], "mass": s["mass"]}


def _verify_own(s, c):
    r, o = _rehip(), s["out"]
    nbytes = r.draft_verify_work_bytes(s["rows"], c["requests"], c["vocab"])
    r.draft_verify_dev(s["x"].data_ptr(), c["vocab"], s["rows"], c["vocab"], c["requests"], s["start"].data_ptr(),
                       s["count"].data_ptr(), s["tokens"].data_ptr(), s["q"].data_ptr() if c["probs"] else None, c["vocab"],
                       s["t"].data_ptr(), s["u"].data_ptr(), s["r"].data_ptr(), o["accepted"].data_ptr(),
                       o["back"].data_ptr(), o["tokens"].data_ptr(), _work(s, nbytes), nbytes)
    return o


def _rewind_own(s, c):
    o = s["out"]
    _rehip().kv_rewind_dev(c["requests"], c["page"], s["back"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(), s["ld"],
                           s["free"].data_ptr(), s["pages"], s["nfree"].data_ptr(), o["len"].data_ptr(),
                           o["nfree"].data_ptr())
    return {**o, "free": s["free"]}


# ---- the plain forms -----------------------------------------------------------------------------
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


def _seen_pages(s, c):
    """Numbers of the table's columns that some row of each request may see: (requests, columns)."""
    page, ld = c["page"], s["ld"]
    if not c["window"]:
        return torch.arange(ld, device="cuda").expand(c["requests"], -1)
    few, many = -(-c["sinks"] // page), (c["window"] + c["max_rows"] - 2) // page + 2
    first = (s["len"] - s["count"] - c["window"] + 1).clamp(min=0) // page
    late = first.clamp(min=few)[:, None] + torch.arange(min(many, ld), device="cuda")
    return torch.cat([torch.arange(few, device="cuda").expand(c["requests"], -1), late], 1)


def _page_values(s, columns, which):
    """K's or V's values of these pages of each request, (requests, kv, tokens, hd)."""
    table = s["table"].long().gather(1, columns.clamp(max=s["ld"] - 1)).clamp(min=0)
    x = (_k_rows, _v_rows)[which](s["codes"][which][table]).float() * s["scales"][which][table][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _scores(s, c, columns):
    """scale q . k of every row and the tokens of these pages, -inf where it sees none: (requests, kv, rows, group, tokens)."""
    n, top, hd, kv, page = c["requests"], c["max_rows"], c["hd"], c["kv_heads"], c["page"]
    grp, i = c["heads"] // kv, torch.arange(top, device="cuda")
    count, lens = s["count"].long()[:, None], s["len"].long()[:, None]
    row = (s["start"].long()[:, None] + i).clamp(max=s["rows"] - 1)         # (n, top)
    q = s["q"][row].reshape(n, top, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, top * grp, hd)
    k = _page_values(s, columns, 0)
    x = (q @ k.transpose(-1, -2).contiguous()).reshape(n, kv, top, grp, -1) * hd ** -0.5
    j = (columns[..., None] * page + torch.arange(page, device="cuda")).flatten(1)[:, None]     # (n, 1, tokens)
    pos = (lens - count + i)[..., None]
    seen = (j <= pos) & (i[:, None] < count[..., None])
    if c["window"]:
        seen = seen & ((j > pos - c["window"]) | (j < c["sinks"]))
    return x.masked_fill(~seen[:, None, :, None], -math.inf), row


def _attention_plain(s, c):
    n, top, hd, kv = c["requests"], c["max_rows"], c["hd"], c["kv_heads"]
    columns = _seen_pages(s, c)
    x, _ = _scores(s, c, columns)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    p = (p / z).reshape(n, kv, -1, p.shape[-1])
    y = (p @ _page_values(s, columns, 1)).reshape(n, kv, top, -1, hd).permute(0, 2, 1, 3, 4).reshape(n, top, -1, hd)
    lse = (m + torch.log(z))[..., 0].permute(0, 2, 1, 3).reshape(n, top, -1)
    at = s["seq"].long()
    i = torch.arange(s["rows"], device="cuda") - s["start"].long()[at]
    return {"ctx": y[at, i], "lse": lse[at, i]}


def _mass_plain(s, c):
    n, kv, page = c["requests"], c["kv_heads"], c["page"]
    columns = _seen_pages(s, c)
    x, row = _scores(s, c, columns)
    lse = s["lse"][row].reshape(n, c["max_rows"], kv, -1).permute(0, 2, 1, 3)[..., None]
    new = torch.exp(x - lse).sum((2, 3)).reshape(n, kv, -1, page).transpose(1, 2)          # (n, columns, kv, page)
    j = columns[..., None] * page + torch.arange(page, device="cuda")
    lens, count = s["len"].long()[:, None, None], s["count"].long()[:, None, None]
    pid = s["table"].long().gather(1, columns.clamp(max=s["ld"] - 1))
    pid = torch.where((columns < s["ld"]) & (pid >= 0), pid, s["pages"])[..., None, None]
    g = torch.arange(kv, device="cuda")[:, None]
    at = ((pid * kv + g) * page + torch.arange(page, device="cuda")).reshape(-1)
    mass = torch.cat([s["mass"].reshape(-1), torch.zeros(kv * page, device="cuda")])
    old = mass[at].reshape(new.shape)
    old = torch.where(((j >= lens - count) & (j < lens))[:, :, None], 0.0, old)
    mass[at] = (old + new).reshape(-1)
    s["mass"].copy_(mass[:-kv * page].reshape(s["mass"].shape))
    return s["mass"]


def _evict_plan_plain(s, c):
    n, page, keep, ld, pages = c["requests"], c["page"], c["keep"], s["ld"], s["pages"]
    lens, table, free, nfree = s["len"].long(), s["table"].long(), s["free"].long(), s["nfree"].long()
    fresh = -(-keep // page)
    over = lens > c["limit"]
    rank = torch.cumsum(over, 0) - 1
    ok = over & ((rank + 1) * fresh <= nfree)
    taken = ok.sum() * fresh
    j = torch.arange(ld, device="cuda")
    mine = (nfree - 1 - (rank[:, None] * fresh + j)).clamp(0, pages - 1)
    new = torch.where(j < fresh, free[mine], -1)
    held = ok[:, None] & (j < ((lens + page - 1) // page)[:, None]) & (table >= 0) & (table < pages)
    order = torch.cumsum(held.reshape(-1), 0) - 1
    at = torch.where(held.reshape(-1), nfree - taken + order, pages)
    free = torch.cat([s["free"], s["free"][:1]]).scatter(0, at, s["table"].reshape(-1))[:pages]
    s["dropped"].copy_(torch.where(ok, s["dropped"] + lens - keep, torch.where(lens == 0, 0, s["dropped"])))
    return {"len": torch.where(ok, keep, lens).int(), "nfree": (nfree - taken + held.sum()).int(),
            "table": torch.where(ok[:, None], new, table).int(), "free": free, "from_len": torch.where(ok, lens, 0).int(),
            "status": torch.stack([(over & ~ok).sum(), ok.sum()]).int()}


def _evict_plain(s, c):
    o = _evict_plan_plain(s, c)
    n, page, keep, ld, kv, pages = c["requests"], c["page"], c["keep"], s["ld"], c["kv_heads"], s["pages"]
    lens, fresh = o["from_len"].long()[:, None, None], -(-c["keep"] // c["page"])
    table = s["table"].long()
    valid = ((table >= 0) & (table < pages)).repeat_interleave(page, 1)[:, None]           # (n, 1, tokens)
    mass = s["mass"][table.clamp(0, pages - 1)].transpose(1, 2).reshape(n, kv, -1)
    bits = mass.view(torch.int32).long()                    # ordered as the weights, which are not negative
    t = torch.arange(ld * page, device="cuda")
    key = torch.where(valid, bits + 1, 0) * 2 ** 22 + (2 ** 22 - 1 - t)
    key = torch.where((t < c["first"]) | (t >= lens - c["recent"]), 2 ** 60 - t, key)
    key = torch.where(t < lens, key, -1 - t)
    kept = torch.topk(key, keep, -1)[1].sort(-1)[0]         # (n, kv, keep)
    pad = fresh * page - keep
    live = torch.nn.functional.pad(torch.ones_like(kept, dtype=torch.bool), (0, pad))
    src = torch.nn.functional.pad(kept, (0, pad))
    pid = table.gather(1, (src // page).reshape(n, -1)).reshape(src.shape)
    live = live & (pid >= 0) & (pid < pages)
    pid = pid.clamp(0, pages - 1)
    g = torch.arange(kv, device="cuda")[:, None]
    done = lens[..., 0] > 0                                 # (n, 1)
    # places of the new pages (of requests that are not cut: a page behind the pool's)
    to = torch.where(done, o["table"].long()[:, :fresh], pages)
    for codes, scale, rows, blocks in zip(s["codes"], s["scales"], (_k_rows, _v_rows), (_k_blocks, _v_blocks)):
        old = torch.where(live, scale[pid, g], 0.0)
        new = old.reshape(n, kv, fresh, page).amax(-1)
        ratio = old.reshape(n, kv, fresh, page) / torch.where(new > 0, new, 1.0)[..., None]
        c8 = rows(codes)[pid, g, src % page].reshape(n, kv, fresh, page, -1)
        c8 = torch.round(c8.float() * torch.where(live.reshape(ratio.shape), ratio, 0.0)[..., None]).to(torch.int8)
        every = torch.cat([codes, codes[:1]])
        every[to] = blocks(c8).transpose(1, 2)
        codes.copy_(every[:pages])
        every = torch.cat([scale, scale[:1]])
        every[to] = new.transpose(1, 2)
        scale.copy_(every[:pages])
    m = torch.where(live, s["mass"][pid, g, src % page], 0.0).reshape(n, kv, fresh, page)
    every = torch.cat([s["mass"], s["mass"][:1]])
    every[to] = m.transpose(1, 2)
    s["mass"].copy_(every[:pages])
    s["kept"].copy_(torch.where(done[..., None], kept, s["kept"]))
    return {**o, "dropped": s["dropped"], "kept": s["kept"], "codes": s["codes"], "scales": s["scales"], "mass": s["mass"]}


def _first_largest(x):
    at = torch.arange(x.shape[-1], device="cuda")
    return torch.where(x == x.amax(-1, keepdim=True), at, x.shape[-1]).amin(-1)


def _verify_plain(s, c):
    """In 64 bits: a token is chosen by where a random number falls between sums over the vocabulary."""
    n, vocab, top = c["requests"], c["vocab"], c["drafts"] + 1
    start, count = s["start"].long(), s["count"].long()
    i = torch.arange(top, device="cuda")
    row = (start[:, None] + i).clamp(max=s["rows"] - 1)     # (n, top)
    seq = torch.searchsorted(start, torch.arange(s["rows"], device="cuda"), right=True) - 1
    t = s["t"].double()
    greedy = ~(t > 0)
    x = s["x"].double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, t)[seq][:, None])
    p = e / e.sum(-1, keepdim=True)
    draft = s["tokens"].long()[(row + 1).clamp(max=s["rows"] - 1)]
    best = _first_largest(s["x"])
    q = s["q"].double()[row, draft] if c["probs"] else 1.0
    ok = torch.where(greedy[:, None], best[row] == draft, s["u"].double()[row] * q < p[row, draft])
    ok = ok & (i < (count - 1)[:, None])
    accepted = torch.cumprod(ok.long(), -1).sum(-1)
    b = torch.arange(n, device="cuda")
    last = start + accepted
    rejected = accepted < count - 1
    w = p[last]
    if c["probs"]:
        w = torch.where(rejected[:, None], (w - s["q"].double()[last]).clamp(min=0), w)
    else:
        d = draft[b, accepted.clamp(max=top - 1)]
        w[b, d] = torch.where(rejected, 0.0, w[b, d])
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[last])
    upto = torch.cumsum(w, -1)
    chosen = (upto <= s["r"].double()[:, None] * upto[:, -1:]).sum(-1).clamp(max=vocab - 1)
    chosen = torch.where(greedy, best[last], chosen)
    k = torch.arange(s["rows"], device="cuda") - start[seq]
    tokens = torch.where(k < accepted[seq], torch.roll(s["tokens"], -1).long(), torch.where(k == accepted[seq], chosen[seq], -1))
    return {"accepted": accepted.int(), "back": (count - 1 - accepted).int(), "tokens": tokens.int()}


def _rewind_plain(s, c):
    n, page, ld, pages = c["requests"], c["page"], s["ld"], s["pages"]
    lens, table = s["len"].long(), s["table"].long()
    left = lens - torch.minimum(s["back"].long().clamp(min=0), lens)
    j = torch.arange(ld, device="cuda")
    pages_of = lambda v: ((v + page - 1) // page)[:, None]  # noqa: E731
    gone = (j >= pages_of(left)) & (j < pages_of(lens)) & (table >= 0) & (table < pages)
    order = torch.cumsum(gone.reshape(-1), 0) - 1
    at = torch.where(gone.reshape(-1), s["nfree"].long() + order, pages)
    free = torch.cat([s["free"], s["free"][:1]]).scatter(0, at, s["table"].reshape(-1))[:pages]
    s["free"].copy_(free)
    return {"len": left.int(), "nfree": (s["nfree"].long() + gone.sum()).int(), "free": s["free"]}


PLAIN = {"attention": _attention_plain, "mass": _mass_plain, "evict": _evict_plain, "verify": _verify_plain,
         "rewind": _rewind_plain}
OWN = {"attention": _attention_own, "mass": _mass_own, "evict": _evict_own, "verify": _verify_own, "rewind": _rewind_own}


def run(s):
    return (OWN if own else PLAIN)[s["case"]["kind"]](s, s["case"])


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("attention", "mass"):
        rows, lens = _sizes(case)
        w, sinks = case["window"] or 1 << 40, case["sinks"]
        kv, width = case["kv_heads"] * case["hd"], case["heads"] * case["hd"]
        seen, keys = 0, 0
        for r, n in zip(rows, lens):
            p = np.arange(n - r, n) + 1
            seen += int((np.minimum(p, w) + np.minimum(sinks, np.maximum(p - w, 0))).sum())
            late = min(n, w + r - 1)
            keys += int(late + min(sinks, n - late))
        total = int(rows.sum())
        if kind == "attention":
            return {"bytes": 8 * total * width + 4 * total * case["heads"] + 2 * keys * kv, "flops": 4 * seen * width}
        return {"bytes": 4 * total * width + 4 * total * case["heads"] + keys * kv + 8 * keys * case["kv_heads"],
                "flops": 2 * seen * width}
    if kind == "evict":                 # weights in, codes, weights and indexes of what stays, tables
        lens = _long(case)
        cut = lens > case["limit"]
        tokens, stay = int(lens[cut].sum()), int(cut.sum()) * case["keep"]
        return {"bytes": case["kv_heads"] * (4 * tokens + stay * (4 * case["hd"] + 8)) + 16 * len(lens),
                "flops": case["kv_heads"] * (tokens + 2 * stay * case["hd"])}
    if kind == "verify":                # the rows up to a request's last, and one row of the draft's
        drafts = _drafts(case)
        rows = int((drafts + 1).sum())
        return {"bytes": 4 * case["vocab"] * (rows + (case["requests"] if case["probs"] else 0)) + 16 * rows,
                "flops": 8 * case["vocab"] * rows}
    return {"bytes": 16 * case["requests"], "flops": 4 * case["requests"]}


# ---- the same in 64 bits -----------------------------------------------------------------------
def _values64(s, case, b, which):
    """K's or V's values of request b, (kv, tokens, hd)."""
    pages = torch.as_tensor(s["host"]["table"][b, :-(-int(s["host"]["lens"][b]) // case["page"])], device="cuda")
    t, d = torch.arange(32, device="cuda")[:, None], torch.arange(32, device="cuda")[None]
    where = [d // 8 * 256 + t % 16 * 16 + t // 16 * 8 + d % 8,
             t // 4 % 4 * 256 + d % 16 * 16 + d // 16 * 8 + t // 16 * 4 + t % 4][which]
    x = s["codes"][which][pages][..., where].double()       # (pages, kv, page / 32, hd / 32, 32, 32)
    x = x.transpose(-3, -2).reshape(len(pages), case["kv_heads"], case["page"], case["hd"])
    x = x * s["scales"][which][pages].double()[..., None, None]
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["hd"])[:, :int(s["host"]["lens"][b])]


def _exact_rows(s, case):
    h, grp = s["host"], case["heads"] // case["kv_heads"]
    out = {"ctx": torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64),
           "lse": torch.zeros(s["lse"].shape, device="cuda", dtype=torch.float64)}
    mass = s["mass"].double() if "mass" in s else None
    for b in range(case["requests"]):
        n, to, r = int(h["rows"][b]), int(h["lens"][b]), int(h["start"][b])
        k = _values64(s, case, b, 0)
        v = _values64(s, case, b, 1) if mass is None else None
        pos = torch.arange(to - n, to, device="cuda")[:, None]
        j = torch.arange(to, device="cuda")[None]
        hide = j > pos
        if case["window"]:
            hide = hide | ((pos - j >= case["window"]) & (j >= case["sinks"]))
        if mass is not None:
            got = torch.zeros(case["kv_heads"], to, device="cuda", dtype=torch.float64)
        for i in range(case["heads"]):
            x = s["q"][r:r + n, i].double() @ k[i // grp].T.contiguous() / math.sqrt(case["hd"])
            x = x.masked_fill(hide, -math.inf)
            if mass is None:
                out["lse"][r:r + n, i] = torch.logsumexp(x, -1)
                out["ctx"][r:r + n, i] = torch.softmax(x, -1) @ v[i // grp]
            else:
                got[i // grp] += torch.exp(x - s["lse"][r:r + n, i].double()[:, None]).sum(0)
        if mass is not None:
            for p in range(-(-to // case["page"])):
                lo, hi = p * case["page"], min(to, (p + 1) * case["page"])
                place = mass[int(h["table"][b, p])]
                begun = max(0, min(hi, to - n) - lo)        # tokens of this page that earlier steps brought
                place[:, begun:hi - lo] = 0
                place[:, :hi - lo] += got[:, lo:hi]
    return out if mass is None else mass


def _exact_evict(s, case):
    """The scales and the weights, request after request."""
    h, page, keep, kv = s["host"], case["page"], case["keep"], case["kv_heads"]
    fresh, top = -(-keep // page), h["spare"]
    mass, scales = s["mass"].double().cpu().numpy(), [x.double().cpu().numpy() for x in s["scales"]]
    for b in range(case["requests"]):
        to = int(h["lens"][b])
        if to <= case["limit"]:
            continue
        if top < fresh:
            break
        new, top = h["free"][top - fresh:top][::-1], top - fresh
        pages = h["table"][b, :-(-to // page)]
        for g in range(kv):
            m = mass[pages, g].reshape(-1)[:to]
            order = m.copy()
            order[:case["first"]] = np.inf
            order[to - case["recent"]:] = np.inf
            stay = np.sort(np.argsort(-order, kind="stable")[:keep])
            for p in range(fresh):
                some = stay[p * page:(p + 1) * page]
                for scale in scales:
                    scale[new[p], g] = scale[pages[some // page], g].max()
                mass[new[p], g] = 0
                mass[new[p], g, :len(some)] = m[some]
    return {"codes": [None, None], "scales": scales, "mass": mass}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("verify", "rewind"):    # whole numbers alone
        return None
    s = prepare(case, seed)
    return _exact_evict(s, case) if kind == "evict" else _exact_rows(s, case)
