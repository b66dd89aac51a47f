"""Plain restatements of the batched serving step (include/rehip.h, "batched serving"), in numpy: float64, or
float32 operation by operation where the result is defined bit by bit. Nothing here calls the library."""
import numpy as np

F32 = np.float32


# ---- the cache's layout ------------------------------------------------------------------------
def block_bytes(is_v):
    t, d = np.meshgrid(np.arange(32), np.arange(32), indexing="ij")
    if is_v:
        return 256 * (t // 4 % 4) + 16 * (d % 16) + 8 * (d // 16) + 4 * (t // 16) + t % 4
    return 256 * (d // 8) + 16 * (t % 16) + 8 * (t // 16) + d % 8


def unpack(codes, n_pages, kv_heads, page, hd, is_v):
    """(pages, heads, page, hd) codes of the flat cache."""
    c = np.asarray(codes, np.int8).reshape(n_pages, kv_heads, page // 32, hd // 32, 1024)[..., block_bytes(is_v)]
    return c.transpose(0, 1, 2, 4, 3, 5).reshape(n_pages, kv_heads, page, hd)


def pack(codes, is_v):
    n, h, page, hd = codes.shape
    c = codes.reshape(n, h, page // 32, 32, hd // 32, 32).transpose(0, 1, 2, 4, 3, 5)
    out = np.empty((n, h, page // 32, hd // 32, 1024), np.int8)
    out[..., block_bytes(is_v)] = c
    return out


# ---- plan --------------------------------------------------------------------------------------
def plan(page, new_len, kv_len, table, free, n_free, cap):
    """Request after request; table and free are changed in place."""
    n, ld = table.shape
    need_pages = lambda t: -(-t // page)  # noqa: E731
    for b in range(n):
        if new_len[b] < 0:
            for j in range(need_pages(kv_len[b])):
                if n_free < len(free):
                    free[n_free] = table[b, j]
                    n_free += 1
    left, asked = n_free, 0
    out_len, start, count = kv_len.copy(), np.zeros(n, np.int32), np.zeros(n, np.int32)
    refused = row = 0
    for b in range(n):
        new = max(int(new_len[b]), 0)
        start[b] = row
        row += new
        if new_len[b] < 0:
            out_len[b] = 0
            continue
        fits = kv_len[b] + new <= ld * page
        held = need_pages(kv_len[b])
        need = need_pages(kv_len[b] + new) - held if fits and new else 0
        asked += need
        if not fits or (need and asked > n_free):
            refused += new > 0
            continue
        for j in range(need):
            table[b, held + j] = free[n_free - 1 - (asked - need) - j]
        left -= need
        out_len[b] = kv_len[b] + new
        count[b] = new
    seq, pos, slot = (np.full(cap, -1, np.int32) for _ in range(3))
    for b in range(n):
        for i in range(count[b]):
            t = start[b] + i
            if t < cap:
                seq[t], pos[t] = b, out_len[b] - count[b] + i
                slot[t] = table[b, pos[t] // page] * page + pos[t] % page
    return dict(len=out_len, n_free=left, start=start, count=count, seq=seq, pos=pos, slot=slot,
                status=[refused, row])


# ---- rotary positions --------------------------------------------------------------------------
def rope(x, pos, freqs, mscale, rot, interleaved):
    """float64, x (rows, heads, hd)."""
    y = x.astype(np.float64).copy()
    a = pos[:, None].astype(np.float64) * freqs
    c, s = (f(a)[:, None] * mscale for f in (np.cos, np.sin))
    i0 = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    i1 = i0 + 1 if interleaved else i0 + rot // 2
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    y[pos < 0] = x[pos < 0]
    return y


# ---- append ------------------------------------------------------------------------------------
def append(x, start, count, kv_len, table, page, codes, scale):
    """codes (pages, heads, page, hd) int8 and scale (pages, heads) f32 in place; x (rows, heads, hd)."""
    n_pages, heads = scale.shape
    with np.errstate(all="ignore"):
        for b in range(len(start)):
            first = int(kv_len[b]) - int(count[b])
            if count[b] <= 0 or first < 0 or kv_len[b] > table.shape[1] * page:
                continue
            for p in range(first // page, -(-int(kv_len[b]) // page)):
                pid = table[b, p]
                if not 0 <= pid < n_pages:
                    continue
                lo, hi = max(p * page, first), min((p + 1) * page, int(kv_len[b]))
                o0, o1 = lo - p * page, hi - p * page
                for h in range(heads):
                    v = x[start[b] + lo - first:start[b] + hi - first, h]
                    amax = np.max(np.abs(np.where(np.isfinite(v), v, F32(0))))
                    s = F32(amax) * F32(F32(1) / F32(127))
                    s = F32(0) if s < np.finfo(F32).tiny else s
                    old = scale[pid, h] if o0 else F32(0)
                    s = max(s, old)
                    if o0 and s > old:
                        codes[pid, h, :o0] = np.rint(codes[pid, h, :o0].astype(F32) * F32(old / s)).astype(np.int8)
                    q = np.rint(v / s) if s > 0 else np.zeros_like(v)
                    codes[pid, h, o0:o1] = np.clip(np.nan_to_num(np.where(np.isnan(v), 0, q), posinf=127,
                                                                 neginf=-127), -127, 127).astype(np.int8)
                    scale[pid, h] = s


# ---- attention ---------------------------------------------------------------------------------
def attention(q, start, count, kv_len, table, page, kcodes, vcodes, kscale, vscale, scale, window, ctx):
    """float64 results of the batch's rows written over `ctx` (rows, heads, hd) in float64, and a bound of
    what f32-accurate arithmetic may be off by, per (row, head) (0 for rows that are left).

    A score is a sum of hd products (each rounded, q in parts good to 2^-22, then added one after the
    other at worst) and two factors: off by at most delta = (hd + 16) 2^-24 scale sum |q k|. All scores
    off by delta change a probability by a factor of at most exp(2 delta), so the output by at most
    4 delta max |v| for the small deltas here; exp, the sums over n keys (chains of n / 16 steps and a few
    joins), the split and the final division add (n / 16 + 64) 2^-24 max |v|."""
    n_pages, kv_heads, _, hd = kcodes.shape
    heads = q.shape[1]
    grp = heads // kv_heads
    tol = np.zeros(ctx.shape[:2])
    for b in range(len(start)):
        n = int(count[b])
        for i in range(n):
            r, p = int(start[b]) + i, int(kv_len[b]) - n + i
            j = np.arange(max(0, p - window + 1) if window else 0, p + 1)
            pid = table[b, j // page] if len(j) else np.empty(0, int)
            j, pid = j[(pid >= 0) & (pid < n_pages)], pid[(pid >= 0) & (pid < n_pages)]
            if len(j) == 0:
                ctx[r] = 0
                continue
            for h in range(kv_heads):
                k = kcodes[pid, h, j % page].astype(np.float64) * kscale[pid, h].astype(np.float64)[:, None]
                v = vcodes[pid, h, j % page].astype(np.float64) * vscale[pid, h].astype(np.float64)[:, None]
                for g in range(h * grp, (h + 1) * grp):
                    x = q[r, g].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        s = k @ x * scale
                        e = np.exp(s - s.max())
                        ctx[r, g] = (e / e.sum()) @ v
                        delta = (hd + 16) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(x)).max()
                    tol[r, g] = np.abs(v).max() * (4 * delta + (len(j) / 16 + 64) * 2.0 ** -24)
    return tol


# ---- log probabilities -------------------------------------------------------------------------
def logprobs(x, targets, k):
    """float64 (logprob, entropy, ids, top); x (rows, vocab) float32."""
    x64 = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x64.max(-1, keepdims=True)
        d = x64 - m
        e = np.exp(d)
        z = e.sum(-1, keepdims=True)
        lp = d - np.log(z)
        ent = (np.log(z) - np.where(e == 0, 0, e * d).sum(-1, keepdims=True) / z)[:, 0]
    rank = np.where(np.isnan(x), -np.inf, x)
    ids = np.argsort(-rank, axis=-1, kind="stable")[:, :k]
    rows = np.arange(len(x))
    inside = (targets >= 0) & (targets < x.shape[1])
    logp = np.where(inside, lp[rows, np.where(inside, targets, 0)], 0)
    return logp, ent, ids, np.take_along_axis(lp, ids, -1)
