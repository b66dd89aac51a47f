"""Plain restatements, in numpy, of serving long conversations (include/rehip.h): attention with sinks, the weights of a
step, eviction, drafts verified and tokens taken back. float64, or float32 operation by operation where the result is
defined bit by bit. Nothing here calls the library."""
import numpy as np

F32 = np.float32
EPS = 2.0 ** -24                 # half a step of f32, relative


def seen_tokens(p, window, sinks):
    """The tokens that a row at position p sees."""
    j = np.arange(p + 1)
    return j[(j > p - window) | (j < sinks)] if window else j


def _row_scores(q, b, i, batch, codes, scales, scale, window, sinks):
    """Of row i of request b: its row number, the seen tokens' numbers, pages and, per head, scores and their error bound."""
    start, count, kv_len, table, page = batch
    n_pages, kv_heads, _, hd = codes.shape
    r, p = int(start[b]) + i, int(kv_len[b]) - int(count[b]) + i
    j = seen_tokens(p, window, sinks)
    j = j[j < table.shape[1] * page]
    pid = table[b, j // page] if len(j) else np.empty(0, int)
    there = (pid >= 0) & (pid < n_pages)
    j, pid = j[there], pid[there]
    heads = q.shape[1]
    grp = heads // kv_heads
    s, delta = np.zeros((heads, len(j))), np.zeros(heads)
    for h in range(kv_heads if len(j) else 0):
        k = codes[pid, h, j % page].astype(np.float64) * scales[pid, h].astype(np.float64)[:, None]
        for g in range(h * grp, (h + 1) * grp):
            x = q[r, g].astype(np.float64)
            with np.errstate(invalid="ignore"):
                s[g] = k @ x * scale
                # a sum of hd products and two factors (see serving_ref.attention)
                delta[g] = (hd + 16) * EPS * abs(scale) * (np.abs(k) @ np.abs(x)).max()
    return r, j, pid, s, delta


def attention(q, batch, cache, scale, window, sinks, ctx, lse):
    """float64 results over `ctx` (rows, heads, hd) and `lse` (rows, heads), and what f32-accurate arithmetic may be off by
    in each (serving_ref.attention has the context's derivation). lse = m + ln l: the scores' delta, l's relative error (n / 16 + 64) EPS,
    and the roundings of m (of the size of lse and of log2 l, below 32), of log2 l, of their sum and of the product with ln 2: 8."""
    start, count, kv_len, table, page = batch
    kc, vc, ks, vs = cache
    heads, hd = q.shape[1:]
    grp = heads // kc.shape[1]
    tol, tol_lse = np.zeros(ctx.shape[:2]), np.zeros(lse.shape)
    for b in range(len(start)):
        for i in range(int(count[b])):
            r, j, pid, s, delta = _row_scores(q, b, i, batch, kc, ks, scale, window, sinks)
            if len(j) == 0:
                ctx[r], lse[r] = 0, -np.inf
                continue
            for g in range(heads):
                h = g // grp
                v = vc[pid, h, j % page].astype(np.float64) * vs[pid, h].astype(np.float64)[:, None]
                with np.errstate(invalid="ignore"):
                    m = s[g].max()
                    e = np.exp(s[g] - m)
                    ctx[r, g] = (e / e.sum()) @ v
                    lse[r, g] = m + np.log(e.sum())
                tol[r, g] = np.abs(v).max() * (4 * delta[g] + (len(j) / 16 + 64) * EPS)
                tol_lse[r, g] = delta[g] + (len(j) / 16 + 64) * EPS + 8 * EPS * (abs(lse[r, g]) + 32)
    return tol, tol_lse


def mass(q, lse, batch, kc, ks, scale, window, sinks, masses):
    """Adds to `masses` (pages, heads, page) in float64; what f32-accurate arithmetic may be off by. A weight exp(s - lse): the
    scores' delta, the roundings of lse log2 e, of s log2 e - that (sizes |lse|, |s|: 4) and exp2's 2 units of the last place; its sum over
    the vectors: a chain of a sixteenth of them and a tree; then one sum with what was there."""
    start, count, kv_len, table, page = batch
    n_pages, kv_heads = masses.shape[:2]
    heads = q.shape[1]
    grp = heads // kv_heads
    tol = np.zeros(masses.shape)
    for b in range(len(start)):
        n, to = int(count[b]), min(int(kv_len[b]), table.shape[1] * page)
        if n <= 0:
            continue
        for j in range(max(0, int(kv_len[b]) - n), to):
            if 0 <= table[b, j // page] < n_pages:
                masses[table[b, j // page], :, j % page] = 0
        added, off = np.zeros(masses.shape), np.zeros(masses.shape)
        for i in range(n):
            r, j, pid, s, delta = _row_scores(q, b, i, batch, kc, ks, scale, window, sinks)
            for g in range(heads):
                if len(j) == 0 or not np.isfinite(lse[r, g]) or not np.all(np.isfinite(q[r, g])):
                    continue
                p = np.exp(s[g] - float(lse[r, g]))
                np.add.at(added, (pid, g // grp, j % page), p)
                np.add.at(off, (pid, g // grp, j % page),
                          p * (delta[g] + 4 * EPS * (abs(float(lse[r, g])) + np.abs(s[g]) + 2)))
        tol += off + added * (n * grp / 16 + 24) * EPS + np.where(added > 0, np.abs(masses) * EPS, 0)
        masses += added
    return tol


def evict_plan(page, limit, keep, kv_len, table, free, n_free, dropped):
    """New (lengths, table, stack, its height, from_len, from_table rows by request, status); `dropped` in place."""
    n, ld = table.shape
    fresh = -(-keep // page)
    out_len, out_table, stack = kv_len.copy(), table.copy(), list(free[:n_free])
    from_len, rows, cut, left = np.zeros(n, np.int32), {}, [], 0
    for b in range(n):
        if dropped is not None and kv_len[b] == 0:
            dropped[b] = 0
        if not limit < kv_len[b] <= ld * page:
            continue
        if len(stack) < fresh:
            left += 1
            continue
        rows[b] = table[b].copy()
        out_table[b] = -1
        for j in range(fresh):
            out_table[b, j] = stack.pop()
        from_len[b], out_len[b] = kv_len[b], keep
        if dropped is not None:
            dropped[b] += kv_len[b] - keep
        cut.append(b)
    for b in cut:
        stack += [e for e in rows[b][:-(-int(from_len[b]) // page)] if 0 <= e < len(free)]
    return out_len, out_table, np.array(stack, np.int32), from_len, rows, [left, len(cut)]


def evict(from_len, rows, table, page, cache, masses, keep, first, recent, kept):
    """The move in place: cache is (kcodes, vcodes, kscale, vscale) with codes (pages, heads, page, hd)."""
    kc, vc, ks, vs = cache
    n_pages, kv_heads = ks.shape
    fresh = -(-keep // page)
    old = [x.copy() for x in cache], None if masses is None else masses.copy()
    for b, row in rows.items():
        to = int(from_len[b])
        pid = row[np.arange(to) // page]
        there = (pid >= 0) & (pid < n_pages)
        at = np.where(there, pid, 0)
        for h in range(kv_heads):
            if masses is None:
                stay = np.r_[np.arange(first), np.arange(to - recent, to)]
            else:
                m = old[1][at, h, np.arange(to) % page].astype(np.float64)
                rank = np.where(there, np.where(np.isnan(m), -np.inf, m), 0)
                middle = np.arange(first, to - recent)
                order = sorted(middle, key=lambda t: (not there[t], -rank[t], t))
                stay = np.sort(np.r_[np.arange(first), order[:keep - first - recent],
                                     np.arange(to - recent, to)]).astype(int)
            kept[b, h] = stay
            for p in range(fresh):
                new = table[b, p]
                some = stay[p * page:(p + 1) * page]
                for codes, scale, oc, os in ((kc, ks, old[0][0], old[0][2]), (vc, vs, old[0][1], old[0][3])):
                    s = np.where(there[some], os[at[some], h], F32(0)).astype(F32)
                    top = s.max()
                    scale[new, h] = top
                    codes[new, h] = 0
                    if top > 0:
                        ratio = (s / top).astype(F32)[:, None]
                        c = np.rint(oc[at[some], h, some % page].astype(F32) * ratio)
                        codes[new, h, :len(some)] = c.astype(np.int8)
                if masses is not None:
                    masses[new, h] = 0
                    masses[new, h, :len(some)] = np.where(there[some], old[1][at[some], h, some % page], F32(0))


def rewind(page, back, kv_len, table, free, n_free, n_pages):
    """(lengths, stack)."""
    out, stack = kv_len.copy(), list(free[:n_free])
    for b in range(len(kv_len)):
        if not 0 <= kv_len[b] <= table.shape[1] * page:
            continue
        out[b] = kv_len[b] - min(max(int(back[b]), 0), int(kv_len[b]))
        gone = table[b, -(-int(out[b]) // page):-(-int(kv_len[b]) // page)]
        stack += [e for e in gone if 0 <= e < n_pages]
    return out, np.array(stack, np.int32)


def verify(x, start, count, tokens, probs, temperature, accept_u, sample_u, out):
    """(accepted, back), the tokens into `out`."""
    vocab = x.shape[1]
    accepted, back = np.zeros(len(start), np.int32), np.zeros(len(start), np.int32)
    for b in range(len(start)):
        n, r0 = int(count[b]), int(start[b])
        if n <= 0:
            continue
        t = 1.0 if temperature is None else float(temperature[b])
        token = -1
        for i in range(n):
            row = x[r0 + i].astype(np.float64)
            fine = not np.any(np.isnan(row)) and not np.any(row == np.inf) and np.any(row > -np.inf)
            draft = int(tokens[r0 + i + 1]) if i < n - 1 else None
            p = None
            if fine and t > 0:
                with np.errstate(all="ignore"):
                    p = np.exp((row - row.max()) / t)
                p = np.where(row == -np.inf, 0.0, p)
                p /= p.sum()
            ok = False
            if draft is not None and fine and 0 <= draft < vocab:
                if t > 0:
                    q = 1.0 if probs is None else float(probs[r0 + i, draft])
                    ok = float(accept_u[r0 + i]) * q < p[draft]
                else:
                    ok = draft == int(np.argmax(row))
            if ok:
                out[r0 + i] = draft
                continue
            if fine and t > 0:
                w = p.copy()
                if draft is not None:
                    if probs is not None:
                        w = np.maximum(p - probs[r0 + i].astype(np.float64), 0)
                    elif 0 <= draft < vocab:
                        w[draft] = 0
                    if not w.sum() > 0:
                        w = p
                upto = np.cumsum(w)
                above = np.nonzero((upto > float(sample_u[b]) * upto[-1]) & (w > 0))[0]
                token = int(above[0]) if len(above) else int(np.nonzero(w > 0)[0][-1])
            elif fine:
                token = int(np.argmax(row))
            accepted[b], back[b] = i, n - 1 - i
            out[r0 + i] = token
            out[r0 + i + 1:r0 + n] = -1
            break
    return accepted, back
