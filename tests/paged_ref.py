"""Plain 64-bit statements of the paged-cache and beam-search operators, one
token, head or row at a time, for the tests."""

from __future__ import annotations

import math

import numpy as np

# Half a step of each type, relative to the value (round to nearest).
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rotate(x, pos, rotary_dim, base, interleaved, scale):
    """x [heads, head_dim] float64 turned at `pos`."""
    y = x.copy()
    for d in range(rotary_dim // 2):
        a = pos * scale * base ** (-2.0 * d / rotary_dim)
        i, j = (2 * d, 2 * d + 1) if interleaved else (d, d + rotary_dim // 2)
        y[:, i] = x[:, i] * math.cos(a) - x[:, j] * math.sin(a)
        y[:, j] = x[:, j] * math.cos(a) + x[:, i] * math.sin(a)
    return y


def append(q, k, v, kc, vc, q_start, kv_len, table, rotary_dim, base, interleaved, scale):
    """-> rotated q (rows of no sequence as they were) and the caches, float64.
    q [tokens, heads, hd] or None; caches [pages, page_size, kv_heads, hd]."""
    kc, vc = kc.copy(), vc.copy()
    qo = None if q is None else q.copy()
    pages, ps = kc.shape[:2]
    for b in range(len(kv_len)):
        for t in range(q_start[b], q_start[b + 1]):
            pos = kv_len[b] - (q_start[b + 1] - t)
            if q is not None:
                qo[t] = rotate(q[t], pos, rotary_dim, base, interleaved, scale)
            if pos < 0 or pos // ps >= table.shape[1]:
                continue
            page = table[b, pos // ps]
            if 0 <= page < pages:
                kc[page, pos % ps] = rotate(k[t], pos, rotary_dim, base, interleaved, scale)
                vc[page, pos % ps] = v[t]
    return qo, kc, vc


def rotation_bound(x, rotary_dim, interleaved):
    """Per element, |x1| + |x2| of its pair (0 where nothing turns)."""
    s = np.zeros_like(x)
    for d in range(rotary_dim // 2):
        i, j = (2 * d, 2 * d + 1) if interleaved else (d, d + rotary_dim // 2)
        s[..., i] = s[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    return s


def attention(q, kc, vc, q_start, kv_len, table, scale, out, rounds_p):
    """-> (out float64, bound on |kernel - out| before the output's rounding).
    q [tokens, heads, hd]; rows of no sequence keep `out`.

    The bound: scores sum hd products in fp32 (each partial sum off by at most
    2^-23 of the sum of magnitudes), which moves a weight by twice that,
    relatively; exp2 and the running rescaling are off by 2^-22 a step; sums
    over len weights in fp32 by len * 2^-23; weights that are rounded to the
    type by half a step.  All of it is relative to sum_j p_j |v_j|."""
    out = out.copy()
    tol = np.zeros_like(out)
    pages, ps, kvh, hd = kc.shape
    nq = q.shape[1]
    group = nq // kvh
    for b in range(len(kv_len)):
        n = q_start[b + 1] - q_start[b]
        for i in range(n):
            t = q_start[b] + i
            seen = kv_len[b] - n + i + 1
            out[t] = 0.0
            if seen <= 0:
                continue
            K = np.zeros((seen, kvh, hd))
            V = np.zeros((seen, kvh, hd))
            for p in range(seen):
                page = table[b, p // ps]
                if 0 <= page < pages:
                    K[p], V[p] = kc[page, p % ps], vc[page, p % ps]
            for h in range(nq):
                s = K[:, h // group] @ q[t, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h] = w @ V[:, h // group]
                mags = (np.abs(K[:, h // group]) @ np.abs(q[t, h])).max() * scale
                rel = 2 * hd * 2.0 ** -23 * mags + (seen + hd) * 2.0 ** -23 + 2.0 ** -20
                tol[t, h] = (rel + rounds_p) * (w @ np.abs(V[:, h // group]))
    return out, tol


def select(logits, scores, finished, eos, pad, beams):
    """logits [batch * beams, vocab] float64 -> tokens, parents, values, ended
    and the smallest gap between values that are not equal."""
    batch, vocab = scores.shape[0], logits.shape[1]
    tokens = np.full((batch, beams), pad, np.int64)
    parents = np.tile(np.arange(beams, dtype=np.int32), (batch, 1))
    values = np.full((batch, beams), -np.inf)
    ended = np.ones((batch, beams), bool)
    gap = np.inf
    for e in range(batch):
        found = []
        for b in range(beams):
            s = float(scores[e, b])
            if finished is not None and finished[e, b]:
                if s > -np.inf:
                    found.append((-s, b * vocab + pad))
                continue
            x = logits[e * beams + b]
            m = np.max(x)
            if not np.isfinite(m):
                continue
            lse = m + np.log(np.sum(np.exp(x - m)))
            if not np.isfinite(lse):
                continue
            for v in range(vocab):
                val = s + x[v] - lse
                if val > -np.inf:
                    found.append((-val, b * vocab + v))
        found.sort()
        top = found[:beams + 1]
        for (x, _), (y, _) in zip(top, top[1:]):
            if x != y:
                gap = min(gap, y - x)
        for k, (val, at) in enumerate(found[:beams]):
            tokens[e, k], parents[e, k], values[e, k] = at % vocab, at // vocab, -val
            ended[e, k] = (finished is not None and bool(finished[e, at // vocab])) \
                or at % vocab in eos
    return tokens, parents, values, ended, gap


def reorder(table, parents, kv_len, pool_start, pool_pages, kc, vc):
    """Caches [layers, pages, page_size, ...] (copied).  -> tables, lengths,
    caches, whether anything was out of range."""
    batch, beams = parents.shape
    ps, num_pages, width = kc.shape[2], kc.shape[1], table.shape[1]
    kc, vc = kc.copy(), vc.copy()
    out = np.full_like(table, -1)
    lens = np.zeros_like(kv_len)
    bad = False
    for e in range(batch):
        lo, hi = int(pool_start[e]), int(pool_start[e]) + pool_pages
        range_ok = lo >= 0 and hi <= num_pages
        bad |= not range_ok
        src = []
        for i in range(beams):
            p = parents[e, i]
            n = int(kv_len[e * beams + p]) if 0 <= p < beams else -1
            ok = 0 <= n <= width * ps
            bad |= not ok
            src.append((e * beams + p, n) if ok else None)
        mine = lambda page: range_ok and lo <= page < hi  # noqa: E731
        held = set()
        for i, s in enumerate(src):
            if s is None:
                continue
            lens[e * beams + i] = s[1]
            for j in range(s[1] // ps):
                page = table[s[0], j]
                if 0 <= page < num_pages:
                    out[e * beams + i, j] = page
                    if mine(page):
                        held.add(int(page))
                else:
                    bad = True
        read = set(held)
        parts, kept = {}, set()
        for i, s in enumerate(src):
            if s is None or s[1] % ps == 0 or s[1] // ps >= width:
                continue
            page = int(table[s[0], s[1] // ps])
            if not 0 <= page < num_pages:
                bad = True
                parts[i] = None
                continue
            first = page not in [x for x in parts.values()]
            parts[i] = page
            if mine(page) and page not in read and first:
                kept.add(i)
                held.add(page)
        free = [page for page in range(lo, hi) if page not in held] if range_ok else []
        for i, s in enumerate(src):
            if s is None or s[1] // ps >= width:
                continue
            at, fill = divmod(s[1], ps)
            if i in kept:
                out[e * beams + i, at] = parts[i]
            elif fill and parts[i] is None:
                pass
            elif not free:
                bad = True
            else:
                page = free.pop(0)
                out[e * beams + i, at] = page
                if fill:
                    kc[:, page, :fill] = kc[:, parts[i], :fill]
                    vc[:, page, :fill] = vc[:, parts[i], :fill]
    return out, lens, kc, vc, bad
