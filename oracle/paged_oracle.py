"""float64 and whole-number restatement of the key-value cache in pages: attention over it, and the
handing out, sharing, freeing and moving of its pages, one sequence and one page after another.

A cache is (k_pages, v_pages [L, P, H, ps, D], refs [P], page_table [N, M]), CPU tensors; the functions
return new ones.
"""
import math

import torch


def rows_of(cache, layer, kv, b, h, n):
    """(float64 [n, D], bool [n]): the first n rows of a sequence and whether they have a page."""
    pages, refs, table = cache[kv][layer], cache[2], cache[3]
    ps, D = pages.shape[2:]
    rows, held = torch.zeros(n, D, dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    for c in range(-(-n // ps)):
        p = int(table[b, c])
        if 0 <= p < refs.numel():
            part = slice(c * ps, min(n, (c + 1) * ps))
            rows[part], held[part] = pages[p, h, :part.stop - part.start].double(), True
    return rows, held


def attend(q, cache, k=None, v=None, lens=0, causal=False, softmax_scale=None, layer=0):
    """(out float64 [B, S, Hq, D], sum of p |v| of the same shape, the new cache)."""
    B, S, Hq, D = q.shape
    new = [x.clone() for x in cache]
    _, P, H, ps, _ = cache[0].shape
    cap = cache[3].shape[1] * ps
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else softmax_scale
    lens = [min(max(int(x), 0), cap) for x in ([lens] * B if isinstance(lens, int) else lens.tolist())]
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b, n in enumerate(lens):
        s_new = S if k is not None else 0
        end = min(cap, n + s_new)
        for h in range(H):
            (kr, held), (vr, _) = (rows_of(cache, layer, i, b, h, n) for i in range(2))
            if k is not None:
                kr, vr = (torch.cat((r, x[b, :end - n, h].double())) for r, x in ((kr, k), (vr, v)))
                held = torch.cat((held, torch.ones(end - n, dtype=torch.bool)))
            for i in range(S):
                limit = max(0, min(end, n + s_new - S + i + 1) if causal else end)
                see = held[:limit].nonzero()[:, 0]
                if not see.numel():
                    continue
                for g in range(Hq // H):
                    hq = h * (Hq // H) + g
                    p = torch.softmax(kr[see] @ q[b, i, hq].double() * scale, 0)
                    out[b, i, hq] = p @ vr[see]
                    mag[b, i, hq] = p @ vr[see].abs()
        for j in range(n, end):
            p = int(cache[3][b, j // ps])
            if 0 <= p < P and int(cache[2][p]) == 1:
                new[0][layer, p, :, j % ps], new[1][layer, p, :, j % ps] = k[b, j - n], v[b, j - n]
    return out, mag, new


def _each(x, n):
    return [int(x)] * n if isinstance(x, int) else [int(y) for y in x.tolist()]


def reserve(cache, lens, new_rows):
    """(the new cache, [N] columns left without a page of their own)."""
    new = [x.clone() for x in cache]
    kp, vp, refs, table = new
    P, ps = kp.shape[1], kp.shape[3]
    N, M = table.shape
    before = cache[2].tolist()
    cap = M * ps
    asked, askers = [], {}
    lens = [min(max(x, 0), cap) for x in _each(lens, N)]
    for n, (a, m) in enumerate(zip(lens, _each(new_rows, N))):
        end = min(cap, a + max(m, 0))
        asked.append(range(a // ps, -(-end // ps)) if end > a else range(0))
        for c in asked[n]:
            p = int(table[n, c])
            if 0 <= p < P:
                askers.setdefault(p, []).append((n, c))
    free = iter([p for p in range(P) if before[p] == 0])
    for n, cols in enumerate(asked):
        for c in cols:
            p = int(table[n, c])
            held = 0 <= p < P
            if held and (before[p] <= 1 or (len(askers[p]) == before[p] and askers[p][0] == (n, c))):
                continue
            to = next(free, None)
            if to is None:
                continue
            table[n, c], refs[to] = to, 1
            if held:
                refs[p] -= 1
                if c == lens[n] // ps:
                    for x in (kp, vp):
                        x[:, to, :, :lens[n] % ps] = x[:, p, :, :lens[n] % ps]
    short = [sum(not 0 <= int(table[n, c]) < P or int(refs[table[n, c]]) > 1 for c in cols) for n, cols in enumerate(asked)]
    return new, torch.tensor(short, dtype=torch.int32)


def fork(cache, parents):
    new = [x.clone() for x in cache]
    table, refs = cache[3].tolist(), cache[2].tolist()
    for n, p in enumerate(parents.tolist()):
        if 0 <= p < len(table) and p != n:
            for old, e in zip(table[n], table[p]):
                if 0 <= old < len(refs):
                    refs[old] -= 1
                if 0 <= e < len(refs):
                    refs[e] += 1
            new[3][n] = cache[3][p]
    new[2][:] = torch.tensor(refs)
    return new


def free(cache, keep):
    new = [x.clone() for x in cache]
    refs, table, ps = new[2], new[3], cache[0].shape[3]
    for n, rows in enumerate(_each(keep, table.shape[0])):
        for c in range(table.shape[1]):
            if c * ps >= rows:
                if 0 <= int(table[n, c]) < refs.numel():
                    refs[table[n, c]] -= 1
                table[n, c] = -1
    return new


def compact(cache):
    """(the new cache, pages in use)."""
    new = [x.clone() for x in cache]
    kp, vp, refs, table = new
    used = int((refs > 0).sum())
    holes = [p for p in range(used) if refs[p] == 0]
    for dst, src in zip(holes, [p for p in range(used, refs.numel()) if refs[p] > 0]):
        for x in (kp, vp):
            x[:, dst] = x[:, src]
        refs[dst], refs[src] = int(refs[src]), 0
        table[table == src] = dst
    return new, used


def copy(cache, src, dst, source=None):
    new = [x.clone() for x in cache]
    source = cache if source is None else source
    for a, b in zip(src.tolist(), dst.tolist()):
        if 0 <= a < source[0].shape[1] and 0 <= b < new[0].shape[1]:
            for i in range(2):
                new[i][:, b] = source[i][:, a]
    return new


def dealt(L, P, H, ps, D, N, M, lens, g, scale=2.0):
    """A cache of random rows in which sequence n holds the pages of its first lens[n] rows, anywhere."""
    kp, vp = ((torch.randn(L, P, H, ps, D, generator=g) * s).bfloat16() for s in (scale, 1.0))
    table, refs = torch.full((N, M), -1, dtype=torch.int32), torch.zeros(P, dtype=torch.int32)
    order = torch.randperm(P, generator=g).int()
    at = 0
    for n, rows in enumerate(lens):
        c = min(M, -(-max(int(rows), 0) // ps))
        table[n, :c] = order[at:at + c]
        refs[order[at:at + c].long()] = 1
        at += c
    assert at <= P
    return [kp, vp, refs, table]
