"""A key-value cache in pages, and the attention that reads it, as measurable cases.

* ``decode`` ``extend``  attention over the pages that a table gives each sequence: one new token per
             sequence, or several (draft tokens, a turn, a piece of a prompt), with query heads that
             share key-value heads. The pages take the call's new rows.
* ``fork``   sequences become copies of others by sharing their pages (beams that go on from other
             beams, samples of one prompt), and get pages of their own for the next rows; an
             incomplete page that others hold is copied first.
* ``admit``  pages for prompts that enter a running batch.
* ``retire`` sequences that ended give up their pages, and the pages in use move to the pool's front.
* ``copy``   pages copied into another pool.

The page operators change a few small integer tensors (the table, how many sequences hold a page);
``run`` gives them copies of these, so that a pass finds what the one before it found. With ``own``
false a pass computes the plain form, with ``own`` true it makes the package's public calls.
``exact(case, seed)`` is the attention in float64, and the page operators' outcome from a walk over the
sequences one after another. Import it with the repository's root as the working directory.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
HEADS = ((8, 8), (16, 16), (12, 12), (16, 4), (16, 2), (10, 5), (16, 1))     # query heads, key-value heads
PAGES = (16, 32, 64, 128, 256)


def listed():
    return [
        # one user: latency
        dict(name="decode_single", kind="decode", B=1, S=1, Hq=16, Hkv=16, D=128, page=64, rows=1536, fill=0.6, len_seed=2,
             causal=False),
        # a full serving batch, each sequence at its own length
        dict(name="decode_batch", kind="decode", B=64, S=1, Hq=16, Hkv=16, D=128, page=64, rows=4096, fill=0.75, len_seed=1,
             causal=False),
        # eight query heads a key-value head, small pages, longer texts
        dict(name="decode_grouped", kind="decode", B=48, S=1, Hq=16, Hkv=2, D=128, page=16, rows=16384, fill=0.6, len_seed=3,
             causal=False),
        # a few long documents
        dict(name="decode_long", kind="decode", B=3, S=1, Hq=12, Hkv=12, D=128, page=256, rows=32768, fill=0.7, len_seed=4,
             causal=False),
        # five draft tokens a sequence to be verified
        dict(name="extend_draft", kind="extend", B=24, S=5, Hq=16, Hkv=4, D=128, page=32, rows=4096, fill=0.6, len_seed=5,
             causal=True),
        # a piece of a long prompt on what came before it
        dict(name="extend_prompt", kind="extend", B=4, S=509, Hq=16, Hkv=16, D=128, page=64, rows=4096, fill=0.5, len_seed=6,
             causal=True),
        # sixteen prompts with four beams each, which go on from one another
        dict(name="fork_beams", kind="fork", groups=16, width=4, layers=4, Hkv=16, D=128, page=64, rows=2048, own_rows=200,
             rest=41, spare=0.1, len_seed=7),
        # one prompt, eight samples of it
        dict(name="fork_samples", kind="fork", groups=1, width=8, layers=8, Hkv=4, D=128, page=32, rows=1021, own_rows=0,
             rest=29, spare=0.5, len_seed=8),
        # thirty prompts enter a batch of 256 slots
        dict(name="admit_prompts", kind="admit", N=256, new=30, prompt=1000, running=0.8, layers=1, Hkv=4, D=64, page=32,
             rows=4096, spare=0.3, len_seed=9),
        # the end of a batch's shortest answers, pages of four layers
        dict(name="retire_batch", kind="retire", N=64, ended=0.3, layers=4, Hkv=8, D=128, page=64, rows=2048, spare=0.1,
             len_seed=10),
        # a few sequences of a small model
        dict(name="retire_small", kind="retire", N=13, ended=0.5, layers=2, Hkv=2, D=64, page=16, rows=500, spare=0.5,
             len_seed=11),
        # the pages of a long text into another pool
        dict(name="copy_text", kind="copy", n=301, layers=8, Hkv=8, D=128, page=64, pool=700),
        ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "decode", "decode", "extend", "extend", "fork", "fork", "admit", "retire", "copy"))
    Hq, Hkv = rng.choice(HEADS)
    D, page = rng.choice((128, 128, 64)), rng.choice(PAGES)
    if kind == "decode":
        B = _log_int(rng, 1, 64)
        most = min(32768, 64 * 4096 * 16 // (B * Hkv))      # rows a sequence, as many values as the largest case
        return dict(kind=kind, B=B, S=1, Hq=Hq, Hkv=Hkv, D=D, page=page, rows=_log_int(rng, 100, most),
                    fill=rng.choice((0.3, 0.6, 0.75)), len_seed=rng.randrange(1 << 20), causal=rng.random() < 0.5)
    if kind == "extend":
        B, S = rng.randint(1, 8), _log_int(rng, 2, 512)
        return dict(kind=kind, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, page=page,
                    rows=S + _log_int(rng, 100, min(8000, 7000000 // (B * S))), fill=rng.choice((0.3, 0.6)),
                    len_seed=rng.randrange(1 << 20), causal=rng.random() < 0.7)
    layers, Hkv = rng.choice((1, 2, 4, 8)), min(Hkv, 8)
    if kind == "fork":
        beams = rng.random() < 0.6
        return dict(kind=kind, groups=rng.randint(1, 16) if beams else 1, width=rng.randint(2, 8), layers=layers, Hkv=Hkv, D=D,
                    page=page, rows=_log_int(rng, 30, 2048), own_rows=rng.randint(1, 300) if beams else 0,
                    rest=rng.choice((-1, 0, rng.randrange(page))), spare=rng.choice((0.1, 0.5)),
                    len_seed=rng.randrange(1 << 20))
    if kind == "admit":
        N = rng.randint(8, 256)
        return dict(kind=kind, N=N, new=rng.randint(1, max(1, N // 4)), prompt=_log_int(rng, 20, 1000),
                    running=rng.choice((0.5, 0.8)), layers=1, Hkv=min(Hkv, 4), D=64, page=page,
                    rows=_log_int(rng, 1100, 4096), spare=rng.choice((0.1, 0.5)), len_seed=rng.randrange(1 << 20))
    if kind == "retire":
        return dict(kind=kind, N=rng.randint(2, 64), ended=rng.choice((0.2, 0.5)), layers=min(layers, 4), Hkv=Hkv, D=D,
                    page=page, rows=_log_int(rng, 50, 2048), spare=rng.choice((0.1, 0.5)), len_seed=rng.randrange(1 << 20))
    n = _log_int(rng, 1, 76800 // (layers * page))
    return dict(kind=kind, n=n, layers=layers, Hkv=Hkv, D=D, page=page, pool=n + rng.randint(1, n + 20))


# ---- inputs ---------------------------------------------------------------------------
def _randn(g, *shape, scale=1.0):
    # a layer at a time: float32 normals of a whole pool would be twice its size
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    for part in (out if len(shape) > 4 else (out,)):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV) * scale)
    return out


def _len_gen(case):
    """Lengths, and with them the tensors' sizes, go with the case and not with the seed."""
    return torch.Generator().manual_seed(case["len_seed"])


def _lens(case):
    """Rows already in each sequence's pages; the new rows still fit."""
    g = _len_gen(case)
    most = case["rows"] - case["S"]
    top = max(1, min(most, int(case["rows"] * case["fill"] * 1.3)))
    low = max(0, min(top - 1, int(case["rows"] * case["fill"] * 0.7)))
    return torch.randint(low, top + 1, (case["B"],), generator=g, dtype=torch.int32)


def _columns(rows, page):
    return -(-rows // page)


def _deal(pages, counts, columns, host):
    """A table whose row n holds counts[n] of the pool's pages, which lie anywhere in it, and how many
    sequences hold each page."""
    order = torch.randperm(pages, generator=host)
    table = torch.full((len(counts), columns), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for n, c in enumerate(counts):
        table[n, :c] = order[at:at + c].int()
        refs[order[at:at + c]] = 1
        at += c
    return table, refs


def _attend_tables(case, host):
    lens = _lens(case)
    counts = [_columns(int(n) + case["S"], case["page"]) for n in lens]
    # pages of other sequences and free ones lie between these
    table, refs = _deal(sum(counts) * 5 // 4 + 3, counts, _columns(case["rows"], case["page"]), host)
    return dict(table=table, refs=refs, lens=lens)


def _fork_tables(case, host):
    """Groups of `width` sequences that share their prompt's pages, all but an incomplete one. With
    own_rows each has generated that many rows in pages of its own; else only the group's first holds the
    prompt, and the others are empty."""
    page, W, G = case["page"], case["width"], case["groups"]
    prompt = torch.randint(case["rows"] // 2, case["rows"] + 1, (G,), generator=_len_gen(case))
    if case["rest"] >= 0:      # how far into a page the sequences are
        prompt = torch.clamp(prompt - (prompt + case["own_rows"]) % page + case["rest"], min=1)
    lens = (prompt + case["own_rows"]).tolist()
    shared = [int(p) // page for p in prompt]
    fresh = [_columns(n, page) - a for n, a in zip(lens, shared)]
    holders = W if case["own_rows"] else 1
    need = sum(a + holders * f for a, f in zip(shared, fresh))
    pages = int(need * (1 + case["spare"])) + G * W + 1
    order = torch.randperm(pages, generator=host).int()
    table = torch.full((G * W, max(_columns(n + 1, page) for n in lens) + 2), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for i in range(G):
        common = order[at:at + shared[i]]
        at += shared[i]
        for w in range(holders):
            mine = torch.cat((common, order[at:at + fresh[i]]))
            at += fresh[i]
            table[i * W + w, :mine.numel()] = mine
            refs[mine.long()] += 1
    parents = (torch.arange(G * W, dtype=torch.int32) // W * W).view(G, W)
    if case["own_rows"]:
        parents = parents + torch.randint(0, W, (G, W), generator=host, dtype=torch.int32)
    return dict(table=table, refs=refs, parents=parents.reshape(-1),
                lens=torch.tensor(lens, dtype=torch.int32).repeat_interleave(W), new=torch.ones(G * W, dtype=torch.int32))


def _admit_tables(case, host):
    """Slots in any order: new prompts, running sequences that bring a row, and empty ones."""
    N, page = case["N"], case["page"]
    sizes = _len_gen(case)
    what = torch.randperm(N, generator=sizes)
    is_new, is_running = what < case["new"], (what >= case["new"]) & (what < case["new"] + int(case["running"] * N))
    lens = torch.where(is_running, torch.randint(1, 1000, (N,), generator=sizes), 0)
    new = torch.where(is_new, torch.randint(case["prompt"] // 2 + 1, case["prompt"] + 2, (N,), generator=sizes),
                      torch.where(is_running, 1, 0))
    counts = [_columns(int(n), page) for n in lens]
    wanted = sum(_columns(int(n + m), page) for n, m in zip(lens, new)) - sum(counts)
    table, refs = _deal(sum(counts) + int(wanted * (1 + case["spare"])) + 1, counts, _columns(case["rows"], page), host)
    return dict(table=table, refs=refs, lens=lens.int(), new=new.int())


def _retire_tables(case, host):
    N, page, rows = case["N"], case["page"], case["rows"]
    lens = torch.randint(rows // 4 + 1, rows + 1, (N,), generator=_len_gen(case))
    counts = [_columns(int(n), page) for n in lens]
    table, refs = _deal(int(sum(counts) * (1 + case["spare"])) + 1, counts, _columns(rows, page), host)
    keep = torch.where(torch.rand(N, generator=host) < case["ended"], 0, lens)
    return dict(table=table, refs=refs, keep=keep.int())


def _copy_tables(case, host):
    n, pool = case["n"], case["pool"]
    return dict(src=torch.randperm(pool, generator=host)[:n].int(), dst=torch.randperm(n + 7, generator=host)[:n].int(),
                refs=torch.ones(pool, dtype=torch.int32), to_refs=torch.ones(n + 7, dtype=torch.int32),
                table=torch.arange(pool, dtype=torch.int32)[None], to_table=torch.arange(n + 7, dtype=torch.int32)[None])


_TABLES = dict(decode=_attend_tables, extend=_attend_tables, fork=_fork_tables, admit=_admit_tables, retire=_retire_tables,
               copy=_copy_tables)


def _tables(case, seed):
    return _TABLES[case["kind"]](case, torch.Generator().manual_seed(int(seed) & 0x7fffffff))


def prepare(case, seed):
    s = {name: x.to(DEV) for name, x in _tables(case, seed).items()}
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7fffffff)
    layers, Hkv, page, D = case.get("layers", 1), case["Hkv"], case["page"], case["D"]
    s["k_pages"], s["v_pages"] = (_randn(g, layers, s["refs"].numel(), Hkv, page, D, scale=x) for x in (2.0, 1.0))
    if case["kind"] in ("decode", "extend"):
        s["q"] = _randn(g, case["B"], case["S"], case["Hq"], D)
        s["k"], s["v"] = (_randn(g, case["B"], case["S"], Hkv, D, scale=x) for x in (2.0, 1.0))
    if case["kind"] == "copy":
        s["to_k"], s["to_v"] = (torch.zeros(layers, s["to_refs"].numel(), Hkv, page, D, dtype=torch.bfloat16, device=DEV)
                                for _ in range(2))
    return dict(s, case=case)


# ---- one pass: the plain forms ---------------------------------------------------------------
def _plain_attend(s):
    case = s["case"]
    B, S, Hq, Hkv, D, page = (case[n] for n in ("B", "S", "Hq", "Hkv", "D", "page"))
    lens, table = s["lens"].long(), s["table"].long()
    cap = table.shape[1] * page
    # the new rows into their pages
    at = lens[:, None] + torch.arange(S, device=DEV)
    into = torch.gather(table, 1, (at // page).clamp_max(table.shape[1] - 1))
    for name in ("k", "v"):
        s[name + "_pages"][0][into, :, at % page] = s[name]
    rows = []
    for name in ("k", "v"):
        x = s[name + "_pages"][0][table.clamp_min(0)]                        # [B, columns, Hkv, page, D]
        rows.append(x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, cap, D).float())
    q = s["q"].float().view(B, S, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = torch.matmul(q, rows[0].transpose(-1, -2)) * (1.0 / math.sqrt(D))
    last = lens[:, None] + (torch.arange(S, device=DEV) + 1 if case["causal"] else S)      # keys that a query sees
    seen = torch.arange(cap, device=DEV) < last[:, :, None]                  # [B, S, cap]
    score = score.view(B, Hkv, -1, S, cap).masked_fill(~seen[:, None, None], -math.inf).view(B, Hkv, -1, cap)
    del q
    score = torch.exp(score - score.amax(-1, keepdim=True))
    rows[1] = torch.where(torch.arange(cap, device=DEV)[:, None] < (lens + S)[:, None, None, None], rows[1], 0.0)
    out = torch.matmul(score, rows[1]) / score.sum(-1, keepdim=True)
    out = out.view(B, Hkv, Hq // Hkv, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, Hq, D)
    return dict(out=out.to(torch.bfloat16), k_pages=s["k_pages"], v_pages=s["v_pages"])


def _count(table, pages):
    held = (table >= 0).reshape(-1)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    return refs.index_add_(0, table.reshape(-1).clamp_min(0).long(), held.int())


def _plain_reserve(s, table, refs):
    """Pages for rows lens .. lens + new: missing ones, and those that others hold too. The lowest free
    pages go to the sequences in order. A page whose holders are all among these stays with the first."""
    page, (N, M), P = s["case"]["page"], table.shape, refs.numel()
    lens, new = s["lens"].long(), s["new"].long()
    end = torch.clamp(lens + new, max=M * page)
    col = torch.arange(M, device=DEV)
    first = lens // page
    inside = (col >= first[:, None]) & (col < ((end + page - 1) // page)[:, None]) & (end > lens)[:, None]
    at = table.long().clamp_min(0)
    shared = inside & (table >= 0) & (refs[at] > 1)
    item = torch.arange(N * M, device=DEV).view(N, M)
    asked = torch.zeros(P, dtype=torch.int32, device=DEV).index_add_(0, at.view(-1), shared.view(-1).int())
    lowest = torch.full((P,), N * M, device=DEV)
    lowest.scatter_reduce_(0, at.view(-1), torch.where(shared, item, N * M).view(-1), "amin")
    leaves = shared & ~((asked[at] == refs[at]) & (lowest[at] == item))
    needs = (inside & (table < 0)) | leaves
    rank = torch.cumsum(needs.view(-1).int(), 0).view(N, M).long() - 1
    free = torch.argsort((refs != 0).int(), stable=True)
    granted = needs & (rank < (refs == 0).sum())
    page_of = free[rank.clamp(0, P - 1)]
    n, c = torch.nonzero(granted & leaves & (col == first[:, None]), as_tuple=True)
    row = torch.arange(page, device=DEV) < (lens % page)[n][:, None]
    for name in ("k_pages", "v_pages"):
        for x in s[name]:
            x[page_of[n, c]] = torch.where(row[:, None, :, None], x[table[n, c].long()], x[page_of[n, c]])
    table = torch.where(granted, page_of.int(), table)
    refs = _count(table, P)
    short = (inside & ((table < 0) | (refs[table.long().clamp_min(0)] > 1))).sum(-1).int()
    return dict(page_table=table, refs=refs, short=short, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _plain_fork(s):
    table = s["table"][s["parents"].long()]
    return _plain_reserve(s, table, _count(table, s["refs"].numel()))


def _plain_retire(s):
    page, P = s["case"]["page"], s["refs"].numel()
    col = torch.arange(s["table"].shape[1], device=DEV)
    kept = col < ((s["keep"].long() + page - 1) // page)[:, None]
    table = torch.where(kept, s["table"], -1)
    refs = _count(table, P)
    used = (refs > 0).sum()
    ids = torch.arange(P, device=DEV)
    src, dst = ids[(refs > 0) & (ids >= used)], ids[(refs == 0) & (ids < used)]
    to = ids.int()
    to[src] = dst.int()
    for name in ("k_pages", "v_pages"):
        for x in s[name]:
            x[dst] = x[src]
    refs[dst] = refs[src]
    refs[src] = 0
    table = torch.where(table >= 0, to[table.long().clamp_min(0)], -1)
    return dict(page_table=table, refs=refs, used=used.int()[None], k_pages=s["k_pages"], v_pages=s["v_pages"])


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name in ("k", "v"):
        for x, y in zip(s[name + "_pages"], s["to_" + name]):
            y[dst] = x[src]
    return dict(k_pages=s["to_k"], v_pages=s["to_v"])


# ---- one pass ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind in ("decode", "extend"):
            return _plain_attend(s)
        if kind == "admit":
            return _plain_reserve(s, s["table"], s["refs"])
        return {"fork": _plain_fork, "retire": _plain_retire, "copy": _plain_copy}[kind](s)
    prefixlm = _package()
    if kind in ("decode", "extend"):
        cache = prefixlm.PagedKVCache(s["k_pages"], s["v_pages"], s["refs"], s["table"])
        out = prefixlm.flash_attn_with_paged_kvcache(s["q"], cache, k=s["k"], v=s["v"], cache_seqlens=s["lens"],
                                                     causal=case["causal"])
        return dict(out=out, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if kind == "copy":
        source = prefixlm.PagedKVCache(s["k_pages"], s["v_pages"], s["refs"], s["table"])
        cache = prefixlm.PagedKVCache(s["to_k"], s["to_v"], s["to_refs"], s["to_table"])
        prefixlm.paged_kvcache_copy(cache, s["src"], s["dst"], source=source)
        return dict(k_pages=s["to_k"], v_pages=s["to_v"])
    cache = prefixlm.PagedKVCache(s["k_pages"], s["v_pages"], s["refs"].clone(), s["table"].clone())
    out = dict(page_table=cache.page_table, refs=cache.refs, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if kind == "retire":
        prefixlm.paged_kvcache_free(cache, s["keep"])
        out["used"] = prefixlm.paged_kvcache_compact(cache)
        return out
    if kind == "fork":
        prefixlm.paged_kvcache_fork(cache, s["parents"])
    out["short"] = prefixlm.paged_kvcache_reserve(cache, s["lens"], s["new"])
    return out


def _package():
    """The framework, found as its users find it: its folder on the path."""
    at = os.path.join(os.getcwd(), "hrm-text_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import prefixlm
    return prefixlm


# ---- what a pass cannot do without ------------------------------------------------------
def work(case):
    kind, D = case["kind"], case["D"]
    row = 4 * case["Hkv"] * D                     # a key and a value row of all heads
    if kind in ("decode", "extend"):
        B, S, Hq, lens = case["B"], case["S"], case["Hq"], _lens(case).tolist()
        pairs = sum(S * n + (S * (S + 1) // 2 if case["causal"] else S * S) for n in lens)
        tables = sum(4 * _columns(n + S, case["page"]) for n in lens)
        # the cached rows, the new rows in and out, queries in and results out
        return dict(bytes=row * (sum(lens) + 2 * B * S) + tables + 4 * B * S * Hq * D, flops=4 * D * Hq * pairs)
    if kind == "copy":
        moved = 2 * row * case["layers"] * case["page"] * case["n"]
        return dict(bytes=moved + 8 * case["n"], flops=case["n"])
    # the tables in and out and the rows that have to be copied, counted on the inputs of one seed
    s = _OUTCOMES[kind](case, _tables(case, 0))
    moved = 2 * row * case["layers"] * s["rows_copied"]
    return dict(bytes=moved + 8 * (s["page_table"].numel() + s["refs"].numel()), flops=s["page_table"].numel())


# ---- the same outputs, by another way ------------------------------------------------------------
def _exact_attend(case, s):
    B, S, Hq, Hkv, D, page = (case[n] for n in ("B", "S", "Hq", "Hkv", "D", "page"))
    out = torch.empty(B, S, Hq, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case).tolist()):
        pages = s["table"][b, :_columns(n, page)].long()
        k, v = (torch.cat((s[x + "_pages"][0, pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :n], s[x][b].transpose(0, 1)), 1)
                for x in ("k", "v"))
        hide = torch.ones(S, n + S, dtype=torch.bool, device=DEV).triu(n + 1) if case["causal"] else None
        for h in range(Hq):
            score = s["q"][b, :, h].double() @ k[h * Hkv // Hq].double().t() / math.sqrt(D)
            if hide is not None:
                score = score.masked_fill(hide, -math.inf)
            out[b, :, h] = torch.softmax(score, -1) @ v[h * Hkv // Hq].double()
    # the pages hold rows as they were given: no value in more bits
    return dict(out=out, k_pages=None, v_pages=None)


def _reserve_walk(case, table, refs, lens, new):
    """Sequence after sequence, each asking for its pages; returns the copies (from, to, rows)."""
    page, P, cap = case["page"], len(refs), len(table[0]) * case["page"]
    before, held = list(refs), {}
    asked = []
    for n, (a, m) in enumerate(zip(lens, new)):
        end = min(a + m, cap)
        asked.append(range(a // page, _columns(end, page)) if end > a else range(0))
        for c in asked[n]:
            if table[n][c] >= 0:
                held.setdefault(table[n][c], []).append((n, c))
    free = iter([p for p in range(P) if before[p] == 0])
    copies = []
    for n, cols in enumerate(asked):
        for c in cols:
            p = table[n][c]
            if p >= 0 and (before[p] == 1 or (len(held[p]) == before[p] and held[p][0] == (n, c))):
                continue
            to = next(free, None)
            if to is None:
                continue
            if p >= 0:
                refs[p] -= 1
                if c == lens[n] // page and lens[n] % page:
                    copies.append((p, to, lens[n] % page))
            table[n][c], refs[to] = to, 1
    short = [sum(table[n][c] < 0 or refs[table[n][c]] > 1 for c in cols) for n, cols in enumerate(asked)]
    return copies, short


def _outcome(table, refs, rows_copied, **more):
    return dict(page_table=torch.tensor(table, dtype=torch.int32), refs=torch.tensor(refs, dtype=torch.int32),
                rows_copied=rows_copied, **more)


def _fork_outcome(case, s):
    before = s["table"].tolist()
    if case["kind"] == "fork":
        table = [list(before[p]) for p in s["parents"].tolist()]
    else:
        table = before
    refs = [0] * s["refs"].numel()
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    copies, short = _reserve_walk(case, table, refs, s["lens"].tolist(), s["new"].tolist())
    return _outcome(table, refs, sum(r for _, _, r in copies), copies=copies, short=torch.tensor(short, dtype=torch.int32))


def _retire_outcome(case, s):
    table, page = s["table"].tolist(), case["page"]
    refs = [0] * s["refs"].numel()
    for row, keep in zip(table, s["keep"].tolist()):
        for c in range(len(row)):
            if c * page >= keep:
                row[c] = -1
            elif row[c] >= 0:
                refs[row[c]] += 1
    used = sum(r > 0 for r in refs)
    high = [p for p in range(used, len(refs)) if refs[p]]
    low = [p for p in range(used) if not refs[p]]
    to = dict(zip(high, low))
    table = [[to.get(p, p) for p in row] for row in table]
    for a, b in to.items():
        refs[a], refs[b] = 0, refs[a]
    return _outcome(table, refs, page * len(to), copies=[(a, b, page) for a, b in to.items()],
                    used=torch.tensor([used], dtype=torch.int32))


_OUTCOMES = dict(fork=_fork_outcome, admit=_fork_outcome, retire=_retire_outcome)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("decode", "extend"):
        return _exact_attend(case, s)
    if case["kind"] == "copy":
        for i, j in zip(s["src"].tolist(), s["dst"].tolist()):
            s["to_k"][:, j], s["to_v"][:, j] = s["k_pages"][:, i], s["v_pages"][:, i]
        return dict(k_pages=s["to_k"], v_pages=s["to_v"])
    out = _OUTCOMES[case["kind"]](case, s)
    out.pop("rows_copied")
    for a, b, rows in out.pop("copies"):
        for x in (s["k_pages"], s["v_pages"]):
            x[:, b, :, :rows] = x[:, a, :, :rows]
    return {**{n: x.to(DEV) for n, x in out.items()}, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
