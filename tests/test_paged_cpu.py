"""The key-value cache in pages without a GPU: the oracle against the contiguous cache's, what its page
functions keep true, and the refusals of the operators and the C entry points."""
import ctypes
import os
import re
import subprocess
import tempfile

import pytest
import torch

import prefixlm
from oracle import paged_oracle as oracle
from oracle.kvcache_oracle import kvcache_attention
from prefixlm import PagedKVCache, _build, _capi, paged_kvcache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rows(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S", [1, 3, 40])
def test_oracle_matches_the_contiguous_cache(S, causal):
    B, H, ps, D, Smax = 3, 2, 16, 64, 96
    lens = torch.tensor([0, 17, Smax - S], dtype=torch.int32)
    g = torch.Generator().manual_seed(S)
    cache = oracle.dealt(2, 24, H, ps, D, B, Smax // ps, [Smax] * B, g)
    q, k, v = (_rows(B, S, H, D, seed=i) for i in range(3))
    flat = [torch.stack([torch.stack([oracle.rows_of(cache, 1, i, b, h, Smax)[0] for h in range(H)], 1) for b in range(B)]).bfloat16()
            for i in range(2)]
    out, mag, new = oracle.attend(q, cache, k, v, lens, causal, layer=1)
    want, kn, vn = kvcache_attention(q, *flat, k, v, lens, causal)
    assert (out - want.double()).abs().max() < 1e-5 and (mag >= out.abs() - 1e-12).all()
    for i, x in ((0, kn), (1, vn)):
        rows = torch.stack([torch.stack([oracle.rows_of(new, 1, i, b, h, Smax)[0] for h in range(H)], 1) for b in range(B)])
        assert torch.equal(rows.bfloat16(), x)
        assert torch.equal(new[i][0], cache[i][0])


def test_grouped_heads_are_repeated_ones():
    B, H, G, ps, D = 2, 2, 3, 16, 64
    cache = oracle.dealt(1, 12, H, ps, D, B, 4, [50, 20], torch.Generator().manual_seed(1))
    q, k, v = _rows(B, 2, H * G, D), _rows(B, 2, H, D, seed=1), _rows(B, 2, H, D, seed=2)
    lens = torch.tensor([50, 20], dtype=torch.int32)
    out, _, _ = oracle.attend(q, cache, k, v, lens)
    many = [x.repeat_interleave(G, 2) for x in cache[:2]] + cache[2:]
    want, _, _ = oracle.attend(q, many, k.repeat_interleave(G, 2), v.repeat_interleave(G, 2), lens)
    assert torch.equal(out, want)


def _counts(cache):
    table, P = cache[3], cache[2].numel()
    return torch.bincount(table[table >= 0].long().reshape(-1), minlength=P).int()


def test_pages_stay_counted_and_rows_stay_with_their_sequences():
    """A long run of forks, reserves, appends, frees and compactions: refs are what the table holds, and each
    sequence reads back what it took."""
    g = torch.Generator().manual_seed(7)
    L, P, H, ps, D, N, M = 2, 40, 1, 16, 64, 6, 8
    cache = oracle.dealt(L, P, H, ps, D, N, M, [0] * N, g)
    lens, said = [0] * N, [[] for _ in range(N)]
    for step in range(60):
        new = [int(x) for x in torch.randint(0, 20, (N,), generator=g)]
        new = [m if a + m <= M * ps else 0 for a, m in zip(lens, new)]
        cache, short = oracle.reserve(cache, torch.tensor(lens), torch.tensor(new))
        for n in range(N):
            if short[n]:
                new[n] = 0
            for j in range(new[n]):
                p = int(cache[3][n, (lens[n] + j) // ps])
                assert int(cache[2][p]) == 1
                x = float(torch.randint(0, 200, (), generator=g))
                cache[0][:, p, :, (lens[n] + j) % ps] = x
                said[n].append(x)
            lens[n] += new[n]
        if step % 3 == 0:
            parents = torch.randint(-1, N, (N,), generator=g)
            cache = oracle.fork(cache, parents)
            old = list(zip(lens, said))
            for n, p in enumerate(parents.tolist()):
                if p >= 0:
                    lens[n], said[n] = old[p][0], list(old[p][1])
        if step % 5 == 0:
            n = int(torch.randint(0, N, (), generator=g))
            lens[n] = lens[n] // 2
            said[n] = said[n][:lens[n]]
            cache = oracle.free(cache, torch.tensor([lens[i] if i == n else 1 << 30 for i in range(N)]))
        if step % 7 == 0:
            cache, used = oracle.compact(cache)
            assert (cache[2][:used] > 0).all() and not cache[2][used:].any()
        assert torch.equal(_counts(cache), cache[2])
        for n in range(N):
            rows, held = oracle.rows_of(cache, 0, 0, n, 0, lens[n])
            assert held.all() and rows[:, 0].tolist() == said[n], (step, n)


def test_planted_mistake_is_caught():
    """A page left behind without its rows gives other attention."""
    g = torch.Generator().manual_seed(3)
    cache = oracle.dealt(1, 12, 1, 16, 64, 2, 3, [20, 0], g)
    cache = oracle.fork(cache, torch.tensor([0, 0]))
    right, short = oracle.reserve(cache, 20, 1)
    assert not short.any() and int(right[3][0, 1]) != int(right[3][1, 1])
    q = _rows(2, 1, 1, 64)
    a, mag, _ = oracle.attend(q, right, lens=20)
    right[1][0, right[3][1, 1]] = 0
    b, _, _ = oracle.attend(q, right, lens=20)
    assert torch.equal(a[0], b[0]) and ((a[1] - b[1]).abs() > 2.0 ** -8 * mag[1]).any()


def test_cache_maker():
    c = paged_kvcache(5, 32, 3, 100, 4, head_dim=64, layers=2, device="cpu")
    assert c.k_pages.shape == (2, 5, 4, 32, 64) and c.v_pages.dtype == torch.bfloat16
    assert c.page_table.shape == (3, 4) and (c.page_table == -1).all() and c.refs.tolist() == [0] * 5
    assert PagedKVCache._fields == ("k_pages", "v_pages", "refs", "page_table")
    for kw, needle in ((dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=2048), "page_size"),
                       (dict(head_dim=96), "head_dim"), (dict(batch=0), "batch"), (dict(layers=0), "layers")):
        with pytest.raises(ValueError, match=needle):
            paged_kvcache(**{**dict(num_pages=4, page_size=16, batch=1, max_seqlen=64, num_kv_heads=1, device="cpu"), **kw})


def test_cpu_tensors_are_refused():
    c = paged_kvcache(4, 16, 2, 64, 1, device="cpu")
    one = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: prefixlm.flash_attn_with_paged_kvcache(_rows(2, 1, 1, 128), c),
                 lambda: prefixlm.paged_kvcache_reserve(c, 0, 1), lambda: prefixlm.paged_kvcache_fork(c, one),
                 lambda: prefixlm.paged_kvcache_free(c), lambda: prefixlm.paged_kvcache_compact(c),
                 lambda: prefixlm.paged_kvcache_copy(c, one, one)):
        with pytest.raises(ValueError, match="GPU"):
            call()


# ---- the C entry points: refused before the GPU is touched ------------------------------------
@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


FAKE = 1 << 20   # never dereferenced


def _pool(**kw):
    a = dict(k_pages=FAKE, v_pages=FAKE, refs=FAKE, page_table=FAKE, table_stride=64, layers=2, num_pages=100, num_kv_heads=2,
             page_size=64, head_dim=128, batch=3, columns=64)
    return _capi.PagePool(**{**a, **kw})


BAD_POOLS = [(dict(head_dim=96), "head_dim"), (dict(page_size=48), "page_size"), (dict(page_size=8), "page_size"),
             (dict(page_size=2048), "page_size"), (dict(layers=0), "layers"), (dict(num_pages=0), "num_pages"),
             (dict(batch=0), "batch"), (dict(columns=0), "columns"), (dict(columns=1 << 25, table_stride=1 << 25), "2\\^30"),
             (dict(num_kv_heads=1 << 20), "2\\^30")]


@pytest.mark.parametrize("pool,kw,needle", [
    *((p, {}, n) for p, n in BAD_POOLS), (dict(k_pages=FAKE + 8), {}, "aligned"), (dict(v_pages=0), {}, "null"),
    (dict(refs=0), {}, "refs"), (dict(page_table=FAKE + 2), {}, "page_table"), (dict(table_stride=63), {}, "table_stride"),
    ({}, dict(v=0), "together"), ({}, dict(q=0), "null"), ({}, dict(out=FAKE + 4), "aligned"), ({}, dict(seqlen_q=0), "seqlen_q"),
    ({}, dict(seqlen_q=0x7fffffff), "seqlen_q"), ({}, dict(num_heads=5), "multiple"), ({}, dict(num_heads=0), "multiple"),
    ({}, dict(layer=2), "layer"), ({}, dict(layer=-1), "layer"), ({}, dict(q_stride_h=4), "stride"),
    ({}, dict(v_stride_s=-8), "stride"), ({}, dict(cache_seqlen=-1), "cache_seqlen"), ({}, dict(cache_seqlen=4097), "cache_seqlen"),
    ({}, dict(workspace=0), "workspace"), ({}, dict(workspace_bytes=8), "workspace"),
    (dict(batch=1 << 20, num_kv_heads=1 << 10, page_size=16), dict(num_heads=1 << 10), "too large"),
    ({}, dict(seqlen_q=1 << 30, num_heads=1 << 20), "too large"),
])
def test_attention_rejects(lib, pool, kw, needle):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, cache_seqlen=3, layer=1, seqlen_q=1, num_heads=4, softmax_scale=0.1, workspace=FAKE,
             workspace_bytes=1 << 62)
    for n in ("q", "k", "v", "out"):
        a.update({f"{n}_stride_b": 512, f"{n}_stride_s": 512, f"{n}_stride_h": 128})
    a = _capi.PagedArgs(pool=_pool(**pool), **{**a, **kw})
    assert lib.prefixlm_paged_fwd(ctypes.byref(a), None) == 1
    assert re.search(needle, _capi.last_error()), _capi.last_error()


@pytest.mark.parametrize("name,pool,kw,needle", [
    *((f, p, {}, n) for f in ("reserve", "fork", "free", "compact", "copy") for p, n in BAD_POOLS),
    *((f, dict(refs=0), {}, "refs") for f in ("reserve", "fork", "free", "compact")),
    *((f, dict(table_stride=3), {}, "table_stride") for f in ("reserve", "fork", "free", "compact")),
    *((f, dict(v_pages=FAKE + 2), {}, "aligned") for f in ("reserve", "compact", "copy")),
    *((f, dict(batch=8193), {}, "8192") for f in ("reserve", "fork")),
    *((f, {}, dict(workspace=0), "workspace") for f in ("reserve", "compact")),
    *((f, {}, dict(workspace_bytes=16), "workspace") for f in ("reserve", "compact")),
    *((f, {}, dict(result=0), "result") for f in ("reserve", "compact")),
    ("fork", {}, dict(src=0), "src"), ("copy", {}, dict(src=0), "src"), ("copy", {}, dict(dst=FAKE + 1), "dst"),
    ("copy", {}, dict(n=-1), "n="), ("copy", {}, dict(n=1 << 40), "n="),
    ("free", dict(batch=1 << 30, columns=64), {}, "too large"),
    ("copy", dict(num_kv_heads=1 << 16), dict(n=1 << 20), "too many"),
])
def test_page_calls_reject(lib, name, pool, kw, needle):
    a = dict(src=FAKE, dst=FAKE, n=5, result=FAKE, workspace=FAKE, workspace_bytes=1 << 62)
    a = _capi.PagesArgs(pool=_pool(**pool), **{**a, **kw})
    assert getattr(lib, f"prefixlm_pages_{name}")(ctypes.byref(a), None) == 1
    assert re.search(needle, _capi.last_error()), _capi.last_error()


def test_pools_that_differ_null_args_and_workspaces(lib):
    for kw in (dict(layers=3), dict(num_kv_heads=1), dict(page_size=32), dict(head_dim=64)):
        other = _pool(**kw)
        a = _capi.PagesArgs(pool=_pool(), from_=ctypes.pointer(other), src=FAKE, dst=FAKE, n=1)
        assert lib.prefixlm_pages_copy(ctypes.byref(a), None) == 1 and "differ" in _capi.last_error()
    for f in ("prefixlm_paged_fwd", *(f"prefixlm_pages_{n}" for n in ("reserve", "fork", "free", "compact", "copy"))):
        assert getattr(lib, f)(None, None) == 1
    assert lib.prefixlm_pages_copy(ctypes.byref(_capi.PagesArgs(pool=_pool())), None) == 0    # n = 0: nothing to do
    assert lib.prefixlm_pages_workspace_size(None) == 0
    # the free pages' list, three words a page, the copies; or the moves and where they go
    assert lib.prefixlm_pages_workspace_size(ctypes.byref(_pool())) == (4 * (100 + 300 + 1 + 9) + 255) // 256 * 256
    assert lib.prefixlm_paged_workspace_size(1, 1, 5, 2, 128, 16, 4) == 0
    assert lib.prefixlm_paged_workspace_size(1, 1, 16, 16, 128, 64, 64) > 0
    # 256 sequences of 2^30 rows are 2^32 tiles of 64, which no 32 bits add up: a workgroup for each
    assert lib.prefixlm_paged_workspace_size(256, 1, 1, 1, 128, 1024, 1 << 20) == 0
    assert lib.prefixlm_paged_workspace_size(64, 1, 1, 1, 128, 1024, 1 << 20) > 0


@pytest.mark.parametrize("cname,cls", [("prefixlm_page_pool", _capi.PagePool), ("prefixlm_paged_args", _capi.PagedArgs),
                                       ("prefixlm_pages_args", _capi.PagesArgs)])
def test_struct_layout_matches_header(cname, cls):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "prefixlm.h"', "int main(void){",
             f'printf("size %zu\\n", sizeof({cname}));']
    lines += [f'printf("{f} %zu\\n", offsetof({cname}, {f.rstrip("_")}));' for f, _ in cls._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(src, "w") as out:
            out.write("\n".join(lines + ["return 0;}"]))
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(got[f]) == getattr(cls, f).offset, f
