"""GPU: the native host path of the paged cache's calls against the Python path: bitwise the same results, the same
refusals, modes, the profiler and a compiler."""
import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import (PagedKVCache, _native, flash_attn_with_paged_kvcache, paged_kvcache_compact, paged_kvcache_copy,
                      paged_kvcache_fork, paged_kvcache_free, paged_kvcache_reserve)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
N, H, G, D, PS, M, L = 5, 2, 2, 64, 16, 40, 2
LENS = torch.tensor([0, 17, 64, 300, 620], dtype=torch.int32)


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def _cache():
    g = torch.Generator().manual_seed(1)
    return PagedKVCache(*(x.to(DEV) for x in oracle.dealt(L, 100, H, PS, D, N, M, LENS.tolist(), g)))


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


CALLS = {
    "decode": lambda c: flash_attn_with_paged_kvcache(_rand(N, 1, H * G, D), c, _rand(N, 1, H, D, seed=1), _rand(N, 1, H, D, seed=2),
                                                      LENS.to(DEV)),
    "decode_int": lambda c: flash_attn_with_paged_kvcache(_rand(N, 1, H, D), c, cache_seqlens=17, softmax_scale=0.2, layer=1),
    "decode_none": lambda c: flash_attn_with_paged_kvcache(_rand(N, 3, H, D), c, _rand(N, 3, H, D, seed=1), _rand(N, 3, H, D, seed=2)),
    "extend": lambda c: flash_attn_with_paged_kvcache(_rand(N, 20, H * G, D), c, _rand(N, 20, H, D, seed=1), _rand(N, 20, H, D, seed=2),
                                                      LENS.to(DEV).long(), causal=True, layer=1),
    "strided": lambda c: flash_attn_with_paged_kvcache(_rand(9, N, H, D).transpose(0, 1), c, _rand(9, N, 2 * H, D, seed=1).transpose(0, 1)[:, :, H:],
                                                       _rand(9, N, H, D, seed=2).transpose(0, 1), LENS.to(DEV), causal=True),
    "off_alignment": lambda c: flash_attn_with_paged_kvcache(
        _rand(N, 1, H, D), c, _rand(N * H * D + 1, seed=1)[1:].view(N, 1, H, D), _rand(N, 1, H, D, seed=2), LENS.to(DEV)),
    "reserve": lambda c: paged_kvcache_reserve(c, LENS.to(DEV), _ints(3, 0, 1, 30, 20)),
    "reserve_ints": lambda c: paged_kvcache_reserve(c, 10, 7),
    "reserve_long": lambda c: paged_kvcache_reserve(c, LENS.to(DEV).long(), 2**40),
    "reserve_none": lambda c: paged_kvcache_reserve(c, None, 5),
    "fork": lambda c: paged_kvcache_fork(c, _ints(3, 3, -1, 0, 7)),
    "fork_long": lambda c: paged_kvcache_fork(c, _ints(3, 3, -1, 0, 7).long()),
    "free": lambda c: paged_kvcache_free(c, _ints(0, 1, 16, 17, 1000)),
    "free_int": lambda c: paged_kvcache_free(c, 32),
    "free_far": lambda c: paged_kvcache_free(c, -2**70),
    "free_all": lambda c: paged_kvcache_free(c),
    "compact": lambda c: paged_kvcache_compact(c),
    "copy": lambda c: paged_kvcache_copy(c, _ints(1, 2, 100), _ints(50, 60, 1)),
    "copy_long": lambda c: paged_kvcache_copy(c, _ints(1, 2).long(), _ints(50, 60).long()),
    "copy_none": lambda c: paged_kvcache_copy(c, _ints(), _ints()),
    "copy_from": lambda c: paged_kvcache_copy(c, _ints(4, 99), _ints(0, 7), source=_cache()),
}
OPS = {"decode": "paged_kvcache_attn", "decode_int": "paged_kvcache_attn", "decode_none": "paged_kvcache_attn", "extend": "paged_kvcache_attn",
       "strided": "paged_kvcache_attn", "off_alignment": "paged_kvcache_attn"}


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    assert _native.calls() is not None, "the native host path is not built"
    if request.param == "python":
        monkeypatch.setattr(_native, "_module", None)
    return request.param


def _run(name):
    c = _cache()
    if name == "compact":
        paged_kvcache_free(c, _ints(0, 0, 64, 0, 620))
    return [CALLS[name](c), *c]


@pytest.mark.parametrize("name", CALLS)
def test_bitwise(name, monkeypatch):
    a = _run(name)
    with monkeypatch.context() as m:
        m.setattr(_native, "_module", None)
        b = _run(name)
    for x, y in zip(a, b):
        assert x is y is None or (x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y))


@pytest.mark.parametrize("name", CALLS)
def test_modes_see_the_operators(name):
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    want = _run(name)
    c = _cache()
    if name == "compact":
        paged_kvcache_free(c, _ints(0, 0, 64, 0, 620))
    with Dispatch():
        got = [CALLS[name](c), *c]
    for x, y in zip(want, got):
        assert x is y is None or torch.equal(x, y)
    op = OPS.get(name, "paged_kvcache_" + name.split("_")[0])
    assert sum(s.startswith(f"prefixlm.{op}") for s in seen) == 1, seen


def test_the_profiler_sees_the_calls(path):
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        for name in ("decode", "reserve", "fork", "free", "compact", "copy"):
            CALLS[name](_cache())
    seen = {e.key: e.count for e in prof.key_averages() if e.key.startswith("prefixlm::")}
    assert seen == {f"prefixlm::paged_kvcache_{n}": 1 for n in ("attn", "reserve", "fork", "free", "compact", "copy")}


def test_versions_count_what_is_written(path):
    """Autograd must know that a saved tensor was overwritten."""
    for name, written in (("decode", "kv"), ("reserve", "kvrt"), ("fork", "rt"), ("free", "rt"), ("compact", "kvrt"), ("copy", "kv")):
        c = _cache()
        before = [x._version for x in c]
        CALLS[name](c)
        for x, n, letter in zip(c, before, "kvrt"):
            assert (x._version > n) == (letter in written), (name, letter)


def test_inference_mode_and_side_streams(path):
    want = _run("decode")
    with torch.inference_mode():
        got = _run("decode")
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_run(n) for n in ("decode", "reserve", "compact")]
    torch.cuda.synchronize()
    for n, r in zip(("decode", "reserve", "compact"), got):
        for x, y in zip(_run(n), r):
            assert torch.equal(x, y), n


def test_refusals(path):
    """The same errors on both paths."""
    c, q, k = _cache(), _rand(N, 1, H * G, D), _rand(N, 1, H, D)
    att = flash_attn_with_paged_kvcache
    for call, needle in (
            (lambda: att(q[:, :, :3], c), "multiple"), (lambda: att(q, c, k), "together"), (lambda: att(q, c, k, k, -1), "cache_seqlens"),
            (lambda: att(q, c, k, k, M * PS + 1), "cache_seqlens"), (lambda: att(q, c, layer=L), "layer"), (lambda: att(q.cpu(), c), "GPU tensor"),
            (lambda: att(q, c._replace(v_pages=c.k_pages), k, k), "overlap"), (lambda: att(q, c._replace(refs=c.refs[:5])), "refs"),
            (lambda: att(c.k_pages[0, :N, :, :1].transpose(1, 2), c), "overlap"),
            (lambda: paged_kvcache_reserve(c, LENS, 1), "cache_seqlens"), (lambda: paged_kvcache_reserve(c, 0, _ints(1, 2)), "new_rows"),
            (lambda: paged_kvcache_fork(c, _ints(1)), "parents"), (lambda: paged_kvcache_free(c, _ints(1).float()), "keep_rows"),
            (lambda: paged_kvcache_compact(c._replace(page_table=c.page_table.long())), "page_table"),
            (lambda: paged_kvcache_copy(c, _ints(1, 2), _ints(3)), "lists"),
            (lambda: paged_kvcache_copy(c, _ints(1), _ints(3), source=c), "overlap")):
        before = [x.clone() for x in c]
        with pytest.raises(ValueError, match=needle):
            call()
        for x, y in zip(before, c):
            assert torch.equal(x, y)


def test_a_compiler_traces_a_step():
    def step(q, k, v, kp, vp, refs, table, lens, new):
        c = PagedKVCache(kp, vp, refs, table)
        short = paged_kvcache_reserve(c, lens, new)
        return short, flash_attn_with_paged_kvcache(q, c, k, v, lens, causal=True) * 2

    args = _rand(N, 1, H * G, D), _rand(N, 1, H, D, seed=1), _rand(N, 1, H, D, seed=2)
    a, b = _cache(), _cache()
    lens, new = torch.clamp(LENS, max=600).to(DEV), _ints(1, 1, 1, 1, 1)
    want = step(*args, *a, lens, new)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*args, *b, lens, new)
    for x, y in zip((*want, *a), (*got, *b)):
        assert torch.equal(x, y)
