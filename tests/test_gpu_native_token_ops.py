"""GPU: the native host path of the log probabilities, the embedding and the 8-bit cache against the
Python path: bitwise the same results and gradients, the same refusals, and the calls it hands back
(operands that need a copy, recorded and batched backwards, modes, saved-tensor hooks)."""
import pytest
import torch

from prefixlm import _native, embedding, flash_attn_with_kvcache_q8, kvcache_q8, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    assert _native.calls() is not None, "the native host path is not built"
    if request.param == "python":
        monkeypatch.setattr(_native, "_module", None)
    return request.param


def _rand(*shape, seed=0, dtype=BF):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _ids(*shape, n=50, seed=0):
    return torch.randint(0, n, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _both(fn, monkeypatch):
    assert _native.calls() is not None
    a = fn()
    with monkeypatch.context() as m:
        m.setattr(_native, "_module", None)
        b = fn()
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape
            u, v = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (x, y))
            assert torch.equal(u, v)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("targets,entropy,top", [(True, False, 0), (True, True, 3), (False, True, 0), (False, False, 2), (True, False, 2)])
def test_logprob_bitwise(targets, entropy, top, dtype, monkeypatch):
    logits, t = _rand(6, 50, 333, dtype=dtype), _ids(6, 50, n=333)
    t[0, :9] = -100
    g, h = _rand(6, 50, seed=3, dtype=F32), _rand(6, 50, seed=4, dtype=F32)

    def run():
        out = []
        for x in (logits.clone().requires_grad_(), logits.transpose(0, 1).clone().transpose(0, 1).requires_grad_()):
            for tt in ((t, t.int()) if targets else (None,)):
                r = token_logprobs(x, tt, entropy=entropy, top_k=top)
                heads, given = [y for y in r[:2] if y is not None], [y for y, w in zip((g, h), r[:2]) if w is not None]
                out += list(r)
                if heads:
                    out += torch.autograd.grad(heads, (x,), given, retain_graph=True)
                    out += torch.autograd.grad(sum(y.sum() for y in heads), (x,), retain_graph=True)
                    out += torch.autograd.grad(heads[0].sum(), (x,))
                else:
                    assert not any(y.requires_grad for y in r if y is not None)
            with torch.no_grad():
                out += list(token_logprobs(x, t if targets else None, entropy=entropy, top_k=top))
        return out
    _both(run, monkeypatch)


@pytest.mark.parametrize("table,out", [(BF, BF), (F32, BF), (F32, F32), (BF, F32)])
def test_embedding_bitwise(table, out, monkeypatch):
    ids, t, dy = _ids(3, 70), _rand(50, 64, dtype=table), _rand(3, 70, 64, seed=1, dtype=out)

    def run():
        res = []
        for i in (ids, ids.int(), ids.t().contiguous().t()):
            for p in (None, 7):
                x = t.clone().requires_grad_()
                y = embedding(i, x, 1.5, dtype=out, padding_idx=p)
                res += [y, *torch.autograd.grad(y, (x,), dy, retain_graph=True), *torch.autograd.grad(y.float().sum(), (x,))]
        return res + [embedding(ids, t, 1.5), embedding(ids[0, 0], t)]
    _both(run, monkeypatch)


@pytest.mark.parametrize("S", [1, 5, 70])
@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_cache_bitwise_and_in_place(S, code, monkeypatch):
    B, H = 2, 3
    q, k, v = (_rand(B, S, H, 128, seed=i) for i in range(3))
    lens = torch.tensor([20, 140], dtype=torch.int32, device=DEV)

    def run():
        cache = kvcache_q8(B, 256, H, dtype=code)
        o = [flash_attn_with_kvcache_q8(q, cache, k, v)]
        before = [x._version for x in cache]
        o.append(flash_attn_with_kvcache_q8(q, cache, k, v, lens, causal=True))
        assert [x._version for x in cache] == [n + 1 for n in before]
        o.append(flash_attn_with_kvcache_q8(q, cache, cache_seqlens=30, softmax_scale=0.3))
        return (*o, *cache)
    _both(run, monkeypatch)


def test_refusals(path):
    x, t = _rand(8, 40), _ids(8, n=40)
    for bad in (dict(top_k=41), dict(top_k=65), dict(targets=t[:5]), dict(targets=t.float()), dict(targets=t.cpu())):
        with pytest.raises(ValueError):
            token_logprobs(x, **{"targets": t, **bad})
    with pytest.raises(ValueError):
        token_logprobs(x)
    w = _rand(50, 64)
    for ids, table, kw in ((t.float(), w, {}), (t.cpu(), w, {}), (t, w[:, :60], {}), (t, w.half(), {}), (t, w, {"dtype": torch.float16}),
                           (t, w, {"padding_idx": 50}), (t, w.view(-1), {})):
        with pytest.raises((ValueError, IndexError)):
            embedding(ids, table, **kw)
    q, cache = _rand(2, 1, 2, 128), kvcache_q8(2, 128, 2)
    for args, kw in (((q.float(), cache), {}), ((q, cache, q), {}), ((q, cache, q, q[:1]), {}), ((q, cache, q, q, 129), {}),
                     ((q, cache._replace(v_codes=cache.k_codes)), {})):
        with pytest.raises((ValueError, TypeError)):
            flash_attn_with_kvcache_q8(*args, **kw)
    xg = x.clone().requires_grad_()
    r = token_logprobs(xg, t)
    with torch.no_grad():
        xg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprob.sum().backward()


def _call(name):
    """(leaf, call, output gradient) of one differentiable call."""
    if name == "embedding":
        ids = _ids(90)
        return _rand(50, 64, dtype=F32).requires_grad_(), lambda t: embedding(ids, t, 2.0, dtype=BF), _rand(90, 64, seed=2)
    t = _ids(90, n=200)
    x = _rand(90, 200, dtype=BF if name == "logprob" else F32).requires_grad_()
    if name == "logprob":
        return x, lambda y: token_logprobs(y, t).logprob, _rand(90, seed=2, dtype=F32)
    return x, lambda y: token_logprobs(y, t, entropy=True, top_k=2).entropy, _rand(90, seed=2, dtype=F32)


CALLS = ["logprob", "entropy", "embedding"]


@pytest.mark.parametrize("name", CALLS)
def test_recorded_backwards_give_the_same_gradient(name, path):
    x, f, dy = _call(name)
    want, = torch.autograd.grad(f(x), x, dy)
    got, = torch.autograd.grad(f(x), x, dy.clone().requires_grad_(), create_graph=True)
    assert got.requires_grad and torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError):
        got.float().sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_hooks_checkpoint_streams_and_inference(name, path):
    x, f, dy = _call(name)
    y = f(x)
    want, = torch.autograd.grad(y, x, dy)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.clone(), lambda t: t):
        out = f(x)
    assert torch.equal(torch.autograd.grad(out, x, dy)[0], want) and packed
    out = torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(out, x, dy)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(f(x), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with torch.inference_mode():
        assert torch.equal(f(x.detach()), y.detach())


def _shifted(t):
    return torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)


# which saved tensor (dtype, dimensions, the n-th such), what a hook gives back for it, and what the
# backward then does: the same gradient, or this error
HOOKS = {
    "logits_off_alignment": ("logprob", (BF, 2, 0), _shifted, None),
    "logits_wide": ("logprob", (BF, 2, 0), lambda t: torch.cat((t, t), -1)[:, :t.shape[1]], None),
    "logits_cpu": ("logprob", (BF, 2, 0), lambda t: t.cpu(), ValueError),
    "logits_half": ("logprob", (BF, 2, 0), lambda t: t.half(), ValueError),
    "targets_int": ("logprob", (torch.int64, 1, 0), lambda t: t.int(), None),
    "targets_strided": ("logprob", (torch.int64, 1, 0), lambda t: torch.stack((t, t), -1)[:, 0], None),
    "targets_short": ("logprob", (torch.int64, 1, 0), lambda t: t[:-1], ValueError),
    "stats_strided": ("logprob", (F32, 2, 0), lambda t: t.t().contiguous().t(), None),
    "stats_short": ("logprob", (F32, 2, 0), lambda t: t[:-1], ValueError),
    "stats_double": ("logprob", (F32, 2, 0), lambda t: t.double(), ValueError),
    "entropy_strided": ("entropy", (F32, 1, 0), lambda t: torch.stack((t, t), -1)[:, 0], None),
    "entropy_short": ("entropy", (F32, 1, 0), lambda t: t[:-1], ValueError),
    "ids_int": ("embedding", (torch.int64, 1, 0), lambda t: t.int(), None),
    "ids_strided": ("embedding", (torch.int64, 1, 0), lambda t: torch.stack((t, t), -1)[:, 0], None),
    "ids_short": ("embedding", (torch.int64, 1, 0), lambda t: t[:-1], ValueError),
    "ids_float": ("embedding", (torch.int64, 1, 0), lambda t: t.float(), ValueError),
    "ids_cpu": ("embedding", (torch.int64, 1, 0), lambda t: t.cpu(), ValueError),
}


@pytest.mark.parametrize("name", HOOKS)
def test_hooks_that_give_back_other_tensors(name, path):
    print(f"[case] hook {name} {path}", flush=True)
    call, which, change, error = HOOKS[name]
    x, f, dy = _call(call)
    want, = torch.autograd.grad(f(x), x, dy)
    seen, given = {}, []

    def pack(t):
        key = (t.dtype, t.dim())
        n = seen.get(key, 0)
        seen[key] = n + 1
        return t, (*key, n) == which

    def unpack(p):
        given.append(p[1])
        return change(p[0].detach()) if p[1] else p[0]

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = f(x)
    if error is None:
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    else:
        with pytest.raises(error):
            torch.autograd.grad(y, x, dy)
    assert given.count(True) == 1


@pytest.mark.parametrize("name", CALLS)
def test_modes_see_the_operators(name):
    from torch.utils._python_dispatch import TorchDispatchMode
    assert _native.calls() is not None
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, f, dy = _call(name)
    y = f(x)
    want, = torch.autograd.grad(y, x, dy)
    with Dispatch():
        z = f(x)
        got, = torch.autograd.grad(z, x, dy)
    assert torch.equal(z, y) and torch.equal(got, want)
    assert sum(op.startswith("prefixlm.") for op in seen) == 2


@pytest.mark.parametrize("name", CALLS)
def test_batched_gradients_as_on_the_python_path(name, monkeypatch):
    def run():
        x, f, dy = _call(name)
        try:
            return torch.autograd.grad(f(x), x, torch.stack((dy, 2 * dy)), is_grads_batched=True)[0]
        except Exception as e:
            return type(e)
    assert _native.calls() is not None
    a = run()
    with monkeypatch.context() as m:
        m.setattr(_native, "_module", None)
        b = run()
    assert torch.equal(a, b) if isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor) else a is b


def test_the_profiler_sees_the_calls(path):
    x, ids, w = _rand(40, 256).requires_grad_(), _ids(40), _rand(50, 64).requires_grad_()
    q, cache = _rand(1, 1, 2, 128), kvcache_q8(1, 64, 2)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        torch.autograd.grad(token_logprobs(x, ids).logprob.sum(), x)
        torch.autograd.grad(embedding(ids, w).sum(), w)
        flash_attn_with_kvcache_q8(q, cache, q, q, 0)
    seen = {e.key: e.count for e in prof.key_averages() if e.key.startswith("prefixlm::")}
    assert seen == {f"prefixlm::{n}": 1 for n in ("token_logprobs_fwd", "token_logprobs_bwd", "embedding_fwd", "embedding_bwd",
                                                  "kvcache_q8_attn")}


def test_parameters_accumulate_over_steps():
    """Leaves that are Parameters, two backwards into .grad."""
    w, head = torch.nn.Parameter(_rand(50, 64, dtype=F32)), torch.nn.Parameter(_rand(50, 64, seed=1))
    ids = _ids(33)
    for _ in range(2):
        token_logprobs(torch.nn.functional.linear(embedding(ids, w, 0.5, dtype=BF), head), ids).logprob.mean().backward()
    once = [p.grad.clone() for p in (w, head)]
    w.grad = head.grad = None
    token_logprobs(torch.nn.functional.linear(embedding(ids, w, 0.5, dtype=BF), head), ids).logprob.mean().backward()
    assert torch.equal(once[0], 2 * w.grad) and torch.equal(once[1], 2 * head.grad)


def test_two_streams_at_once():
    """The same operators on two streams, whose workspaces must be their own."""
    xs, ids = [_rand(3, 200000, seed=i) for i in range(2)], [_ids(20000, n=3000, seed=i) for i in range(2)]
    dys = [_rand(20000, 64, seed=i) for i in range(2)]
    from prefixlm.embedding import embedding_bwd
    caches = [kvcache_q8(1, 8192, 4) for _ in range(2)]
    for c in caches:
        c.k_codes.view(torch.uint8).random_(0, 100)
        c.v_codes.view(torch.uint8).random_(0, 100)
        c.k_scale.fill_(0.01)
        c.v_scale.fill_(0.01)
    qs = [_rand(1, 1, 4, 128, seed=i) for i in range(2)]

    def work(i):
        r = token_logprobs(xs[i], None, entropy=True, top_k=5)
        return (r.entropy, r.top_logprobs, r.top_ids, embedding_bwd(ids[i], dys[i], 3000, 1.0, F32, -1),
                flash_attn_with_kvcache_q8(qs[i], caches[i], cache_seqlens=8000))

    want = [work(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_cache_operands_that_share_memory_are_refused(path):
    """Queries or rows that lie in the cache would be read while it is written."""
    cache = kvcache_q8(2, 128, 2)
    q, k, v = (_rand(2, 3, 2, 128, seed=i) for i in range(3))
    inside = cache.k_recent.transpose(1, 2)[:, :3]     # [B, 3, H, 128]
    for args in ((inside, k, v), (q, inside, v), (q, k, inside), (inside, None, None)):
        with pytest.raises(ValueError, match="overlap"):
            flash_attn_with_kvcache_q8(args[0], cache, args[1], args[2], 0)
    # one allocation that holds all, without sharing
    whole = torch.zeros(2 * cache.k_recent.numel() + q.numel(), dtype=BF, device=DEV)
    n = cache.k_recent.numel()
    beside = cache._replace(k_recent=whole[:n].view_as(cache.k_recent), v_recent=whole[n + q.numel():].view_as(cache.k_recent))
    row = whole[n:n + q.numel()].view_as(q)
    row.copy_(k)
    assert torch.equal(flash_attn_with_kvcache_q8(q, beside, row, v, 0), flash_attn_with_kvcache_q8(q, cache, k, v, 0))
    assert torch.equal(beside.k_recent, cache.k_recent)


def test_wide_lengths_and_rows_off_alignment(path):
    q, k, v = (_rand(3, 2, 2, 128, seed=i) for i in range(3))
    off = torch.cat((k.flatten()[:1], k.flatten()))[1:].view_as(k)
    assert off.data_ptr() % 16
    lens = torch.tensor([2 ** 32 + 7, -(2 ** 33), 100], device=DEV)
    out = []
    for n, kk in ((lens, off), (torch.tensor([128, 0, 100], dtype=torch.int32, device=DEV), k)):
        cache = kvcache_q8(3, 128, 2)
        for j in range(0, 100, 50):
            flash_attn_with_kvcache_q8(_rand(3, 50, 2, 128, seed=j), cache, _rand(3, 50, 2, 128, seed=j + 1),
                                       _rand(3, 50, 2, 128, seed=j + 2), j)
        out.append((flash_attn_with_kvcache_q8(q, cache, kk, v, n), *cache))
    for a, b in zip(*out):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
