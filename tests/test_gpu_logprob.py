"""GPU: token log probabilities, entropy, alternatives and the logits' gradient against the fp64 oracle.

Tolerances (u = 2^-24, fp32's half step). A thread adds at most V / 512 + 8 of the weights and 17 more
sums join them, each off by u; a weight e^(x - m) is off by (2 |x - m| + 4) u relative, which weighted
is at most 5 u; so S is off by (V / 512 + 32) u relative and ln S by that much. logprob adds the
rounding of its terms, (|x_t - m| + ln S) 4 u; W / S is off by twice S's error relative, plus 2 u.
p = e^((x - m) - ln S) has ln S's error and (3 |x - m| + 2 ln S + 4) u, relative; bf16 gradients
another half step, 2^-8 relative. Indices are equal.
"""
import math

import pytest
import torch

from oracle import logprob_oracle as oracle
from prefixlm import token_logprobs
from prefixlm.logprob import token_logprobs_bwd, token_logprobs_fwd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _close(tag, got, want, tol):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), tag
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), tag
    ok = torch.isfinite(want)
    over = ((got - want).abs() - tol)[ok]
    assert not over.numel() or over.max().item() <= 0, (tag, (got - want).abs()[ok].max().item())


def _sum_tol(V):
    return (V / 512 + 32) * U


def _check(x, t, top=0, ignore=-100, entropy=True, with_grad=True):
    """x, t on the CPU."""
    V = x.shape[-1]
    xd = x.to(DEV).requires_grad_(with_grad)
    r = token_logprobs(xd, t.to(DEV) if t is not None else None, entropy=entropy, top_k=top, ignore_index=ignore)
    x2, t2 = x.reshape(-1, V), t.reshape(-1) if t is not None else None
    lp, ent, lse, tv, ti = oracle.forward(x2, t2, top, ignore)
    m = x2.double().amax(-1)
    m = torch.where(torch.isinf(m), 0.0, m)
    span = (x2.double() - m[:, None]).exp().sum(-1).log().abs().nan_to_num(0, 0, 0)   # ln S
    if t is not None:
        far = (lp + span).abs().nan_to_num(0, 0, 0) + span
        _close("logprob", r.logprob.reshape(-1), lp, _sum_tol(V) + 4 * U * far)
    if entropy:
        _close("entropy", r.entropy.reshape(-1), ent, _sum_tol(V) * (1 + 2 * (ent.abs() + span).nan_to_num(0)) + 4 * U)
    if top:
        _close("top", r.top_logprobs.reshape(-1, top), tv, _sum_tol(V) + 4 * U * (span + (tv + span[:, None]).abs().nan_to_num(
            0, 0, 0).amax(-1))[:, None])
        assert torch.equal(r.top_ids.reshape(-1, top).cpu(), ti)
    if not with_grad or (t is None and not entropy):
        return r
    g = torch.randn(x2.shape[0], generator=torch.Generator().manual_seed(3)) if t is not None else None
    h = torch.randn(x2.shape[0], generator=torch.Generator().manual_seed(4)) if entropy else None
    heads = [y for y in (r.logprob, r.entropy) if y is not None]
    given = [y.to(DEV).reshape(heads[0].shape) for y in (g, h) if y is not None]
    d, = torch.autograd.grad(heads, (xd,), given)
    assert d.dtype == x.dtype and d.shape == x.shape
    want = oracle.backward(x2, t2, g, h, ignore)
    logp = (x2.double() - m[:, None]) - (x2.double() - m[:, None]).exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    rel = _sum_tol(V) + (3 * (logp.abs().clamp_max(200) + span[:, None]) + 2 * span[:, None] + 8) * U
    w = (g.abs().double()[:, None] if g is not None else 0.0)
    if h is not None:
        w = w + h.abs().double()[:, None] * (logp.abs().clamp_max(200) + ent.abs()[:, None] + 2)
    tol = (p * w * rel).nan_to_num(0) * 2 + want.abs().nan_to_num(0) * (2.0 ** -8 if x.dtype == torch.bfloat16 else 4 * U) + 1e-37
    _close("grad", d.reshape(-1, V), want, tol)
    return r


def _random(rows, V, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * scale).to(dtype), torch.randint(0, V, (rows,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 5), (2, 8), (7, 63), (260, 129), (5, 4096), (3, 4099), (300, 1001),
                                    (2, 20011), (1, 50257), (1, 131072)])
def test_matches_oracle(rows, V, dtype):
    x, t = _random(rows, V, dtype, rows + V)
    t[0] = V - 1
    _check(x, t, top=min(5, V))
    _check(x, t, top=0, entropy=False)


@pytest.mark.parametrize("top", [1, 2, 20, 64])
@pytest.mark.parametrize("rows,V", [(3, 64), (300, 700), (2, 30000)])
def test_tops_of_every_length(rows, V, top):
    x, t = _random(rows, V, torch.float32, top)
    _check(x, t, top=top, entropy=False, with_grad=False)
    _check(x.bfloat16(), None, top=top, entropy=True)


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("V", [40, 3000, 20000])
def test_equal_logits_go_by_index(rows, V):
    """Rows of one value, of two, and of few: more equal values than a workgroup ranks at once."""
    x = torch.zeros(rows, V)
    x[0, V // 2:] = 1.0
    x[1] = (torch.arange(V) % 7).float()
    x[1, 5] = -0.0
    x[1, 7] = 0.0
    for dtype in (torch.bfloat16, torch.float32):
        _check(x.to(dtype), torch.full((rows,), V - 1), top=min(33, V), with_grad=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [6, 300])
def test_masked_logits(rows, dtype):
    """-inf and the type's lowest value beside ordinary logits, in most of a row and in all of it."""
    V = 9001
    x, t = _random(rows, V, dtype, 5)
    low = torch.finfo(dtype).min
    x[0, 10:] = -math.inf
    x[1, :V - 1] = low
    x[2] = low
    x[3] = -math.inf
    x[4, ::2] = -math.inf
    t[0], t[1], t[4] = 3, V - 1, 1
    xd = x.to(DEV)
    r = token_logprobs(xd, t.to(DEV), entropy=True, top_k=4)
    assert torch.isnan(r.logprob[3]) and torch.isnan(r.entropy[3])    # as log_softmax
    assert r.top_ids[3].tolist() == [0, 1, 2, 3] and r.top_ids[2].tolist() == [0, 1, 2, 3]
    assert r.top_ids[0, :4].tolist() == x[0, :10].float().topk(4).indices.tolist()
    keep = [i for i in range(rows) if i != 3]
    _check(x[keep], t[keep], top=4)
    hidden = t[0].item() + 100
    assert token_logprobs(xd[:1], torch.tensor([hidden], device=DEV)).logprob.item() == -math.inf


def test_nan_and_infinite_logits_spread_over_their_row_only():
    x, t = _random(300, 5000, torch.float32, 6)
    x[1, 17], x[2, 40] = math.nan, math.inf
    r = token_logprobs(x.to(DEV), t.to(DEV), entropy=True, top_k=3)
    assert torch.isnan(r.logprob[[1, 2]]).all() and torch.isnan(r.entropy[[1, 2]]).all()
    assert torch.isnan(r.top_logprobs[[1, 2]]).all() and r.top_ids[1].tolist()[0] == 17 and r.top_ids[2].tolist()[0] == 40
    keep = [0] + list(range(3, 300))
    lp, ent, _, _, ti = oracle.forward(x[keep], t[keep], 3)
    _close("logprob", r.logprob[keep], lp, 1e-5)
    assert torch.equal(r.top_ids[keep].cpu(), ti)
    assert ((r.top_ids >= 0) & (r.top_ids < 5000)).all()
    every = token_logprobs(torch.full((2, 3000), math.nan, device=DEV), None, top_k=64)
    assert ((every.top_ids >= 0) & (every.top_ids < 3000)).all()


@pytest.mark.parametrize("rows", [4, 400])
def test_ignored_and_outside_targets(rows):
    x, t = _random(rows, 3001, torch.bfloat16, 7)
    t[0], t[1], t[2] = -100, -1, 3001
    r = _check(x, t, top=2)
    assert r.logprob[0].item() == 0.0 and torch.isnan(r.logprob[1:3]).all()
    _check(x, t, entropy=False)
    t[t == -100] = 7
    t[3] = 5
    _check(x, t, ignore=5, entropy=False)
    # an ignored row has no gradient, whatever it holds
    x[3] = math.nan
    xd = x.to(DEV).requires_grad_()
    token_logprobs(xd, t.to(DEV), ignore_index=5).logprob[3:].sum().backward()
    assert torch.equal(xd.grad[3], torch.zeros(3001, dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_offsets_and_shapes(dtype):
    base, t = _random(12, 1013, dtype, 8)
    wide = torch.zeros(12, 1200, dtype=dtype)
    wide[:, 3:1016] = base
    _check(base.reshape(3, 4, 1013), t.reshape(3, 4), top=3)
    got = token_logprobs(wide.to(DEV)[:, 3:1016], t.to(DEV).int(), entropy=True, top_k=3)
    want = token_logprobs(base.to(DEV), t.to(DEV), entropy=True, top_k=3)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    cols = token_logprobs(base.t().contiguous().to(DEV).t(), t.to(DEV))            # strided over V: copied
    assert torch.equal(cols.logprob, want.logprob)
    same = token_logprobs(base[:1].to(DEV).expand(5, 1013), t[:1].to(DEV).expand(5))   # one row, five times
    assert torch.equal(same.logprob, want.logprob[:1].expand(5))
    xd = wide.to(DEV).requires_grad_()
    token_logprobs(xd[:, 3:1016], t.to(DEV)).logprob.sum().backward()
    xe = base.to(DEV).requires_grad_()
    token_logprobs(xe, t.to(DEV)).logprob.sum().backward()
    assert torch.equal(xd.grad[:, 3:1016], xe.grad) and not xd.grad[:, :3].any() and not xd.grad[:, 1016:].any()
    empty = token_logprobs(torch.zeros(0, 7, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 2)
    one = token_logprobs(base[0].to(DEV), t[0].to(DEV))
    assert one.logprob.shape == () and torch.equal(one.logprob, want.logprob[0])


def test_large_logits_keep_their_precision():
    x, t = _random(4, 2000, torch.float32, 9, scale=1.0)
    x += 20000.0
    _check(x, t, top=3)


def test_rows_past_32_bits():
    """Logits of more than 2^32 elements: the last rows, at odd offsets."""
    V, rows = 1 << 20, 4100
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.randn(2, V, device=DEV).bfloat16()
    t = torch.full((rows,), 5, device=DEV)
    got = token_logprobs(x, t, top_k=2)
    lp = torch.log_softmax(x[-2:].double(), -1)
    tol = _sum_tol(V) + 100 * U
    assert (got.logprob[-2:].double() - lp[:, 5]).abs().max().item() <= tol
    assert torch.equal(got.top_ids[-2:], torch.sort(lp, descending=True, stable=True).indices[:, :2])   # topk: any order of ties
    assert (got.logprob[0].double() + math.log(V)).abs().item() <= tol
    lse = torch.logsumexp(x[-2:].double(), -1)
    f, dx = token_logprobs_fwd(x, t, False, 0, -100), None
    dx = token_logprobs_bwd(x, t, f[2], f[1], torch.ones(rows, device=DEV), None, -100)
    want = -torch.exp(x[-2:].double() - lse[:, None])
    want[:, 5] += 1
    assert ((dx[-2:].double() - want).abs() <= want.abs() * 2.0 ** -8 + want.abs() * tol + 1e-37).all()


def test_gradient_matches_differences():
    x, t = _random(2, 40, torch.float32, 10)
    xd = x.to(DEV).requires_grad_()
    r = token_logprobs(xd, t.to(DEV), entropy=True)
    d, = torch.autograd.grad((r.logprob.sum() + 0.5 * r.entropy.sum()), (xd,))

    def f(y):
        lp, e, _, _, _ = oracle.forward(y, t)
        return lp.sum() + 0.5 * e.sum()

    for j in range(0, 40, 7):
        step = torch.zeros(2, 40, dtype=torch.float64)
        step[1, j] = 1e-6
        diff = (f(x.double() + step) - f(x.double() - step)) / 2e-6
        assert abs(diff.item() - d[1, j].item()) < 1e-5   # 1e-9 of differences, 1e-6 of fp32


def test_one_of_two_gradients():
    x, t = _random(300, 500, torch.bfloat16, 11)
    xd = x.to(DEV).requires_grad_()
    r = token_logprobs(xd, t.to(DEV), entropy=True, top_k=2)
    assert not r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    d, = torch.autograd.grad(r.entropy.sum(), (xd,), retain_graph=True)
    want = oracle.backward(x, t, None, torch.ones(300))
    assert ((d.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
    d, = torch.autograd.grad(r.logprob.sum(), (xd,))
    want = oracle.backward(x, t, torch.ones(300), None)
    assert ((d.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()


def test_repeats_bitwise_and_both_host_paths_agree():
    x, t = _random(3, 60000, torch.bfloat16, 12)
    xd, td = x.to(DEV), t.to(DEV)
    a = token_logprobs(xd, td, entropy=True, top_k=9)
    for _ in range(3):
        for u, v in zip(a, token_logprobs(xd, td, entropy=True, top_k=9)):
            assert torch.equal(u, v)
    lp, ent, _, top, ids = token_logprobs_fwd(xd, td, True, 9, -100)
    for u, v in zip(a, (lp, ent, top, ids)):
        assert torch.equal(u, v)


def test_graph_replays():
    """Captured forward and backward, replayed on new inputs between eager calls."""
    rows, V = 5, 33000
    xs, t = _random(rows, V, torch.bfloat16, 13)
    x, t = xs.to(DEV).requires_grad_(), t.to(DEV)
    g = torch.ones(rows, device=DEV)

    def step():
        r = token_logprobs(x, t, entropy=True, top_k=5)
        return (*r, *torch.autograd.grad((r.logprob, r.entropy), (x,), (g, g)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(_random(rows, V, torch.bfloat16, 20 + k)[0].to(DEV))
            t.copy_(torch.randint(0, V, (rows,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream_and_compile():
    x, t = _random(40, 2000, torch.bfloat16, 14)
    xd, td = x.to(DEV), t.to(DEV)
    want = token_logprobs(xd, td, entropy=True, top_k=3)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = token_logprobs(xd, td, entropy=True, top_k=3)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)

    @torch.compile(dynamic=False, fullgraph=True)
    def loss(x, t):
        r = token_logprobs(x, t, entropy=True, top_k=3)
        return r.logprob.sum() + r.entropy.sum(), r.top_ids

    xe, xc = xd.clone().requires_grad_(), xd.clone().requires_grad_()
    r = token_logprobs(xe, td, entropy=True)
    (r.logprob.sum() + r.entropy.sum()).backward()
    y, ids = loss(xc, td)
    y.backward()
    assert torch.equal(ids, want.top_ids) and torch.equal(xe.grad, xc.grad)


def test_refusals_on_the_gpu():
    x, t = torch.zeros(4, 10, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad, needle in ((dict(targets=t[:3]), "targets"), (dict(targets=t.cpu()), "targets"),
                        (dict(targets=t.float()), "targets"), (dict(targets=t, top_k=11), "top_k"),
                        (dict(targets=t, top_k=-1), "top_k")):
        with pytest.raises(ValueError, match=needle):
            token_logprobs(x, **bad)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        token_logprobs(x.half(), t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("equal", [3, 600, 1022, 1023, 1024, 1025, 2048])
def test_alternatives_among_many_equal_ones(equal, dtype):
    """The largest value at `equal` places, each in another thread's vectors: as many places as are
    ranked at once, one more, and fewer; the lowest ids win. A row alone and a row among others."""
    print(f"[case] equal {equal} {dtype}", flush=True)
    V, g = 65543, torch.Generator().manual_seed(equal)
    x = torch.randn(3, V, generator=g).clamp_(max=3.0).to(dtype)
    turn, thread = torch.arange(2048) // 512, torch.arange(2048) % 512
    at = (8 * (turn * 2048 + thread))[torch.randperm(2048, generator=g)[:equal]]
    x[1, at] = 4.0
    x[2, at] = 4.0
    x[2, V - 1] = 5.0
    for top in (1, 7, 64):
        _check(x, torch.zeros(3, dtype=torch.int64), top=top, with_grad=False)


@pytest.mark.parametrize("rows,V,top", [(1, 98304, 8), (16, 98307, 3), (2, 131072, 9), (64, 131073, 20), (3, 262145, 64),
                                        (65, 131072, 2), (5, 140001, 0)])
def test_split_rows(rows, V, top):
    """Rows in several workgroups, with as few and as many alternatives as their join ranks."""
    print(f"[case] split {rows} {V} {top}", flush=True)
    x, t = _random(rows, V, torch.bfloat16, rows + top)
    x[0, -5:] = 60.0
    x[-1, :V // 2] = -math.inf
    _check(x, t, top=top, with_grad=False)
