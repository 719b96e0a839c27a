"""GPU: the scaled embedding against float32 torch (bitwise) and its gradient against the fp64 oracle.

Tolerances: the lookup is one fp32 product and one rounding, torch's own: equal bits. An element of
the gradient that n rows go into is off by at most (n + 2) 2^-24 of the sum of their magnitudes
(n additions and the scale), and by half a step of its type: 2^-8 relative in bf16, 2^-24 in fp32.
"""
import pytest
import torch

from oracle import embedding_oracle as oracle
from prefixlm import embedding
from prefixlm.embedding import embedding_bwd, embedding_fwd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32


def _data(T, V, D, table, out, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=g) if ids is None else ids
    return ids, torch.randn(V, D, generator=g).to(table), torch.randn(*ids.shape, D, generator=g).to(out)


def _tol(ids, dtype, mag, want):
    n = torch.bincount(ids.reshape(-1).clamp(0, want.shape[0] - 1), minlength=want.shape[0]).double()[:, None]
    return (n + 2) * 2.0 ** -24 * mag + want.abs() * (2.0 ** -8 if dtype == BF else 2.0 ** -24) + 1e-40


def _check(ids, table, dy, scale, padding=None):
    t = table.to(DEV).requires_grad_()
    y = embedding(ids.to(DEV), t, scale, dtype=dy.dtype, padding_idx=padding)
    ok = (ids >= 0) & (ids < table.shape[0])
    want = (table[ids.clamp(0, table.shape[0] - 1)].float() * torch.tensor(scale, dtype=F32)).to(dy.dtype)
    assert y.shape == want.shape and torch.equal(y.detach().cpu()[ok], want[ok])
    assert torch.isnan(y.detach().cpu()[~ok]).all()
    grad, = torch.autograd.grad(y, (t,), dy.to(DEV))
    ref, mag = oracle.backward(ids, dy, table.shape[0], scale, -1 if padding is None else padding)
    assert grad.dtype == table.dtype and grad.shape == table.shape
    over = (grad.double().cpu() - ref).abs() - _tol(ids, table.dtype, mag, ref)
    assert over.max().item() <= 0, over.max().item()
    untouched = mag.sum(-1) == 0
    assert not grad.cpu()[untouched].any()
    return grad


@pytest.mark.parametrize("table,out", [(BF, BF), (F32, BF), (F32, F32), (BF, F32)])
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (5, 3, 8), (63, 10, 24), (64, 512, 512), (65, 511, 520), (129, 513, 128),
                                   (700, 40, 1032), (2047, 5000, 64), (2049, 300000, 8), (6000, 700, 136)])
def test_matches_oracle(T, V, D, table, out):
    ids, t, dy = _data(T, V, D, table, out, T + V)
    _check(ids, t, dy, 3.25)


@pytest.mark.parametrize("table", [BF, F32])
def test_long_runs(table):
    """One id for every token; runs that begin and end at every place of a chunk of sorted tokens."""
    ids = torch.full((1000,), 6)
    _check(*_data(1000, 9, 40, table, BF, 1, ids), 1.0)
    ids = torch.repeat_interleave(torch.arange(12), torch.tensor([1, 63, 64, 65, 1, 62, 128, 129, 191, 3, 300, 1]))
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(2))]
    _check(*_data(0, 13, 72, table, BF, 2, ids), 0.5)
    half = torch.where(torch.arange(4096) % 2 == 0, 3, torch.arange(4096) % 4000)
    _check(*_data(0, 4000, 16, table, BF, 3, half), 1.0)


def test_padding_and_outside_ids():
    ids, t, dy = _data(500, 30, 16, F32, BF, 4)
    ids[::7] = 5
    grad = _check(ids, t, dy, 2.0, padding=5)
    assert not grad[5].any()
    ids[0], ids[1], ids[2], ids[3] = -1, 30, 1 << 40, -(1 << 62)
    _check(ids, t, dy, 2.0)
    _check(torch.full((100,), 99), t, dy[:100], 1.0)      # no token has a gradient
    _check(torch.full((100,), 29), t, dy[:100], 1.0, padding=29)


def test_shapes_strides_and_int32():
    ids, t, dy = _data(24, 50, 32, BF, BF, 5)
    a = _check(ids, t, dy, 1.5)
    b = _check(ids.reshape(2, 3, 4), t, dy.reshape(2, 3, 4, 32), 1.5)
    assert torch.equal(a, b)
    wide = torch.zeros(50, 48, dtype=BF)
    wide[:, 8:40] = t
    td, wd = t.to(DEV), wide.to(DEV)
    want = embedding(ids.to(DEV), td, 1.5)
    assert torch.equal(embedding(ids.to(DEV).int(), wd[:, 8:40], 1.5), want)
    assert torch.equal(embedding(ids.to(DEV), wd[:, 8:40].t().contiguous().t(), 1.5), want)       # copied
    assert torch.equal(embedding(ids.to(DEV), td[:1].expand(50, 32), 1.5), embedding(ids.to(DEV) * 0, td, 1.5))
    assert torch.equal(embedding(ids.to(DEV).reshape(4, 6).t(), td, 1.5), want.reshape(4, 6, 32).transpose(0, 1))
    one = embedding(ids[0].to(DEV), td)
    assert one.shape == (32,) and torch.equal(one, td[ids[0]])
    # gradients of other layouts: expanded, strided, and off 16 bytes
    flat = dy.to(DEV)
    base = embedding_bwd(ids.to(DEV), flat, 50, 1.5, BF, -1)
    assert torch.equal(embedding_bwd(ids.to(DEV).int(), flat.t().contiguous().t(), 50, 1.5, BF, -1), base)
    off = torch.zeros(24 * 32 + 1, dtype=BF, device=DEV)[1:].view(24, 32).copy_(flat)
    assert torch.equal(embedding_bwd(ids.to(DEV), off, 50, 1.5, BF, -1), base)
    tt = td.clone().requires_grad_()
    embedding(ids.to(DEV), tt, 1.5).sum().backward()                                               # stride 0
    ref, mag = oracle.backward(ids, torch.ones(24, 32), 50, 1.5)
    assert ((tt.grad.double().cpu() - ref).abs() <= _tol(ids, BF, mag, ref)).all()


def test_no_tokens():
    t = torch.randn(20, 16, device=DEV, requires_grad=True)
    ids = torch.zeros(0, dtype=torch.int64, device=DEV)
    y = embedding(ids, t)
    assert y.shape == (0, 16)
    grad, = torch.autograd.grad(y, (t,), torch.zeros(0, 16, device=DEV))
    assert torch.equal(grad, torch.zeros_like(t))


def test_infinities_stay_in_their_rows():
    ids, t, dy = _data(300, 20, 16, F32, BF, 6)
    dy[ids == 3] = float("inf")
    t[7] = float("nan")
    td = t.to(DEV).requires_grad_()
    y = embedding(ids.to(DEV), td, 1.0)
    assert torch.isfinite(y.cpu()[ids != 7]).all()
    grad, = torch.autograd.grad(y, (td,), dy.to(DEV).float())
    keep = torch.arange(20) != 3
    assert torch.isfinite(grad.cpu()[keep]).all() and torch.isinf(grad.cpu()[3]).all()


def test_tables_past_32_bits():
    """A table and a gradient of more than 2^32 bytes, ids at both ends."""
    V, D = 600000, 2048
    t = torch.zeros(V, D, dtype=F32, device=DEV)
    t[-3:] = torch.randn(3, D, device=DEV)
    ids = torch.tensor([V - 1, 0, V - 3, V - 1], device=DEV)
    assert torch.equal(embedding(ids, t, 2.0), t[ids] * 2.0)
    dy = torch.randn(4, D, device=DEV)
    grad = embedding_bwd(ids, dy, V, 1.0, F32, -1)
    assert torch.equal(grad[V - 1], dy[0] + dy[3]) and torch.equal(grad[0], dy[1]) and torch.equal(grad[V - 3], dy[2])
    grad[V - 1], grad[0], grad[V - 3] = 0, 0, 0
    assert not grad.any()


def test_many_tokens():
    """More tokens than the sort's smallest tiles cover; the order of the sum is the tokens'."""
    T, V = 400001, 70000
    g = torch.Generator(device=DEV).manual_seed(7)
    ids = (torch.rand(T, generator=g, device=DEV) ** 3 * V).long()
    dy = torch.randn(T, 8, generator=g, device=DEV)
    grad = embedding_bwd(ids, dy, V, 1.0, F32, -1)
    order = torch.argsort(ids, stable=True)
    want = torch.zeros(V, 8, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
    mag = torch.zeros(V, 8, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double().abs())
    n = torch.bincount(ids, minlength=V)[:, None]
    assert ((grad.double() - want).abs() <= (n + 2) * 2.0 ** -24 * mag + 1e-40).all()
    few = (n[:, 0] <= 3) & (n[:, 0] > 1)          # runs of two and three, added one after another
    first = torch.cumsum(n[:, 0], 0) - n[:, 0]
    v = int(torch.nonzero(few)[0])
    acc = torch.zeros(8, device=DEV)
    for i in order[first[v]:first[v] + n[v, 0]]:
        acc = acc + dy[i]
    if int(first[v]) // 64 == (int(first[v] + n[v, 0]) - 1) // 64:
        assert torch.equal(grad[v], acc)


def test_repeats_bitwise_and_both_host_paths_agree():
    ids, t, dy = _data(5000, 300, 256, F32, BF, 8)
    td, i, d = t.to(DEV).requires_grad_(), ids.to(DEV), dy.to(DEV)
    y = embedding(i, td, 1.5, dtype=BF)
    grads = [torch.autograd.grad(y, (td,), d, retain_graph=True)[0] for _ in range(3)]
    grads.append(embedding_bwd(i, d, 300, 1.5, F32, -1))
    assert all(torch.equal(grads[0], x) for x in grads[1:])
    assert torch.equal(embedding_fwd(i, t.to(DEV), 1.5, BF), y)


def test_graph_replays():
    ids, t, dy = _data(3000, 900, 128, BF, BF, 9)
    i, td, d = ids.to(DEV), t.to(DEV).requires_grad_(), dy.to(DEV)

    def step():
        y = embedding(i, td, 2.0)
        return y, torch.autograd.grad(y, (td,), d)[0]

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
        i.copy_(torch.randint(0, 900 if k % 2 else 5, (3000,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream_and_compile():
    ids, t, dy = _data(300, 90, 64, F32, BF, 10)
    i, td, d = ids.to(DEV), t.to(DEV), dy.to(DEV)
    want = embedding_bwd(i, d, 90, 1.0, F32, -1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = embedding_bwd(i, d, 90, 1.0, F32, -1)
    s.synchronize()
    assert torch.equal(got, want)

    @torch.compile(dynamic=False, fullgraph=True)
    def f(i, t):
        return embedding(i, t, 1.0, dtype=BF)

    tc = td.clone().requires_grad_()
    f(i, tc).backward(d)
    assert torch.equal(tc.grad, want)


def test_refusals_on_the_gpu():
    t, i = torch.zeros(10, 16, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for ids, table, kw, needle in ((i.cpu(), t, {}, "ids"), (i.float(), t, {}, "ids"), (i, t.half(), {}, "bf16 or fp32"),
                                   (i, t[:, :12], {}, "multiple of 8"), (i, t[0], {}, "table"), (i, t, {"dtype": torch.float16}, "dtype"),
                                   (i, t[:0], {}, "V in")):
        with pytest.raises(ValueError, match=needle):
            embedding(ids, table, **kw)


@pytest.mark.parametrize("T", [15, 16, 17, 32, 33, 1023, 1024, 1025, 2048, 4095, 4097, 5119, 6144, 6145, 8192, 8193, 9727, 12288,
                               12289, 16383, 16384, 16385])
def test_sorts_of_every_size(T):
    """Small whole numbers, whose sums are exact in any order: the gradient is the integer sum. Ids at
    both ends, some outside the table; the largest table of the one-launch sort and the next."""
    print(f"[case] sort {T}", flush=True)
    for V in (7, 262143, 262144):
        g = torch.Generator().manual_seed(T)
        ids = torch.randint(-1, V + 1, (T,), generator=g)
        ids[0], ids[-1] = V - 1, 0
        dy = torch.randint(-8, 9, (T, 8), generator=g)
        want = torch.zeros(V + 2, 8, dtype=torch.int64).index_add_(0, ids + 1, dy)[1:-1]
        got = embedding_bwd(ids.to(DEV), dy.to(BF).to(DEV), V, 1.0, F32, -1)
        assert torch.equal(got.cpu(), want.float())
