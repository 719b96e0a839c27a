"""GPU: the order in which the table's gradient is added, bit for bit.

The tokens are sorted by id, those of one id in their order, and cut into chunks: 16 sorted tokens
where T times the number of 512-column blocks is below 65536, else 32. A chunk adds an id's rows one
after another in float32, and an id that goes on over several chunks has the chunks' sums added in
their order; then the scale, then the rounding."""
import numpy as np
import pytest
import torch

from prefixlm.embedding import embedding_bwd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _emulate(ids, dy, V, scale, run):
    order = np.argsort(ids, kind="stable")
    grad = np.zeros((V, dy.shape[1]), np.float32)
    whole, last = None, -1                     # the id so far, over chunks
    for c in range(0, len(order), run):
        part, key = None, -1
        for i in list(order[c:c + run]) + [None]:
            k = ids[i] if i is not None else -2
            if k != key:
                if part is not None:           # the run of `key` in this chunk has ended
                    whole = part if key != last else whole + part
                    last = key
                    grad[key] = whole
                part, key = np.zeros(dy.shape[1], np.float32), k
            if i is not None:
                part = part + dy[i]
    return grad * np.float32(scale)


@pytest.mark.parametrize("T,D,run", [(7, 8, 16), (1000, 24, 16), (16384, 8, 16), (16385, 8, 16), (40000, 16, 16),
                                     (33000, 520, 32), (65535, 8, 16), (65536, 8, 32), (70001, 8, 32)])
def test_chunks_and_their_joins(T, D, run):
    print(f"[case] {T} {D}", flush=True)
    V = 4000
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, V, (T,), generator=g)
    ids[torch.rand(T, generator=g) < 0.33] = 1234                  # a third of the tokens is one id
    ids[torch.rand(T, generator=g) < 0.01] = V - 1
    dy = torch.randn(T, D, generator=g)
    want = torch.from_numpy(_emulate(ids.numpy(), dy.numpy(), V, 1.75, run))
    got = embedding_bwd(ids.to(DEV), dy.to(DEV), V, 1.75, torch.float32, -1).cpu()
    assert torch.equal(got, want), (got != want).nonzero()[:4].tolist()
    half = embedding_bwd(ids.to(DEV), dy.to(DEV), V, 1.75, torch.bfloat16, -1).cpu()
    assert torch.equal(half, want.bfloat16())


def test_runs_at_every_place_of_a_chunk():
    """Ids of 1 to 70 tokens in turn: each length begins at most places of a chunk."""
    n = torch.arange(1, 71).repeat(6)
    ids = torch.repeat_interleave(torch.arange(n.numel()), n)
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))]
    dy = torch.randn(ids.numel(), 8, generator=torch.Generator().manual_seed(2))
    want = torch.from_numpy(_emulate(ids.numpy(), dy.numpy(), n.numel(), 1.0, 16))
    got = embedding_bwd(ids.to(DEV), dy.to(DEV), n.numel(), 1.0, torch.float32, -1).cpu()
    assert torch.equal(got, want)
