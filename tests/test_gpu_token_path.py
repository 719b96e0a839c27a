"""GPU: the token ends and the 8-bit cache together, as a model uses them: the stack from tokens to log
probabilities with its gradients, and a decode loop (embedding, attention over the cache, log
probability and the best next token) eager and captured.

Each stage is held to its oracle on the inputs that the stage before it gave. Tolerances: the log
probabilities' are those of fp32 sums over V logits, (V / 512 + 32 + 4 (|x_t - m| + ln S)) 2^-24;
the attention's half a bf16 step and, of the sum of p |v|, 2 * 140 * 2^-24 of a score's magnitudes
(here below 2^6) and 1e-4 for its sums; a gradient of n bf16 rows half a step of its type and (n + 2)
2^-24 of their magnitudes.
"""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import embedding_oracle, kvcache8_oracle, logprob_oracle
from prefixlm import (KVCacheQ8, embedding, flash_attn_with_kvcache_q8, fused_attention_layer, kvcache_q8,
                      token_logprobs)
from prefixlm.hrm_stack import FusedLayer, HRMStack, HRMStackConfig, packed_position_ids
from prefixlm.synth import metadata_tensors

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _lp_tol(logits, t):
    x = logits.double()
    m = x.amax(-1)
    ln_s = (x - m[:, None]).exp().sum(-1).log()
    far = (x.gather(1, t.clamp_min(0)[:, None])[:, 0] - m).abs() + ln_s
    return (x.shape[-1] / 512 + 32 + 4 * far) * U


@pytest.mark.parametrize("embed_f32", [False, True])
def test_stack_scores_tokens(embed_f32):
    prefix, causal = np.array([5, 0, 40]), np.array([70, 33, 20])
    T, V = 180, 1003
    cfg = HRMStackConfig(hidden_size=256, num_heads=2, fused_elementwise=True, vocab_size=V)
    model = HRMStack(cfg).init_weights(3).to(DEV).to(torch.bfloat16)
    if embed_f32:
        model.embed = torch.nn.Parameter(model.embed.detach().float())
    st, ss = metadata_tensors(prefix, causal, T, DEV)
    info = {**st, **ss}
    pos = packed_position_ids(prefix, causal, T, DEV)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (T,), generator=g)
    ids[::9] = 7
    targets = torch.cat((ids[1:], torch.tensor([-100])))
    targets[:5] = -100
    attn = FusedLayer(fused_attention_layer)
    args = (pos, attn, info)
    r = model.score(ids.to(DEV), targets.to(DEV), *args, bp_steps=None, entropy=True, top_k=3)
    loss = -r.logprob.sum() / (targets != -100).sum() - 0.01 * r.entropy.mean()
    loss.backward()
    # the same hidden states and logits again (every kernel is deterministic)
    x = model.embed_tokens(ids.to(DEV)).detach().requires_grad_()
    assert torch.equal(x, (model.embed.detach()[ids.to(DEV)].float() * 16.0).bfloat16())
    z = model(x, *args, bp_steps=None)
    logits = F.linear(z, model.head.detach())
    lp, ent, _, top, tid = logprob_oracle.forward(logits.detach().cpu(), targets, 3)
    tol = _lp_tol(logits.detach().cpu(), targets)
    assert ((r.logprob.detach().double().cpu() - lp).abs() <= tol).all()
    assert ((r.entropy.detach().double().cpu() - ent).abs() <= tol * (1 + 4 * ent)).all()
    assert torch.equal(r.top_ids.cpu(), tid)
    # the gradients of the two ends, from the gradient of the logits
    n = int((targets != -100).sum())
    d = logprob_oracle.backward(logits.detach().cpu(), targets, torch.full((T,), -1.0 / n), torch.full((T,), -0.01 / T))
    zd = z.detach().double().cpu()
    head = d.t() @ zd
    # its elements are rounded to bf16, the products' sums too
    bound = 2.0 ** -8 * (d.abs().t() @ zd.abs()) * 1.01 + 2.0 ** -8 * head.abs() + 1e-9
    assert ((model.head.grad.double().cpu() - head).abs() <= bound).all()
    again = token_logprobs(logits, targets.to(DEV), entropy=True)
    dx, = torch.autograd.grad(-again.logprob.sum() / (targets != -100).sum() - 0.01 * again.entropy.mean(), (x,))
    table, mag = embedding_oracle.backward(ids, dx.cpu(), V, 16.0)
    count = torch.bincount(ids, minlength=V).double()[:, None]
    seen = model.embed.grad.double().cpu()
    assert ((seen - table).abs() <= (count + 2) * U * mag + (U if embed_f32 else 2.0 ** -8) * table.abs() + 1e-40).all()
    assert table.abs().max() > 0 and not seen[mag.sum(-1) == 0].any()


def test_the_plain_ends_of_the_stack_agree():
    """The same model with PyTorch's elementwise operations, in float32 on the CPU, at the token ends."""
    V, T = 211, 30
    cfg = HRMStackConfig(hidden_size=64, num_heads=2, vocab_size=V, max_seq_len=64)
    model = HRMStack(cfg).init_weights(5)
    ids = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(2))
    attn = lambda q, k, v, c, **_: v  # noqa: E731
    r = model.score(ids, ids, torch.arange(T), attn, {}, entropy=True, top_k=2)
    logits = F.linear(model(F.embedding(ids, model.embed) * 8.0, torch.arange(T), attn, {}), model.head)
    lp, ent, _, _, tid = logprob_oracle.forward(logits.detach(), ids, 2)
    assert ((r.logprob.detach().double() - lp).abs() <= 1e-5).all() and torch.equal(r.top_ids, tid)
    assert ((r.entropy.detach().double() - ent).abs() <= 1e-5 * (1 + ent)).all()


class _Decoder:
    """One attention layer between an embedding and a head, with a cache."""

    def __init__(self, B, H, V, Smax, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        D = 128 * H
        w = lambda n, m: (torch.randn(n, m, generator=g) / math.sqrt(m)).bfloat16().to(DEV)  # noqa: E731
        self.table, self.qkv, self.head = w(V, D), w(3 * D, D), w(V, D)
        self.cache = kvcache_q8(B, Smax, H, dtype=dtype)
        self.H, self.scale = H, math.sqrt(D)

    def rows(self, ids):
        x = embedding(ids, self.table, self.scale)
        return F.linear(x, self.qkv).view(*ids.shape, 3 * self.H, 128).split(self.H, dim=2)

    def step(self, ids, lens, cache=None):
        """(attention, logits, log probabilities of the best and of one other token) for ids [B, S]."""
        q, k, v = self.rows(ids)
        o = flash_attn_with_kvcache_q8(q, self.cache if cache is None else cache, k, v, lens, causal=True)
        logits = F.linear(o[:, -1].reshape(ids.shape[0], -1), self.head)
        return o, logits, token_logprobs(logits, ids[:, -1].contiguous(), entropy=True, top_k=4)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_decode_loop(dtype):
    B, H, V, Smax, prompt, steps = 3, 2, 1009, 256, 60, 80
    m = _Decoder(B, H, V, Smax, dtype, 7)
    ids = torch.randint(0, V, (B, prompt), generator=torch.Generator().manual_seed(8)).to(DEV)
    want = [x.cpu() for x in m.cache]
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    n, tokens = 0, ids
    for i in range(steps):
        q, k, v = (x.cpu() for x in m.rows(tokens))
        o, logits, r = m.step(tokens, lens)
        ref, mag, want = kvcache8_oracle.attend(q, want, k, v, n, True)
        if i % 8 < 2 or i in (3, 4, 5, 67, 68, 69):
            tol = 2.0 ** -8 * ref.abs() + (2 * 140 * U * 64 + 1e-4) * mag + 1e-9
            assert ((o.double().cpu() - ref).abs() <= tol).all(), i
            t = tokens[:, -1].cpu()
            lp, _, _, _, tid = logprob_oracle.forward(logits.cpu(), t, 4)
            assert ((r.logprob.double().cpu() - lp).abs() <= _lp_tol(logits.cpu(), t)).all() and torch.equal(r.top_ids.cpu(), tid)
        lens.add_(tokens.shape[1])
        n += tokens.shape[1]
        tokens = r.top_ids[:, :1].contiguous()
    for name, a, b in zip(KVCacheQ8._fields, m.cache, want):
        a, b = (x.view(torch.uint8) if x.element_size() == 1 else x for x in (a.cpu(), b))
        assert torch.equal(a, b), name


def test_a_captured_decode_step_gives_the_eager_tokens():
    B, H, V, Smax = 2, 2, 5003, 256
    m = _Decoder(B, H, V, Smax, torch.float8_e4m3fn, 9)
    first = torch.randint(0, V, (B, 1), generator=torch.Generator().manual_seed(10)).to(DEV)

    def run(cache, steps, step):
        for x in cache:
            x.zero_()
        ids, lens = first.clone(), torch.zeros(B, dtype=torch.int32, device=DEV)
        return [step(ids, lens) for _ in range(steps)]

    def advance(cache, ids, lens):
        _, _, r = m.step(ids, lens, cache)
        ids.copy_(r.top_ids[:, :1])
        lens.add_(1)
        return r

    eager = run(m.cache, 70, lambda ids, lens: (advance(m.cache, ids, lens).logprob.clone(), ids.clone()))
    other = kvcache_q8(B, Smax, H)
    ids, lens = first.clone(), torch.zeros(B, dtype=torch.int32, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        advance(other, ids, lens)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = advance(other, ids, lens)
    for again in range(2):
        for x in other:
            x.zero_()
        ids.copy_(first)
        lens.zero_()
        for i, (lp, token) in enumerate(eager):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.logprob, lp) and torch.equal(ids, token), (again, i)
    for a, b in zip(m.cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
