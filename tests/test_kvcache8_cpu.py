"""The 8-bit KV cache without a GPU: the oracle against the bf16 cache's oracle, its rounding, and the
refusals of the operator and of the C entry point."""
import ctypes
import os

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from oracle.kvcache_oracle import kvcache_attention
from prefixlm import KVCacheQ8, _build, _capi, flash_attn_with_kvcache_q8, kvcache_q8


def _rows(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S,lens", [(1, [0, 5, 63]), (3, [2, 60, 0]), (70, [0, 1, 50])])
def test_oracle_matches_the_bf16_cache_where_nothing_is_rounded(S, lens, causal):
    """Rows of the incomplete block, the call's new rows, and codes that hold their rows exactly."""
    B, H, Smax = 3, 2, 192
    q, k, v, kc, vc = (_rows(B, n, H, 128, seed=i) for i, n in enumerate((S, S, S, Smax, Smax)))
    cache = oracle.empty(B, H, Smax, torch.int8)
    for c, x in enumerate((kc, vc)):
        cache[4 + c][:] = x.transpose(1, 2)[:, :, :128]
    t = torch.tensor(lens)
    out, mag, new = oracle.attend(q, cache, k, v, t, causal)
    want, kn, _ = kvcache_attention(q, kc, vc, k, v, t, causal)
    assert (out - want.double()).abs().max() < 1e-5 and (mag >= out.abs() - 1e-12).all()
    for b, n in enumerate(lens):
        end = n + S
        for j in range(max(0, end // 64 * 64 - 64), end):
            assert torch.equal(new[4][b, :, j % 128], kn[b, j]), (b, j)


def test_exact_codes_are_the_bf16_cache():
    """Integer rows with 127 in every block are held exactly."""
    B, H, Smax, n = 2, 2, 256, 200
    g = torch.Generator().manual_seed(3)
    kc, vc = (torch.randint(-127, 128, (B, Smax, H, 128), generator=g).bfloat16() for _ in range(2))
    kc[:, ::64], vc[:, ::64] = 127.0, -127.0
    kc = kc / 128
    q = _rows(B, 2, H, 128)
    cache = oracle.empty(B, H, Smax, torch.int8)
    empty, lens = torch.zeros(B, 1, H, 128).bfloat16(), torch.full((B,), 0)
    _, _, cache = oracle.attend(empty.expand(B, n, H, 128), cache, kc[:, :n], vc[:, :n], lens)
    out, _, _ = oracle.attend(q, cache, lens=n)
    want, _, _ = kvcache_attention(q, kc.float(), vc.float(), cache_seqlens=n)
    assert (out - want.double()).abs().max() < 1e-4


@pytest.mark.parametrize("dtype,half", [(torch.int8, 0.5 / 127), (torch.float8_e4m3fn, 2.0 ** -4)])
def test_rounding_is_off_by_half_a_step(dtype, half):
    x = _rows(64, 128, seed=4)
    codes, scale = oracle.round_block(x, dtype)
    err = (codes.float() * scale - x.float()).abs()
    # int8: half a step of amax / 127; e4m3: 2^-4 of the value, or half its smallest step
    limit = x.float().abs().max() * half if dtype == torch.int8 else torch.maximum(x.float().abs() * half, scale * 2.0 ** -10)
    assert (err <= limit * (1 + 1e-5)).all()
    zero, s = oracle.round_block(torch.zeros(64, 128).bfloat16(), dtype)
    assert s == 2.0 ** -126 and not zero.float().any()


def test_planted_mistake_is_caught():
    """Scales of the blocks exchanged are ten times as far from the bf16 cache as the rounding is."""
    B, H = 1, 1
    k = _rows(B, 128, H, 128) * torch.where(torch.arange(128) < 64, 1.0, 30.0)[None, :, None, None].bfloat16()
    _, _, cache = oracle.attend(k, oracle.empty(B, H, 128, torch.int8), k, k, 0)
    q = _rows(B, 1, H, 128, seed=9)
    right, _, _ = oracle.attend(q, cache, lens=128)
    want, _, _ = kvcache_attention(q, k, k, cache_seqlens=128)
    cache[3] = cache[3].roll(1, -1)
    wrong, _, _ = oracle.attend(q, cache, lens=128)
    assert (wrong - want.double()).abs().max() > 10 * (right - want.double()).abs().max()


def test_cache_maker():
    c = kvcache_q8(2, 100, 3, device="cpu")
    assert c.k_codes.shape == (2, 3, 128, 128) and c.k_codes.dtype == torch.float8_e4m3fn
    assert c.v_scale.shape == (2, 3, 2) and c.v_recent.shape == (2, 3, 128, 128) and c.v_recent.dtype == torch.bfloat16
    assert kvcache_q8(1, 64, 1, dtype=torch.int8, device="cpu").v_codes.dtype == torch.int8
    for kw, needle in ((dict(head_dim=64), "head_dim"), (dict(dtype=torch.uint8), "dtype"), (dict(max_seqlen=0), "max_seqlen"),
                       (dict(batch=0), "batch")):
        with pytest.raises(ValueError, match=needle):
            kvcache_q8(**{**dict(batch=1, max_seqlen=64, num_heads=1, device="cpu"), **kw})


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU tensor"):
        flash_attn_with_kvcache_q8(_rows(1, 1, 1, 128), kvcache_q8(1, 64, 1, device="cpu"))


def test_fields_of_the_cache_follow_the_operator():
    assert KVCacheQ8._fields == ("k_codes", "v_codes", "k_scale", "v_scale", "k_recent", "v_recent")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def _args(**kw):
    fake = 1 << 20   # never dereferenced: validation fails first
    a = dict(q=fake, k=fake, v=fake, k_codes=fake, v_codes=fake, k_scale=fake, v_scale=fake, k_recent=fake, v_recent=fake,
             out=fake, cache_seqlen=3, batch=2, seqlen_q=1, num_heads=2, head_dim=128, max_seqlen_cache=1024,
             softmax_scale=0.1, workspace=fake, workspace_bytes=1 << 30)
    for n in ("q", "k", "v", "out"):
        a.update({f"{n}_stride_b": 256, f"{n}_stride_s": 256, f"{n}_stride_h": 128})
    a.update(kw)
    return _capi.Kvcache8Args(**a)


@pytest.mark.parametrize("kw,needle", [
    (dict(head_dim=64), "head_dim"), (dict(batch=0), "batch"), (dict(seqlen_q=0), "seqlen_q"), (dict(num_heads=0), "num_heads"),
    (dict(max_seqlen_cache=100), "multiple of 64"), (dict(max_seqlen_cache=0), "multiple of 64"), (dict(v=0), "together"),
    (dict(cache_seqlen=-1), "cache_seqlen"), (dict(cache_seqlen=1025), "cache_seqlen"), (dict(q=0), "null"),
    (dict(k_codes=(1 << 20) + 8), "aligned"), (dict(k_scale=(1 << 20) + 2), "aligned"), (dict(v_recent=0), "null"),
    (dict(k=(1 << 20) + 2), "aligned"), (dict(q_stride_h=4), "stride"), (dict(v_stride_s=-8), "stride"),
    (dict(workspace_bytes=8, max_seqlen_cache=4096), "workspace"),
    (dict(workspace=0, max_seqlen_cache=4096), "workspace"), (dict(seqlen_q=0x7fffffff), "too large"),
])
def test_entry_point_rejects(lib, kw, needle):
    assert lib.prefixlm_kvcache8_fwd(ctypes.byref(_args(**kw)), None) == 1
    assert needle in _capi.last_error()


def test_null_args_and_workspace(lib):
    assert lib.prefixlm_kvcache8_fwd(None, None) == 1
    assert lib.prefixlm_kvcache8_workspace_size(0, 1, 1, 64) == 0
    assert lib.prefixlm_kvcache8_workspace_size(1, 1, 1, 64) == 0          # one split
    assert lib.prefixlm_kvcache8_workspace_size(1, 1, 16, 4096) > 0
