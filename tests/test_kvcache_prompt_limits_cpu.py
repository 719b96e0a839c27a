"""Prompts into an empty KV cache whose rows lie too far apart for the forward's 32-bit offsets are
not refused and take the extend kernel. Without a GPU a call ends where its path first needs the
device, and says where: the forward at its kernels' attributes, the 8-bit cache's extend at the device's
number."""
import ctypes
import os

import pytest
import torch

from prefixlm import _build, _capi

INVALID = 1


@pytest.fixture(scope="module")
def lib():
    if torch.cuda.is_available():
        pytest.skip("the calls below have no memory behind their pointers: they must end at the missing device")
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def _strides(names, S, far, stride):
    a = {}
    for n in names:
        a.update({f"{n}_stride_b": S * 128, f"{n}_stride_s": 128, f"{n}_stride_h": 128})
    a.update({f"{far}_stride_b": S * stride, f"{far}_stride_s": stride})
    return a


@pytest.mark.parametrize("far", ["q", "k", "v", "out"])
@pytest.mark.parametrize("stride,S", [(8192, 130815), (8192, 130816), (2048, 524031), (2048, 524032), (128, 100),
                                      (1 << 40, 2), (1 << 60, 2)])
def test_prompts_on_both_sides_of_the_limit(lib, far, stride, S):
    fake = 1 << 20   # never dereferenced
    Smax = (S + 63) // 64 * 64
    shared = dict(q=fake, k=fake, v=fake, out=fake, cache_seqlen=0, batch=1, seqlen_q=S, num_heads=1, head_dim=128,
                  max_seqlen_cache=Smax, softmax_scale=0.1, workspace=fake, workspace_bytes=1 << 62)
    a = _capi.Kvcache8Args(**shared, **_strides(("q", "k", "v", "out"), S, far, stride), k_codes=fake, v_codes=fake,
                           k_scale=fake, v_scale=fake, k_recent=fake, v_recent=fake)
    rc = lib.prefixlm_kvcache8_fwd(ctypes.byref(a), None)
    assert rc not in (0, INVALID), _capi.last_error()
    fits = (S + 256) * stride * 2 < 1 << 31
    assert ("hipGetDevice" in _capi.last_error()) != fits, _capi.last_error()
    caches = {f"{n}_cache_stride_{d}": x for n in "kv" for d, x in (("b", Smax * 128), ("s", 128), ("h", 128))}
    a = _capi.KvcacheArgs(**shared, **_strides(("q", "k", "v", "out"), S, far, stride), k_cache=fake, v_cache=fake, **caches)
    rc = lib.prefixlm_kvcache_fwd(ctypes.byref(a), None)
    assert rc not in (0, INVALID), _capi.last_error()
