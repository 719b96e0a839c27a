"""The C entry points of the cache in pages refuse by name what no launch can hold, before the GPU is touched."""
import ctypes
import os

import pytest

from prefixlm import _build, _capi

FAKE = 1 << 20   # never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def _pool(**kw):
    a = dict(k_pages=FAKE, v_pages=FAKE, refs=FAKE, page_table=FAKE, table_stride=1 << 26, layers=1, num_pages=4, num_kv_heads=16,
             page_size=16, head_dim=128, batch=1, columns=64)
    return _capi.PagePool(**{**a, **kw})


# one row a unit in workgroups of 512 threads, up to 16 and blocks of 128 in workgroups of 256
@pytest.mark.parametrize("B,Hkv,G,S", [(1 << 19, 16, 1, 1), (1 << 20, 16, 4, 1), (1, 16, 1, 1 << 27), (512, 16, 2, 1 << 17)])
def test_attention_past_a_launch(lib, B, Hkv, G, S):
    a = _capi.PagedArgs(pool=_pool(batch=B, num_kv_heads=Hkv), q=FAKE, out=FAKE, cache_seqlen=3, seqlen_q=S, num_heads=G * Hkv,
                        softmax_scale=0.1, workspace=FAKE, workspace_bytes=1 << 62)
    assert lib.prefixlm_paged_fwd(ctypes.byref(a), None) == 1 and "too large" in _capi.last_error()


@pytest.mark.parametrize("N,columns", [(600, 1 << 26), (1024, 1 << 26), (8192, 1 << 24)])
def test_fork_past_a_launch(lib, N, columns):
    a = _capi.PagesArgs(pool=_pool(batch=N, columns=columns), src=FAKE)
    assert lib.prefixlm_pages_fork(ctypes.byref(a), None) == 1 and "too large" in _capi.last_error()
