"""The argument structs of the log probabilities, the embedding and the 8-bit KV cache: the ctypes
mirrors against the header's layout, as gcc lays it out."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from prefixlm import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cname,cls", [("prefixlm_logprob_args", _capi.LogprobArgs),
                                       ("prefixlm_embedding_args", _capi.EmbeddingArgs),
                                       ("prefixlm_kvcache8_args", _capi.Kvcache8Args)])
def test_struct_layout_matches_header(cname, cls):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "prefixlm.h"', "int main(void){",
             f'printf("size %zu\\n", sizeof({cname}));']
    lines += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(src, "w") as out:
            out.write("\n".join(lines + ["return 0;}"]))
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(got[f]) == getattr(cls, f).offset, f


@pytest.fixture(scope="module")
def lib():
    from prefixlm import _build
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def test_calls_past_a_launch_are_refused(lib):
    """A launch has fewer than 2^32 threads: a call that needs more is refused before it."""
    fake = 1 << 20   # never dereferenced
    a = _capi.LogprobArgs(x=fake, targets=fake, logprob=fake, stats=fake, dx=fake, dlogprob=fake, x_stride=8, dx_stride=8,
                          rows=1 << 33, vocab=8)
    for rows in (1 << 23, 1 << 31, 1 << 62):
        a.rows = rows
        assert lib.prefixlm_logprob_fwd(ctypes.byref(a), None) == 1 and "too many" in _capi.last_error()
    for rows in (1 << 24, 1 << 31, 1 << 62):
        a.rows = rows
        assert lib.prefixlm_logprob_bwd(ctypes.byref(a), None) == 1 and "too many" in _capi.last_error()
    e = _capi.EmbeddingArgs(ids=fake, table=fake, y=fake, dy=fake, grad=fake, table_stride=8192, y_stride=8192, dy_stride=0,
                            tokens=1 << 22, vocab=100, padding_id=-1, cols=8192, scale=1.0, workspace=fake,
                            workspace_bytes=1 << 62)
    assert lib.prefixlm_embedding_fwd(ctypes.byref(e), None) == 1 and "too many" in _capi.last_error()
    e.tokens, e.cols, e.dy_stride = 0x7fffffff, 1 << 20, 1 << 20
    assert lib.prefixlm_embedding_bwd(ctypes.byref(e), None) == 1 and "too many" in _capi.last_error()
    c = _capi.Kvcache8Args(q=fake, k=fake, v=fake, k_codes=fake, v_codes=fake, k_scale=fake, v_scale=fake, k_recent=fake,
                           v_recent=fake, out=fake, cache_seqlen=3, batch=1 << 14, seqlen_q=1, num_heads=1 << 10,
                           head_dim=128, max_seqlen_cache=64, softmax_scale=0.1)
    assert lib.prefixlm_kvcache8_fwd(ctypes.byref(c), None) == 1 and "too large" in _capi.last_error()
