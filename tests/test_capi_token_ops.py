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
