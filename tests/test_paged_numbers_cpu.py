"""What the calls on a cache in pages take for a number of rows: whole numbers, of any kind, and tensors."""
import numpy
import pytest
import torch

import prefixlm
from prefixlm import paged_kvcache
from prefixlm.paged import _rows


def test_what_is_no_number_of_rows_is_refused():
    """None in particular, which would give up every page of every sequence."""
    c = paged_kvcache(4, 16, 2, 64, 1, device="cpu")
    q = torch.zeros(2, 1, 1, 128, dtype=torch.bfloat16)
    for x in (None, 2.5, "3", [1, 2]):
        for call, name in ((lambda: prefixlm.paged_kvcache_free(c, x), "keep_rows"), (lambda: prefixlm.paged_kvcache_reserve(c, 0, x), "new_rows")):
            with pytest.raises(ValueError, match=name):
                call()
        if x is not None:
            for call in (lambda: prefixlm.paged_kvcache_reserve(c, x, 1), lambda: prefixlm.flash_attn_with_paged_kvcache(q, c, cache_seqlens=x)):
                with pytest.raises(ValueError, match="cache_seqlens"):
                    call()


def test_whole_numbers():
    dev = torch.device("cpu")
    assert [_rows(x, 2, dev, "x") for x in (3, True, numpy.int64(7), numpy.int32(-4), 2**40, -2**70)] == [
        (None, n) for n in (3, 1, 7, -1, 2**31 - 1, -1)]
    assert _rows(torch.tensor([2**40, -2**40]), 2, dev, "x")[0].tolist() == [2**31 - 1, -2**31]
