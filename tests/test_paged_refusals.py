"""Misaligned and overlapping arguments of the paged cache operators, refused before a device is asked (no GPU needed)."""
from __future__ import annotations

import pytest

from test_paged_args import pages, query, refused, rows


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import build
    build.build()
    from voxcpm2_b200 import runtime
    runtime.lib()
    return runtime


@pytest.mark.parametrize("off", [1, 2, 3])
def test_lists_of_the_page_calls(rt, off):
    p, at, bad = pages(rt), 4096, 4096 + off
    for call in (lambda: rt.pages_extend(p, bad, 4, at, at), lambda: rt.pages_extend(p, at, 4, bad, at),
                 lambda: rt.pages_extend(p, at, 4, at, bad), lambda: rt.pages_free(p, bad), lambda: rt.pages_fork(p, bad),
                 lambda: rt.pages_compact(p, bad)):
        refused(rt, call, "misaligned")


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("field", ["row_seq", "row_pos", "status"])
def test_lists_of_the_rows(rt, field, off):
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, **{field: 32768 + off}), pages(rt)), "boundaries")
    if field != "status":
        refused(rt, lambda: rt.sparse_attention(query(rt, **{field: 32768 + off}), pages(rt)), "boundaries")


@pytest.mark.parametrize("stride", [264, 512, 1 << 40])
def test_rows_in_place_of_another_stride(rt, stride):
    """Row r would be written where another row, which may not have been read, stands."""
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, q_out=4096, q_out_stride=stride), pages(rt)), "same strides")
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, q_stride=stride, q_out=4096), pages(rt)), "same strides")
    free = dict(k_out=8192, k_out_stride=stride)
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, **free), None), "same strides")
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, q_out=4096, q_out_stride=stride, **free), None), "same strides")


def test_no_device_is_an_error_of_every_call(rt):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    p = pages(rt)
    for call in (lambda: rt.pages_extend(p, 4096, 4, 4096, 4096), lambda: rt.pages_free(p, 4096), lambda: rt.pages_fork(p, 4096),
                 lambda: rt.pages_compact(p), lambda: rt.pages_compact(p, 4096),
                 lambda: rt.qk_norm_rope(rows(rt), p),
                 lambda: rt.qk_norm_rope(rows(rt, k_out=8192, k_out_stride=128), None),
                 lambda: rt.sparse_attention(query(rt), p)):
        with pytest.raises(rt.VxcError) as e:
            call()
        assert e.value.status == 5
