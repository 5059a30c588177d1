"""What the paged cache operators refuse before they touch a device (no GPU needed)."""
from __future__ import annotations

import pytest


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import build
    build.build()
    from voxcpm2_b200 import runtime
    runtime.lib()
    return runtime


def pages(rt, **change):
    f = dict(dtype=rt.DTYPES["f16"], layers=2, n_pages=10, kv_heads=2, page_size=16, head_dim=64, n_seqs=3, max_pages=5,
             k=4096, v=8192, bounds=12288, table=16384, lens=20480, refs=24576, status=28672, work=32768)
    return rt.Pages(**{**f, **change})


def rows(rt, **change):
    f = dict(dtype=rt.DTYPES["f16"], rows=4, q_heads=4, kv_heads=2, head_dim=64, q=4096, k=8192, v=12288, q_out=16384,
             q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, q_gain=20480, k_gain=20480, cos=24576,
             sin=28672, positions=80, eps=1e-5, row_seq=32768, row_pos=36864, status=40960)
    return rt.QkRows(**{**f, **change})


def query(rt, **change):
    f = dict(rows=4, q_heads=4, q=4096, out=8192, q_stride=256, out_stride=256, row_seq=12288, row_pos=16384, scale=0.0,
             top_pages=4, sink_pages=1, local_pages=1)
    return rt.SparseQuery(**{**f, **change})


def refused(rt, call, *words):
    with pytest.raises(rt.VxcError) as e:
        call()
    assert e.value.status == 1, e.value
    for w in words:
        assert w in str(e.value)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(layers=0), "layers"), (dict(n_pages=0), "n_pages"),
    (dict(n_pages=(1 << 20) + 1), "n_pages"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=257), "kv_heads"),
    (dict(page_size=48), "page_size"), (dict(page_size=0), "page_size"), (dict(head_dim=96), "head_dim"),
    (dict(n_seqs=0), "n_seqs"), (dict(n_seqs=4097), "n_seqs"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=16385), "max_pages"),
])
def test_cache_sizes(rt, change, word):
    p = pages(rt, **change)
    refused(rt, lambda: rt.pages_work_ints(p), word)
    refused(rt, lambda: rt.pages_extend(p, 4096, 4, 4096, 4096), word)
    refused(rt, lambda: rt.pages_free(p, 4096), word)
    refused(rt, lambda: rt.pages_fork(p, 4096), word)
    refused(rt, lambda: rt.pages_compact(p), word)
    refused(rt, lambda: rt.sparse_attention(query(rt), p), word)
    if "dtype" not in change and "head_dim" not in change and "kv_heads" not in change:
        refused(rt, lambda: rt.qk_norm_rope(rows(rt), p), word)


def test_work_ints(rt):
    assert rt.pages_work_ints(pages(rt)) >= 3 * 10 + 3 + 1
    assert rt.pages_work_ints(pages(rt, k=None, work=None)) == rt.pages_work_ints(pages(rt))  # before there are arrays


@pytest.mark.parametrize("field", ["k", "v", "bounds", "table", "lens", "refs", "status", "work"])
def test_cache_arrays(rt, field):
    refused(rt, lambda: rt.pages_free(pages(rt, **{field: None}), 4096), "null")
    off = 2 if field in ("table", "lens", "status") else 8
    refused(rt, lambda: rt.pages_free(pages(rt, **{field: 4096 + off}), 4096), "align" if off == 2 else "16-byte")
    if field in "kv":
        refused(rt, lambda: rt.pages_free(pages(rt, **{field: 4096 + 16}), 4096), "32-byte")


def test_null_arguments(rt):
    L = rt.lib()
    p = pages(rt)
    assert L.vxc_pages_work_ints(None) == 0
    assert L.vxc_pages_extend(None, 4096, 1, 4096, 4096, None) == 1
    assert L.vxc_pages_extend(p, None, 1, 4096, 4096, None) == 1
    assert L.vxc_pages_extend(p, 4096, 1, None, 4096, None) == 1
    assert L.vxc_pages_extend(p, 4096, 1, 4096, None, None) == 1
    assert L.vxc_pages_extend(p, 4096, 0, 4096, 4096, None) == 1
    assert L.vxc_pages_extend(p, 4096, (1 << 30) + 1, 4096, 4096, None) == 1
    assert L.vxc_pages_free(p, None, None) == 1 and L.vxc_pages_free(None, 4096, None) == 1
    assert L.vxc_pages_fork(p, None, 1, None) == 1 and L.vxc_pages_fork(None, 4096, 1, None) == 1
    assert L.vxc_pages_compact(None, None, None) == 1
    assert L.vxc_qk_norm_rope(None, p, 0, None) == 1
    assert L.vxc_sparse_attention(None, p, 0, None) == 1 and L.vxc_sparse_attention(query(rt), None, 0, None) == 1


@pytest.mark.parametrize("change,word", [
    (dict(dtype=7), "dtype"), (dict(rows=0), "rows"), (dict(q_heads=0), "q_heads"), (dict(q_heads=1025), "q_heads"),
    (dict(kv_heads=0), "kv_heads"), (dict(head_dim=80), "head_dim"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(q_out=None), "null"), (dict(row_pos=None), "null"), (dict(row_seq=None), "null"),
    (dict(status=None), "null"), (dict(sin=None), "together"), (dict(positions=0), "positions"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q=4104), "16-byte"), (dict(v=4104), "v must"), (dict(k_gain=4104), "16-byte"),
    (dict(cos=4104), "16-byte"), (dict(q_stride=255), "stride"), (dict(q_stride=260), "stride"),
    (dict(k_stride=120), "stride"), (dict(v_stride=132), "v must"), (dict(q_out_stride=248), "stride"),
    (dict(dtype=0), "differ"), (dict(kv_heads=1), "differ"),
    (dict(head_dim=128, q_stride=512, q_out_stride=512, k_stride=256, v_stride=256), "differ"),
])
def test_qk_rows(rt, change, word):
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, **change), pages(rt)), word)


def test_qk_rows_layer_and_no_cache(rt):
    refused(rt, lambda: rt.qk_norm_rope(rows(rt), pages(rt), 2), "layer")
    refused(rt, lambda: rt.qk_norm_rope(rows(rt), pages(rt), -1), "layer")
    refused(rt, lambda: rt.qk_norm_rope(rows(rt), None), "null")  # no k_out
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, k_out=4096, k_out_stride=100), None), "k_out")
    refused(rt, lambda: rt.qk_norm_rope(rows(rt, k_out=4104, k_out_stride=128), None), "k_out")


@pytest.mark.parametrize("change,word", [
    (dict(rows=0), "rows"), (dict(q_heads=5), "q_heads"), (dict(q_heads=34), "q_heads"), (dict(q_heads=0), "q_heads"),
    (dict(top_pages=0), "top_pages"), (dict(top_pages=257), "top_pages"), (dict(local_pages=0), "local_pages"),
    (dict(sink_pages=-1), "sink_pages"), (dict(sink_pages=4), "sink_pages"), (dict(local_pages=4), "sink_pages"),
    (dict(local_pages=2 ** 31 - 1), "sink_pages"), (dict(scale=-0.5), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(row_seq=None), "null"),
    (dict(row_pos=None), "null"), (dict(q=4100), "16-byte"), (dict(out=4100), "16-byte"), (dict(selected=4097), "16-byte"),
    (dict(q_stride=248), "stride"), (dict(out_stride=252), "stride"), (dict(rows=2 ** 31 - 1), "rows"),
])
def test_sparse_query(rt, change, word):
    refused(rt, lambda: rt.sparse_attention(query(rt, **change), pages(rt)), word)


def test_sparse_query_layer(rt):
    refused(rt, lambda: rt.sparse_attention(query(rt), pages(rt), 2), "layer")
    refused(rt, lambda: rt.sparse_attention(query(rt), pages(rt), -1), "layer")


def test_no_device_is_an_error(rt):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    for call in (lambda: rt.pages_free(pages(rt), 4096), lambda: rt.qk_norm_rope(rows(rt), pages(rt)),
                 lambda: rt.sparse_attention(query(rt), pages(rt))):
        with pytest.raises(rt.VxcError) as e:
            call()
        assert e.value.status == 5
