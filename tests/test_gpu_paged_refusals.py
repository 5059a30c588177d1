"""Every array of the paged cache operators that is not memory of the current device is refused before anything runs."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

from paged_model import Cache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import runtime
    return runtime


PAGES = ["k", "v", "bounds", "table", "lens", "refs", "status", "work"]
ROWS = ["q", "k", "v", "q_out", "q_gain", "k_gain", "cos", "sin", "row_seq", "row_pos", "status"]
QUERY = ["q", "out", "row_seq", "row_pos", "selected"]


def host(kind):
    """Aligned memory of the host: (owner, address)."""
    t = torch.zeros(1 << 16, dtype=torch.uint8, pin_memory=kind == "pinned")
    return t, (t.data_ptr() + 63) // 64 * 64


def copy_of(s, **change):
    c = type(s).from_buffer_copy(s)
    for name, value in change.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("kind", ["paged", "pinned"])
def test_arrays_of_the_host(rt, kind):
    c = Cache(rt, "f16", n_pages=8, n_seqs=2, max_pages=4)
    dev = torch.zeros(8, 1024, dtype=torch.float16, device="cuda")
    ints = torch.full((5, 64), -1, dtype=torch.int32, device="cuda")
    at = [t.data_ptr() for t in dev] + [t.data_ptr() for t in ints]
    rows = rt.QkRows(dtype=1, rows=2, q_heads=2, kv_heads=2, head_dim=64, q=at[0], k=at[1], v=at[2], q_out=at[3], k_out=at[4],
                     q_stride=128, k_stride=128, v_stride=128, q_out_stride=128, k_out_stride=128, q_gain=at[5], k_gain=at[5],
                     cos=at[6], sin=at[7], positions=1, row_seq=at[8], row_pos=at[9], status=c.status.data_ptr())
    query = rt.SparseQuery(rows=2, q_heads=2, q=at[0], out=at[1], q_stride=128, out_stride=128, row_seq=at[8], row_pos=at[9],
                           top_pages=2, local_pages=1, selected=at[10])
    keep, h = host(kind)
    x, y, z = at[10:13]
    cases = []
    for f in PAGES:
        p = copy_of(c.p, **{f: h})
        cases += [("pages." + f, call) for call in (
            lambda p=p: rt.pages_extend(p, x, 4, y, z), lambda p=p: rt.pages_free(p, x), lambda p=p: rt.pages_fork(p, x),
            lambda p=p: rt.pages_compact(p), lambda p=p: rt.qk_norm_rope(rows, p), lambda p=p: rt.sparse_attention(query, p))]
    cases += [("counts", lambda: rt.pages_extend(c.p, h, 4, y, z)), ("row_seq", lambda: rt.pages_extend(c.p, x, 4, h, z)),
              ("row_pos", lambda: rt.pages_extend(c.p, x, 4, y, h)), ("flags", lambda: rt.pages_free(c.p, h)),
              ("parents", lambda: rt.pages_fork(c.p, h)), ("used", lambda: rt.pages_compact(c.p, h))]
    for f in ROWS:
        r = copy_of(rows, **{f: h})
        cases.append((f, lambda r=r: rt.qk_norm_rope(r, c.p)))
        if f != "v":
            cases.append((f, lambda r=r: rt.qk_norm_rope(r, None)))
    cases.append(("k_out", lambda: rt.qk_norm_rope(copy_of(rows, k_out=h), None)))
    for f in QUERY:
        a = copy_of(query, **{f: h})
        cases.append((f, lambda a=a: rt.sparse_attention(a, c.p)))
    before = [t.clone() for t in (*c.state(), dev, ints, c.status)]
    for name, call in cases:
        with pytest.raises(rt.VxcError) as e:
            call()
        assert e.value.status == 1 and f": {name} is not memory of the current device" in str(e.value), (name, e.value)
    torch.cuda.synchronize()
    assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(before, (*c.state(), dev, ints, c.status)))
    assert not bool(keep.any())


def test_arrays_of_separate_allocations_and_managed_memory(rt):
    """Arrays far apart, each an allocation of its own (more than a call remembers), and managed ones are taken."""
    big = [torch.zeros(24 << 20, dtype=torch.uint8, device="cuda") for _ in range(8)]
    c = Cache(rt, "f16", n_pages=8, n_seqs=2, max_pages=4)
    p = copy_of(c.p)
    for f, t in zip(PAGES, big):
        setattr(p, f, t.data_ptr())
    big[3].view(torch.int32).fill_(-1)
    p.work = c.work.data_ptr()
    counts, seq, pos = c.ints([20, 3]), c.ints([7] * 24), c.ints([7] * 24)
    rt.pages_extend(p, counts.data_ptr(), 24, seq.data_ptr(), pos.data_ptr(), c.stream())
    assert big[6].view(torch.int32)[0].item() == 0 and big[4].view(torch.int32)[:2].tolist() == [20, 3]
    assert seq.tolist() == [0] * 20 + [1] * 3 + [-1]
    cuda = ctypes.CDLL("libcuda.so.1")
    at = ctypes.c_uint64()
    assert cuda.cuMemAllocManaged(ctypes.byref(at), ctypes.c_size_t(4096), 1) == 0
    rt.pages_compact(p, at.value, c.stream())
    torch.cuda.synchronize()
    assert ctypes.c_int32.from_address(at.value).value == 3
    assert cuda.cuMemFree_v2(at) == 0
