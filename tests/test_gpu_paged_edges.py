"""The paged cache operators at their edges: values that are not finite, calls that fail as a whole, rows in bulk."""
from __future__ import annotations

import math
import random

import pytest

torch = pytest.importorskip("torch")

from paged_model import DTYPES, Cache, attend, choose, norm_rope  # noqa: E402
from test_gpu_paged import ask, close, gen, half_ulp, rows_of, tables  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import runtime
    return runtime


def unchanged(before, c):
    return all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(before, c.state()))


# ------------------------------------------------------------------ values that are not finite
def held_with_infinities(c, q, seq, pos, out):
    """Rows that see all their pages: NaN and infinities where the 64-bit softmax has them, the rest within the bound
    of finite values (scores off by 2^-20 of their terms' sum, weights by twice that and 2^-16, one rounding)."""
    G, dt = q.shape[1] // c.kv_heads, q.dtype
    for r, (s, n) in enumerate(zip(seq.tolist(), pos.tolist())):
        k, v = c.history(0, s, n + 1)
        for h in range(c.kv_heads):
            want, _ = attend(q[r, h * G:(h + 1) * G].double().cpu(), k[h], v[h], 1 / math.sqrt(c.dim))
            _, terms = attend(q[r, h * G:(h + 1) * G].double().cpu(), k[h].nan_to_num(0, 0, 0), v[h], 1 / math.sqrt(c.dim))
            got = out[r, h * G:(h + 1) * G].double().cpu()
            fin = want.isfinite()
            assert torch.equal(got.isnan(), want.isnan()), (r, h)
            assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), (r, h)
            bound = 2 * (2.0 ** -20 * (terms + 4) + (0 if dt == torch.float32 else 2.0 ** -16)) * float(
                v[h].nan_to_num(0, 0, 0).abs().max())
            err = (got - want)[fin].abs() - half_ulp(dt) * want[fin].abs() * 1.01
            assert bool((err <= bound).all()), (r, h, float(err.max()), bound)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,G", [(64, 2, 8), (128, 1, 16), (64, 1, 1), (128, 3, 5)])
@pytest.mark.parametrize("rows", [2, 400])
def test_infinite_values(rt, dtype, dim, kv_heads, G, rows):
    """Infinities among the values make their element of the output infinite, both signs not a number; the other
    elements, heads and sequences are as without them, and infinities past a row's end do not count."""
    g = gen(dim + G)
    c = Cache(rt, dtype, 1, 90, kv_heads, 16, dim, 2, 40)
    c.fill_random([16 * 37 - 3, 16 * 37 - 3], g)
    q = torch.randn(2, kv_heads * G, dim, generator=g).to(DTYPES[dtype]).cuda()
    where = random.Random(dim)

    def put(s, t, h, d, x):
        c.v[0, c.table[s, t // 16].long(), h, t % 16, d] = x

    for t in where.sample(range(500), 9):
        put(0, t, kv_heads - 1, 3, math.inf)       # many of one sign
    put(0, 0, 0, 7, -math.inf)                     # the first key
    put(0, 588, 0, dim - 1, math.inf)              # the row's own
    put(0, 17, 0, 20, math.inf)                    # both signs
    put(0, 333, 0, 20, -math.inf)
    put(0, 40, 0, 21, math.nan)                    # and one that is none
    put(0, 400, 0, 21, math.inf)
    k, _ = c.history(0, 0, 589)
    best = int((q[0, 0].double().cpu() @ k[0].T).argmax())
    put(0, best, 0, 30, math.inf)                  # the key of the largest weight
    put(1, 580, 0, 9, math.inf)                    # past the second row's end
    many = q[torch.arange(rows) % 2].contiguous()
    seq, pos = c.ints([i % 2 for i in range(rows)]), c.ints([588 if i % 2 == 0 else 570 for i in range(rows)])
    out, _ = ask(rt, c, many, seq, pos, 40, 1, 1)
    assert c.status.tolist() == [0]
    held_with_infinities(c, many[:2], seq[:2], pos[:2], out[:2])
    assert bool(out[1].isfinite().all())
    assert all(torch.equal(out[i].nan_to_num(9), out[i % 2].nan_to_num(9)) for i in range(rows))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 400])
def test_infinite_values_of_little_weight(rt, dtype, rows):
    """A weight of e^-200 is below what 32 bits hold and still positive; one of a score of -infinity is none, and
    none times infinity is not a number."""
    c = Cache(rt, dtype, 1, 20, 1, 16, 64, 1, 20)
    c.fill_random([320], gen(3), spread=0.0)
    first, last = c.table[0, 0].long(), c.table[0, 19].long()
    c.k[0, first, 0, 2, 0], c.v[0, first, 0, 2, 5] = -200.0, math.inf
    c.k[0, last, 0, 3, 0], c.v[0, last, 0, 3, 6] = -200.0, -math.inf
    c.k[0, first, 0, 9, 0], c.v[0, first, 0, 9, 7] = -math.inf, math.inf
    c.k[0, last, 0, 9, 0] = -math.inf                                      # counts for nothing
    c.bounds[0, first, 0, 0, 0] = c.bounds[0, last, 0, 0, 0] = -math.inf
    q = torch.randn(1, 4, 64, generator=gen(4))
    q[:, :, 0] = 8.0
    q = q.to(DTYPES[dtype]).cuda().expand(rows, 4, 64).contiguous()
    seq, pos = c.ints([0] * rows), c.ints([319] * rows)
    out, _ = ask(rt, c, q, seq, pos, 20, 1, 1)
    held_with_infinities(c, q[:1], seq[:1], pos[:1], out[:1])
    assert bool((out[:, :, 5] == math.inf).all() and (out[:, :, 6] == -math.inf).all() and out[:, :, 7].isnan().all())
    assert bool(out[:, :, :5].isfinite().all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,dim,page", [(1, 64, 16), (8, 128, 16), (16, 64, 16), (5, 64, 128)])
@pytest.mark.parametrize("rows,n", [(1, 60), (1, 400), (340, 100), (340, 400), (340, 700)])
def test_infinite_bounds(rt, dtype, G, dim, page, rows, n):
    """Bounds that are infinite on the side that no query of the KV head looks at do not change a page's score; on
    the other side they decide it, and a zero in a query makes them not a number."""
    if page * n > 30000:
        pytest.skip("the same scores as with small pages")
    g = gen(n + G)
    c = Cache(rt, dtype, 1, n, 1, page, dim, 1, n)
    c.fill_random([page * n], g)
    q = torch.randn(1, G, dim, generator=g)
    q[:, :, 0], q[:, :, 1] = q[:, :, 0].abs() + 0.1, -q[:, :, 1].abs() - 0.1
    q[:, 0, 2] = 0.0
    q[:, 1:, 2] = -q[:, 1:, 2].abs() - 0.1
    q = q.to(DTYPES[dtype])
    low, high = c.bounds[0, :, 0, 0], c.bounds[0, :, 0, 1]
    page_of = lambda j: c.table[0, j].long()  # noqa: E731
    some = random.Random(G).sample(range(1, n - 1), 30)
    for j in some[:12]:
        low[page_of(j), 0] = -math.inf       # queries there are positive
        high[page_of(j), 1] = math.inf       # and negative
    low[page_of(some[12]), 1] = -math.inf    # score +infinity
    high[page_of(some[13]), 0] = math.inf
    low[page_of(some[14]), 0] = high[page_of(some[14]), 0] = -math.inf  # score -infinity
    low[page_of(some[15]), 2] = -math.inf    # zero times infinity
    high[page_of(some[16]), 2] = math.inf
    low[page_of(some[17]), 0] = high[page_of(some[17]), 0] = -math.inf  # both infinities
    low[page_of(some[17]), 1] = -math.inf
    high[page_of(some[18]), 1] = math.nan    # not a number, on either side
    seen = c.table[0, :n].long()
    b = c.bounds[0, seen, 0].double().cpu()
    for top in (20, 45):
        want = choose(q[0].double(), b[:, 0], b[:, 1], n, top, 1, 1)
        assert {some[12], some[13], some[15], some[16], some[17], some[18]} <= set(want)
        _, sel = ask(rt, c, q.cuda().expand(rows, G, dim).contiguous(), c.ints([0] * rows), c.ints([page * n - 1] * rows), top, 1, 1)
        assert c.status.tolist() == [0]
        assert sel[0, 0].tolist() == want
        assert torch.equal(sel, sel[:1].expand_as(sel))


@pytest.mark.parametrize("rows", [1, 400])
def test_sixteen_heads_that_round_alike(rt, rows):
    """Sums of 16 heads whose 15 roundings all go one way, up in half of the dimensions and down in the others, and
    bounds that turn every rounding of a plain fp32 sum the same way: page 3 beats page 1 by 2^-19 of what one dimension
    adds to a score, and plain sums have it the other way round by 2304 / 2^24."""
    steps = [12, 10, 59, 31, 46, 20, 0, 33, 20, 36, 43, 5, 43, 6, 11, 7, 35, 30, 8, 39, 46, 20, 0, 33, 36, 44, 23, 9, 9,
             36, 0, 46, 50, 12, 29, 13, 9, 36, 0, 46, 36, 44, 23, 9, 9, 62, 56, 12, 3, 20, 14, 3, 38, 28, 59, 22, 10, 31,
             25, 46, 27, 28, 15, 13]
    c = Cache(rt, "f32", 1, 6, 1, 16, 64, 1, 6)
    c.fill_random([96], gen(1))
    up = (torch.arange(64) // 4) % 2 == 0
    edge = (1 + torch.tensor(steps, dtype=torch.float64) * 2.0 ** -23) * torch.where(up, 1.0, -1.0)
    low, high = c.bounds[0, :, 0, 0], c.bounds[0, :, 0, 1]
    high[:], low[:] = -0.5, -1.0
    for page, sign in ((1, 1), (3, -1)):
        high[c.table[0, page].long()] = (sign * edge).float().cuda()
        low[c.table[0, page].long()] = -2.0
    q = torch.where(up, 2.0 ** -24 * 1.0001, 2.0 ** -24 * 0.9999).expand(1, 16, 64).clone()
    q[0, 0] = 1.0
    b = c.bounds[0, c.table[0, :6].long(), 0].double().cpu()
    assert choose(q[0].double(), b[:, 0], b[:, 1], 6, 2, 0, 1) == [3, 5]
    _, sel = ask(rt, c, q.cuda().expand(rows, 16, 64).contiguous(), c.ints([0] * rows), c.ints([95] * rows), 2, 0, 1)
    assert all(s == [3, 5] for s in sel[:, 0].tolist())


# ------------------------------------------------------------------ calls that fail as a whole
@pytest.mark.parametrize("length", [-1, 3 * 16 + 1])
def test_compact_with_a_bad_length_changes_nothing(rt, length):
    c = Cache(rt, n_pages=9, n_seqs=3, max_pages=3)
    c.extend([20, 40, 17])
    c.free([1, 0, 0])
    good = c.lens.clone()
    c.lens[2] = length
    before = c.state()
    used = c.compact()
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and used.tolist() == [-5]
    assert unchanged(before, c)
    c.status.zero_()
    c.lens.copy_(good)
    assert c.compact().tolist() == [5] and c.status.tolist() == [0]
    assert sorted(c.table[c.table >= 0].tolist()) == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("column,bad", [(0, -1), (1, 40), (2, 2 ** 31 - 1), (2, -2 ** 31), (2, 40)])
def test_fork_of_a_bad_table_changes_nothing(rt, share, column, bad):
    """Parents with a page outside the pool, a full one or the last: no child is made, theirs or another's."""
    c = Cache(rt, n_pages=40, n_seqs=6, max_pages=5)
    c.extend([40, 33, 0, 0, 0, 0])
    good = c.table.clone()
    c.table[0, column] = bad
    before = c.state()
    c.fork([-1, -1, 1, 0, 0, -1], share)
    assert c.status.tolist() == [rt.PAGES_BAD_ID]
    assert unchanged(before, c)
    c.status.zero_()
    c.fork([-1, -1, 1, -1, -1, 1], share)  # nothing of the other parent is looked at
    assert c.status.tolist() == [0] and c.lens.tolist() == [40, 33, 33, 0, 0, 33]
    c.table[0] = good[0]
    c.fork([-1, -1, -1, 0, 0, -1], share)
    assert c.status.tolist() == [0] and c.lens.tolist() == [40, 33, 33, 40, 40, 33]


def test_fork_does_not_look_past_a_parents_end(rt):
    c = Cache(rt, n_pages=20, n_seqs=4, max_pages=5)
    c.extend([32, 0, 0, 0])
    c.table[0, 2:] = 99
    c.fork([-1, 0, 1 << 20, -1])
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and c.lens.tolist() == [32, 0, 0, 0]
    c.status.zero_()
    c.fork([-1, 0, -1, 0])
    assert c.status.tolist() == [0] and c.lens.tolist() == [32, 32, 0, 32]


def test_free_leaves_a_sequence_of_bad_length(rt):
    c = Cache(rt, n_pages=20, n_seqs=4, max_pages=3)
    c.extend([20, 33, 40, 5])
    rows, refs = c.table.clone(), c.refs.clone()
    c.lens[1], c.lens[2] = 49, -3
    c.free([1, 1, 1, 0])
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and c.lens.tolist() == [0, 49, -3, 5]
    assert c.table[0].tolist() == [-1] * 3 and torch.equal(c.table[1:], rows[1:])
    gone = rows[0, :2].long()
    assert c.refs[gone].tolist() == [0, 0] and int(c.refs.sum()) == int(refs.sum()) - 2


# ------------------------------------------------------------------ rows in bulk
def bulk(dtype, dim):
    """Query heads and rows beyond the one-launch form (8 CTAs an SM of 256 threads, 16 bytes a thread)."""
    slots = 256 * 16 // (dim * DTYPES[dtype].itemsize)
    rows = 1300
    limit = 8 * torch.cuda.get_device_properties(0).multi_processor_count * slots
    heads = limit // rows + 1
    while heads % 4 != 3:
        heads += 1
    assert heads * rows > limit
    return heads, rows


def row_lists(rng, n_seqs, rows, page, past):
    """Prompts of n_seqs sequences, rows of nobody before, between and behind them."""
    seq, pos = [-1] * 2, [7] * 2
    left = rows - 2
    for s in range(n_seqs):
        n = left // (n_seqs - s) - rng.randint(3, 9)
        seq += [s] * n + [-4] * 3
        pos += list(range(past[s], past[s] + n)) + [-1, 0, 1 << 30]
        left -= n + 3
    assert left >= 0
    return seq + [-1] * left, pos + [-1] * left


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,page", [(64, 3, 16), (128, 1, 64), (64, 2, 128), (128, 5, 32)])
@pytest.mark.parametrize("norm,turn,interleaved,in_place", [("qk", True, False, False), ("k", True, True, True), ("q", False, False, False),
                                                            ("", True, False, True)])
def test_rows_in_bulk_into_the_cache(rt, dtype, dim, kv_heads, page, norm, turn, interleaved, in_place):
    g, rng = gen(dim + kv_heads), random.Random(page)
    heads, R = bulk(dtype, dim)
    n, past = 3, [5, 0, page + 1]
    each = -(-(R // n + 30) // page) + 4
    c = Cache(rt, dtype, 2, n * each + 4, kv_heads, page, dim, n, each)
    c.fill_random(past, g)
    before_keys = [c.history(1, s, past[s]) for s in range(n)]
    seq, pos = row_lists(rng, n, R, page, past)
    count = [seq.count(s) for s in range(n)]
    c.extend(count)
    cos, sin = (t.cuda() for t in tables(each * page, dim)) if turn else (None, None)
    gain = [(torch.randn(dim, generator=g) * 0.3 + 1).to(DTYPES[dtype]).cuda() if x in norm else None for x in "qk"]
    x = torch.randn(R, heads + 2 * kv_heads + 1, dim, generator=g).mul_(1.5).to(DTYPES[dtype])
    qkv = x.cuda()[:, :-1]
    x = x[:, :-1]
    out = qkv[:, :heads] if in_place else torch.full((R, heads, dim), 5.0, dtype=DTYPES[dtype], device="cuda")
    before = c.state()
    dseq, dpos = c.ints(seq), c.ints(pos)
    rt.qk_norm_rope(rows_of(rt, c, dtype, qkv, heads, kv_heads, dseq, dpos, out, cos, sin, gain, interleaved=int(interleaved)),
                    c.p, 1, c.stream())
    assert c.status.tolist() == [0]
    sq, ps = torch.tensor(seq), torch.tensor(pos)
    live = sq >= 0
    cpu = [None if t is None else t.cpu() for t in (*gain, cos, sin)]
    size = lambda part, gain: norm_rope(part, gain, None, None, None, 1e-5, False).norm(dim=-1, keepdim=True)  # noqa: E731
    xq, xk, xv = x[live][:, :heads], x[live][:, heads:heads + kv_heads], x[live][:, heads + kv_heads:]
    want = norm_rope(xq, cpu[0], cpu[2], cpu[3], ps[live], 1e-5, interleaved)
    close(out.cpu()[live], want, DTYPES[dtype], size(xq, cpu[0]))
    idle = x[~live][:, :heads] if in_place else torch.full_like(x[~live][:, :heads], 5.0)
    assert torch.equal(out.cpu()[~live], idle)
    assert torch.equal(qkv[:, heads:].cpu(), x[:, heads:])
    k = norm_rope(xk, cpu[1], cpu[2], cpu[3], ps[live], 1e-5, interleaved)
    for s in range(n):
        mine = sq[live] == s
        total = past[s] + count[s]
        got_k, got_v = c.history(1, s, total)
        assert torch.equal(got_k[:, :past[s]], before_keys[s][0]) and torch.equal(got_v[:, :past[s]], before_keys[s][1])
        want_k = k[mine].transpose(0, 1)
        close(got_k[:, past[s]:], want_k, DTYPES[dtype], size(xk, cpu[1])[mine].transpose(0, 1))
        assert torch.equal(got_v[:, past[s]:], xv[mine].double().transpose(0, 1))
        ids = c.table[s, :-(-total // page)].long()
        b = c.bounds[1, ids].double().cpu()
        for j in range(len(ids)):
            part = got_k[:, j * page:(j + 1) * page]
            assert torch.equal(b[j, :, 0], part.amin(1)) and torch.equal(b[j, :, 1], part.amax(1)), (s, j)
    for i in range(3):
        assert torch.equal(before[i][0].nan_to_num(9), c.state()[i][0].nan_to_num(9))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads", [(64, 3), (128, 6)])
@pytest.mark.parametrize("norm,turn,interleaved,in_place", [("qk", True, False, True), ("q", True, True, False), ("k", False, False, True)])
def test_rows_in_bulk_without_a_cache(rt, dtype, dim, kv_heads, norm, turn, interleaved, in_place):
    g = gen(dim + kv_heads + 1)
    heads, R = bulk(dtype, dim)
    c = Cache(rt, dtype)
    cos, sin = (t.cuda() for t in tables(900, dim)) if turn else (None, None)
    gain = [(torch.rand(dim, generator=g) + 0.5).to(DTYPES[dtype]).cuda() if x in norm else None for x in "qk"]
    x = torch.randn(R, heads + 2 * kv_heads, dim, generator=g).to(DTYPES[dtype])
    qkv = x.cuda()
    seq = torch.randint(-1, 3, (R,), generator=g)
    pos = torch.randint(0, 900, (R,), generator=g)
    pos[seq < 0] = -5
    live = seq >= 0
    dseq, dpos = seq.int().cuda(), pos.int().cuda()
    make = lambda n: torch.full((R, n, dim), 5.0, dtype=DTYPES[dtype], device="cuda")  # noqa: E731
    out, k_out = (qkv[:, :heads], qkv[:, heads:heads + kv_heads]) if in_place else (make(heads), make(kv_heads))
    rt.qk_norm_rope(rows_of(rt, c, dtype, qkv, heads, kv_heads, dseq, dpos, out, cos, sin, gain, interleaved=int(interleaved),
                            k_out=k_out.data_ptr(), k_out_stride=k_out.stride(0)), None, 0, c.stream())
    assert c.status.tolist() == [0]
    for got, part, gn in ((out, x[:, :heads], gain[0]), (k_out, x[:, heads:heads + kv_heads], gain[1])):
        gn = None if gn is None else gn.cpu()
        want = norm_rope(part[live], gn, *(None if t is None else t.cpu() for t in (cos, sin)), pos[live], 1e-5, interleaved)
        size = norm_rope(part[live], gn, None, None, None, 1e-5, False).norm(dim=-1, keepdim=True)
        close(got.cpu()[live], want, DTYPES[dtype], size)
        assert torch.equal(got.cpu()[~live], part[~live] if in_place else torch.full_like(part[~live], 5.0))
    assert torch.equal(qkv[:, heads + kv_heads:].cpu(), x[:, heads + kv_heads:])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("captured", [False, True])
def test_bulk_rows_written_just_before(rt, dtype, captured):
    """Rows, their places and the gains are written by the kernels right before the call, and the attention reads its
    outputs right after it: chunk after chunk of a prompt with nothing waited for in between."""
    dim, kv_heads, page, chunks = 64, 2, 64, 6
    heads, R = bulk(dtype, dim)
    heads += -heads % kv_heads
    c = Cache(rt, dtype, 1, chunks * (R // page + 2) + 2, kv_heads, page, dim, 1, chunks * (R // page + 2))
    g = gen(17)
    cos, sin = (t.cuda() for t in tables(chunks * R, dim))
    x = torch.randn(chunks, R, heads + 2 * kv_heads, dim, generator=g).to(DTYPES[dtype])
    gain = (torch.rand(chunks, dim, generator=g) + 0.5).to(DTYPES[dtype])
    dx, dgain, counts = x.cuda(), gain.cuda(), c.ints([R])
    qkv, now = torch.zeros_like(dx[0]), torch.zeros_like(dgain[0])
    q = qkv[:, :heads]
    seq, pos = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2))
    some = 3  # query heads of a KV head that attend
    out = torch.zeros(R, kv_heads * some, dim, dtype=DTYPES[dtype], device="cuda")
    a = rt.SparseQuery(rows=R, q_heads=kv_heads * some, q=q.data_ptr(), q_stride=q.stride(0), out=out.data_ptr(),
                       out_stride=out.stride(0), row_seq=seq.data_ptr(), row_pos=pos.data_ptr(), top_pages=4, sink_pages=1,
                       local_pages=3)
    rows = rows_of(rt, c, dtype, qkv, heads, kv_heads, seq, pos, q, cos, sin, (now, now))

    def step():
        s = torch.cuda.current_stream().cuda_stream
        rt.pages_extend(c.p, counts.data_ptr(), R, seq.data_ptr(), pos.data_ptr(), s)
        rt.qk_norm_rope(rows, c.p, 0, s)
        rt.sparse_attention(a, c.p, 0, s)

    counts.zero_()
    step()  # rows of nobody
    counts.fill_(R)
    run = step
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        run = graph.replay
    got = []
    for i in range(chunks):
        qkv.mul_(0).add_(dx[i])
        now.mul_(0).add_(dgain[i])
        run()
        got.append((q.clone(), out.clone()))
    assert c.status.tolist() == [0] and c.lens.tolist() == [chunks * R]
    keys, values = c.history(0, 0, chunks * R)
    cs = [t.cpu() for t in (cos, sin)]
    for i in range(chunks):
        p = torch.arange(i * R, (i + 1) * R)
        part = x[i][:, :heads]
        size = norm_rope(part, gain[i], None, None, None, 1e-5, False).norm(dim=-1, keepdim=True)
        close(got[i][0].cpu(), norm_rope(part, gain[i], *cs, p, 1e-5, False), DTYPES[dtype], size)
        part = x[i][:, heads:heads + kv_heads]
        size = norm_rope(part, gain[i], None, None, None, 1e-5, False).norm(dim=-1, keepdim=True).transpose(0, 1)
        close(keys[:, p], norm_rope(part, gain[i], *cs, p, 1e-5, False).transpose(0, 1), DTYPES[dtype], size)
        assert torch.equal(values[:, p], x[i][:, heads + kv_heads:].double().transpose(0, 1))
        for r in (0, 77, R - 1):  # top pages 1 + 3: the first and the last ones
            t = i * R + r
            seen = t // page + 1
            pages = range(seen) if seen <= 4 else [0, seen - 3, seen - 2, seen - 1]
            at = [j for b in pages for j in range(b * page, min(b * page + page, t + 1))]
            for h in range(kv_heads):
                hq = got[i][0][r, h * some:(h + 1) * some].double().cpu()
                want, terms = attend(hq, keys[h, at], values[h, at], 1 / math.sqrt(dim))
                bound = 2 * (2.0 ** -20 * (terms + 4) + (0 if dtype == "f32" else 2.0 ** -16)) * float(values[h, at].abs().max())
                err = (got[i][1][r, h * some:(h + 1) * some].double().cpu() - want).abs() - half_ulp(DTYPES[dtype]) * want.abs() * 1.01
                assert bool((err <= bound).all()), (i, r, h)
