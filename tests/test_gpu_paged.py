"""The paged cache operators on the GPU against host tables and 64-bit formulas."""
from __future__ import annotations

import math
import random

import pytest

torch = pytest.importorskip("torch")

from paged_model import DTYPES, Cache, Model, attend, choose, norm_rope  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import runtime
    return runtime


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ pages
def stamp(c, seq, pos, value):
    """Writes one token's keys and values (all layers) as its page holds them: a number of its own."""
    page = c.table[seq.long(), (pos // c.page).long()].long()
    slot = (pos % c.page).long()
    for x, sign in ((c.k, 1), (c.v, -1)):
        x.transpose(2, 3)[:, page, slot] = (sign * value.to(c.k.device))[None, :, None, None].to(c.dtype)


@pytest.mark.parametrize("seed,dtype,page,kv_heads,dim,layers,pool,seqs,most", [
    (1, "f16", 16, 2, 64, 2, 60, 9, 12), (2, "f32", 16, 1, 128, 1, 90, 33, 5), (3, "bf16", 128, 3, 64, 3, 31, 6, 9),
    (4, "f16", 32, 8, 128, 1, 41, 12, 7), (5, "bf16", 64, 1, 64, 1, 9001, 5, 3000),
])
def test_pages_follow_the_tables_of_a_plain_allocator(rt, seed, dtype, page, kv_heads, dim, layers, pool, seqs, most):
    """Random calls in a row: tables, holders and rows equal the host's after each, and every token of every
    sequence is still what was written for it (the host keeps the sequences' contents apart from any page)."""
    rng = random.Random(seed)
    c = Cache(rt, dtype, layers, pool, kv_heads, page, dim, seqs, most)
    m = Model(pool, seqs, most, page)
    content = [[] for _ in range(seqs)]
    tag = 0
    for step in range(30):
        op = rng.choice(["extend", "extend", "fork", "copy", "free", "compact"])
        if op == "extend":
            counts = [rng.choice([0, 0, 1, 1, page, rng.randint(0, 3 * page)]) for _ in range(seqs)]
            counts = [min(n, most * page - len(t)) for n, t in zip(counts, content)]
            if step == 0 and pool > 1000:
                counts[1] = 2900 * page + 1
            room = sum(counts) + rng.choice([0, 1, 40])
            if room == 0:
                continue
            seq, pos = c.extend(counts, room)
            code, rows = m.extend(counts, room)
            assert list(zip(seq.tolist(), pos.tolist())) == rows
            assert c.status.tolist() == [code]
            c.status.zero_()
            if code == 0 and sum(counts):
                # at most 2^11 values, whole numbers in every type's range (bf16 holds 256 of them exactly)
                value = torch.tensor([float((tag + i) % 251) for i in range(sum(counts))], dtype=torch.float32)
                stamp(c, seq[:sum(counts)], pos[:sum(counts)], value)
                for (s, _), x in zip(rows, value.tolist()):
                    content[s].append(x)
                tag += sum(counts)
        elif op in ("fork", "copy"):
            parents = [-1] * seqs
            for d in range(seqs):
                if not m.lens[d] and rng.random() < 0.5:
                    s = rng.randrange(seqs)
                    if s != d and parents[s] < 0 and d not in parents:
                        parents[d] = s
            c.fork(parents, op == "fork")
            code = m.fork(parents, op == "fork")
            assert c.status.tolist() == [code]
            c.status.zero_()
            if code == 0:
                for d, s in enumerate(parents):
                    if s >= 0:
                        content[d] = list(content[s])
        elif op == "free":
            flags = [int(rng.random() < 0.3) for _ in range(seqs)]
            c.free(flags)
            m.free(flags)
            content = [[] if f else t for f, t in zip(flags, content)]
        else:
            used = c.compact()
            assert used.tolist() == [m.compact()]
        assert c.status.tolist() == [0]
        m.check(c)
        for s in range(seqs):
            assert m.lens[s] == len(content[s])
            if content[s]:
                k, v = c.history(layers - 1, s, m.lens[s])
                want = torch.tensor(content[s], dtype=torch.float64)[None, :, None].expand_as(k)
                assert torch.equal(k, want) and torch.equal(v, -want), (step, op, s)


def test_a_full_pool_changes_nothing(rt):
    c = Cache(rt, n_pages=7, n_seqs=3, max_pages=8)
    c.extend([33, 16, 0])  # 3 + 1 pages
    before = c.state()
    seq, pos = c.extend([1, 64, 0], 70)  # 4 more where 3 are free
    assert c.status.tolist() == [rt.PAGES_FULL] and set(seq.tolist()) == set(pos.tolist()) == {-1}
    c.status.zero_()
    c.fork([-1, -1, 0], share=False)  # 3 pages: these fit
    assert c.status.tolist() == [0] and c.lens.tolist() == [33, 16, 33]
    c.free([0, 0, 1])
    c.extend([16 * 2 - 1, 0, 0])  # 1 page left
    c.free([0, 0, 0])
    before = c.state()
    c.fork([-1, -1, 0], share=False)
    assert c.status.tolist() == [rt.PAGES_FULL]
    assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(before, c.state()))


@pytest.mark.parametrize("call", [
    lambda c: c.extend([-1, 0, 0], 4), lambda c: c.extend([5, 0, 0], 4), lambda c: c.extend([0, 81, 0], 100),
    lambda c: c.extend([0, 2 ** 31 - 1, 2 ** 31 - 1], 100), lambda c: c.fork([-1, 0, -1]), lambda c: c.fork([0, -1, -1]),
    lambda c: c.fork([-1, -1, 2]), lambda c: c.fork([-1, -1, 3]), lambda c: c.fork([-1, -1, 2 ** 31 - 1]),
    lambda c: c.fork([2, -1, 1]),
])
def test_bad_counts_and_parents_change_nothing(rt, call):
    c = Cache(rt, n_pages=30, n_seqs=3, max_pages=5)
    c.extend([20, 3, 0])
    before = c.state()
    call(c)
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ]
    assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(before, c.state()))
    c.extend([500, 0, 0], 600)
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ]  # the first code stays, later calls still run
    c.extend([1, 0, 1])
    assert c.lens.tolist() == [21, 3, 1]


def test_tables_with_ids_outside_the_pool_are_reported_and_skipped(rt):
    c = Cache(rt, n_pages=6, n_seqs=3, max_pages=3)
    c.extend([30, 17, 0])
    c.table[0, 1], c.table[1, 0] = 6, -7
    c.compact()
    assert c.status.tolist() == [rt.PAGES_BAD_ID]
    c.status.zero_()
    c.fork([-1, -1, 0], share=True)
    assert c.status.tolist() == [rt.PAGES_BAD_ID]
    c.status.zero_()
    c.free([1, 1, 1])
    assert c.status.tolist() == [rt.PAGES_BAD_ID] and c.lens.tolist() == [0, 0, 0]
    assert int(c.refs.min()) >= 0


def test_a_page_freed_too_often_is_reported(rt):
    c = Cache(rt, n_pages=6, n_seqs=2, max_pages=3)
    c.extend([16, 16])
    c.table[1, 0] = c.table[0, 0]
    c.free([1, 1])
    assert c.status.tolist() == [rt.PAGES_BAD_ID] and int(c.refs.min()) == 0


def test_many_sequences(rt):
    c = Cache(rt, n_pages=9000, n_seqs=4096, max_pages=2, kv_heads=1)
    m = Model(9000, 4096, 2, 16)
    counts = [s % 33 for s in range(4096)]
    seq, pos = c.extend(counts)
    _, rows = m.extend(counts, sum(counts))
    assert list(zip(seq.tolist(), pos.tolist())) == rows
    flags = [int(s % 3 == 0) for s in range(4096)]
    c.free(flags)
    m.free(flags)
    parents = [s + 1 if s % 3 == 0 and s < 4095 else -1 for s in range(4096)]
    c.fork(parents)
    assert m.fork(parents, True) == 0
    m.check(c)
    assert c.status.tolist() == [0]


# ------------------------------------------------------------------ norm and rotation
def tables(n, dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    a = torch.arange(n, dtype=torch.float64)[:, None] * torch.cat([inv, inv])
    return a.cos().float(), a.sin().float()


def rows_of(rt, c, dtype, qkv, heads, kv_heads, seq, pos, q_out, cos=None, sin=None, gains=(None, None), **more):
    """QkRows over a fused [rows, (heads + 2 kv_heads), dim] tensor (any row stride)."""
    dim, size, row = qkv.shape[-1], qkv.element_size(), qkv.stride(0)
    q = qkv.data_ptr()
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return rt.QkRows(dtype=rt.DTYPES[dtype], rows=qkv.shape[0], q_heads=heads, kv_heads=kv_heads, head_dim=dim, q=q,
                     k=q + heads * dim * size, v=q + (heads + kv_heads) * dim * size, q_stride=row, k_stride=row,
                     v_stride=row, q_out=q_out.data_ptr(), q_out_stride=q_out.stride(0), q_gain=ptr(gains[0]),
                     k_gain=ptr(gains[1]), eps=1e-5, cos=ptr(cos), sin=ptr(sin),
                     positions=0 if cos is None else cos.shape[0], row_seq=ptr(seq), row_pos=ptr(pos),
                     status=c.status.data_ptr(), **more)


def close(got, want, dtype, magnitude):
    """Within the one rounding and 24 fp32 ones (sum of squares, rsqrt, gain, two products and their sum) of the
    magnitude that goes into an element."""
    got, want = got.double().cpu(), want.double().cpu()
    err = (got - want).abs()
    bound = half_ulp(dtype) * want.abs() * 1.01 + 24 * 2.0 ** -24 * magnitude + 2.0 ** -25
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 16, 2, 64), (128, 7, 1, 16), (64, 3, 3, 128), (128, 24, 8, 32)])
@pytest.mark.parametrize("norm,turn,interleaved", [(True, True, False), (True, True, True), (False, True, False),
                                                   (True, False, False)])
def test_norm_rope_into_the_cache(rt, dtype, dim, heads, kv_heads, page, norm, turn, interleaved):
    """Prompts, then single tokens and short pieces that end anywhere in a page: q, keys, values and bounds after
    each call; garbage, other sequences, the other layer and the rows of no sequence stay."""
    g = gen(heads * dim + page)
    n, layer, longest = 5, 1, 3 * page + 9
    c = Cache(rt, dtype, 2, 40, kv_heads, page, dim, n, 6)
    cos, sin = (t.cuda() for t in tables(6 * page, dim)) if turn else (None, None)
    gains = [(torch.randn(dim, generator=g) * 0.3 + 1).to(DTYPES[dtype]).cuda() for _ in range(2)] if norm else [None] * 2
    history = [torch.zeros(0, kv_heads, dim, dtype=torch.float64) for _ in range(n)], [
        torch.zeros(0, kv_heads, dim, dtype=torch.float64) for _ in range(n)]
    for counts in ([longest, 1, page, 0, page - 1], [1, 1, 1, 1, 1], [2, page + 1, 0, 33, 1], [1, 0, 1, 1, 0]):
        pad = 3
        seq, pos = c.extend(counts, sum(counts) + pad)
        R = sum(counts) + pad
        wide = torch.randn(R, heads + 2 * kv_heads + 1, dim, generator=g).mul_(1.5).to(DTYPES[dtype]).cuda()
        qkv = wide[:, :-1]  # rows further apart than they are wide
        out = torch.full((R, heads, dim), 5.0, dtype=DTYPES[dtype], device="cuda")
        before = c.state()
        rt.qk_norm_rope(rows_of(rt, c, dtype, qkv, heads, kv_heads, seq, pos, out, cos, sin, gains,
                                interleaved=int(interleaved)), c.p, layer, c.stream())
        assert c.status.tolist() == [0]
        x, sq, ps = qkv.cpu(), seq.cpu().long(), pos.cpu().long()
        live = sq >= 0
        cpu = [None if t is None else t.cpu() for t in (*gains, cos, sin)]
        size = lambda part, gain: norm_rope(part[live], gain, None, None, None, 1e-5, False).norm(dim=-1, keepdim=True)  # noqa: E731
        want = norm_rope(x[live][:, :heads], cpu[0], cpu[2], cpu[3], ps[live], 1e-5, interleaved)
        close(out.cpu()[live], want, DTYPES[dtype], size(x[:, :heads], cpu[0]))
        assert bool((out.cpu()[~live] == 5.0).all())
        k = norm_rope(x[live][:, heads:heads + kv_heads], cpu[1], cpu[2], cpu[3], ps[live], 1e-5, interleaved)
        for s in range(n):
            mine = sq[live] == s
            history[0][s] = torch.cat([history[0][s], k[mine]])
            history[1][s] = torch.cat([history[1][s], x[live][:, heads + kv_heads:][mine].double()])
            if not len(history[0][s]):
                continue
            got_k, got_v = c.history(layer, s, len(history[0][s]))
            want_k = history[0][s].transpose(0, 1)
            close(got_k, want_k, DTYPES[dtype], want_k.norm(dim=-1, keepdim=True))
            assert torch.equal(got_v, history[1][s].transpose(0, 1))
            for j in range(-(-len(history[0][s]) // page)):
                part = got_k[:, j * page:(j + 1) * page]
                b = c.bounds[layer, c.table[s, j].long()].double().cpu()
                assert torch.equal(b[:, 0], part.amin(1)) and torch.equal(b[:, 1], part.amax(1)), (s, j)
        after = c.state()
        for i in range(3):
            assert torch.equal(before[i][0].nan_to_num(9), after[i][0].nan_to_num(9))
        # nothing but the new tokens' cells has changed
        cells = torch.zeros(c.n_pages, page, dtype=torch.bool, device="cuda")
        cells[c.table[seq[:-pad].long(), (pos[:-pad] // page).long()].long(), (pos[:-pad] % page).long()] = True
        for i in range(2):
            a, b = (t[i][layer].transpose(1, 2)[~cells].nan_to_num(9) for t in (before, after))
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim,in_place,gains", [(1, 64, False, "qk"), (77, 128, True, "q"), (300, 64, True, "k"),
                                                     (5, 128, False, "")])
def test_norm_rope_without_a_cache(rt, dtype, rows, dim, in_place, gains):
    g = gen(rows)
    heads, kv_heads = 6, 2
    c = Cache(rt, dtype)
    cos, sin = (t.cuda() for t in tables(1000, dim))
    gq, gk = ((torch.rand(dim, generator=g) + 0.5).to(DTYPES[dtype]).cuda() if x in gains else None for x in "qk")
    x = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g).to(DTYPES[dtype])
    qkv = x.cuda()
    pos = torch.randint(0, 1000, (rows,), generator=g)
    dpos = pos.int().cuda()
    out = qkv[:, :heads] if in_place else torch.empty(rows, heads, dim, dtype=DTYPES[dtype], device="cuda")
    k_out = qkv[:, heads:heads + kv_heads] if in_place else torch.empty(rows, kv_heads, dim, dtype=DTYPES[dtype], device="cuda")
    rt.qk_norm_rope(rows_of(rt, c, dtype, qkv, heads, kv_heads, None, dpos, out, cos, sin, (gq, gk),
                            k_out=k_out.data_ptr(), k_out_stride=k_out.stride(0)), None, 0, c.stream())
    for got, part, gain in ((out, x[:, :heads], gq), (k_out, x[:, heads:heads + kv_heads], gk)):
        gain = None if gain is None else gain.cpu()
        want = norm_rope(part, gain, cos.cpu(), sin.cpu(), pos, 1e-5, False)
        close(got.cpu(), want, DTYPES[dtype], want.norm(dim=-1, keepdim=True))
    assert torch.equal(qkv[:, heads + kv_heads:].cpu(), x[:, heads + kv_heads:])
    assert c.status.tolist() == [0]


def test_norm_rope_skips_and_reports_bad_rows(rt):
    c = Cache(rt, n_pages=8, n_seqs=3, max_pages=2)
    c.extend([20, 20, 0])
    c.table[1, 1] = 8  # outside the pool
    g = gen(3)
    qkv = torch.randn(6, 8, 64, generator=g).half().cuda()
    cos, sin = (t.cuda() for t in tables(19, 64))
    for seq, pos, code, written in (([0] * 6, [13, 14, 15, 16, 17, 18], 0, 6), ([0, 3, 0, 0, 0, 0], [0, 0, 32, -1, 19, 1], 4, 2),
                                    ([1] * 6, [13, 14, 15, 16, 17, 18], 3, 6)):
        c.status.zero_()
        out = torch.full((6, 4, 64), 5.0, dtype=torch.float16, device="cuda")
        before = c.state()
        rt.qk_norm_rope(rows_of(rt, c, "f16", qkv, 4, 2, c.ints(seq), c.ints(pos), out, cos, sin), c.p, 0, c.stream())
        assert c.status.tolist() == [code]
        assert int((out != 5.0).flatten(1).any(1).sum()) == written
        assert torch.equal(before[0][0, 4:].nan_to_num(9), c.k[0, 4:].nan_to_num(9))  # pages of nobody


# ------------------------------------------------------------------ sparse attention
def ask(rt, c, q, seq, pos, top, sink, local, layer=0, scale=0.0, out=None, selected=True):
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device=q.device) if out is None else out
    sel = torch.full((q.shape[0], c.kv_heads, top), -9, dtype=torch.int32, device=q.device) if selected else None
    a = rt.SparseQuery(rows=q.shape[0], q_heads=q.shape[1], q=q.data_ptr(), q_stride=q.stride(0), out=out.data_ptr(),
                       out_stride=out.stride(0), row_seq=seq.data_ptr(), row_pos=pos.data_ptr(), scale=scale,
                       top_pages=top, sink_pages=sink, local_pages=local, selected=None if sel is None else sel.data_ptr())
    rt.sparse_attention(a, c.p, layer, c.stream())
    return out, sel


def held_to_64_bits(c, q, seq, pos, top, sink, local, layer, scale, out, sel):
    """The pages taken are equal; outputs within: scores off by at most 2^-20 of their terms' sum (fp32 sums, products
    of two pieces), weights by twice that (numerator and sum) and 2^-16 (16-bit pieces of the weights), one rounding."""
    P, G, dt = c.page, q.shape[1] // c.kv_heads, q.dtype
    scale = scale or 1 / math.sqrt(c.dim)
    for r, (s, n) in enumerate(zip(seq.tolist(), pos.tolist())):
        if s < 0:
            assert bool((out[r] == 5.0).all()) and (sel is None or bool((sel[r] == -9).all()))
            continue
        k, v = c.history(layer, s, n + 1)
        seen = n // P + 1
        b = c.bounds[layer, c.table[s, :seen].long()].double().cpu()
        for h in range(c.kv_heads):
            qh = q[r, h * G:(h + 1) * G].double().cpu()
            pages = choose(qh, b[:, h, 0], b[:, h, 1], seen, top, sink, local)
            if sel is not None:
                assert sel[r, h].tolist() == pages + [-1] * (top - len(pages)), (r, h)
            at = [t for j in pages for t in range(j * P, min(j * P + P, n + 1))]
            want, terms = attend(qh, k[h, at], v[h, at], scale)
            got = out[r, h * G:(h + 1) * G].double().cpu()
            bound = 2 * (2.0 ** -20 * (terms + 4) + (0 if dt == torch.float32 else 2.0 ** -16)) * float(v[h, at].abs().max())
            err = (got - want).abs() - half_ulp(dt) * want.abs() * 1.01
            assert bool((err <= bound).all()), (r, h, float(err.max()), bound)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,G,page,lens,top,sink,local", [
    (64, 2, 8, 64, [1, 63, 64, 65, 1000, 513], 4, 1, 1),
    (128, 1, 16, 16, [1, 16, 17, 700, 333], 8, 2, 2),
    (64, 3, 1, 32, [2, 31, 320, 321], 3, 0, 1),
    (128, 2, 5, 128, [129, 128, 1500], 2, 1, 1),     # nothing left for the scores
    (64, 1, 3, 16, [3000, 4001], 100, 1, 3),
    (128, 8, 4, 64, [70, 900], 256, 0, 1),           # more room than pages: every key
])
def test_sparse_attention_single_tokens(rt, dtype, dim, kv_heads, G, page, lens, top, sink, local):
    g = gen(dim + page + G)
    pool = sum(-(-n // page) for n in lens) + 3
    c = Cache(rt, dtype, 2, pool, kv_heads, page, dim, len(lens) + 1, max(-(-n // page) for n in lens) + 1)
    c.fill_random(lens, g)
    seq, pos = c.ints([-1] + list(range(len(lens))) + [-3]), c.ints([0] + [n - 1 for n in lens] + [5])
    wide = torch.randn(len(lens) + 2, kv_heads * G + 1, dim, generator=g).to(DTYPES[dtype]).cuda()
    q = wide[:, :-1]
    for scale in (0.0, 0.31):
        out, sel = ask(rt, c, q, seq, pos, top, sink, local, 1, scale)
        assert c.status.tolist() == [0]
        held_to_64_bits(c, q, seq, pos, top, sink, local, 1, scale, out, sel)
    again, _ = ask(rt, c, q, seq, pos, top, sink, local, 1, 0.31, selected=False)
    assert torch.equal(again, out)  # sums run in a fixed order


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,G,top,sink,local,past,new", [(64, 8, 4, 1, 1, 500, 150), (16, 2, 12, 0, 2, 0, 200),
                                                            (32, 16, 5, 1, 3, 1000, 40)])
def test_sparse_attention_prompt_rows(rt, dtype, page, G, top, sink, local, past, new):
    """Rows of a piece of a prompt: each sees the keys up to its own, though later ones are in the cache already."""
    g = gen(page + G)
    n = past + new
    c = Cache(rt, dtype, 1, 2 * (-(-n // page)) + 2, 2, page, 64, 2, -(-n // page))
    c.fill_random([n, n - 7], g, shared=past // page // 2)
    some = sorted(random.Random(page).sample(range(new), 25) + [0, new - 1])
    seq, pos = c.ints([0] * len(some) + [1]), c.ints([past + i for i in some] + [n - 8])
    q = torch.randn(len(some) + 1, 2 * G, 64, generator=g).to(DTYPES[dtype]).cuda()
    out, sel = ask(rt, c, q, seq, pos, top, sink, local)
    assert c.status.tolist() == [0]
    held_to_64_bits(c, q, seq, pos, top, sink, local, 0, 0.0, out, sel)


@pytest.mark.parametrize("rows", [1, 3, 40, 700])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_sparse_attention_does_not_depend_on_the_batch(rt, rows, dtype):
    """The same rows alone and in batches of any size take the same pages and agree within fp32 sums."""
    g = gen(rows)
    c = Cache(rt, dtype, 1, 200, 2, 16, 64, 2, 130)
    c.fill_random([2000, 1000], g)
    q = torch.randn(2, 16, 64, generator=g).to(DTYPES[dtype]).cuda()
    many = q[torch.arange(rows) % 2].contiguous()
    out, sel = ask(rt, c, many, c.ints([i % 2 for i in range(rows)]), c.ints([1999 - 1000 * (i % 2) for i in range(rows)]), 9, 1, 2)
    seq, pos = c.ints([0, 1])[:rows], c.ints([1999, 999])[:rows]
    held_to_64_bits(c, q[:rows], seq, pos, 9, 1, 2, 0, 0.0, out[:2], sel[:2])
    assert all(torch.equal(out[i], out[i % 2]) and torch.equal(sel[i], sel[i % 2]) for i in range(rows))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,top,G", [(1, 700, 40, 3), (3, 2100, 200, 8), (400, 540, 30, 1), (400, 300, 9, 16), (350, 1300, 256, 2)])
def test_every_way_to_the_best_pages(rt, dtype, rows, n, top, G):
    """Histories of n pages by few rows (clusters that share the scores) and by many (plain sums up to 512 pages, full
    ones above): the same pages as the 64-bit scores give."""
    g = gen(rows + n)
    c = Cache(rt, dtype, 1, n + 1, 1, 16, 64, 1, n)
    c.fill_random([16 * n - 3], g)
    q = torch.randn(rows, G, 64, generator=g).to(DTYPES[dtype]).cuda()
    seq, pos = c.ints([0] * rows), c.ints([16 * n - 4 - 7 * (r % 50) for r in range(rows)])
    out, sel = ask(rt, c, q, seq, pos, top, 2, 3)
    assert c.status.tolist() == [0]
    some = torch.tensor(sorted({0, rows - 1, rows // 2, rows // 3}), device="cuda")
    held_to_64_bits(c, q[some], seq[some], pos[some], top, 2, 3, 0, 0.0, out[some], sel[some])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,dim", [(16, 128), (8, 64)])
@pytest.mark.parametrize("rows", [1, 400])
def test_the_longest_tables(rt, dtype, G, dim, rows):
    """16384 pages a sequence, all but a few of them the same page of the pool: equal scores, the first ones win."""
    c = Cache(rt, dtype, 1, 40, 1, 16, dim, 2, 16384)
    c.fill_random([40 * 16], gen(20))
    c.table[0, 40:] = c.table[0, 0]
    c.table[1] = c.table[0]
    q = torch.randn(rows, G, dim, generator=gen(21)).to(DTYPES[dtype]).cuda()
    seq, pos = c.ints([1] * rows), c.ints([16384 * 16 - 1 - r for r in range(rows)])
    out, sel = ask(rt, c, q, seq, pos, 50, 1, 1)
    assert c.status.tolist() == [0]
    held_to_64_bits(c, q[:1], seq[:1], pos[:1], 50, 1, 1, 0, 0.0, out[:1], sel[:1])
    held_to_64_bits(c, q[-1:], seq[-1:], pos[-1:], 50, 1, 1, 0, 0.0, out[-1:], sel[-1:])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_too_close_to_call_among_many(rt, dtype):
    """Hundreds of pages whose scores lie within the plain sums' error of one another, in every number of rows."""
    n = 400
    c = Cache(rt, dtype, 1, n, 1, 16, 64, 1, n)
    c.fill_random([16 * n], gen(22))
    low, high = c.bounds[0, :, :, 0], c.bounds[0, :, :, 1]
    low[:], high[:] = -1.0, 1.0
    tiny = {"f32": 2.0 ** -23, "f16": 2.0 ** -10}[dtype]
    order = random.Random(5).sample(range(1, n - 1), 60)
    for i, j in enumerate(order):
        high[c.table[0, j].long(), 0, 7] = 1.0 + tiny * (60 - i)
    q = torch.full((1, 4, 64), 8.0, dtype=DTYPES[dtype])
    q[:, :, 7] = 2.0 ** -9
    for rows in (1, 350):
        _, sel = ask(rt, c, q.cuda().expand(rows, 4, 64).contiguous(), c.ints([0] * rows), c.ints([16 * n - 1] * rows), 33, 1, 1)
        assert all(r == sorted([0, n - 1] + order[:31]) for r in sel.flatten(1).tolist())


def test_equal_scores_take_the_first_pages(rt):
    c = Cache(rt, "f16", 1, 40, 1, 16, 64, 1, 40)
    c.fill_random([640], gen(1))
    c.bounds[:] = c.bounds[:, 3:4]
    q = torch.randn(1, 4, 64, generator=gen(2)).half().cuda()
    _, sel = ask(rt, c, q, c.ints([0]), c.ints([639]), 9, 2, 1)
    assert sel.flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 39]
    c.bounds[0, c.table[0, 30].long()] += 0.5  # this one page beats them, and zero queries make all equal again
    _, sel = ask(rt, c, q.abs(), c.ints([0]), c.ints([639]), 9, 2, 1)
    assert sel.flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 30, 39]
    _, sel = ask(rt, c, q * -0.0, c.ints([0]), c.ints([639]), 9, 2, 1)
    assert sel.flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 39]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_close_scores_are_told_apart(rt, dtype):
    """Two kinds of page whose scores differ by a few parts in 2^22 of their terms, below what fp32 sums keep apart."""
    c = Cache(rt, dtype, 1, 70, 1, 16, 64, 1, 64)
    c.fill_random([1024], gen(4))
    low, high = c.bounds[0, :, :, 0], c.bounds[0, :, :, 1]
    low[:] = -1.0
    high[:] = 1.0
    tiny = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[dtype]
    order = [9, 40, 41, 50, 17]
    for i, j in enumerate(order):
        high[c.table[0, j].long(), 0, 5] = 1.0 + tiny * (len(order) - i)
    q = torch.full((1, 2, 64), 8.0, dtype=DTYPES[dtype])
    q[:, :, 5] = 2.0 ** -9
    _, sel = ask(rt, c, q.cuda(), c.ints([0]), c.ints([1023]), 4, 0, 1)
    assert sel.flatten().tolist() == [9, 40, 41, 63]


def test_numbers_that_are_none_stay_in_their_place(rt):
    c = Cache(rt, "f32", 1, 40, 2, 16, 64, 2, 20)
    c.fill_random([320, 320], gen(5))
    q = torch.randn(3, 4, 64, generator=gen(6)).cuda()
    seq, pos = c.ints([0, 1, 1]), c.ints([319, 319, 100])
    clean, chosen = ask(rt, c, q, seq, pos, 5, 1, 1)
    bad = c.table[0, 7].long()
    c.k[0, bad, 1, 3], c.bounds[0, bad, 1] = math.nan, math.nan  # one key of sequence 0, KV head 1
    out, sel = ask(rt, c, q, seq, pos, 5, 1, 1)
    assert torch.equal(out[1:], clean[1:]) and torch.equal(out[0, :2], clean[0, :2]) and torch.equal(sel[0, 0], chosen[0, 0])
    assert 7 in sel[0, 1].tolist() and bool(out[0, 2:].isnan().all())
    q[1, 0, 0] = math.nan  # a query of NaN: its own head only
    out, _ = ask(rt, c, q, seq, pos, 20, 0, 1)
    assert bool(out[1, 0].isnan().all()) and not bool(out[1, 1:].isnan().any()) and not bool(out[2].isnan().any())


def test_large_scores_do_not_overflow(rt):
    """Scores of thousands, among them only very low ones: the running maximum keeps the weights in range."""
    c = Cache(rt, "f16", 1, 20, 1, 16, 64, 1, 20)
    c.fill_random([300], gen(7))
    for sign in (1, -1):
        base = torch.ones(64, dtype=torch.float16, device="cuda")
        q = (base * 60 * sign).expand(1, 2, 64).contiguous()
        c.k[:] = torch.where(c.k.isnan(), c.k, 12 + c.k * 0.25)
        out, sel = ask(rt, c, q, c.ints([0]), c.ints([299]), 20, 0, 1)
        held_to_64_bits(c, q, c.ints([0]), c.ints([299]), 20, 0, 1, 0, 0.0, out, sel)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 400])
def test_many_small_weights_add_up(rt, dtype, rows):
    """One key of weight 1 and 32767 of e^-17.5 each, less than half of fp16's smallest step: they carry the output
    (400 rows: a warp has a quarter of the keys, and that share beside the large one)."""
    c = Cache(rt, dtype, 1, 256, 1, 128, 64, 1, 256)
    c.fill_random([256 * 128], gen(24))
    c.k[:], c.v[:] = 0.0, 1.0
    first = c.table[0, 0].long()
    c.k[0, first, 0, 5], c.v[0, first, 0, 5] = 2.1875, 0.0
    q = torch.ones(rows, 8, 64, dtype=DTYPES[dtype], device="cuda")
    seq, pos = c.ints([0] * rows), c.ints([256 * 128 - 1] * rows)
    out, sel = ask(rt, c, q, seq, pos, 256, 1, 1)
    held_to_64_bits(c, q[-1:], seq[-1:], pos[-1:], 256, 1, 1, 0, 0.0, out[-1:], None)
    assert 7e-4 < float(out.float().mean()) < 9e-4  # 32767 e^-17.5 = 8.2e-4


def test_bad_rows_and_pages_are_reported_and_skipped(rt):
    c = Cache(rt, "f16", 1, 30, 1, 16, 64, 2, 10)
    c.fill_random([160, 160], gen(8))
    q = torch.randn(4, 2, 64, generator=gen(9)).half().cuda()
    out, _ = ask(rt, c, q, c.ints([2, 0, 1, 0]), c.ints([0, 160, -1, 159]), 4, 1, 1)
    assert c.status.tolist() == [rt.PAGES_BAD_ROW]
    assert bool((out[:3] == 5.0).all()) and not bool((out[3] == 5.0).any())
    c.status.zero_()
    c.table[0, 0], c.table[1] = 30, -1
    out, _ = ask(rt, c, q[:2], c.ints([0, 1]), c.ints([159, 159]), 4, 1, 1)
    assert c.status.tolist() == [rt.PAGES_BAD_ID] and bool(out.isfinite().all())


def test_pages_past_two_to_the_31_elements(rt):
    """Keys that lie further than 2^31 elements (and 2^32 bytes) into the pool."""
    n = 70000  # 70000 pages x 8 heads x 64 tokens x 64 = 2.29e9 elements
    c = Cache(rt, "bf16", 1, n, 8, 64, 64, 2, 4, fill=False)
    ids = [n - 1, n - 77, 2, n // 2]
    c.table[0] = c.ints(ids)
    c.refs[torch.tensor(ids).cuda()] = 1
    c.lens[0] = 250
    g = gen(10)
    qkv = torch.randn(250, 16 + 16, 64, generator=g).bfloat16().cuda()
    seq, pos = c.ints([0] * 250), torch.arange(250, dtype=torch.int32, device="cuda")
    out = torch.empty(250, 16, 64, dtype=torch.bfloat16, device="cuda")
    rt.qk_norm_rope(rows_of(rt, c, "bf16", qkv, 16, 8, seq, pos, out), c.p, 0, c.stream())
    k, v = c.history(0, 0, 250)
    assert torch.equal(k, qkv[:, 16:24].transpose(0, 1).double().cpu())
    some = torch.tensor([0, 63, 64, 249]).cuda()
    o, sel = ask(rt, c, out[some].contiguous(), seq[some], pos[some], 2, 0, 1)
    held_to_64_bits(c, out[some], seq[some], pos[some], 2, 0, 1, 0, 0.0, o, sel)
    c.fork([-1, 0], share=False)
    c.free([1, 0])
    assert c.compact().tolist() == [4]
    k2, v2 = c.history(0, 1, 250)
    assert torch.equal(k, k2) and torch.equal(v, v2) and c.status.tolist() == [0]


# ------------------------------------------------------------------ together
class Decoder:
    """One layer's attention of a few utterances through the operators, as a server would run it; the host keeps
    every utterance's rows in 64 bits."""

    def __init__(self, rt, dtype, page=16, dim=64, heads=8, kv_heads=2, seqs=4, top=6):
        self.rt, self.dtype, self.heads, self.kv_heads, self.dim, self.top = rt, dtype, heads, kv_heads, dim, top
        self.c = Cache(rt, dtype, 1, 120, kv_heads, page, dim, seqs, 20)
        self.cos, self.sin = (t.cuda() for t in tables(20 * page, dim))
        g = gen(11)
        self.gains = [(torch.rand(dim, generator=g) + 0.5).to(DTYPES[dtype]).cuda() for _ in range(2)]

    def buffers(self, rows):
        shape, dt = (rows, self.heads, self.dim), DTYPES[self.dtype]
        self.qkv = torch.zeros(rows, self.heads + 2 * self.kv_heads, self.dim, dtype=dt, device="cuda")
        self.q, self.out = (torch.zeros(shape, dtype=dt, device="cuda") for _ in range(2))
        self.seq, self.pos = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
        self.counts = torch.zeros(self.c.n_seqs, dtype=torch.int32, device="cuda")

    def step(self):
        c, rt, s = self.c, self.rt, torch.cuda.current_stream().cuda_stream
        rt.pages_extend(c.p, self.counts.data_ptr(), self.seq.numel(), self.seq.data_ptr(), self.pos.data_ptr(), s)
        rt.qk_norm_rope(rows_of(rt, c, self.dtype, self.qkv, self.heads, self.kv_heads, self.seq, self.pos, self.q,
                                self.cos, self.sin, self.gains), c.p, 0, s)
        a = rt.SparseQuery(rows=self.seq.numel(), q_heads=self.heads, q=self.q.data_ptr(), q_stride=self.q.stride(0),
                           out=self.out.data_ptr(), out_stride=self.out.stride(0), row_seq=self.seq.data_ptr(),
                           row_pos=self.pos.data_ptr(), scale=0.0, top_pages=self.top, sink_pages=1, local_pages=2)
        rt.sparse_attention(a, c.p, 0, s)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_utterances_from_one_prompt(rt, dtype):
    """A prompt, forked to three utterances that go on by themselves (one by a copy), the pool drawn together in
    between and the parent ended: every step's outputs against all the rows each utterance has been given."""
    d = Decoder(rt, dtype, top=20)
    c = d.c
    g = gen(12)
    text = [torch.zeros(0, d.heads + 2 * d.kv_heads, d.dim, dtype=DTYPES[dtype]) for _ in range(c.n_seqs)]
    G = d.heads // d.kv_heads

    def go(counts):
        d.buffers(sum(counts) + 2)
        d.counts.copy_(c.ints(counts))
        new = torch.randn(d.qkv.shape, generator=g).to(DTYPES[dtype])
        d.qkv.copy_(new)
        d.step()
        assert c.status.tolist() == [0]
        at = 0
        for s, n in enumerate(counts):
            text[s] = torch.cat([text[s], new[at:at + n]])
            if n:
                x, T = text[s], len(text[s])
                p = torch.arange(T)
                cpu = [t.cpu() for t in (*d.gains, d.cos, d.sin)]
                q = norm_rope(x[:, :d.heads], cpu[0], cpu[2], cpu[3], p, 1e-5, False)
                k = norm_rope(x[:, d.heads:d.heads + d.kv_heads], cpu[1], cpu[2], cpu[3], p, 1e-5, False)
                v = x[:, d.heads + d.kv_heads:].double()
                for h in range(d.heads):
                    for i in range(n):
                        t = T - n + i + 1
                        want, terms = attend(q[t - 1, h][None], k[:t, h // G], v[:t, h // G], 1 / math.sqrt(d.dim))
                        # q and k are rounded to the type before the scores, the output after
                        u = half_ulp(DTYPES[dtype])
                        bound = (2 * (2 * u + 2.0 ** -18) * terms + 2.0 ** -15) * float(v[:t, h // G].abs().max()) + u * want.abs()
                        assert bool(((d.out[at + i, h].double().cpu() - want[0]).abs() <= bound).all()), (s, h, i)
            at += n

    go([70, 0, 0, 0])
    c.fork([-1, 0, 0, -1])
    text[1], text[2] = text[0], text[0]
    go([1, 1, 1, 0])
    c.fork([-1, -1, -1, 2], share=False)
    text[3] = text[2]
    go([0, 17, 1, 1])
    c.free([1, 0, 0, 0])
    text[0] = text[0][:0]
    c.compact()
    go([33, 1, 1, 16])
    go([1, 1, 1, 1])


def test_a_captured_step_is_replayed(rt):
    """extend, norm and attention captured once and replayed token by token give what calls one by one give, to the
    bit; a second graph of other buffers on the same cache too."""
    runs = []
    for captured in (False, True):
        d = Decoder(rt, "f16")
        g = gen(13)
        d.buffers(90)
        d.counts.copy_(d.c.ints([80, 0, 9, 0]))
        d.qkv.copy_(torch.randn(d.qkv.shape, generator=g))
        d.step()
        torch.cuda.synchronize()
        steps = []
        for rows in (5, 3):
            d.buffers(rows)
            kept = {x: getattr(d, x) for x in ("qkv", "q", "out", "seq", "pos", "counts")}
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    d.step()
                steps.append((kept, graph.replay, graph))
            else:
                steps.append((kept, d.step, None))
        got = []
        for i in range(40):
            kept, run, _ = steps[i % 2]
            for x, t in kept.items():
                setattr(d, x, t)
            d.counts.copy_(d.c.ints([1, 0, 1, int(i > 5)]))
            d.qkv.copy_(torch.randn(d.qkv.shape, generator=g))
            run()
            got.append(d.out.clone())
        runs.append((got, [d.c.k.clone(), d.c.table.clone(), d.c.lens.clone(), d.c.status.clone()]))
    assert runs[0][1][3].tolist() == [0] and runs[0][1][2].tolist() == [120, 0, 49, 34]
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a.nan_to_num(9), b.nan_to_num(9))


def test_streams_of_the_callers(rt):
    """Readers of one cache on several streams at once, each ordered after the writer by its own stream's events."""
    c = Cache(rt, "f16", 1, 300, 2, 16, 64, 4, 70)
    c.fill_random([1000, 900, 1100, 16], gen(14))
    q = torch.randn(4, 16, 64, generator=gen(15)).half().cuda()
    seq, pos = c.ints([0, 1, 2, 3]), c.ints([999, 899, 1099, 15])
    want, _ = ask(rt, c, q, seq, pos, 8, 1, 2)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ask(rt, c, q, seq, pos, 8, 1, 2)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_calls_from_several_threads(rt):
    """Host threads whose calls need different amounts of shared memory for the same kernels, at the same time."""
    import threading
    jobs = []
    for i, (most, page) in enumerate(((40, 16), (9000, 16), (16384, 16), (60, 128))):
        c = Cache(rt, "f32", 1, 45, 1, page, 128, 1, most)
        c.fill_random([40 * page], gen(30 + i))
        q = torch.randn(2, 4, 128, generator=gen(40 + i)).cuda()
        seq, pos = c.ints([0, 0]), c.ints([40 * page - 1, 33])
        want, _ = ask(rt, c, q, seq, pos, 7, 1, 1)
        jobs.append((c, q, seq, pos, want))
    torch.cuda.synchronize()
    wrong = []

    def work(c, q, seq, pos, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = []
                for _ in range(150):
                    outs.append(ask(rt, c, q, seq, pos, 7, 1, 1)[0])
                    rows = torch.zeros(1, 6, 128, device="cuda")
                    rt.qk_norm_rope(rows_of(rt, c, "f32", rows, 4, 1, c.ints([-1]), c.ints([0]), torch.zeros(1, 4, 128, device="cuda")),
                                    c.p, 0, c.stream())
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(o, want) for o in outs):
                    wrong.append("outputs differ")
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_memory_of_the_host_is_refused(rt):
    c = Cache(rt)
    host = torch.zeros(64 * 1024, dtype=torch.float16)
    keep, c.p.k = c.p.k, (host.data_ptr() + 15) // 16 * 16
    for call in (lambda: c.free([0] * 4), lambda: c.fork([-1] * 4), lambda: c.compact(), lambda: c.extend([0] * 4, 1)):
        with pytest.raises(rt.VxcError) as e:
            call()
        assert e.value.status == 1 and "current device" in str(e.value)
    c.p.k = keep
    ints = torch.zeros(8, dtype=torch.int32)
    at, dev = ints.data_ptr(), c.lens.data_ptr()
    for call in (lambda: rt.pages_free(c.p, at), lambda: rt.pages_fork(c.p, at), lambda: rt.pages_extend(c.p, at, 1, dev, dev),
                 lambda: rt.pages_extend(c.p, dev, 1, at, dev), lambda: rt.pages_extend(c.p, dev, 1, dev, at)):
        with pytest.raises(rt.VxcError) as e:
            call()
        assert e.value.status == 1 and "current device" in str(e.value)
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(rt.VxcError) as e:
        rt.sparse_attention(rt.SparseQuery(rows=1, q_heads=2, q=(q.data_ptr() + 15) // 16 * 16, out=c.k.data_ptr(), q_stride=128,
                                           out_stride=128, row_seq=c.lens.data_ptr(), row_pos=c.lens.data_ptr(),
                                           top_pages=1, local_pages=1), c.p, 0, 0)
    assert e.value.status == 1 and "current device" in str(e.value)
