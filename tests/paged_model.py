"""A paged KV cache in plain host code and 64-bit formulas: what the operators are held to."""
from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Cache:
    """The arrays of a vxc_pages on the GPU, garbage (not a number) in every page."""

    def __init__(self, rt, dtype="f16", layers=1, n_pages=16, kv_heads=2, page=16, dim=64, n_seqs=4, max_pages=8,
                 device="cuda", fill=True):
        self.rt, self.dtype, self.page, self.dim, self.kv_heads, self.layers = rt, DTYPES[dtype], page, dim, kv_heads, layers
        self.n_pages, self.n_seqs, self.max_pages = n_pages, n_seqs, max_pages
        shape = (layers, n_pages, kv_heads, page, dim)
        make = (lambda s: torch.full(s, math.nan, device=device, dtype=self.dtype)) if fill else (
            lambda s: torch.empty(s, device=device, dtype=self.dtype))
        self.k, self.v, self.bounds = make(shape), make(shape), make((layers, n_pages, kv_heads, 2, dim))
        ints = dict(device=device, dtype=torch.int32)
        self.table = torch.full((n_seqs, max_pages), -1, **ints)
        self.lens, self.refs = torch.zeros(n_seqs, **ints), torch.zeros(n_pages, **ints)
        self.status = torch.zeros(1, **ints)
        self.p = rt.Pages(dtype=rt.DTYPES[dtype], layers=layers, n_pages=n_pages, kv_heads=kv_heads, page_size=page,
                          head_dim=dim, n_seqs=n_seqs, max_pages=max_pages, k=self.k.data_ptr(), v=self.v.data_ptr(),
                          bounds=self.bounds.data_ptr(), table=self.table.data_ptr(), lens=self.lens.data_ptr(),
                          refs=self.refs.data_ptr(), status=self.status.data_ptr())
        self.work = torch.full((rt.pages_work_ints(self.p),), 0x3fffffff, **ints)  # nothing may hang on what it held
        self.p.work = self.work.data_ptr()

    def stream(self):
        return torch.cuda.current_stream(self.k.device).cuda_stream

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.k.device)

    def extend(self, counts, max_rows=None):
        n = sum(c for c in counts if c > 0) if max_rows is None else max_rows
        seq, pos = (torch.full((n,), 77, dtype=torch.int32, device=self.k.device) for _ in range(2))
        c = self.ints(counts)
        self.rt.pages_extend(self.p, c.data_ptr(), n, seq.data_ptr(), pos.data_ptr(), self.stream())
        return seq, pos

    def free(self, flags):
        f = self.ints(flags)
        self.rt.pages_free(self.p, f.data_ptr(), self.stream())

    def fork(self, parents, share=True):
        f = self.ints(parents)
        self.rt.pages_fork(self.p, f.data_ptr(), share, self.stream())

    def compact(self):
        used = self.ints([-5])
        self.rt.pages_compact(self.p, used.data_ptr(), self.stream())
        return used

    def state(self):
        return [x.clone() for x in (self.k, self.v, self.bounds, self.table, self.lens, self.refs)]

    def fill_random(self, lens, g, shared=0, spread=1.0):
        """Sequences of the given lengths in pages from all over the pool, the first `shared` full pages in
        common; bounds as the operator keeps them. What lies past a sequence's end stays garbage."""
        P, at = self.page, shared
        ids = torch.randperm(self.n_pages, generator=g).tolist()
        table, refs, filled = torch.full((self.n_seqs, self.max_pages), -1, dtype=torch.int32), [0] * self.n_pages, {}
        for s, n in enumerate(lens):
            need = -(-n // P)
            common = min(shared, n // P)
            take = ids[:common] + ids[at:at + need - common]
            assert len(take) == need, "the pool is too small"
            at += need - common
            for j, i in enumerate(take):
                table[s, j] = i
                refs[i] += 1
                filled[i] = min(P, n - j * P)
        pages = torch.tensor(list(filled))
        cells = (self.layers, len(pages), self.kv_heads, P, self.dim)
        k = torch.randn(cells, generator=g, dtype=torch.float64) + spread * torch.randn(
            (*cells[:3], 1, self.dim), generator=g, dtype=torch.float64)
        v = torch.randn(cells, generator=g, dtype=torch.float64)
        k, v = k.to(self.dtype), v.to(self.dtype)
        empty = torch.arange(P)[None] >= torch.tensor(list(filled.values()))[:, None]
        empty = empty[None, :, None, :, None].expand(cells)
        low = k.masked_fill(empty, math.inf).amin(3)
        high = k.masked_fill(empty, -math.inf).amax(3)
        dev = self.k.device
        self.k[:, pages.to(dev)] = k.masked_fill(empty, math.nan).to(dev)
        self.v[:, pages.to(dev)] = v.masked_fill(empty, math.nan).to(dev)
        self.bounds[:, pages.to(dev)] = torch.stack([low, high], 3).to(dev)
        self.table.copy_(table)
        self.refs.copy_(torch.tensor(refs, dtype=torch.int32))
        self.lens.zero_()
        self.lens[:len(lens)] = torch.tensor(lens, dtype=torch.int32)

    def history(self, layer, seq, n):
        """Keys and values [kv_heads, n, dim] of a sequence's first n tokens, in 64 bits on the host."""
        ids = self.table[seq, :-(-n // self.page)].long()
        return [x[layer][ids].transpose(0, 1).flatten(1, 2)[:, :n].double().cpu() for x in (self.k, self.v)]


class Model:
    """The same cache's tables, by lists."""

    def __init__(self, n_pages, n_seqs, max_pages, page):
        self.refs, self.rows, self.lens = [0] * n_pages, [[] for _ in range(n_seqs)], [0] * n_seqs
        self.max_pages, self.page = max_pages, page

    def lowest(self, n):
        free = [i for i, r in enumerate(self.refs) if r == 0]
        return free[:n] if len(free) >= n else None

    def extend(self, counts, max_rows):
        need = [-(-(n + c) // self.page) - len(r) for n, c, r in zip(self.lens, counts, self.rows)]
        if min(counts) < 0 or sum(counts) > max_rows or any(
                n + c > self.max_pages * self.page for n, c in zip(self.lens, counts)):
            return 2, [(-1, -1)] * max_rows
        ids = self.lowest(sum(need))
        if ids is None:
            return 1, [(-1, -1)] * max_rows
        rows = []
        for s, c in enumerate(counts):
            for _ in range(need[s]):
                self.refs[ids[0]] = 1
                self.rows[s].append(ids.pop(0))
            rows += [(s, self.lens[s] + i) for i in range(c)]
            self.lens[s] += c
        return 0, rows + [(-1, -1)] * (max_rows - len(rows))

    def free(self, flags):
        for s, f in enumerate(flags):
            if f:
                for i in self.rows[s]:
                    self.refs[i] -= 1
                self.rows[s], self.lens[s] = [], 0

    def fork(self, parents, share):
        for d, s in enumerate(parents):
            if s >= 0 and (s >= len(parents) or parents[s] >= 0 or self.lens[d]):
                return 2
        fresh = {d: (self.lens[s] % self.page != 0) if share else len(self.rows[s])
                 for d, s in enumerate(parents) if s >= 0}
        ids = self.lowest(sum(fresh.values()))
        if ids is None:
            return 1
        for d, n in fresh.items():
            s = parents[d]
            common = self.rows[s][:len(self.rows[s]) - n]
            for i in common:
                self.refs[i] += 1
            self.rows[d] = common + ids[:n]
            for i in ids[:n]:
                self.refs[i] = 1
            ids = ids[n:]
            self.lens[d] = self.lens[s]
        return 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [i for i in range(used) if self.refs[i] == 0]
        high = [i for i in range(used, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(high, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(i, i) for i in r] for r in self.rows]
        return used

    def check(self, c):
        assert c.lens.tolist() == self.lens
        assert c.refs.tolist() == self.refs
        want = [r + [-1] * (self.max_pages - len(r)) for r in self.rows]
        assert c.table.tolist() == want


def norm_rope(x, gain, cos, sin, pos, eps, interleaved):
    """[rows, heads, dim] in 64 bits."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    if cos is None:
        return x
    h = x.shape[-1] // 2
    c, s = (t.double()[pos][:, None, :h] for t in (cos, sin))
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    a, b = a * c - b * s, b * c + a * s
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def choose(q, low, high, seen, top, sink, local):
    """Pages one KV head takes for q [group, dim] (64 bits) among `seen` with bounds [seen, dim]."""
    if seen <= top:
        return list(range(seen))
    score = torch.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2))
    score = torch.where(score.isnan(), math.inf, score).tolist()
    must = set(range(sink)) | set(range(seen - local, seen))
    rest = sorted((i for i in range(seen) if i not in must), key=lambda i: (-score[i], i))
    return sorted(list(must) + rest[:top - len(must)])


def attend(q, k, v, scale):
    """q [group, dim], k and v [n, dim], in 64 bits: the output, and the largest sum |q||k| of a score."""
    s = q @ k.T * scale
    return torch.softmax(s, -1) @ v, float((q.abs() @ k.abs().T).max()) * scale
