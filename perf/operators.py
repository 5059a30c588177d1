"""The paged KV cache operators: what is timed and compared, in plain torch and through the library.

Three kinds of case, told apart by "op":

  norm_rope   vxc_qk_norm_rope: the RMS norm of every query and key head and the position rotation in one
              pass, keys and values written into the pages of a cache, the pages' key bounds kept up to date.
  fork, copy, compact, turnover
              vxc_pages_fork (pages shared, or copied one by one), vxc_pages_compact, vxc_pages_free with
              vxc_pages_extend: the pages themselves.
  attention   vxc_sparse_attention: every query row scores the pages of its sequence by their key bounds,
              takes the best of them and attends over those.

A case's dtype is that of the rows, the cache and the outputs. Where `own` is false, run() computes the same in
elementary torch operations, in 32 bits (page scores, whose order decides, in 64).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of a lone utterance through the benchmark model's heads
        {"name": "norm_rope_one_f16", "op": "norm_rope", "dtype": "f16", "q_heads": 16, "kv_heads": 2, "head_dim": 64,
         "page": 64, "seqs": 1, "new": 1, "past": 300, "pad": 0, "interleaved": False, "norm": True},
        # one new token of each of 61 utterances, the batch padded to 64 rows
        {"name": "norm_rope_batch_bf16", "op": "norm_rope", "dtype": "bf16", "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 32, "seqs": 61, "new": 1, "past": 500, "pad": 3, "interleaved": False, "norm": True},
        # prompts of three utterances in 32 bits, as the decoders' rows are
        {"name": "norm_rope_prompt_f32", "op": "norm_rope", "dtype": "f32", "q_heads": 16, "kv_heads": 2,
         "head_dim": 64, "page": 64, "seqs": 3, "new": 333, "past": 37, "pad": 1, "interleaved": False, "norm": True},
        # a long prefill of wide heads, neighbouring elements rotated in pairs
        {"name": "norm_rope_prefill_bf16", "op": "norm_rope", "dtype": "bf16", "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "seqs": 4, "new": 2001, "past": 0, "pad": 0, "interleaved": True, "norm": True},
        # one voice prompt of 300 tokens leads 8 utterances: its pages are shared, the last one copied
        {"name": "fork_voice_f16", "op": "fork", "dtype": "f16", "kv_heads": 2, "head_dim": 64, "page": 64,
         "layers": 24, "seqs": 12, "parents": 1, "children": 8, "tokens": 300, "pool": 128},
        # four long utterances get copies of their own, for another use of the same history
        {"name": "copy_long_bf16", "op": "copy", "dtype": "bf16", "kv_heads": 2, "head_dim": 64, "page": 64,
         "layers": 24, "seqs": 9, "parents": 4, "children": 4, "tokens": 4000, "pool": 600},
        # a pool of which three fifths have been given back at random is drawn together
        {"name": "compact_pool_f16", "op": "compact", "dtype": "f16", "kv_heads": 2, "head_dim": 64, "page": 64,
         "layers": 8, "seqs": 64, "tokens": 1500, "pool": 3000},
        # 24 of 64 utterances end and others begin with prompts of their own
        {"name": "turnover_f16", "op": "turnover", "dtype": "f16", "kv_heads": 2, "head_dim": 64, "page": 16,
         "layers": 1, "seqs": 64, "ending": 24, "tokens": 900, "pool": 8000},
        # one new token of a lone utterance of ordinary length: most pages are taken
        {"name": "attention_one_f16", "op": "attention", "dtype": "f16", "q_heads": 16, "kv_heads": 2, "head_dim": 64,
         "page": 64, "seqs": 1, "new": 1, "past": 700, "least": 700, "pad": 0, "top": 8, "sink": 1, "local": 2,
         "shared": 0},
        # one new token of 61 long utterances that share a prompt, padded to 64 rows
        {"name": "attention_batch_bf16", "op": "attention", "dtype": "bf16", "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "seqs": 61, "new": 1, "past": 14000, "least": 2000, "pad": 3, "top": 32,
         "sink": 1, "local": 4, "shared": 9},
        # one new token of two very long histories in 32 bits
        {"name": "attention_long_f32", "op": "attention", "dtype": "f32", "q_heads": 16, "kv_heads": 2,
         "head_dim": 64, "page": 64, "seqs": 2, "new": 1, "past": 131000, "least": 90000, "pad": 0, "top": 64,
         "sink": 1, "local": 4, "shared": 0},
        # a chunk of a long prompt, every row with pages of its own choice
        {"name": "attention_prefill_f16", "op": "attention", "dtype": "f16", "q_heads": 16, "kv_heads": 2,
         "head_dim": 64, "page": 64, "seqs": 1, "new": 1023, "past": 9000, "least": 9000, "pad": 1, "top": 16,
         "sink": 1, "local": 2, "shared": 0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "attention", "attention", "attention", "fork", "copy", "compact",
                     "turnover"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([64, 64, 128])
    kv = rng.choice([1, 2, 2, 4, 8] if dim == 64 else [1, 2, 4])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "norm_rope":
        new = rng.choice([1, 1, 2, _spread(rng, 3, 700)])
        return {"op": op, "dtype": dtype, "q_heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv,
                "head_dim": dim, "page": page, "seqs": _spread(rng, 1, 64 if new < 3 else 6), "new": new,
                "past": rng.choice([0, _spread(rng, 1, 600)]), "pad": rng.choice([0, 0, 1, 5]),
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.8}
    if op == "attention":
        new = rng.choice([1, 1, 1, 3, _spread(rng, 4, 300)])
        seqs = _spread(rng, 1, 48 if new == 1 else 3)
        past = _spread(rng, 1, 40000 if seqs < 3 else 6000)
        top = _spread(rng, 4, 48)
        while seqs * new * kv * dim * max(top * page, 8 * past / page) > 130e6:
            seqs, new = (seqs, (new + 1) // 2) if new > 1 else ((seqs + 1) // 2, 1)
        return {"op": op, "dtype": dtype, "q_heads": kv * rng.choice([1, 2, 3, 5, 8, 16]), "kv_heads": kv,
                "head_dim": dim, "page": page, "seqs": seqs, "new": new, "past": past,
                "least": max(1, past // rng.choice([1, 2, 9])), "pad": rng.choice([0, 0, 1, 3]), "top": top,
                "sink": rng.choice([0, 1, 2]), "local": rng.choice([1, 2]), "shared": rng.choice([0, 0, 1, 4])}
    layers = rng.choice([1, 2, 8])
    tokens = _spread(rng, 5, 1500)
    each = tokens // page + 1
    if op in ("fork", "copy"):
        parents, children = rng.choice([1, 2, 3]), _spread(rng, 1, 9)
        return {"op": op, "dtype": dtype, "kv_heads": kv, "head_dim": dim, "page": page, "layers": layers,
                "seqs": parents + children + rng.choice([0, 1, 5]), "parents": parents, "children": children,
                "tokens": tokens, "pool": each * (parents + (children if op == "copy" else 0)) + children + 20}
    seqs = _spread(rng, 4, 40)
    case = {"op": op, "dtype": dtype, "kv_heads": kv, "head_dim": dim, "page": page, "layers": layers, "seqs": seqs}
    if op == "turnover":
        case |= {"layers": 1, "ending": rng.randint(1, seqs)}
    return case | {"tokens": min(tokens, 600), "pool": 4 * seqs * (min(tokens, 600) // page + 1) + rng.randint(0, 40)}


# ------------------------------------------------------------------------------------------------ inputs
def _pool(case, dev, g, layers, n_pages, filled):
    """Keys, values and key bounds of a pool: pages of a centre of their own, `filled` tokens in each (the rest
    holds what an earlier user of the page left, not a number among it)."""
    dt, H, P, D = DTYPES[case["dtype"]], case["kv_heads"], case["page"], case["head_dim"]
    shape = (layers, n_pages, H, P, D)
    k = torch.randn(shape, device=dev, generator=g, dtype=dt)
    k.mul_(0.7).add_(torch.randn((layers, n_pages, H, 1, D), device=dev, generator=g, dtype=dt))
    v = torch.randn(shape, device=dev, generator=g, dtype=dt)
    low, high = k.amin(3), k.amax(3)
    partial = torch.nonzero((filled > 0) & (filled < P))[:, 0]
    if partial.numel():
        empty = torch.arange(P, device=dev)[None, :] >= filled[partial, None]
        empty = empty[None, :, None, :, None]
        part = k[:, partial]
        low[:, partial] = part.masked_fill(empty, math.inf).amin(3)
        high[:, partial] = part.masked_fill(empty, -math.inf).amax(3)
        k[:, partial] = part.masked_fill(empty, math.nan)
        v[:, partial] = v[:, partial].masked_fill(empty, math.nan)
    return k, v, torch.stack([low, high], 3)


def _tables(lens, page, n_pages, max_pages, g, shared=0):
    """Pages for every sequence, from all over the pool; the first `shared` pages are the same ones."""
    n = len(lens)
    need = [-(-t // page) for t in lens]
    ids = torch.randperm(n_pages, generator=g)
    table = torch.full((n, max_pages), -1, dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    filled = torch.zeros(n_pages, dtype=torch.int64)
    at = shared
    for s in range(n):
        common = min(shared, lens[s] // page)
        take = torch.cat([ids[:common], ids[at:at + need[s] - common]])
        at += need[s] - common
        table[s, :need[s]] = take.int()
        refs[take] += 1
        filled[take] = page
        if lens[s] % page:
            filled[take[-1]] = lens[s] % page
    return table, refs, filled


def _sizes(n, high, low, h):
    """n sizes from low to high: the same ones for every seed, so that shapes are, in an order of the seed's own."""
    fixed = torch.Generator().manual_seed(n)
    sizes = torch.randint(low, high + 1, (n,), generator=fixed)
    return sizes[torch.randperm(n, generator=h)].tolist()


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    S = {"case": case}
    page, n = case["page"], case["seqs"]
    if case["op"] in ("norm_rope", "attention"):
        _prepare_rows(case, S, dev, g, h)
    else:
        layers, pool, t = case["layers"], case["pool"], case["tokens"]
        lens = _sizes(n, t, (t + 1) // 2, h)
        if case["op"] in ("fork", "copy"):
            parents, children = case["parents"], case["children"]
            order = torch.randperm(n, generator=h).tolist()
            first = set(order[:parents])
            lens = [lens[s] if s in first else 0 for s in range(n)]
            parent = torch.full((n,), -1, dtype=torch.int32)
            for i, s in enumerate(order[parents:parents + children]):
                parent[s] = order[i % parents]
            S["parent"] = parent.to(dev)
            S["flags"] = (parent >= 0).int().to(dev)
        elif case["op"] == "turnover":
            ending = torch.zeros(n, dtype=torch.int32)
            ending[torch.randperm(n, generator=h)[:case["ending"]]] = 1
            S["flags"] = ending.to(dev)
            begin = torch.zeros(n, dtype=torch.int32)
            begin[ending != 0] = torch.tensor(_sizes(case["ending"], t, 1, h), dtype=torch.int32)
            S["counts"] = begin.to(dev)
            S["max_rows"] = int(S["counts"].sum()) + 3
        S["max_pages"] = -(-case["tokens"] // page) + 1
        table, refs, filled = _tables(lens, page, pool, S["max_pages"], h)
        S["k"], S["v"], S["bounds"] = _pool(case, dev, g, layers, pool, filled.to(dev))
        S["table"], S["refs"] = table.to(dev), refs.to(dev)
        S["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    S["status"] = torch.zeros(1, dtype=torch.int32, device=dev)
    if case["op"] == "turnover":
        S["row_seq"] = torch.empty(S["max_rows"], dtype=torch.int32, device=dev)
        S["row_pos"] = torch.empty(S["max_rows"], dtype=torch.int32, device=dev)
    if case["op"] == "compact":
        S["used"] = torch.zeros(1, dtype=torch.int32, device=dev)
        S["before"] = [S[x].clone() for x in ("table", "refs")]
    if own:
        _handle(case, S)
    return S


def _prepare_rows(case, S, dev, g, h):
    """Rows of a batch as vxc_pages_extend lays them out (sequence by sequence, padding rows last) and their cache."""
    dt, page, n, new = DTYPES[case["dtype"]], case["page"], case["seqs"], case["new"]
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "attention":
        past = _sizes(n, case["past"], case["least"], h)
        count = [new] * n
        shared = case["shared"]
    else:
        # prompts of several lengths follow histories of several lengths
        past = _sizes(n, case["past"], case["past"] // 2, h)
        count = _sizes(n, new, (new + 1) // 2, h)
        shared = 0
    lens = [a + b for a, b in zip(past, count)]
    S["max_pages"] = -(-max(lens) // page) + 2
    pool = sum(a // page + b // page + 2 for a, b in zip(past, count)) + 5
    table, refs, _ = _tables(lens, page, pool, S["max_pages"], h, shared)
    # the cache as it stands before the call: without the new rows for norm_rope, with them for attention
    held = past if case["op"] == "norm_rope" else lens
    filled = torch.zeros(pool, dtype=torch.int64)
    for s in range(n):
        pages = table[s, :-(-lens[s] // page)].long()
        filled[pages] = torch.clamp(held[s] - torch.arange(len(pages)) * page, 0, page)
    layers = 2 if n * case["past"] < 50000 else 1
    S["layer"] = layers - 1
    S["k"], S["v"], S["bounds"] = _pool(case, dev, g, layers, pool, filled.to(dev))
    S["table"], S["refs"] = table.to(dev), refs.to(dev)
    S["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    seq = torch.cat([torch.full((c,), s) for s, c in enumerate(count)] + [torch.full((case["pad"],), -1)])
    pos = torch.cat([torch.arange(c) + a for a, c in zip(past, count)] + [torch.full((case["pad"],), -1)])
    S["row_seq"], S["row_pos"] = seq.int().to(dev), pos.int().to(dev)
    R = seq.numel()
    S["rows"] = R
    if case["op"] == "attention":
        S["q"] = torch.randn((R, Hq, D), device=dev, generator=g).to(dt)
        S["out"] = torch.zeros((R, Hq, D), device=dev, dtype=dt)
        S["selected"] = torch.zeros((R, Hkv, case["top"]), device=dev, dtype=torch.int32)
        return
    # q, k and v as one projection leaves them: a row of (Hq + 2 Hkv) heads
    S["qkv"] = (torch.randn((R, Hq + 2 * Hkv, D), device=dev, generator=g) * 1.7).to(dt)
    S["q_gain"] = (1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(dt)
    S["k_gain"] = (1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(dt)
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    angle = torch.arange(max(lens) + 1, dtype=torch.float64, device=dev)[:, None] * torch.cat([inv, inv])
    S["cos"], S["sin"] = angle.cos().float(), angle.sin().float()
    S["out"] = torch.zeros((R, Hq, D), device=dev, dtype=dt)


def _handle(case, S):
    """What a program keeps between calls: the description of its cache and of its rows."""
    from voxcpm2_b200 import runtime as rt
    L, N, H, P, D = S["k"].shape
    p = rt.Pages(dtype=rt.DTYPES[case["dtype"]], layers=L, n_pages=N, kv_heads=H, page_size=P, head_dim=D,
                 n_seqs=S["table"].shape[0], max_pages=S["max_pages"], k=S["k"].data_ptr(), v=S["v"].data_ptr(),
                 bounds=S["bounds"].data_ptr(), table=S["table"].data_ptr(), lens=S["lens"].data_ptr(),
                 refs=S["refs"].data_ptr(), status=S["status"].data_ptr())
    S["work"] = torch.zeros(rt.pages_work_ints(p), dtype=torch.int32, device=S["k"].device)
    p.work = S["work"].data_ptr()
    S["pages"] = p
    if case["op"] == "norm_rope":
        Hq, size, row = case["q_heads"], S["qkv"].element_size(), S["qkv"].stride(0)
        q = S["qkv"].data_ptr()
        gains = (S["q_gain"].data_ptr(), S["k_gain"].data_ptr()) if case["norm"] else (None, None)
        S["args"] = rt.QkRows(dtype=p.dtype, rows=S["rows"], q_heads=Hq, kv_heads=H, head_dim=D, q=q,
                              k=q + Hq * D * size, v=q + (Hq + H) * D * size, q_stride=row, k_stride=row,
                              v_stride=row, q_out=S["out"].data_ptr(), q_out_stride=Hq * D, q_gain=gains[0],
                              k_gain=gains[1], eps=1e-5, cos=S["cos"].data_ptr(), sin=S["sin"].data_ptr(),
                              positions=S["cos"].shape[0], interleaved=int(case["interleaved"]),
                              row_seq=S["row_seq"].data_ptr(), row_pos=S["row_pos"].data_ptr(),
                              status=S["status"].data_ptr())
    if case["op"] == "attention":
        S["args"] = rt.SparseQuery(rows=S["rows"], q_heads=case["q_heads"], q=S["q"].data_ptr(),
                                   q_stride=S["q"].stride(0), out=S["out"].data_ptr(), out_stride=S["out"].stride(0),
                                   row_seq=S["row_seq"].data_ptr(), row_pos=S["row_pos"].data_ptr(), scale=0.0,
                                   top_pages=case["top"], sink_pages=case["sink"], local_pages=case["local"],
                                   selected=S["selected"].data_ptr())


# ------------------------------------------------------------------------------------------------ one pass
def run(S):
    op = S["case"]["op"]
    if own:
        _run_own(op, S)
    elif op == "norm_rope":
        _plain_norm_rope(S)
    elif op == "attention":
        _plain_attention(S)
    elif op in ("fork", "copy"):
        _plain_free(S)
        _plain_fork(S, share=op == "fork")
    elif op == "compact":
        S["table"].copy_(S["before"][0])
        S["refs"].copy_(S["before"][1])
        _plain_compact(S)
    else:
        _plain_free(S)
        _plain_extend(S)
    if op == "norm_rope":
        at = S["layer"]
        return {"q": S["out"], "k": S["k"][at], "v": S["v"][at], "bounds": S["bounds"][at]}
    if op == "attention":
        return {"out": S["out"], "selected": S["selected"]}
    state = {"table": S["table"], "lens": S["lens"], "refs": S["refs"]}
    if op == "turnover":
        return state | {"row_seq": S["row_seq"], "row_pos": S["row_pos"]}
    return state | {"k": S["k"], "v": S["v"], "bounds": S["bounds"]}


def _run_own(op, S):
    from voxcpm2_b200 import runtime as rt
    stream = torch.cuda.current_stream().cuda_stream
    p = S["pages"]
    if op == "norm_rope":
        rt.qk_norm_rope(S["args"], p, S["layer"], stream)
    elif op == "attention":
        rt.sparse_attention(S["args"], p, S["layer"], stream)
    elif op in ("fork", "copy"):
        rt.pages_free(p, S["flags"].data_ptr(), stream)
        rt.pages_fork(p, S["parent"].data_ptr(), op == "fork", stream)
    elif op == "compact":
        # the fragmented tables of this case come back before every pass (the pages that move are overwritten with
        # what they already hold)
        S["table"].copy_(S["before"][0])
        S["refs"].copy_(S["before"][1])
        rt.pages_compact(p, S["used"].data_ptr(), stream)
    else:
        rt.pages_free(p, S["flags"].data_ptr(), stream)
        rt.pages_extend(p, S["counts"].data_ptr(), S["max_rows"], S["row_seq"].data_ptr(), S["row_pos"].data_ptr(),
                        stream)


def _plain_norm_rope(S):
    case, at = S["case"], S["layer"]
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    live = torch.nonzero(S["row_seq"] >= 0)[:, 0]
    pos, seq = S["row_pos"][live].long(), S["row_seq"][live].long()
    x = S["qkv"][live]
    qk = x[:, :Hq + Hkv].float()
    if case["norm"]:
        gain = torch.cat([S["q_gain"].float().expand(Hq, D), S["k_gain"].float().expand(Hkv, D)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-5) * gain
    c, s = S["cos"][pos, None, :D // 2], S["sin"][pos, None, :D // 2]
    if case["interleaved"]:
        a, b = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = qk[..., :D // 2], qk[..., D // 2:]
        qk = torch.cat([a * c - b * s, b * c + a * s], -1)
    qk = qk.to(x.dtype)
    S["out"][live] = qk[:, :Hq]
    keys = qk[:, Hq:].contiguous()
    page, slot = S["table"][seq, pos // case["page"]].long(), pos % case["page"]
    S["k"][at].transpose(1, 2)[page, slot] = keys
    S["v"][at].transpose(1, 2)[page, slot] = x[:, Hq + Hkv:]
    low, high = S["bounds"][at][:, :, 0], S["bounds"][at][:, :, 1]
    begun = page[slot == 0]
    low[begun], high[begun] = math.inf, -math.inf
    low.index_reduce_(0, page, keys, "amin")
    high.index_reduce_(0, page, keys, "amax")


def _plain_attention(S):
    case, at = S["case"], S["layer"]
    P, Hkv, D, top = case["page"], case["kv_heads"], case["head_dim"], case["top"]
    G = case["q_heads"] // Hkv
    live = torch.nonzero(S["row_seq"] >= 0)[:, 0]
    pos, seq = S["row_pos"][live].long(), S["row_seq"][live].long()
    R, q = live.numel(), S["q"][live].view(-1, Hkv, G, D)
    visible = pos // P + 1
    table = S["table"][seq].long().clamp(min=0)
    # the largest product that a key between the page's bounds can have with each query, summed over the group's heads
    q64 = q.double()
    up, down = q64.clamp(min=0).sum(2), q64.clamp(max=0).sum(2)
    low, high = (S["bounds"][at][:, :, i][table].double() for i in (0, 1))
    score = torch.einsum("rhd,rphd->rhp", up, high) + torch.einsum("rhd,rphd->rhp", down, low)
    score = torch.where(score.isnan(), math.inf, score)
    number = torch.arange(S["max_pages"], device=q.device)
    seen = number < visible[:, None]
    forced = seen & ((number < case["sink"]) | (number >= visible[:, None] - case["local"]))
    rank = torch.where(forced, 2, torch.where(seen, 1, 0))[:, None].expand_as(score)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)
    order = torch.nn.functional.pad(order, (0, max(0, top - S["max_pages"])))[..., :top]
    taken = torch.arange(top, device=q.device) < visible[:, None, None]
    chosen = torch.where(taken, order, 1 << 30).sort(dim=-1).values
    taken = chosen < (1 << 30)
    S["selected"][live] = torch.where(taken, chosen, -1).int()
    chosen = torch.where(taken, chosen, 0)
    ids = table[:, None].expand(R, Hkv, -1).gather(-1, chosen)
    head = torch.arange(Hkv, device=q.device)[:, None]
    keep = taken[..., None] & (chosen[..., None] * P + torch.arange(P, device=q.device) <= pos[:, None, None, None])
    keep = keep.flatten(2)
    k = S["k"][at][ids, head].flatten(2, 3).float().masked_fill(~keep[..., None], 0.0)
    x = torch.matmul(q.float(), k.transpose(-1, -2)) / math.sqrt(D)
    x = x.masked_fill(~keep[:, :, None], -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    v = S["v"][at][ids, head].flatten(2, 3).float().masked_fill(~keep[..., None], 0.0)
    S["out"][live] = (torch.matmul(w, v) / w.sum(-1, keepdim=True)).flatten(1, 2).to(S["out"].dtype)


def _held(S):
    """Which entries of the tables are in use."""
    need = (S["lens"] + S["case"]["page"] - 1) // S["case"]["page"]
    return torch.arange(S["max_pages"], device=need.device) < need[:, None]


def _free_ids(S, n):
    """The n lowest pages that nobody holds."""
    return torch.nonzero(S["refs"] == 0)[:n, 0]


def _plain_free(S):
    gone = _held(S) & (S["flags"] != 0)[:, None]
    ids = S["table"][gone].long()
    S["refs"].index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    S["table"].masked_fill_(gone, -1)
    S["lens"].masked_fill_(S["flags"] != 0, 0)


def _plain_fork(S, share):
    child = torch.nonzero(S["parent"] >= 0)[:, 0]
    parent = S["parent"][child].long()
    S["lens"][child] = S["lens"][parent]
    rows = S["table"][parent]
    held = _held(S)[child]
    if share:
        full = S["lens"][child] // S["case"]["page"]
        fresh = held & (torch.arange(S["max_pages"], device=full.device) >= full[:, None])
    else:
        fresh = held
    source = rows[fresh].long()
    ids = _free_ids(S, source.numel())
    common = rows[held & ~fresh].long()
    S["refs"].index_add_(0, common, torch.ones_like(common, dtype=torch.int32))
    S["refs"][ids] = 1
    rows[fresh] = ids.int()
    S["table"][child] = torch.where(held, rows, -1)
    for x in (S["k"], S["v"], S["bounds"]):
        x[:, ids] = x[:, source]


def _plain_extend(S):
    page, n = S["case"]["page"], S["counts"].numel()
    held = _held(S)
    begin = S["lens"].clone()
    S["lens"].add_(S["counts"])
    fresh = _held(S) & ~held
    need = int(fresh.sum())
    ids = _free_ids(S, need)
    S["refs"][ids] = 1
    S["table"][fresh] = ids.int()
    ends = S["counts"].cumsum(0)
    row = torch.arange(S["max_rows"], device=ends.device)
    seq = torch.searchsorted(ends, row, right=True).clamp(max=n - 1)
    pos = begin[seq] + row - (ends - S["counts"])[seq]
    S["row_seq"].copy_(torch.where(row < ends[-1], seq, -1))
    S["row_pos"].copy_(torch.where(row < ends[-1], pos, -1))


def _plain_compact(S):
    held = S["refs"] > 0
    count = held.sum()
    number = torch.arange(held.numel(), device=held.device)
    to = torch.nonzero(~held & (number < count))[:, 0]
    source = torch.nonzero(held & (number >= count))[:, 0]
    for x in (S["k"], S["v"], S["bounds"]):
        x[:, to] = x[:, source]
    S["refs"][to] = S["refs"][source]
    S["refs"][source] = 0
    number[source] = to
    S["table"].copy_(torch.where(S["table"] >= 0, number[S["table"].long().clamp(min=0)], -1))


# ------------------------------------------------------------------------------------------------ what it takes
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    page = case["page"]
    if case["op"] == "norm_rope":
        D, heads = case["head_dim"], case["q_heads"] + 2 * case["kv_heads"]
        rows = case["seqs"] * max(1, 0.75 * case["new"])
        touched = rows / page + case["seqs"]
        return {"bytes": rows * (2 * heads * D * size + 4 * D) + touched * case["kv_heads"] * 4 * D * size,
                "flops": rows * (case["q_heads"] + case["kv_heads"]) * D * 7}
    if case["op"] == "attention":
        D, Hkv, Hq = case["head_dim"], case["kv_heads"], case["q_heads"]
        rows = case["seqs"] * case["new"]
        pages = (case["past"] + case["least"]) / 2 / page + 1
        taken = min(case["top"], pages)
        each = min(case["seqs"] * pages, rows * taken)
        return {"bytes": rows * (2 * Hq * D * size + Hkv * case["top"] * 4) + case["seqs"] * pages * Hkv * 2 * D * size
                + each * Hkv * page * 2 * D * size,
                "flops": rows * (4 * Hq * taken * page * D + 4 * Hkv * pages * D)}
    one = case["layers"] * case["kv_heads"] * case["head_dim"] * size * (2 * page + 2)
    tokens = 0.75 * case["tokens"]
    table = 4 * case["pool"]
    if case["op"] == "fork":
        return {"bytes": case["children"] * (2 * one + 8 * tokens / page) + table, "flops": 0}
    if case["op"] == "copy":
        return {"bytes": case["children"] * (tokens / page + 0.5) * 2 * one + table, "flops": 0}
    if case["op"] == "compact":
        used = min(case["seqs"] * (tokens / page + 0.5), case["pool"])
        return {"bytes": used * (1 - used / case["pool"]) * 2 * one + 2 * table, "flops": 0}
    return {"bytes": 2 * table + 8 * case["ending"] * case["tokens"] / 2, "flops": 0}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] not in ("norm_rope", "attention"):
        return None  # whole numbers, and values that are only copied
    S = prepare(case, seed)
    P, D, Hkv, Hq, at = case["page"], case["head_dim"], case["kv_heads"], case["q_heads"], S["layer"]
    seqs, poss = S["row_seq"].tolist(), S["row_pos"].tolist()
    table = S["table"].tolist()
    live = [r for r, s in enumerate(seqs) if s >= 0]
    if case["op"] == "norm_rope":
        x = S["qkv"].double()
        if case["norm"]:
            for part, gain in ((x[:, :Hq], S["q_gain"]), (x[:, Hq:Hq + Hkv], S["k_gain"])):
                part /= torch.sqrt(part.square().sum(-1, keepdim=True) / D + 1e-5)
                part *= gain.double()
        # pairs as complex numbers, turned by the table's angle
        pairs = x.view(*x.shape[:2], D // 2, 2) if case["interleaved"] else x.view(*x.shape[:2], 2, D // 2).transpose(2, 3)
        turn = torch.complex(S["cos"].double(), S["sin"].double())[S["row_pos"].long().clamp(min=0), None, :D // 2]
        z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        z = z.flatten(2) if case["interleaved"] else z.transpose(2, 3).flatten(2)
        q, k, v, b = S["out"].double(), S["k"][at].double(), S["v"][at].double(), S["bounds"][at].double()
        q[live] = z[live, :Hq]
        page = torch.tensor([table[seqs[r]][poss[r] // P] for r in live], device=q.device)
        slot = torch.tensor([poss[r] % P for r in live], device=q.device)
        rows = torch.tensor(live, device=q.device)
        for j in range(Hkv):
            k[page, j, slot] = z[rows, Hq + j]
            v[page, j, slot] = x[rows, Hq + Hkv + j]
        last = {}
        for r in live:
            last[table[seqs[r]][poss[r] // P]] = poss[r] % P + 1
        for p, n in last.items():
            b[p, :, 0], b[p, :, 1] = k[p, :, :n].amin(1), k[p, :, :n].amax(1)
        return {"q": q, "k": k, "v": v, "bounds": b}
    out = S["out"].double()
    selected = torch.zeros((S["rows"], Hkv, case["top"]), dtype=torch.int32)
    G = Hq // Hkv
    cache = {}
    for r in live:
        s, p = seqs[r], poss[r]
        n = p // P + 1
        if s not in cache:
            ids = torch.tensor(table[s][:-(-int(S["lens"][s]) // P)], device=out.device)
            cache = {s: [t[at][ids].double() for t in (S["k"], S["v"], S["bounds"])]}
        k, v, b = (t[:n] for t in cache[s])
        q = S["q"][r].double().view(Hkv, G, D)
        reach = torch.maximum(q[None] * b[:, :, 0, None], q[None] * b[:, :, 1, None]).sum((2, 3))  # [n, Hkv]
        must = set(range(min(case["sink"], n))) | set(range(max(0, n - case["local"]), n))
        if n <= case["top"]:
            lists = [list(range(n))] * Hkv
        else:
            ranked = (-reach).T.contiguous().sort(dim=-1, stable=True).indices.tolist()
            lists = [sorted(list(must) + [i for i in order if i not in must][:case["top"] - len(must)])
                     for order in ranked]
        choice = torch.tensor(lists, device=out.device)  # [Hkv, m]
        selected[r] = -1
        selected[r, :, :choice.shape[1]] = choice.int().cpu()
        head = torch.arange(Hkv, device=out.device)[:, None]
        kk, vv = k[choice, head].reshape(Hkv, -1, D), v[choice, head].reshape(Hkv, -1, D)
        where = (choice[:, :, None] * P + torch.arange(P, device=out.device)).reshape(Hkv, -1)
        kk[where > p], vv[where > p] = 0, 0
        x = (q @ kk.transpose(1, 2) / math.sqrt(D)).masked_fill((where > p)[:, None], -math.inf)
        out[r] = (torch.softmax(x, -1) @ vv).reshape(Hq, D)
    return {"out": out, "selected": selected}
