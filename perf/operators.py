"""The paged key-value cache: what is measured of the operators that write and read it.

Sequences of uneven length share one pool of pages ``[pages, kv_heads, page, 128]`` for K and one for V; ``block_table[b, i]``
names the page that holds positions ``i * page .. (i + 1) * page - 1`` of sequence ``b``.

Operators (``op`` of a case):
    append   keys and values of new tokens, RMS-normalised and rotated to their positions, stored in their pages; the tokens'
             queries, normalised and rotated, returned beside them in the pages' type
    decode   one new token of every sequence: attention over the cached rows (the nearest ``window - 1``) and the token's own,
             which is stored
    attend   queries of a chunk of every sequence, whose keys and values are already in the pages, causal over everything
             cached before them (``window`` nearest); the queries have the pages' type
"""
from __future__ import annotations

import math

import torch

own = False

D = 128                      # head dimension of every configuration
SCALE = 0.12                 # the module's attention scale
EPS = 2.0 ** -23             # of the RMS norms
MAX_POSITIONS = 131072       # the module's RoPE table
ROW_HEADS = 64 * 4096 * 16   # cached rows x key heads that the largest decode step reads
PAIRS = 8192 * 61440 * 16    # (query, key, head) triples of the largest chunk


def listed():
    return [
        # the smallest call: one token of one chat on the small model (six heads)
        dict(name="append_token", op="append", seqs=1, tokens=1, ragged=False, start=700, heads=6, kv_heads=6, page=16, f16=False),
        # eleven prompts of uneven length packed in one row, some continuing a cached prefix
        dict(name="append_ragged", op="append", seqs=11, tokens=701, ragged=True, start=300, heads=16, kv_heads=16, page=64, f16=False),
        # whole prompts of a full batch, keys and values kept as float16
        dict(name="append_batch", op="append", seqs=8, tokens=8192, ragged=False, start=0, heads=16, kv_heads=16, page=128, f16=True),
        # a chat turn's next token on the small model, short window: latency
        dict(name="decode_token", op="decode", seqs=1, ctx=700, ragged=False, heads=6, kv_heads=6, window=512, page=16, f16=False),
        # a handful of conversations of uneven length, float16 cache
        dict(name="decode_few", op="decode", seqs=5, ctx=5003, ragged=True, heads=16, kv_heads=16, window=4096, page=64, f16=True),
        # batched serving: 64 conversations past the window
        dict(name="decode_batch", op="decode", seqs=64, ctx=9001, ragged=False, heads=16, kv_heads=16, window=4097, page=64, f16=False),
        # query heads in groups of four over shared key heads, lengths between a few tokens and the longest
        dict(name="decode_grouped", op="decode", seqs=24, ctx=16384, ragged=True, heads=32, kv_heads=8, window=0, page=32, f16=False),
        # one long document: a single sequence has to be split over the whole device
        dict(name="decode_long", op="decode", seqs=1, ctx=131071, ragged=False, heads=16, kv_heads=16, window=0, page=256, f16=False),
        # a short, ragged prompt on the small model, nothing cached before it
        dict(name="attend_short", op="attend", seqs=1, tokens=131, prior=0, ragged=False, heads=6, kv_heads=6, window=512, page=16, f16=False, bounded=True),
        # a few drafted tokens of each conversation, to be verified together
        dict(name="attend_draft", op="attend", seqs=8, tokens=5, prior=9001, ragged=True, heads=16, kv_heads=16, window=4096, page=64, f16=False, bounded=True),
        # pieces of several prompts packed together, each behind its cached prefix
        dict(name="attend_ragged", op="attend", seqs=7, tokens=2048, prior=8192, ragged=True, heads=16, kv_heads=16, window=4096, page=64, f16=False, bounded=True),
        # the last piece of a long document
        dict(name="attend_long", op="attend", seqs=1, tokens=8192, prior=57344, ragged=False, heads=16, kv_heads=16, window=0, page=128, f16=False, bounded=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "decode", "attend"])
    kv = rng.choice([1, 2, 6, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 1, 2, 4, 8])
    if heads > 48:
        heads = kv
    case = dict(op=op, seqs=1, ragged=rng.random() < 0.6, heads=heads, kv_heads=kv, page=rng.choice([16, 32, 64, 128, 256]), f16=rng.random() < 0.4)
    if op == "append":
        tokens = _log(rng, 1, 8192)
        most = 65536 * 48 // (heads + 2 * kv)                     # rows of q, k and v of the largest listed call
        case.update(tokens=tokens, seqs=_log(rng, 1, max(1, min(256, most // tokens))), start=rng.choice([0, _log(rng, 1, 32768)]))
    elif op == "decode":
        ctx, window = _log(rng, 1, MAX_POSITIONS - 1), rng.choice([0, _log(rng, 128, 8192)])
        rows = min(ctx, window - 1) if window else ctx
        case.update(ctx=ctx, window=window, seqs=_log(rng, 1, max(1, min(128, ROW_HEADS // (rows * kv)))))
    else:
        tokens, prior, window = _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 57344)]), rng.choice([0, _log(rng, 128, 8192)])
        keys = prior + tokens
        rows = min(keys, window + tokens) if window else keys
        most = min(PAIRS // (tokens * rows * heads), 2 * ROW_HEADS // (keys * kv), 65536 // tokens)
        case.update(tokens=tokens, prior=prior, window=window, seqs=_log(rng, 1, max(1, min(32, most))), bounded=rng.random() < 0.7)
    return case


# ---------------------------------------------------------------------------------------------- lengths
def _spread(case, most, least, row=0):
    """A length for every sequence: all ``most``, or uneven ones between (multiples of the golden ratio)."""
    n = case["seqs"]
    if not case["ragged"]:
        return [most] * n
    return [max(least, int(round(most * ((0.6180339887 * (i + 1) + 0.31 * row) % 1.0)))) for i in range(n)]


def _lengths(case):
    """-> (tokens already cached, new tokens) of every sequence."""
    if case["op"] == "append":
        return _spread(case, case["start"], 0, 1), _spread(case, case["tokens"], 1)
    if case["op"] == "decode":
        return _spread(case, case["ctx"], 0), [1] * case["seqs"]
    return _spread(case, case["prior"], 0, 1), _spread(case, case["tokens"], 1)


def _first(case, p):
    """First position that a query at position ``p`` sees."""
    w = case.get("window", 0)
    return max(0, p - w + 1) if w else 0


# ---------------------------------------------------------------------------------------------- preparation
def _unit(shape, dtype):
    """Rows as the norm leaves them: root mean square one."""
    x = torch.randn(shape, dtype=torch.float32, device="cuda")
    x *= (x.square().mean(-1, keepdim=True) + EPS).rsqrt_()
    return x.to(dtype)


def _tables():
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _pool(case, cached, new):
    """Pages in a shuffled order, as an allocator in use hands them out; none where no later query looks (pages behind the window
    have been given back).  Cached rows are normalised keys and values, rows that nobody wrote yet are zero."""
    page, kv = case["page"], case["kv_heads"]
    dtype = torch.float16 if case["f16"] else torch.bfloat16
    spans = []                                                    # pages [first, end) of every sequence
    for c, n in zip(cached, new):
        first = 0 if case["op"] == "append" else _first(case, c)
        spans.append((first // page if case["op"] != "append" else c // page, -(-(c + n) // page)))
    total = sum(e - f for f, e in spans)
    order = torch.randperm(total + 3, device="cuda").to(torch.int32)
    table = torch.full((case["seqs"], max(e for _, e in spans)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (f, e) in enumerate(spans):
        table[b, f:e] = order[at:at + e - f]
        at += e - f
    k = torch.zeros(total + 3, kv, page, D, dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    if case["op"] != "append":
        plain = case["op"] == "attend" and not case["bounded"]    # a model without a norm on q and k
        for pool in (k, v):
            for i in range(0, pool.shape[0], 256):
                part = pool[i:i + 256]
                part.copy_(torch.randn(part.shape, device="cuda") * 0.7 if plain else _unit(part.shape, dtype))
    return k, v, table


def prepare(case, seed):
    torch.manual_seed(seed)
    cached, new = _lengths(case)
    n, H, KV = sum(new), case["heads"], case["kv_heads"]
    k_pages, v_pages, table = _pool(case, cached, new)
    ints = dict(dtype=torch.int32, device="cuda")
    s = dict(op=case["op"], k_pages=k_pages, v_pages=v_pages, table=table, cached=cached, new=new, window=case.get("window", 0))
    normal = lambda *shape: torch.randn(*shape, device="cuda").bfloat16()
    if case["op"] == "attend":
        s["bounded"] = case["bounded"]
        q = _unit((n, H, D), k_pages.dtype) if case["bounded"] else (torch.randn(n, H, D, device="cuda") * 1.5).to(k_pages.dtype)
        s["lens"] = torch.tensor([c + m for c, m in zip(cached, new)], **ints)
    else:
        # views of one merged projection, as the layer's GEMM leaves it
        qkv = normal(n, H + 2 * KV, D)
        q, s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        s["cos"], s["sin"] = _tables()
        s["lens"] = torch.tensor(cached, **ints)
    s["q"], s["cu"] = q, None
    if case["op"] != "decode" and case["ragged"]:                 # packed in one row; a batch of equal lengths is dense
        s["cu"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], **ints)
        shape = (1, n)
    else:
        shape = (case["seqs"], n // case["seqs"])
    for name in ("q", "k", "v"):
        if name in s:
            s[name] = s[name].unflatten(0, shape)
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from daisy_b200 import ops
    window = s["window"] or None
    if s["op"] == "append":
        q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cos"], s["sin"], cu_seqlens=s["cu"], q=s["q"], eps=EPS)
        return s["k_pages"], s["v_pages"], q
    if s["op"] == "decode":
        y = ops.paged_decode_step(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], window, s["cos"], s["sin"], eps=EPS)
        return s["k_pages"], s["v_pages"], y
    y = ops.paged_attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], window, cu_seqlens=s["cu"], bounded_qk=s["bounded"])
    return y


# ---------------------------------------------------------------------------------------------- plain form, 32 bits
def _norm(x):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rotate(x, cos, sin):
    a, b = x[..., :D // 2], x[..., D // 2:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos + b * sin, b * cos - a * sin], -1)


def _store(s, k, v, seq, pos):
    """Rows ``k, v [n, kv_heads, D]`` to the pages of their sequences and positions."""
    page = s["k_pages"].shape[2]
    at = s["table"][seq, pos // page].long()
    s["k_pages"][at, :, pos % page] = k
    s["v_pages"][at, :, pos % page] = v


def _context(s, b, first, end):
    """Rows ``first .. end - 1`` of sequence ``b`` as ``[kv_heads, rows, D]`` in 32 bits."""
    page = s["k_pages"].shape[2]
    at = s["table"][b, first // page:-(-end // page)].long()
    cut = slice(first % page, first % page + end - first)
    return tuple(pool[at].transpose(0, 1).flatten(1, 2)[:, cut].float() for pool in (s["k_pages"], s["v_pages"]))


def _softmax_product(q, k, v, hidden):
    """``q [kv, G, n, D]`` over ``k, v [kv, rows, D]``; ``hidden [n, rows]`` or None."""
    z = torch.matmul(q, k[:, None].transpose(-1, -2)) * SCALE
    if hidden is not None:
        z.masked_fill_(hidden, -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    return torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)


def _plain(s):
    cached, new = s["cached"], s["new"]
    kv = s["k_pages"].shape[1]
    if s["op"] == "attend":
        q = s["q"].flatten(0, 1)
        out = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")
        H, at = q.shape[1], 0
        for b, (c, n) in enumerate(zip(cached, new)):
            step = max(1, (1 << 27) // (H * (c + n)))
            for i in range(0, n, step):
                m = min(step, n - i)
                lo = max(0, c + i - s["window"] + 1) if s["window"] else 0
                k, v = _context(s, b, lo, c + i + m)
                gap = torch.arange(c + i, c + i + m, device="cuda")[:, None] - torch.arange(lo, c + i + m, device="cuda")[None, :]
                hidden = (gap < 0) | (gap >= s["window"]) if s["window"] else gap < 0
                x = q[at + i:at + i + m].float().unflatten(1, (kv, H // kv)).permute(1, 2, 0, 3)
                out[at + i:at + i + m] = _softmax_product(x, k, v, hidden).permute(2, 0, 1, 3).flatten(1, 2).bfloat16()
            at += n
        return out.view_as(s["q"])
    counts = torch.tensor(new, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), counts)
    pos = torch.arange(len(seq), device="cuda") - (counts.cumsum(0) - counts)[seq] + s["lens"].long()[seq]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(_norm(s["q"].flatten(0, 1)), cos, sin)
    k = _rotate(_norm(s["k"].flatten(0, 1)), cos, sin).to(s["k_pages"].dtype)
    v = _norm(s["v"].flatten(0, 1)).to(s["v_pages"].dtype)
    _store(s, k, v, seq, pos)
    if s["op"] == "append":
        return s["k_pages"], s["v_pages"], q.to(s["k_pages"].dtype).view(s["q"].shape)
    out = torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda")
    for b, c in enumerate(cached):
        kc, vc = _context(s, b, max(0, c - s["window"] + 1) if s["window"] else 0, c + 1)
        y = _softmax_product(q[b].unflatten(0, (kv, -1))[:, :, None], kc, vc, None)
        out[b, 0] = y.flatten(0, 2).bfloat16()
    return s["k_pages"], s["v_pages"], out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- 64 bits, from the definition
def exact(case, seed):
    s = prepare(case, seed)
    cached, new = _lengths(case)
    page, KV, H = case["page"], case["kv_heads"], case["heads"]
    G = H // KV
    table = s["table"].tolist()
    keys, values = s["k_pages"], s["v_pages"]
    q = s["q"].flatten(0, 1)
    if case["op"] != "attend":
        def prepared(x, p, turn):
            x = x.double()
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS)
            if not turn:
                return x
            c, t = s["cos"][p].double()[:, None], s["sin"][p].double()[:, None]
            lo, hi = x.split(D // 2, dim=-1)
            return torch.cat((lo * c + hi * t, hi * c - lo * t), dim=-1)
        k_new, v_new = s["k"].flatten(0, 1), s["v"].flatten(0, 1)
        out_q, out_k, out_v, at = [], [], [], 0
        for c, n in zip(cached, new):
            p = torch.arange(c, c + n, device=q.device)
            out_q.append(prepared(q[at:at + n], p, True))
            out_k.append(prepared(k_new[at:at + n], p, True))
            out_v.append(prepared(v_new[at:at + n], p, False))
            at += n
    if case["op"] == "append":
        keys, values = keys.double(), values.double()
        for b, (c, n) in enumerate(zip(cached, new)):
            for i in range(n if n < page else 0):
                keys[table[b][(c + i) // page], :, (c + i) % page] = out_k[b][i]
                values[table[b][(c + i) // page], :, (c + i) % page] = out_v[b][i]
            if n >= page:                                         # page by page
                for j in range(c // page, (c + n - 1) // page + 1):
                    lo, hi = max(c, j * page), min(c + n, (j + 1) * page)
                    keys[table[b][j], :, lo - j * page:hi - j * page] = out_k[b][lo - c:hi - c].transpose(0, 1)
                    values[table[b][j], :, lo - j * page:hi - j * page] = out_v[b][lo - c:hi - c].transpose(0, 1)
        return keys, values, torch.cat(out_q).view(s["q"].shape)
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    at = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        end = c + n
        rows_of = lambda pool, h, lo: torch.cat([pool[table[b][j], h] for j in range(lo // page, -(-end // page))])[lo % page:][:end - lo].double()
        for h in range(KV):
            first = _first(case, c)
            kh, vh = rows_of(keys, h, first), rows_of(values, h, first)
            if case["op"] == "decode":                            # the token's own row, not yet in the pages
                kh[-1], vh[-1] = out_k[b][0, h], out_v[b][0, h]
            step = max(1, (1 << 25) // len(kh))
            for g in range(h * G, (h + 1) * G):
                for i in range(0, n, step):
                    m = min(step, n - i)
                    x = out_q[b][i:i + m, g] if case["op"] == "decode" else q[at + i:at + i + m, g].double()
                    p = torch.arange(c + i, c + i + m, device=q.device).unsqueeze(1)
                    j = torch.arange(first, end, device=q.device).unsqueeze(0)
                    seen = j <= p
                    if case["window"]:
                        seen &= j > p - case["window"]
                    z = torch.where(seen, (x @ kh.t()) * SCALE, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
                    out[at + i:at + i + m, g] = torch.softmax(z, dim=-1) @ vh
        at += n
    out = out.view(s["q"].shape)
    # the pools of a decode step hold what they held but for one row of each sequence: in 64 bits they would not fit beside them
    return (None, None, out) if case["op"] == "decode" else out


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    cached, new = _lengths(case)
    n, H, KV = sum(new), case["heads"], case["kv_heads"]
    row = 2 * D
    if case["op"] == "append":
        # q, k, v read, q' and the stored rows written, a table row of either kind for every position
        positions = len(set(p for c, m in set(zip(cached, new)) for p in range(c, c + m)))
        return dict(bytes=2 * n * (H + 2 * KV) * row + positions * 4 * D + 4 * n / case["page"], flops=n * (H * 7 + KV * 10) * D)
    if case["op"] == "decode":
        rows = [c - _first(case, c) for c in cached]
        return dict(bytes=sum(rows) * KV * 2 * row + n * (2 * H + 4 * KV) * row, flops=4 * D * H * sum(r + 1 for r in rows))
    w, pairs, rows = case["window"], 0, 0
    for c, m in zip(cached, new):
        rows += c + m - _first(case, c)
        full = min(m, max(0, w - c)) if w else m                  # queries that see everything before them
        pairs += full * c + full * (full + 1) // 2 + (m - full) * w
    return dict(bytes=2 * n * H * row + rows * KV * 2 * row, flops=4 * D * H * pairs)
