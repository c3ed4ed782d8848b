"""Calls of the paged cache at the borders of what its documentation allows, against the formula in 64 bits.  Tolerances as in
``test_gpu_paged``; what a case adds to them stands beside it."""
import math

import pytest
import torch

from gpu_util import assert_close_bf16
from test_gpu_paged import (D, EPS, SCALE, Pool, _attend_tol, _attention, _check, _decode_tol, _gen, _ints, _randn, _stack, _status,
                            _tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [0, 3, 40])
def test_float16_weights_far_below_the_largest(T):
    """One key at weight 1 whose value is zero, 4096 behind it at 2^-25.3: all of the result.  T = 0: the one-token step; 3 and 40: chunks of
    either kernel.  As many (sequence, head) pairs as leave every warp a long run of rows."""
    from daisy_b200 import ops
    n, H, page, rows = 64, 16, 256, 4096
    k_pages = torch.zeros(rows // page + n, H, page, D, dtype=torch.float16, device="cuda")
    pattern = 0.5 + torch.arange(D, dtype=torch.float64) % 8 / 8
    v_pages = pattern.half().cuda().expand(k_pages.shape).contiguous()
    k_pages[0, :, 0], v_pages[0, :, 0] = 73 / 64, 0.0
    table = torch.cat([torch.arange(rows // page).expand(n, -1), rows // page + torch.arange(n)[:, None]], 1).int().cuda()
    one = torch.ones(n, max(T, 1), H, D, dtype=torch.float16 if T else torch.bfloat16, device="cuda")
    lens = _ints([rows] * n)
    if T:
        y = ops.paged_attend(one, k_pages, v_pages, table, lens, None)
        tail = rows - T + torch.arange(T)                            # rows behind the first that each query sees
    else:
        own = pattern.bfloat16().cuda().expand(n, 1, H, D).contiguous()
        y = ops.paged_decode_step(one, torch.zeros_like(one), own, k_pages, v_pages, table, lens, None, None, None, flags=0)
        tail = torch.tensor([rows])
    _status()
    top = SCALE * D * 73 / 64
    mass = tail.double() * math.exp(-top)
    ref = (mass / (1 + mass))[:, None] * pattern                     # [T, D]; values are positive: also the mean of |v|
    top_mass = torch.full((len(tail),), D * 73 / 64, dtype=torch.float64)
    tol = _attend_tol(ref, ref, top_mass, 0, torch.float16, 0.0, False) + rows * 2.0 ** -23 * ref if T == 40 else _decode_tol(ref, ref, top_mass, rows)
    # float16 weights have a floor of 2^-32 of the largest, each row's
    tol = tol + rows * 2.0 ** -32 * pattern
    assert (2.0 ** -5 * ref > tol).all()
    over = (y.double().cpu() - ref[None, :, None]).abs() - tol[None, :, None]
    assert (over <= 0).all(), f"{over.max().item():.3g} over the tolerance; off by up to {((y.double().cpu() / ref[None, :, None]) - 1).abs().max().item():.3g} of the value"


def test_tokens_behind_the_rope_table():
    """A block table longer than the RoPE table: what is stored stays stored, refused tokens' queries and their sequences' outputs are zero."""
    from daisy_b200 import _lib, ops
    H, page, T, rope = 2, 16, 20, 50
    cos, sin = (t.cuda() for t in _tables(rope))
    x = _randn(_gen(1), 3, T, 3 * H, D).cuda()
    table = torch.arange(12).view(3, 4).int().cuda()                 # 64 positions a sequence
    start = _ints([0, 40, 60])                                       # inside; across the RoPE table's end; across both ends
    fill = float("nan")
    k_pages = torch.full((12, H, page, D), fill, dtype=torch.bfloat16, device="cuda")
    v_pages = k_pages.clone()
    # the queries' memory comes from the allocator: leave NaN there
    del_me = torch.full((3, T, H, D), fill, dtype=torch.bfloat16, device="cuda")
    del del_me
    q = ops.paged_append(x[:, :, H:2 * H], x[:, :, 2 * H:], k_pages, v_pages, table, start, cos, sin, q=x[:, :, :H], eps=EPS)
    _status(_lib.EINVAL)
    assert torch.isfinite(q.float()).all() and (q[1, 10:] == 0).all() and (q[2] == 0).all() and (q[1, :10] != 0).any(-1).all()
    for T_q in (T, 3):                                               # both kernels
        y = ops.paged_attend(q[:, -T_q:], k_pages, v_pages, table, start + T, None, bounded_qk=True, max_len=rope)
        _status(_lib.EINVAL)
        assert (y[1:] == 0).all() and torch.isfinite(y.float()).all()
        alone = ops.paged_attend(q[:1, -T_q:], k_pages, v_pages, table[:1], start[:1] + T, None, bounded_qk=True)
        _status()
        assert torch.equal(y[:1], alone)
        # up to the limit and no further
        assert (ops.paged_attend(q[:1, -T_q:], k_pages, v_pages, table[:1], _ints([T]), None, bounded_qk=True, max_len=T) == alone).all()
        _status()
        assert (ops.paged_attend(q[:1, -T_q:], k_pages, v_pages, table[:1], _ints([T]), None, bounded_qk=True, max_len=T - 1) == 0).all()
        _status(_lib.EINVAL)
    with pytest.raises(ValueError):
        ops.paged_attend(q[:1], k_pages, v_pages, table[:1], _ints([T]), None, max_len=-1)


def test_layer_prompt_behind_the_rope_table():
    from daisy_b200 import B200CausalSelfAttention, B200PagedKVCache, _lib
    H, dim = 2, 256
    torch.manual_seed(3)
    a = B200CausalSelfAttention(dim, H, D, max_seq_len=64)
    with torch.no_grad():
        a.qkvo_w.copy_(torch.randn(4, dim, dim) * dim ** -0.5)
    a = a.cuda()
    assert a.rotary.cos.shape[0] == 64
    cache = B200PagedKVCache(1, 16, H, D, 2, 128, "cuda", page=16)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    slots = [cache.claim(), cache.claim()]
    cache.reserve(slots, 70)
    x = torch.randn(2, 70, dim, generator=_gen(2)).bfloat16().cuda()
    with torch.inference_mode():
        y = a.prefill_paged(x[:, :64], None, cache, 0, cache.table, _ints([0, 6]), _ints([64, 70]), None)
    _status(_lib.EINVAL)
    assert torch.isfinite(y.float()).all() and (y[1] == 0).all() and (y[0] != 0).any()


@pytest.mark.parametrize("T", [3, 40])
def test_chunks_over_a_very_wide_table(T):
    """A short chunk over a table with more blocks than the form for few queries counts goes by the other one."""
    from daisy_b200 import ops
    n, page, width, lens = 128, 256, 2 ** 22, 300
    g = _gen(7)
    k, v = (_randn(g, 2, 1, page, D) for _ in range(2))
    q = torch.randn(n, T, 1, D, generator=g).bfloat16()
    row = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    row[0, :2] = _ints([1, 0])
    y = ops.paged_attend(q.cuda(), k.cuda(), v.cuda(), row.expand(n, -1), _ints([lens - b for b in range(n)]), None)
    _status()
    kk, vv = (x.flip(0)[:, 0].flatten(0, 1)[None].double() for x in (k, v))
    for b in range(n):
        seen = torch.arange(2 * page)[None] <= (lens - b - T + torch.arange(T))[:, None]
        ref, A, mass = _attention(q[b].double(), kk, vv, seen)
        _check(y[b], ref, _attend_tol(ref, A, mass, lens, torch.bfloat16, 0.0, False), f"sequence {b}")


@pytest.mark.parametrize("window,page", [(None, 16), (90, 32), (33, 64)])
@pytest.mark.parametrize("graph", [False, True])
def test_runner_out_of_pages(window, page, graph):
    """Prompts and steps that the pool has no pages for are refused with nothing changed, and served once a sequence has ended."""
    from daisy_b200 import PagedRunner
    H, dim = 1, D
    runner = PagedRunner(_stack(1, H, dim), window, pages=6, max_seqs=2, max_len=6 * page, page=page)
    if graph:
        runner.capture_step(dim)
    step = runner.step_graph if graph else runner.step
    c = runner.cache
    g = _gen(11)

    def prompt(n):
        return torch.randn(n, dim, generator=g).bfloat16().cuda()

    def state():
        return list(c.length), [list(r) for r in c.book.table], sorted(c.book.free), c.lens.tolist(), c.table.tolist()
    a, b = runner.add(), runner.add()
    runner.prefill([prompt(page), prompt(page)], [a, b])             # full pages: the next token needs one each
    held = {s: c.book.end[s] - c.book.first[s] for s in (a, b)}
    assert held == {a: 1, b: 1}
    before = state()
    with pytest.raises(RuntimeError, match="4 pages left"):
        runner.prefill([prompt(4 * page), prompt(1)], [a, b])
    assert state() == before
    runner.prefill([prompt(3 * page)], [a])
    while c.book.free:                                               # (pages behind a window have come back); a's are full
        c.reserve([b], (c.book.end[b] + 1) * page - c.length[b])
    before = state()
    x = torch.randn(2, 1, dim, generator=g).bfloat16().cuda()
    with pytest.raises(RuntimeError, match="0 pages left"):
        step(x)
    assert state() == before
    runner.drop(b)
    y = step(x)
    assert torch.isfinite(y).all() and (y[a] != 0).any() and (y[b] == 0).all() and c.length == [4 * page + 1, -1]
    _status()


@pytest.mark.parametrize("T", [8, 9, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_and_outputs_are_taken_whatever_a_chunk_goes_by(T, dtype):
    """Broadcast queries and results on 8-byte boundaries: of chunks for either kernel (8 and 9 are the border), with the bits of a plain call."""
    from daisy_b200 import ops
    n, H, page, N = 3, 2, 32, 2 * T
    pool = Pool([70, 100, 64], [0] * n, H, page, dtype, seed=201)
    k_pages, v_pages, table = pool.gpu()
    lens = _ints([70, 100, 64])
    q = (torch.randn(n, T, H, D, generator=_gen(202)) / 3).to(dtype).cuda()
    for view in (q[:1].expand(n, -1, -1, -1), q[:, :1].expand(-1, T, -1, -1), q[:, :, :1].expand(-1, -1, H, -1)):
        plain = ops.paged_attend(view.contiguous(), k_pages, v_pages, table, lens, 50)
        assert torch.equal(ops.paged_attend(view, k_pages, v_pages, table, lens, 50), plain)
    for at in (0, 4):                                                # rows 264 bytes apart, from a 16-byte boundary and from an 8-byte one
        wide = torch.full((n, T, H, D + 4), 3.0, dtype=torch.bfloat16, device="cuda")
        out = wide[..., at:at + D]
        assert ops.paged_attend(view, k_pages, v_pages, table, lens, 50, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, plain) and (wide[..., D:] == 3.0 if at == 0 else wide[..., :4] == 3.0).all()
    # packed, with tokens of nobody behind: their rows stay
    packed, cu = q.flatten(0, 1)[None, :N + 3], _ints([0, T, N, N])
    plain = ops.paged_attend(packed, k_pages, v_pages, table, lens, 50, cu_seqlens=cu, out=torch.full_like(packed, 9.0, dtype=torch.bfloat16))
    out = torch.full((1, N + 3, H, D + 4), 9.0, dtype=torch.bfloat16, device="cuda")[..., 4:]
    ops.paged_attend(packed, k_pages, v_pages, table, lens, 50, cu_seqlens=cu, out=out)
    assert torch.equal(out, plain) and (out[:, N:] == 9.0).all()
    for shared in (torch.empty(1, T, H, D), torch.empty(n, 1, H, D), torch.empty(n, T, 1, D)):
        with pytest.raises(ValueError, match="broadcast"):
            ops.paged_attend(q, k_pages, v_pages, table, lens, 50, out=shared.bfloat16().cuda().expand(n, T, H, D))
    x = _randn(_gen(203), n, 1, 3 * H, D).cuda().split(H, 2)
    for shared in (torch.empty(1, 1, H, D), torch.empty(n, 1, 1, D)):
        with pytest.raises(ValueError, match="broadcast"):
            ops.paged_decode_step(*x, k_pages, v_pages, table, lens, None, None, None, flags=0, out=shared.bfloat16().cuda().expand(n, 1, H, D))
    _status()


def _laid_out(pool, layout):
    """The same pool with other strides: rows of all heads together, heads outermost, or gaps between rows, heads and pages."""
    n, H, page, _ = pool.shape
    if layout == "rows first":
        return pool.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "heads outermost":
        return pool.transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((n, H + 1, page + 1, D + 16), 7.0, dtype=pool.dtype, device="cuda")
    view = big[:, :H, :page, 8:8 + D]
    view.copy_(pool)
    return view


@pytest.mark.parametrize("layout", ["rows first", "heads outermost", "gaps"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pools_of_any_strides(layout, page, dtype):
    """Every call over a pool laid out otherwise has the bits of the same call over the contiguous one, in the results and in the pages."""
    from daisy_b200 import ops
    H, G, lens, T = 3, 2, [300, 0, 77, 530], 90
    pool = Pool(lens, [T + 1] * 4, H, page, dtype, seed=211)
    x = _randn(_gen(212), 4, T, (G + 2) * H, D).cuda()
    one = _randn(_gen(213), 4, 1, (G + 2) * H, D).cuda()
    cos, sin = (t.cuda() for t in _tables())
    got = []
    for relaid in (False, True):
        k, v, table = pool.gpu()
        if relaid:
            k, v = _laid_out(k, layout), _laid_out(v, layout)
            assert not k.is_contiguous()
        q = ops.paged_append(x[:, :, G * H:(G + 1) * H], x[:, :, (G + 1) * H:], k, v, table, _ints(lens), cos, sin, q=x[:, :, :G * H], eps=EPS)
        after = _ints([n + T for n in lens])
        res = [q]
        for window in (None, 100):
            for bounded in (True, False):
                res.append(ops.paged_attend(q, k, v, table, after, window, bounded_qk=bounded))
                res.append(ops.paged_attend(q[:, -3:], k, v, table, after, window, bounded_qk=bounded))
        res.append(ops.paged_decode_step(one[:, :, :G * H], one[:, :, G * H:(G + 1) * H], one[:, :, (G + 1) * H:], k, v, table, after, 100, cos, sin, eps=EPS))
        got.append(res + [k.contiguous().view(torch.int16), v.contiguous().view(torch.int16)])
    _status()
    for i, (a, b) in enumerate(zip(*got)):
        assert torch.isfinite(a.float()).all() and torch.equal(a, b), i


@pytest.mark.parametrize("window,page", [(None, 32), (70, 16)])
@pytest.mark.parametrize("graph", [False, True])
def test_runner_over_float16_pages(window, page, graph):
    """Prompts in pieces and steps through two layers against the dense layers (whose keys and values are bf16, rounded more coarsely)."""
    from daisy_b200 import PagedRunner, WindowMask
    H, L = 2, 2
    dim = H * D
    layers = _stack(L, H, dim)
    runner = PagedRunner(layers, window, pages=40, max_seqs=2, max_len=400, page=page, dtype=torch.float16)
    assert runner.cache.k.dtype == torch.float16
    if graph:
        runner.capture_step(dim)
    g = _gen(221)
    a, b = runner.add(), runner.add()
    fed, got = {a: [], b: []}, {a: [], b: []}
    for counts in ([150, 7], [3, 40], [60, 129]):                    # both kernels
        xs = [torch.randn(n, dim, generator=g).bfloat16().cuda() for n in counts]
        for s, x, y in zip((a, b), xs, runner.prefill(xs, [a, b])):
            fed[s].append(x)
            got[s].append(y.clone())
    for _ in range(20):
        x = torch.randn(2, 1, dim, generator=g).bfloat16().cuda()
        y = (runner.step_graph if graph else runner.step)(x)
        for s in (a, b):
            fed[s].append(x[s])
            got[s].append(y[s].clone())
    _status()
    for s in (a, b):
        x = torch.cat(fed[s])[None]
        for layer in layers:
            with torch.inference_mode():
                x, _, _ = layer.prefill(x, None, attn_mask=WindowMask(window))
        assert_close_bf16(torch.cat(got[s]), x[0], f"sequence {s}")


def test_limits_of_the_library_calls():
    """``max_len`` of the C interface: positions at or behind it are refused by every call."""
    import ctypes as C
    from daisy_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    H, page, n = 2, 16, 3
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = _randn(_gen(241), n, 1, 3 * H, D).cuda()
    table = torch.arange(12).view(n, 4).int().cuda()

    def pool(limit):
        k = torch.full((12, H, page, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        v = k.clone()
        return k, v, _lib.Pages(k=k.data_ptr(), v=v.data_ptr(), p_sb=H * page * D, p_sh=page * D, p_sr=D, table=table.data_ptr(), table_sb=4, n_pages=12, H=H, page=page, width=4, n_seq=n,
                                max_len=limit)

    def raised():
        was = status.item()
        status.zero_()
        return was
    s = 3 * H * D
    for limit, stored in ((0, 3), (64, 3), (1000, 3), (41, 3), (40, 2), (1, 0)):
        start = _ints([30, 40, 1])
        k, v, pages = pool(limit)
        _lib.check(lib.daisy_b200_paged_append(C.byref(pages), x[:, :, H:].data_ptr(), x[:, :, 2 * H:].data_ptr(), None, s, s, D, s, s, D, 0, 0, 0, None, start.data_ptr(), None, None, None, 0,
                                               None, 0, 0, 0, None, n, 1, 0, D, EPS, 0, status.data_ptr(), stream), "append")
        kept = [bool(torch.isfinite(k[b * 4 + p // page, :, p % page].float()).all()) for b, p in enumerate((30, 40, 1))]
        assert sum(kept) == stored and int(torch.isfinite(k.float()).all(-1).sum()) == stored * H and (raised() != 0) == (stored < 3)
        k, v, pages = pool(limit)
        k.zero_(), v.fill_(1.0)
        ws = torch.zeros(lib.daisy_b200_paged_decode_workspace_bytes(n, H, H, D), dtype=torch.uint8, device="cuda")
        out = torch.full((n, 1, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
        _lib.check(lib.daisy_b200_paged_decode_step(C.byref(pages), x.data_ptr(), x[:, :, H:].data_ptr(), x[:, :, 2 * H:].data_ptr(), s, D, s, D, s, D, start.data_ptr(), 0, None, None, 0,
                                                    out.data_ptr(), H * D, D, None, 0, 0, None, H, D, SCALE, EPS, 0, ws.data_ptr(), ws.numel(), status.data_ptr(), stream), "decode")
        assert [bool((out[b] != 0).any()) for b in range(n)] == kept and torch.isfinite(out.float()).all() and (raised() != 0) == (stored < 3)
        assert [bool((v[b * 4 + p // page, :, p % page] != 1).any()) for b, p in enumerate((30, 40, 1))] == kept
